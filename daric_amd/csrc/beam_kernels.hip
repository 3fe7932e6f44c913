// Beam search on MI355X (gfx950): the k best of a request's W x V candidates, and
// the reordering of its beams' pages by them.
//
// A candidate's score is the beam's plus x - lse, lse = log sum exp(x) of its row of
// logits. Within a row scores are ordered as the logits are, so the choice needs one
// pass over them: a wavefront takes a split of a row, 8 KiB, into registers, reduces its
// maximum and its sum of exponentials, and leaves the split's k best logits in order, ties
// to the lower token. select_join_kernel, a workgroup per request, joins the splits' sums to
// each beam's in fp64 and chooses among the lists by score.
//
// Scores of different beams differ by more than what the sums err by, almost always: so
// the exponentials' argument (x - max) log2(e) is one product with log2(e) to 48 bits,
// rounded once, and what follows the splits' fp32 sums is fp64.
//
// MI355X, traced medians, 256 rows of 128000 bf16, 16 candidates of 8 beams: splits 18.5
// us, join 6.2. The splits' loads and maxima alone take 11.3 us (65.5 MB at 5.8 TB/s), the
// exponentials 1.7 more, thresholds, hits and their ranks the rest: vector instructions
// issue for 10 us of the 18 and overlap the loads only in part. One request of four such
// rows: 6.1 + 5.9 us, latency.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "append.h"
#include "beams.h"
#include "elem.h"
#include "kernels.h"
#include "launch.h"

namespace daric {
namespace {

constexpr int kSplitThreads = 256;                     // wavefronts of a workgroup work apart
constexpr int kSplitsPerBlock = kSplitThreads / 64;
constexpr int kListed = 512;                           // candidates that a wavefront ranks
// Candidates up to which thresholds are taken of one maximum a lane, with one test a step:
// the looser, the more of the 64 lanes are asked for. MI355X, splits and join of 32 requests
// of 8 beams of 128000 bf16, by lanes and by units: 8 candidates 24 and 28 us, 16 25 and 29, 32
// 28 and 31, 48 38 and 34, 64 140 and 38; two requests of 32 beams 16 17 and 19, 32 20 and
// 21, 48 28 and 26, 64 77 and 29; 7 of 5 of 50021 fp32 16 12 and 15, 48 17 and 17, 64 72 and 20.
// They cross between 32 and 48.
constexpr int kFewCandidates = 16;

// Order of a type's values as unsigned numbers, in the leading bits that they differ
// in as fp32; -0 as +0, NaN as -inf.
template <int KIND>
struct Rank {
    static constexpr int kBits = KIND == kF32 ? 32 : KIND == kBF16 ? 16 : 19;
    static constexpr uint32_t kMask = ~0u << (32 - kBits);
    static constexpr uint32_t kLeast = 0x00800000u;    // below any finite value's, above -inf's
    static __device__ __forceinline__ uint32_t of(float f) {
        const uint32_t b = f2u(f == f ? f + 0.0f : -__builtin_huge_valf());
        return ((b & 0x80000000u) ? ~b : (b | 0x80000000u)) & kMask;
    }
    static __device__ __forceinline__ float value(uint32_t r) {
        return u2f((r & 0x80000000u) ? r & 0x7fffffffu : ~r & kMask);
    }
    // A value and its place in a split (lower places first) as one number: a rank of 19
    // bits and a place below 2^12 fit in one word.
    static constexpr int kPlaceBits = 12;
    using Key = typename std::conditional<KIND == kF32, uint64_t, uint32_t>::type;
    static __device__ __forceinline__ Key key(uint32_t rank, int place) {
        if constexpr (KIND == kF32) return static_cast<uint64_t>(rank) << 32 | static_cast<uint32_t>(~place);
        else return rank | ((1u << kPlaceBits) - 1 - static_cast<uint32_t>(place));
    }
    static __device__ __forceinline__ uint32_t rank(Key k) {
        if constexpr (KIND == kF32) return static_cast<uint32_t>(k >> 32);
        else return k & kMask;
    }
    static __device__ __forceinline__ int place(Key k) {
        if constexpr (KIND == kF32) return static_cast<int>(~static_cast<uint32_t>(k));
        else return static_cast<int>((1u << kPlaceBits) - 1 - (k & ((1u << kPlaceBits) - 1)));
    }
};
static_assert(kSplitBytes / 2 <= 1 << Rank<kF16>::kPlaceBits && Rank<kF16>::kBits + Rank<kF16>::kPlaceBits <= 32,
              "keys of 16-bit values");

// A lane's share of a split of a row: kSplitBytes / 64, in units of 16 bytes. Value j of unit
// r is value (r * 64 + lane) * kUnit + j of the split; behind its end stands -inf.
template <int KIND>
struct Split {
    static constexpr int kPerReg = KIND == kF32 ? 1 : 2;
    static constexpr int kBytes = 4 / kPerReg;         // of a value
    static constexpr int kUnit = 4 * kPerReg;          // values of a unit
    static constexpr int kUnits = kSplitBytes / 1024;
    static constexpr int kTotal = 64 * kUnits * kUnit;
    const uint8_t* p;                                  // of the split's values, at any element
    int n, lane;                                       // values that are there

    __device__ __forceinline__ int index(int r) const { return (r * 64 + lane) * kUnit; }
    __device__ __forceinline__ u32x4 words(int r) const {
        constexpr uint32_t kNone = KIND == kF32 ? 0xff800000u : KIND == kBF16 ? 0xff80ff80u : 0xfc00fc00u;
        const int i = index(r);
        u32x4 w;
        if (i + kUnit <= n) {
            __builtin_memcpy(&w, p + static_cast<int64_t>(i) * kBytes, 16);
            return w;
        }
        w = u32x4{kNone, kNone, kNone, kNone};
        for (int j = 0; j < kUnit; ++j) {
            if (i + j >= n) break;
            uint32_t x = 0;
            __builtin_memcpy(&x, p + static_cast<int64_t>(i + j) * kBytes, kBytes);
            const int at = j / kPerReg;
            const uint32_t old = at == 0 ? w[0] : at == 1 ? w[1] : at == 2 ? w[2] : w[3];
            const uint32_t mixed = kPerReg == 1 ? x : (j & 1) != 0 ? (old & 0xffffu) | x << 16 : (old & 0xffff0000u) | x;
            w[0] = at == 0 ? mixed : w[0];
            w[1] = at == 1 ? mixed : w[1];
            w[2] = at == 2 ? mixed : w[2];
            w[3] = at == 3 ? mixed : w[3];
        }
        return w;
    }
    // Value j of a unit and its place as one word or two, which cost less than its key.
    using Raw = typename std::conditional<KIND == kF32, uint64_t, uint32_t>::type;
    static __device__ __forceinline__ Raw raw(const u32x4& w, int j, int place) {
        const uint32_t x = w[j / kPerReg];
        if constexpr (KIND == kF32) return static_cast<uint64_t>(static_cast<uint32_t>(place)) << 32 | x;
        else return static_cast<uint32_t>(place) << 16 | ((j & 1) != 0 ? x >> 16 : x & 0xffffu);
    }
    static __device__ __forceinline__ float raw_value(Raw r) {
        return value(u32x4{static_cast<uint32_t>(r), 0, 0, 0}, 0);
    }
    static __device__ __forceinline__ int raw_place(Raw r) { return static_cast<int>(r >> (KIND == kF32 ? 32 : 16)); }
    static __device__ __forceinline__ float value(const u32x4& w, int j) {
        const uint32_t x = w[j / kPerReg];
        if constexpr (KIND == kF32) return u2f(x);
        else if constexpr (KIND == kBF16) return u2f((j & 1) != 0 ? x & 0xffff0000u : x << 16);
        else return f16_to_f32((j & 1) != 0 ? x >> 16 : x & 0xffffu);
    }
};

// Lane i's value of lane i - n of its row of 16 (CTRL row_shr:n), or lane 15's or 31's
// passed on to the rows behind (row_bcast); `old` where there is none.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float old, float x) {
#ifdef __HIP_DEVICE_COMPILE__
    return u2f(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(f2u(old)), static_cast<int>(f2u(x)), CTRL, ROWS, 0xf, false)));
#else
    return old + x;
#endif
}
__device__ __forceinline__ float lane63(float x) {
    return u2f(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(f2u(x)), 63)));
}
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp<0x111>(x, x));
    x = fmaxf(x, dpp<0x112>(x, x));
    x = fmaxf(x, dpp<0x114>(x, x));
    x = fmaxf(x, dpp<0x118>(x, x));
    x = fmaxf(x, dpp<0x142, 0xa>(x, x));
    x = fmaxf(x, dpp<0x143, 0xc>(x, x));
    return lane63(x);
}
__device__ __forceinline__ float wave_sum(float x) {
    x += dpp<0x111>(0.0f, x);
    x += dpp<0x112>(0.0f, x);
    x += dpp<0x114>(0.0f, x);
    x += dpp<0x118>(0.0f, x);
    x += dpp<0x142, 0xa>(0.0f, x);
    x += dpp<0x143, 0xc>(0.0f, x);
    return lane63(x);
}
// Larger of three; a NaN is passed over.
__device__ __forceinline__ float max3(float a, float b, float c) {
#ifdef __HIP_DEVICE_COMPILE__
    float m;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
    return m;
#else
    return fmaxf(fmaxf(a, b), c);
#endif
}

// The largest t of `bits` leading bits for which count(t) >= k (0 if none). UNROLL 1 in a
// kernel that runs through its code once, and waits for the code itself.
template <int UNROLL, class Count>
__device__ __forceinline__ uint32_t largest_with(int bits, int k, Count&& count) {
    uint32_t t = 0;
#pragma unroll UNROLL
    for (int b = 31; b > 31 - bits; --b) {
        const uint32_t u = t | (1u << b);
        if (count(u) >= k) t = u;
    }
    return t;
}

template <int KIND>
__global__ __launch_bounds__(kSplitThreads) void select_split_kernel(SelectArgs a) {
    using S = Split<KIND>;
    using R = Rank<KIND>;
    using Key = typename R::Key;
    __shared__ __align__(16) Key s_list[kSplitsPerBlock][kListed + 4];
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const uint32_t unit = blockIdx.x * kSplitsPerBlock + wave;
    const uint32_t rows = static_cast<uint32_t>(a.B) * a.W;
    if (unit >= rows * a.splits) return;
    const uint32_t row = a.d_splits.div(unit);
    const int split = static_cast<int>(unit - row * a.splits);
    // rows that offer no logit: their beam has ended, or has no score
    if (a.ended != nullptr && a.ended[row] != 0) return;
    if (!(a.scores[row] > -__builtin_huge_valf())) return;
    const uint32_t b = a.d_beams.div(row), w = row - b * a.W;
    const int64_t v0 = static_cast<int64_t>(split) * S::kTotal;
    S v;
    v.p = a.logits + (b * a.batch + w * a.row + v0) * S::kBytes;
    v.n = static_cast<int>(min(a.V - v0, static_cast<int64_t>(S::kTotal)));
    v.lane = lane;
    u32x4 x[S::kUnits];
#pragma unroll
    for (int r = 0; r < S::kUnits; ++r) x[r] = v.words(r);

    float best[S::kUnits], top = -__builtin_huge_valf();   // of each unit, of all
#pragma unroll
    for (int r = 0; r < S::kUnits; ++r) {
        best[r] = -__builtin_huge_valf();
#pragma unroll
        for (int j = 0; j < S::kUnit; j += 2) best[r] = max3(best[r], S::value(x[r], j), S::value(x[r], j + 1));
        top = fmaxf(top, best[r]);
    }
    const float most = wave_max(top);
    // a split of nothing but -inf: 0 in its place, so that the sum is 0, or NaN if it holds one
    const float ref = most > -__builtin_huge_valf() ? most : 0.0f;
    constexpr float kLog2e = 1.44269504088896341f;
    constexpr float kLog2eRest = static_cast<float>(1.44269504088896340736 - static_cast<double>(kLog2e));
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < S::kUnits; ++r) {
#pragma unroll
        for (int j = 0; j < S::kUnit; ++j) {
            const float d = S::value(x[r], j) - ref;
            sum[j % 4] += __builtin_amdgcn_exp2f(__builtin_fmaf(d, kLog2e, d * kLog2eRest));
        }
    }
    const float total = wave_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (lane == 0) {
        a.part_ms[static_cast<int64_t>(unit) * 2] = most;
        a.part_ms[static_cast<int64_t>(unit) * 2 + 1] = total;
    }

    // At least k of the split's values are as large as the k-th largest of the lanes' maxima,
    // few more than k where those are few of the lanes; for larger k, of the units' maxima.
    uint32_t least;
    if (a.k <= kFewCandidates) {
        const uint32_t mine = R::of(top);
        least = largest_with<32>(R::kBits, a.k, [&](uint32_t t) { return __popcll(__ballot(mine >= t)); });
    } else {
        uint32_t mine[S::kUnits];
#pragma unroll
        for (int r = 0; r < S::kUnits; ++r) mine[r] = R::of(best[r]);
        least = largest_with<32>(R::kBits, a.k, [&](uint32_t t) {
            int c = 0;
#pragma unroll
            for (int r = 0; r < S::kUnits; ++r) c += __popcll(__ballot(mine[r] >= t));
            return c;
        });
    }
    least = max(least, R::kLeast);
    Key* const list = s_list[wave];
    const unsigned long long below = (1ull << lane) - 1;
    int found = 0;
    {
        // The units that hold any, each lane's next one at a time, chosen from the registers by
        // selects: read again from memory they kept a wavefront at its end waiting.
        const float bound = R::value(least);
        uint32_t holds = 0;
#pragma unroll
        for (int r = 0; r < S::kUnits; ++r) holds |= best[r] >= bound ? 1u << r : 0u;
        while (__ballot(holds != 0) != 0) {
            const int r = holds != 0 ? __ffs(static_cast<int>(holds)) - 1 : 0;
            const float mine = holds != 0 ? bound : __builtin_nanf("");     // no value is as large
            holds &= holds - 1;
            static_assert(S::kUnits == 8, "a unit is chosen by three bits");
            u32x4 u;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t a0 = (r & 1) != 0 ? x[1][c] : x[0][c], a1 = (r & 1) != 0 ? x[3][c] : x[2][c];
                const uint32_t a2 = (r & 1) != 0 ? x[5][c] : x[4][c], a3 = (r & 1) != 0 ? x[7][c] : x[6][c];
                const uint32_t b0 = (r & 2) != 0 ? a1 : a0, b1 = (r & 2) != 0 ? a3 : a2;
                u[c] = (r & 4) != 0 ? b1 : b0;
            }
            const int at0 = v.index(r);
#pragma unroll
            for (int j = 0; j < S::kUnit; ++j) {
                const bool is = S::value(u, j) >= mine;
                const unsigned long long some = __ballot(is);
                if (some == 0) continue;
                const int at = found + __popcll(some & below);
                if (is && at < kListed) list[at] = S::raw(u, j, at0 + j);
                found += __popcll(some);
            }
        }
        for (int i = lane; i < min(found, kListed); i += 64) {
            const Key k = list[i];
            list[i] = R::key(R::of(S::raw_value(k)), S::raw_place(k));
        }
    }
    if (found > kListed) {
        // Few lanes hold them, or many are alike: the k-th largest value itself, and from the
        // values read again all above it and the first of those equal to it.
        const auto count = [&](int r, auto&& test) {
            const u32x4 u = v.words(r);
            int n = 0;
#pragma unroll
            for (int j = 0; j < S::kUnit; ++j) n += test(R::of(S::value(u, j))) ? 1 : 0;
            return n;
        };
        const auto upto = [&](int n) {                 // sum over the lanes up to this one
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(n, o, 64);
                if (lane >= o) n += y;
            }
            return n;
        };
        least = largest_with<1>(R::kBits, a.k, [&](uint32_t t) {
            if (t < R::kLeast) return a.k;             // all are as large, and enough
            const float from = R::value(t);
            int n = 0;
#pragma unroll
            for (int r = 0; r < S::kUnits; ++r) {
#pragma unroll
                for (int j = 0; j < S::kUnit; ++j) n += __popcll(__ballot(S::value(x[r], j) >= from));
            }
            return n;
        });
        least = max(least, R::kLeast);
        found = 0;
        int open = a.k;                                // places for those equal to it, in order
        for (int r = 0; r < S::kUnits; ++r) open -= __shfl(upto(count(r, [&](uint32_t q) { return q > least; })), 63, 64);
        for (int r = 0; r < S::kUnits; ++r) {
            const u32x4 u = v.words(r);
            const int equal = upto(count(r, [&](uint32_t q) { return q == least; }));
            int before = equal - count(r, [&](uint32_t q) { return q == least; });
#pragma unroll
            for (int j = 0; j < S::kUnit; ++j) {
                const uint32_t q = R::of(S::value(u, j));
                const bool is = q > least || (q == least && before < open);
                before += q == least ? 1 : 0;
                const unsigned long long some = __ballot(is);
                if (is) list[found + __popcll(some & below)] = R::key(q, v.index(r) + j);
                found += __popcll(some);
            }
            open -= min(open, __shfl(equal, 63, 64));
        }
    }
    // a candidate's place is the number of better ones
    if (lane < 4) list[found + lane] = 0;              // read with the last of them, better than none
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
    BeamCandidate* const out = a.part + static_cast<int64_t>(unit) * a.k;
    for (int i = lane; i < found; i += 64) {
        const Key key = list[i];
        int place = 0;
        for (int j = 0; j < found; j += 4) {
            Key o[4];
            __builtin_memcpy(o, __builtin_assume_aligned(list + j, 16), sizeof(o));
#pragma unroll
            for (int e = 0; e < 4; ++e) place += o[e] > key ? 1 : 0;
        }
        if (place < a.k) out[place] = BeamCandidate{R::value(R::rank(key)), static_cast<int32_t>(v0 + R::place(key))};
    }
    for (int i = found + lane; i < a.k; i += 64) out[i].token = -1;
}

// The order of scores as unsigned numbers (-0 as +0), and its leading 32 bits.
__device__ __forceinline__ uint64_t score_key(double s) {
    const uint64_t b = __builtin_bit_cast(uint64_t, s + 0.0);
    return (b >> 63) != 0 ? ~b : (b | 1ull << 63);
}
__device__ __forceinline__ double key_score(uint64_t k) {
    return __builtin_bit_cast(double, (k >> 63) != 0 ? k & ~(1ull << 63) : ~k);
}
__device__ __forceinline__ uint32_t score_rank(double s) { return static_cast<uint32_t>(score_key(s) >> 32); }

// What orders candidates of equal scores, less is better: the beam, then the logit (the larger one
// first), then the token. A score as large as a type's lowest value or infinite swallows the logits
// of its beam in 64 bits, but the lists hold its likeliest tokens: so they stay in the lists' order.
// 6 bits of beam; the tokens of 32-bit logits fit in 26 bits and leave their 32; those of 16-bit
// ones, of which 19 bits differ, take 32 and leave 26.
struct Place {
    int token_bits;
    __device__ explicit Place(int bits) : token_bits(bits) {}
    __device__ __forceinline__ uint64_t of(int w, float x, int token) const {
        const uint32_t b = f2u(x);
        const uint32_t larger_first = (b & 0x80000000u) != 0 ? b : ~(b | 0x80000000u);
        return static_cast<uint64_t>(w) << 58 | static_cast<uint64_t>(larger_first >> (token_bits - 26)) << token_bits |
               static_cast<uint32_t>(token);
    }
    __device__ __forceinline__ int beam(uint64_t p) const { return static_cast<int>(p >> 58); }
    __device__ __forceinline__ int token(uint64_t p) const { return static_cast<int>(p & ((1ull << token_bits) - 1)); }
};
static_assert(kMaxBeams <= 64 && kMaxSplits * (kSplitBytes / 4) <= 1ll << 26 && kMaxSplits * (kSplitBytes / 2) <= 1ll << 32,
              "beams and tokens in a place");

// A workgroup per request. The k-th best of the lists' heads, one or the first few of each,
// is at most the k-th best of all: of the lists whose head is as good, the candidates that
// are as good too, few more than k, are ranked in LDS. Where one beam's lists hold most of
// them they may be many: a rank that leaves few is found then bit by bit, and they are taken
// again from it on. Where they are too many for that (scores alike), each wavefront takes k
// times the best head of its share of the lists, and those are ranked. Bound by latency: three
// rounds of loads. MI355X, two requests of 32 beams of 128000 bf16, 64 candidates: 15 us where
// the scores spread over the beams, 490 where one wavefront took 64 times the best of all heads.
constexpr int kJoinThreads = 512;
constexpr int kJoined = kJoinThreads / 64 * kMaxCandidates;
constexpr int kJoinLists = 2048;      // lists whose candidates are looked through
constexpr int kHalved = 4096;         // candidates of which a few are found so; room for the heads, too
constexpr int kHeadsPerLane = 64;     // of the first wavefront: what is beyond is not asked for the threshold
__global__ __launch_bounds__(kJoinThreads) void select_join_kernel(SelectArgs a, int lists_per_lane, int log2_heads) {
    extern __shared__ uint8_t s_at[];                  // [lists_per_lane][kJoinThreads]: candidates taken from each list
    // A candidate's score is (score - log sum exp(x - most)) + (x - most), most the row's largest
    // logit: logits of any size cancel before a score is added to them, also in rows of nothing
    // but a mask's -3e38.
    __shared__ double s_base[kMaxBeams];               // the first term of each beam; of one at its end, its score
    __shared__ float s_most[kMaxBeams];
    __shared__ uint8_t s_ended[kMaxBeams];
    __shared__ uint32_t s_rank[kHalved];               // of the lists' heads, then of the candidates
    struct Found {
        uint64_t key;                                  // of the score; 0: none
        uint64_t tie;                                  // larger is better among equal scores: ~its Place
    };
    __shared__ __align__(16) Found s_found[kJoined];
    __shared__ uint16_t s_lists[kJoinLists];
    __shared__ uint32_t s_least;
    __shared__ int s_sums[2][kJoinThreads / 64];
    __shared__ int s_count, s_n_lists;
    const int64_t b = blockIdx.x;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int64_t row0 = b * a.W;
    const double kNone = -__builtin_huge_val();
    // what is not above it rounds to -inf in the fp32 that scores are given in
    constexpr double kLeastScore = -0x1.ffffffp+127;
    const int lists = a.W * a.splits;
    const BeamCandidate* const part = a.part + row0 * a.splits * a.k;
    constexpr int kMine = 2;                           // of a lane's samples, read ahead
    // the first 2^log2_heads candidates of each list, from which the threshold is taken
    const int samples = lists << log2_heads;
    const auto sample_at = [&](int i) {
        return static_cast<int64_t>(i >> log2_heads) * a.k + (i & ((1 << log2_heads) - 1));
    };
    BeamCandidate head[kMine];                         // what rows without logits left there is not used
#pragma unroll
    for (int n = 0; n < kMine; ++n)
        if (n * kJoinThreads + tid < samples) head[n] = part[sample_at(n * kJoinThreads + tid)];
    // sixteen lanes a beam
    for (int w = tid >> 4; w < a.W; w += kJoinThreads / 16) {
        const float score = a.scores[row0 + w];
        const bool at_end = a.ended != nullptr && a.ended[row0 + w] != 0;
        double base = score;
        float most = -__builtin_huge_valf();
        if (!at_end) {
            const float* ms = a.part_ms + (row0 + w) * a.splits * 2;
            for (int i = tid & 15; i < a.splits; i += 16) most = fmaxf(most, ms[2 * i]);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
            double sum = 0.0;
            for (int i = tid & 15; i < a.splits; i += 16)
                sum += static_cast<double>(ms[2 * i + 1]) * exp(static_cast<double>(ms[2 * i]) - static_cast<double>(most));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
            // a beam without a score left no sums
            base = score > -__builtin_huge_valf() ? base - log(sum) : kNone;
        }
        if ((tid & 15) == 0) {
            s_base[w] = base;
            s_most[w] = most;
            s_ended[w] = at_end ? 1 : 0;
        }
    }
    if (tid == 0) s_count = s_n_lists = 0;
    __syncthreads();
    const Place place(a.token_bits);
    // A list's candidate (number `at` of it): its score, -inf where there is none (NaN too),
    // and its place.
    const auto score_of = [&](int list, int at, const BeamCandidate& c, double* score, uint64_t* where) {
        const int w = static_cast<int>(a.d_splits.div(static_cast<uint32_t>(list)));
        const bool at_end = s_ended[w] != 0;
        const bool first = list == w * a.splits && at == 0;
        const int token = at_end ? a.end_token : c.token;
        const double v = at_end ? s_base[w] : s_base[w] + (static_cast<double>(c.x) - static_cast<double>(s_most[w]));
        const bool is = (at_end ? first : token >= 0) && v > kLeastScore;
        *score = is ? v : kNone;
        *where = place.of(w, at_end ? 0.0f : c.x, token);
    };
    const auto look = [&](int list, int at, double* score, uint64_t* where) {
        BeamCandidate c{0.0f, -1};
        if (at < a.k) c = part[static_cast<int64_t>(list) * a.k + at];
        score_of(list, at, c, score, where);
    };
    const auto rank_of = [&](int list, int n, const BeamCandidate& c) {
        double s;
        uint64_t at;
        score_of(list, n, c, &s, &at);
        return s > kNone ? score_rank(s) : 0u;
    };
    const auto sample_rank = [&](int i, const BeamCandidate& c) {
        return rank_of(i >> log2_heads, i & ((1 << log2_heads) - 1), c);
    };
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
        const int i = n * kJoinThreads + tid;
        s_rank[i] = i < samples ? sample_rank(i, head[n]) : 0u;
    }
    const int sampled = min(samples, kHeadsPerLane * 64);
    for (int i = kMine * kJoinThreads + tid; i < (sampled + 63) / 64 * 64; i += kJoinThreads)
        s_rank[i] = i < samples ? sample_rank(i, part[sample_at(i)]) : 0u;
    __syncthreads();
    if (wave == 0) {
        // in 20 bits: eight of a score's mantissa; of one maximum a lane, or of four
        uint32_t h[4], least;
        for (int g = 0; g < 4; ++g) h[g] = 0;
        for (int n = 0; n * 64 < samples && n < kHeadsPerLane; n += 4) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if ((n + g) * 64 < samples) h[g] = max(h[g], s_rank[(n + g) * 64 + lane]);
        }
        if (a.k <= kFewCandidates) {
            const uint32_t best = max(max(h[0], h[1]), max(h[2], h[3]));
            least = largest_with<1>(20, a.k, [&](uint32_t t) { return __popcll(__ballot(best >= t)); });
        } else {
            least = largest_with<1>(20, a.k, [&](uint32_t t) {
                return __popcll(__ballot(h[0] >= t)) + __popcll(__ballot(h[1] >= t)) + __popcll(__ballot(h[2] >= t)) +
                       __popcll(__ballot(h[3] >= t));
            });
        }
        if (lane == 0) s_least = max(least, 1u);
    }
    __syncthreads();
    uint32_t least = s_least;
    const auto enlist = [&](int list, uint32_t r) {
        if (r < least) return;
        const int p = atomicAdd(&s_n_lists, 1);
        if (p < kJoinLists) s_lists[p] = static_cast<uint16_t>(list);
    };
    for (int i = tid; i < sampled; i += kJoinThreads)
        if ((i & ((1 << log2_heads) - 1)) == 0) enlist(i >> log2_heads, s_rank[i]);
    for (int i = kHeadsPerLane * 64 + tid; i < lists; i += kJoinThreads)
        enlist(i, rank_of(i, 0, part[static_cast<int64_t>(i) * a.k]));
    __syncthreads();
    // The candidates from `least` on: how many, their ranks, and the first of them.
    const int n_lists = s_n_lists;
    const auto take = [&]() {
        // sixteen lanes a list, which is in order: on while all of them are good enough
        for (int l = tid >> 4; l < n_lists; l += kJoinThreads / 16) {
            for (int at0 = 0; at0 < a.k; at0 += 16) {
                double s;
                uint64_t at;
                look(s_lists[l], at0 + (tid & 15), &s, &at);
                const uint32_t r = s > kNone ? score_rank(s) : 0u;
                const bool is = r >= least;
                if (is) {
                    const int p = atomicAdd(&s_count, 1);
                    if (p < kHalved) s_rank[p] = r;
                    if (p < kJoined) s_found[p] = Found{score_key(s), ~at};
                }
                if ((__ballot(is) >> (lane & 48) & 0xffffull) != 0xffffull) break;
            }
        }
        __syncthreads();
        return s_count;
    };
    int count = n_lists <= kJoinLists ? take() : kHalved + 1;
    if (count > kJoined && count <= kHalved) {
        // the largest t of leading bits that leaves k of them, or the first that leaves few
        uint32_t t = 0;
        for (int bit = 31, turn = 0; bit >= 0; --bit, turn ^= 1) {
            const uint32_t u = t | 1u << bit;
            int c = 0;
            for (int i = tid; i < (count + 63) / 64 * 64; i += kJoinThreads) c += __popcll(__ballot(i < count && s_rank[i] >= u));
            if (lane == 0) s_sums[turn][wave] = c;
            __syncthreads();
            c = 0;
#pragma unroll
            for (int w = 0; w < kJoinThreads / 64; ++w) c += s_sums[turn][w];
            if (c >= a.k) t = u;
            if (c >= a.k && c <= kJoined / 2) break;
        }
        least = t;
        __syncthreads();
        if (tid == 0) s_count = 0;
        __syncthreads();
        count = take();
    }
    if (count > kJoined) {
        // lists n * kJoinThreads + tid are the lane's
        for (int i = 0; i < lists_per_lane; ++i) s_at[i * kJoinThreads + tid] = 0;
        double best = kNone;
        uint64_t where = 0;
        int mine = 0;                                  // which of the lane's lists its best heads
        const auto heads = [&]() {
            best = kNone;
            for (int n = 0; n < lists_per_lane && n * kJoinThreads + tid < lists; ++n) {
                double s;
                uint64_t at;
                look(n * kJoinThreads + tid, s_at[n * kJoinThreads + tid], &s, &at);
                if (s > best || (s == best && s > kNone && at < where)) {
                    best = s;
                    where = at;
                    mine = n;
                }
            }
        };
        heads();
        __syncthreads();                               // the candidates of the first attempt are read no more
        for (int c = 0; c < a.k; ++c) {
            double top = best;
            uint64_t at = where;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const double s = __shfl_xor(top, o, 64);
                const uint64_t p = __shfl_xor(at, o, 64);
                if (s > top || (s == top && p < at)) {
                    top = s;
                    at = p;
                }
            }
            const int to = c * (kJoinThreads / 64) + wave;
            if (lane == 0) s_found[to] = top > kNone ? Found{score_key(top), ~at} : Found{0, static_cast<uint64_t>(to)};
            if (top > kNone && best == top && where == at) {
                ++s_at[mine * kJoinThreads + tid];
                heads();
            }
        }
        __syncthreads();
        count = a.k * (kJoinThreads / 64);
    }
    // a candidate's rank is the number of better ones, counted by eight lanes, four at a time
    const int padded = (count + 31) & ~31;
    if (tid < padded - count) s_found[count + tid] = Found{0, static_cast<uint64_t>(count + tid)};
    __syncthreads();
    const auto write = [&](int c, const Found& f) {
        const int64_t o = b * a.k + c;
        const bool none = f.key == 0;
        a.out_scores[o] = none ? -__builtin_huge_valf() : static_cast<float>(key_score(f.key));
        a.parents[o] = none ? -1 : place.beam(~f.tie);
        a.tokens[o] = none ? -1 : place.token(~f.tie);
    };
    for (int i0 = 0; i0 < count; i0 += kJoinThreads / 8) {
        const int i = i0 + (tid >> 3);
        const Found f = s_found[min(i, count - 1)];
        int better = 0;
        for (int j = tid & 7; j < padded; j += 32) {
            Found o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = s_found[j + 8 * e];
#pragma unroll
            for (int e = 0; e < 4; ++e) better += o[e].key > f.key || (o[e].key == f.key && o[e].tie > f.tie) ? 1 : 0;
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) better += __shfl_xor(better, o, 64);
        if (i < count && (tid & 7) == 0 && better < a.k) write(better, f);
    }
    for (int c = count + tid; c < a.k; c += kJoinThreads) write(c, Found{0, 0});
}

// ------------------------------------------------------------------- reorder
//
// Beam w goes on from beam p_w: the ids of its full pages become p_w's, and its last
// page, its own, takes the rows of p_w's. A lane holds one unit of the rows of all
// the beams of a request: it reads the parents' before it writes any, so beams may
// exchange places, and no other lane touches those bytes. Bound by memory: 80 e4m3 layers of
// 8 requests of 8 beams, 143 MB, 24 us with the pages in the cache behind the L2s (5.9
// TB/s) and 32 without; 32 layers of one request of four 4.8 us.
// The ids of full pages: a lane holds one place of all the lists of a request.
template <int W>
__device__ __forceinline__ void reorder_lists(const BeamLists& s, int32_t* block_table, const int32_t* __restrict__ parents,
                                              int page_size, int block, int* s_from) {
    const int tid = static_cast<int>(threadIdx.x);
    if (tid < s.n_beams) {
        const int p = parents[tid];
        s_from[tid] = p >= 0 && p < s.n_beams && p != tid ? p : -1;
    }
    __syncthreads();
    const int at = block * kReorderThreads + tid;
    if (at >= s.n_tokens / page_size) return;
    int32_t* list = block_table + s.bt_offset + at;
    int32_t id[W];
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < s.n_beams && s_from[w] >= 0) id[w] = list[s_from[w] * s.stride];
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < s.n_beams && s_from[w] >= 0) list[w * s.stride] = id[w];
}

template <typename U, int W>
__global__ __launch_bounds__(kReorderThreads) void reorder_kernel(DescArg d, int layer_off, LayerMinor lm, KVGeom g,
                                                                       int es, int32_t* block_table,
                                                                       const int32_t* __restrict__ parents,
                                                                       int64_t parent_stride, int n_lists,
                                                                       FastDiv inner, FastDiv mid, int token_inner,
                                                                       int head_units, unsigned row_blocks,
                                                                       unsigned page_blocks) {
    __shared__ int s_from[kReorderBeams], s_to[kReorderBeams];       // pages; to 0: beam stays
    __shared__ int s_moves;
    if (blockIdx.x >= row_blocks) {
        const unsigned i = blockIdx.x - row_blocks, list = i / page_blocks;
        reorder_lists<W>(desc_load(desc_at<BeamLists>(d, 0) + list), block_table, parents + list * parent_stride, g.PS,
                         static_cast<int>(i - list * page_blocks), s_from);
        return;
    }
    int l;
    int64_t item;
    lm.at(l, item);
    const DescPtr<BeamLists> lists = desc_at<BeamLists>(d, 0);
    const int li = find_by_tile(lists, n_lists, static_cast<int>(item));
    const BeamLists s = desc_load(lists + li);
    const int full = s.n_tokens / g.PS, rest = s.n_tokens - full * g.PS;
    const int tid = static_cast<int>(threadIdx.x);
    if (tid < W) {
        int from = 0, to = 0;
        if (tid < s.n_beams) {
            const int32_t* last = block_table + s.bt_offset + full;
            const int p = parents[li * parent_stride + tid];
            if (p >= 0 && p < s.n_beams && p != tid) {
                from = last[p * s.stride];
                to = last[tid * s.stride];
                if (from <= 0 || from >= g.num_blocks || to <= 0 || to >= g.num_blocks || from == to) from = to = 0;
            }
        }
        // beams that stay read what the first that moves does, and write nothing: loads
        // without branches, all in flight together
        const unsigned long long moves = __ballot(from != 0);
        const int first = __shfl(from, __ffsll(static_cast<long long>(moves | 1ull << 63)) - 1, 64);
        s_from[tid] = from != 0 ? from : first;
        s_to[tid] = to;
        if (tid == 0) s_moves = moves != 0 ? 1 : 0;
    }
    __syncthreads();
    if (s_moves == 0) return;
    // a workgroup's units are K's or V's: (outer, inner, unit of the row); tokens are the
    // inner index of head-major pages, heads of the others
    const int units = rest * g.H * head_units;
    const int blocks = (units + kReorderThreads - 1) / kReorderThreads;
    int block = static_cast<int>(item) - s.tile_begin;
    const bool v = block >= blocks;
    block -= v ? blocks : 0;
    const int i = block * kReorderThreads + tid;
    if (i >= units) return;
    const int row = static_cast<int>(inner.div(static_cast<uint32_t>(i)));       // head_units
    const int u = i - row * head_units;
    int token, head;
    if (token_inner) {
        head = row / rest;
        token = row - head * rest;
    } else {
        token = static_cast<int>(mid.div(static_cast<uint32_t>(row)));           // H
        head = row - token * g.H;
    }
    uint8_t* const plane = desc_at<uint8_t*>(d, layer_off)[l] + (v ? g.v_off * es : 0);
    const int64_t at = (static_cast<int64_t>(token) * g.ss + static_cast<int64_t>(head) * g.sh) * es +
                       static_cast<int64_t>(u) * static_cast<int>(sizeof(U));
    const int64_t page = g.sb * es;
    U x[W];
#pragma unroll
    for (int w = 0; w < W; ++w)
        x[w] = *reinterpret_cast<const U*>(plane + __builtin_amdgcn_readfirstlane(s_from[w]) * page + at);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int to = __builtin_amdgcn_readfirstlane(s_to[w]);
        if (to != 0) *reinterpret_cast<U*>(plane + to * page + at) = x[w];
    }
}

}  // namespace

void launch_select_beams(const SelectArgs& a, int kind, hipStream_t stream) {
    const int64_t units = static_cast<int64_t>(a.B) * a.W * a.splits;
    const unsigned blocks = static_cast<unsigned>((units + kSplitsPerBlock - 1) / kSplitsPerBlock);
    if (kind == kBF16) DARIC_LAUNCH((select_split_kernel<kBF16>), blocks, kSplitThreads, 0, stream, a);
    else if (kind == kF16) DARIC_LAUNCH((select_split_kernel<kF16>), blocks, kSplitThreads, 0, stream, a);
    else DARIC_LAUNCH((select_split_kernel<kF32>), blocks, kSplitThreads, 0, stream, a);
    check_launch("select_beams");
    const int lists = a.W * a.splits, per_lane = (lists + kJoinThreads - 1) / kJoinThreads;
    // of a beam's few lists more than their best: twice as many as candidates are asked for,
    // since one beam may hold all of them
    int log2_heads = 0;
    while ((a.splits << log2_heads) < 2 * a.k && (2 << log2_heads) <= a.k && (lists << (log2_heads + 1)) <= kHeadsPerLane * 64)
        ++log2_heads;
    DARIC_LAUNCH(select_join_kernel, static_cast<unsigned>(a.B), kJoinThreads, static_cast<size_t>(per_lane) * kJoinThreads, stream, a, per_lane, log2_heads);
    check_launch("select_beams join");
}

void launch_reorder(const DescArg& d, int layer_off, int n_layers, const KVGeom& g, int es, int unit,
                    int32_t* block_table, const int32_t* parents, int64_t parent_stride, int n_lists, int most_beams,
                    int64_t most_pages, int64_t tiles, hipStream_t stream) {
    const int head_units = g.D * es / unit;
    const FastDiv inner(static_cast<uint32_t>(head_units)), mid(static_cast<uint32_t>(g.H));
    const int token_inner = g.ss < g.sh ? 1 : 0;
    // the lists' blocks stand behind the rows' of one launch: they write other places of
    // block_table than the rows' read; a launch that they do not fit in is followed by theirs
    const unsigned page_blocks = static_cast<unsigned>((most_pages + kReorderThreads - 1) / kReorderThreads);
    unsigned list_blocks = page_blocks * static_cast<unsigned>(n_lists);
    const auto launch = [&](const LayerMinor& lm, unsigned row_blocks) {
        const bool fit = static_cast<int64_t>(row_blocks) + list_blocks <= kMaxGridBlocks;
        const unsigned blocks = row_blocks + (fit ? list_blocks : 0);
#define DARIC_RW(U, W) DARIC_LAUNCH((reorder_kernel<U, W>), blocks, kReorderThreads, 0, stream, d, layer_off, lm, g, es, \
                                    block_table, parents, parent_stride, n_lists, inner, mid, token_inner, head_units, \
                                    row_blocks, std::max(1u, page_blocks))
#define DARIC_RU(U)                                 \
    do {                                            \
        if (most_beams <= 4) DARIC_RW(U, 4);        \
        else if (most_beams <= 8) DARIC_RW(U, 8);   \
        else if (most_beams <= 16) DARIC_RW(U, 16); \
        else DARIC_RW(U, 32);                       \
    } while (0)
        if (unit == 16) DARIC_RU(u32x4);
        else if (unit == 8) DARIC_RU(u32x2);
        else if (unit == 4) DARIC_RU(uint32_t);
        else if (unit == 2) DARIC_RU(uint16_t);
        else DARIC_RU(uint8_t);
#undef DARIC_RU
#undef DARIC_RW
        check_launch("reorder_beams");
        if (fit) list_blocks = 0;
    };
    for_layer_minor(n_layers, tiles, launch);
    if (list_blocks > 0) launch(LayerMinor{}, 0);
}

}  // namespace daric
