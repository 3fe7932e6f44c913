// Beam search on MI355X (gfx950): the k best of a request's W x V candidates, and
// the reordering of its beams' pages by them.
//
// A candidate's score is the beam's plus x - lse, lse = log sum exp(x) of its row of
// logits. Within a row scores are ordered as the logits are, so the choice needs one
// pass over them: a wavefront takes a split of a row into registers (`REGS` words a
// lane), reduces its maximum and its sum of exponentials, and leaves the split's k
// best logits in order, ties to the lower token. select_join_kernel, a wavefront per
// request, joins the splits' sums to each beam's lse in fp64 and merges the lists by
// score: k times the best of their heads.
//
// Scores of different beams differ by no less than what the sums err by, almost
// always: so the exponentials' argument (x - max) log2(e) is one product with log2(e)
// to 48 bits, rounded once, and what follows the splits' fp32 sums is fp64.
#include <hip/hip_runtime.h>

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
};

template <int KIND, int REGS>
struct Split {
    static constexpr int kPerReg = KIND == kF32 ? 1 : 2;
    static constexpr int kUnit = 4 * kPerReg;          // values of a 16-byte access
    static constexpr int kValues = REGS * kPerReg;     // of a lane
    uint32_t w[REGS];
    int lane;
    // Value j of the lane is value (j / kUnit * 64 + lane) * kUnit + j % kUnit of the split.
    __device__ __forceinline__ int index(int j) const { return (j / kUnit * 64 + lane) * kUnit + j % kUnit; }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (KIND == kF32) return u2f(w[j]);
        else if constexpr (KIND == kBF16) return u2f((j & 1) != 0 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        else return f16_to_f32((j & 1) != 0 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu);
    }
    // n values from p, of any element-aligned address; -inf behind them.
    __device__ __forceinline__ void load(const uint8_t* p, int64_t n) {
        constexpr uint32_t kNone = KIND == kF32 ? 0xff800000u : KIND == kBF16 ? 0xff80ff80u : 0xfc00fc00u;
        constexpr int kBytes = 4 / kPerReg;
#pragma unroll
        for (int r = 0; r < REGS / 4; ++r) {
            const int64_t i = (static_cast<int64_t>(r) * 64 + lane) * kUnit;
            if (i + kUnit <= n) {
                u32x4 x;
                __builtin_memcpy(&x, p + i * kBytes, 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * r + j] = x[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t x = kNone;
                    if constexpr (KIND == kF32) {
                        if (i + j < n) __builtin_memcpy(&x, p + (i + j) * kBytes, 4);
                    } else {
                        uint16_t h;
                        if (i + 2 * j < n) {
                            __builtin_memcpy(&h, p + (i + 2 * j) * kBytes, 2);
                            x = (x & 0xffff0000u) | h;
                        }
                        if (i + 2 * j + 1 < n) {
                            __builtin_memcpy(&h, p + (i + 2 * j + 1) * kBytes, 2);
                            x = (x & 0xffffu) | static_cast<uint32_t>(h) << 16;
                        }
                    }
                    w[4 * r + j] = x;
                }
            }
        }
    }
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// The largest t of `bits` leading bits for which count(t) >= k (0 if none).
template <class Count>
__device__ __forceinline__ uint32_t largest_with(int bits, int k, Count&& count) {
    uint32_t t = 0;
    for (int b = 31; b > 31 - bits; --b) {
        const uint32_t u = t | (1u << b);
        if (count(u) >= k) t = u;
    }
    return t;
}

template <int KIND, int REGS>
__global__ __launch_bounds__(kSplitThreads) void select_split_kernel(SelectArgs a) {
    __shared__ uint64_t s_list[kSplitsPerBlock][kListed];
    using S = Split<KIND, REGS>;
    constexpr int kBytes = 4 / S::kPerReg;
    constexpr int kTotal = S::kValues * 64;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int lane = static_cast<int>(threadIdx.x) & 63;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * kSplitsPerBlock + wave;
    const int64_t rows = static_cast<int64_t>(a.B) * a.W;
    if (unit >= rows * a.splits) return;
    const int64_t row = unit / a.splits;
    const int split = static_cast<int>(unit - row * a.splits);
    // rows that offer no logit: their beam has ended, or has no score
    if (a.ended != nullptr && a.ended[row] != 0) return;
    if (!(a.scores[row] > -__builtin_huge_valf())) return;
    const int64_t b = row / a.W, w = row - b * a.W;
    const int64_t v0 = static_cast<int64_t>(split) * kTotal;
    S v;
    v.lane = lane;
    v.load(a.logits + (b * a.batch + w * a.row + v0) * kBytes, a.V - v0);

    float top = -__builtin_huge_valf();
#pragma unroll
    for (int j = 0; j < S::kValues; ++j) top = fmaxf(top, v.at(j));
    const float most = wave_max(top);
    // a split of nothing but -inf: 0 in its place, so that the sum is 0, or NaN if it holds one
    const float ref = most > -__builtin_huge_valf() ? most : 0.0f;
    constexpr float kLog2e = 1.44269504088896341f;
    constexpr float kLog2eRest = static_cast<float>(1.44269504088896340736 - static_cast<double>(kLog2e));
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < S::kValues; ++j) {
        const float x = v.at(j) - ref;
        sum[j % 4] += __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, x * kLog2eRest));
    }
    const float total = wave_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (lane == 0) {
        a.part_ms[unit * 2] = most;
        a.part_ms[unit * 2 + 1] = total;
    }

    // At least k of the split's values are as large as the k-th largest of the lanes'
    // maxima: few more than k where they are spread over the lanes.
    using R = Rank<KIND>;
    const uint32_t mine = R::of(top);
    uint32_t least = largest_with(R::kBits, a.k, [&](uint32_t t) { return __popcll(__ballot(mine >= t)); });
    least = max(least, R::kLeast);
    int found = 0;
#pragma unroll
    for (int j = 0; j < S::kValues; ++j) found += __popcll(__ballot(R::of(v.at(j)) >= least));
    uint64_t* const list = s_list[wave];
    const auto entry = [&](int j) { return static_cast<uint64_t>(R::of(v.at(j))) << 32 | static_cast<uint32_t>(~v.index(j)); };
    const unsigned long long below = (1ull << lane) - 1;
    if (found > kListed) {
        // Few lanes hold them, or many are alike: the k-th largest value itself, all
        // above it, and the first of those equal to it.
        least = largest_with(R::kBits, a.k, [&](uint32_t t) {
            int n = 0;
#pragma unroll
            for (int j = 0; j < S::kValues; ++j) n += __popcll(__ballot(R::of(v.at(j)) >= t));
            return n;
        });
        least = max(least, R::kLeast);
        found = 0;
#pragma unroll
        for (int j = 0; j < S::kValues; ++j) {
            const bool is = R::of(v.at(j)) > least;
            const unsigned long long some = __ballot(is);
            if (is) list[found + __popcll(some & below)] = entry(j);
            found += __popcll(some);
        }
        int open = a.k - found;                        // places for those equal to it, in order
#pragma unroll
        for (int r = 0; r < REGS / 4; ++r) {
            int n = 0;
#pragma unroll
            for (int j = 0; j < S::kUnit; ++j) n += R::of(v.at(r * S::kUnit + j)) == least ? 1 : 0;
            int upto = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(upto, o, 64);
                if (lane >= o) upto += x;
            }
            int at = upto - n;
#pragma unroll
            for (int j = 0; j < S::kUnit; ++j) {
                if (R::of(v.at(r * S::kUnit + j)) == least) {
                    if (at < open) list[found + at] = entry(r * S::kUnit + j);
                    ++at;
                }
            }
            const int all = min(__shfl(upto, 63, 64), open);
            found += all;
            open -= all;
        }
    } else {
        int at = 0;
#pragma unroll
        for (int j = 0; j < S::kValues; ++j) {
            const bool is = R::of(v.at(j)) >= least;
            const unsigned long long some = __ballot(is);
            if (some == 0) continue;
            if (is) list[at + __popcll(some & below)] = entry(j);
            at += __popcll(some);
        }
    }
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
    // a candidate's place is the number of better ones
    BeamCandidate* const out = a.part + unit * a.k;
    for (int i = lane; i < found; i += 64) {
        const uint64_t key = list[i];
        int place = 0;
        for (int j = 0; j < found; ++j) place += list[j] > key ? 1 : 0;
        if (place < a.k) {
            out[place].x = R::value(static_cast<uint32_t>(key >> 32));
            out[place].token = static_cast<int32_t>(v0 + static_cast<int32_t>(~static_cast<uint32_t>(key)));
        }
    }
    for (int i = found + lane; i < a.k; i += 64) out[i].token = -1;
}

// The order of scores as unsigned numbers, of their leading 32 bits.
__device__ __forceinline__ uint32_t score_rank(double s) {
    const uint64_t b = __builtin_bit_cast(uint64_t, s);
    return static_cast<uint32_t>(((b >> 63) != 0 ? ~b : (b | 1ull << 63)) >> 32);
}

// A workgroup per request. The k-th best of the lists' heads is at most the k-th best of
// all: the candidates from it on, few more than k, are ranked in LDS. Where they are too
// many (scores alike), the first wavefront takes k times the best of the heads.
constexpr int kJoinThreads = 256;
constexpr int kJoined = 512;
constexpr int kHeadsPerLane = 8;      // of the first wavefront: lists beyond are not asked for the threshold
__global__ __launch_bounds__(kJoinThreads) void select_join_kernel(SelectArgs a, int lists_per_lane) {
    extern __shared__ uint8_t s_at[];                  // [lists_per_lane][64]: candidates taken from each list
    __shared__ double s_base[kMaxBeams];               // score - lse of each beam
    __shared__ double s_score[kJoined];
    __shared__ int64_t s_where[kJoined];
    __shared__ uint32_t s_least;
    __shared__ int s_count;
    const int64_t b = blockIdx.x;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int64_t row0 = b * a.W;
    const double kNone = -__builtin_huge_val();
    const auto ended = [&](int w) { return a.ended != nullptr && a.ended[row0 + w] != 0; };
    const auto alive = [&](int w) { return a.scores[row0 + w] > -__builtin_huge_valf(); };
    for (int w = wave; w < a.W; w += kJoinThreads / 64) {
        double base = a.scores[row0 + w];
        if (!ended(w) && alive(w)) {
            const float* ms = a.part_ms + (row0 + w) * a.splits * 2;
            float most = -__builtin_huge_valf();
            for (int i = lane; i < a.splits; i += 64) most = fmaxf(most, ms[2 * i]);
            most = wave_max(most);
            double sum = 0.0;
            for (int i = lane; i < a.splits; i += 64)
                sum += static_cast<double>(ms[2 * i + 1]) * exp(static_cast<double>(ms[2 * i]) - static_cast<double>(most));
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
            base -= static_cast<double>(most) + log(sum);
        }
        if (lane == 0) s_base[w] = base;
    }
    if (tid == 0) s_count = 0;
    __syncthreads();
    const int lists = a.W * a.splits;
    // Candidate `at` of a list: its score, -inf where there is none (NaN too), and its
    // beam and token in one number, which orders ties.
    const auto look = [&](int list, int at, double* score, int64_t* where) {
        *score = kNone;
        *where = 0;
        const int w = list / a.splits, s = list - w * a.splits;
        int token = a.end_token;
        double x = 0.0;
        if (ended(w)) {
            if (s > 0 || at > 0) return;
        } else {
            if (at >= a.k || !alive(w)) return;
            const BeamCandidate c = a.part[(row0 * a.splits + list) * a.k + at];
            token = c.token;
            if (token < 0) return;
            x = c.x;
        }
        const double v = s_base[w] + x;
        if (!(v > kNone)) return;
        *score = v;
        *where = static_cast<int64_t>(w) << 32 | token;
    };
    if (wave == 0) {
        uint32_t head[kHeadsPerLane];
#pragma unroll
        for (int n = 0; n < kHeadsPerLane; ++n) {
            double s = kNone;
            int64_t at;
            if (n * 64 + lane < lists) look(n * 64 + lane, 0, &s, &at);
            head[n] = s > kNone ? score_rank(s) : 0u;
        }
        // 20 bits: eight of a score's mantissa
        const uint32_t least = largest_with(20, a.k, [&](uint32_t t) {
            int c = 0;
#pragma unroll
            for (int n = 0; n < kHeadsPerLane; ++n) c += __popcll(__ballot(head[n] >= t));
            return c;
        });
        if (lane == 0) s_least = max(least, 1u);
    }
    __syncthreads();
    const uint32_t least = s_least;
    for (int i = tid; i < lists * a.k; i += kJoinThreads) {
        const int list = i / a.k;
        double s;
        int64_t at;
        look(list, i - list * a.k, &s, &at);
        if (s > kNone && score_rank(s) >= least) {
            const int p = atomicAdd(&s_count, 1);
            if (p < kJoined) {
                s_score[p] = s;
                s_where[p] = at;
            }
        }
    }
    __syncthreads();
    const int count = s_count;
    const auto write = [&](int c, double s, int64_t at) {
        const int64_t o = b * a.k + c;
        const bool none = !(s > kNone);
        a.out_scores[o] = none ? -__builtin_huge_valf() : static_cast<float>(s);
        a.parents[o] = none ? -1 : static_cast<int32_t>(at >> 32);
        a.tokens[o] = none ? -1 : static_cast<int32_t>(at);
    };
    if (count <= kJoined) {
        for (int i = tid; i < count; i += kJoinThreads) {
            const double s = s_score[i];
            const int64_t at = s_where[i];
            int place = 0;
            for (int j = 0; j < count; ++j) place += s_score[j] > s || (s_score[j] == s && s_where[j] < at) ? 1 : 0;
            if (place < a.k) write(place, s, at);
        }
        for (int c = count + tid; c < a.k; c += kJoinThreads) write(c, kNone, 0);
        return;
    }
    if (wave != 0) return;
    for (int i = 0; i < lists_per_lane; ++i) s_at[i * 64 + lane] = 0;
    double best = kNone;
    int64_t where = 0;
    int mine = 0;                                      // which of the lane's lists its best heads
    const auto heads = [&]() {
        best = kNone;
        for (int n = 0; n < lists_per_lane && n * 64 + lane < lists; ++n) {
            double s;
            int64_t at;
            look(n * 64 + lane, s_at[n * 64 + lane], &s, &at);
            if (s > best || (s == best && s > kNone && at < where)) {
                best = s;
                where = at;
                mine = n;
            }
        }
    };
    heads();
    for (int c = 0; c < a.k; ++c) {
        double top = best;
        int64_t at = where;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double s = __shfl_xor(top, o, 64);
            const int64_t p = __shfl_xor(at, o, 64);
            if (s > top || (s == top && p < at)) {
                top = s;
                at = p;
            }
        }
        if (lane == 0) write(c, top, at);
        if (top > kNone && best == top && where == at) {
            ++s_at[mine * 64 + lane];
            heads();
        }
    }
}

// ------------------------------------------------------------------- reorder
//
// Beam w goes on from beam p_w: the ids of its full pages become p_w's, and its last
// page, its own, takes the rows of p_w's. A lane holds one unit of the rows of all
// the beams of a request: it reads the parents' before it writes any, so beams may
// exchange places, and no other lane touches those bytes. Bound by memory.
template <typename U, int W>
__global__ __launch_bounds__(kReorderThreads) void reorder_rows_kernel(DescArg d, int layer_off, LayerMinor lm, KVGeom g,
                                                                       int es, const int32_t* block_table,
                                                                       const int32_t* __restrict__ parents,
                                                                       int64_t parent_stride, int n_lists,
                                                                       FastDiv inner, FastDiv mid, int token_inner,
                                                                       int head_units) {
    __shared__ int64_t s_from[kReorderBeams], s_to[kReorderBeams];   // bytes of the pages, -1: beam stays
    int l;
    int64_t item;
    lm.at(l, item);
    const DescPtr<BeamLists> lists = desc_at<BeamLists>(d, 0);
    const int li = find_by_tile(lists, n_lists, static_cast<int>(item));
    const BeamLists s = desc_load(lists + li);
    const int full = s.n_tokens / g.PS, rest = s.n_tokens - full * g.PS;
    const int tid = static_cast<int>(threadIdx.x);
    if (tid < s.n_beams) {
        const int32_t* last = block_table + s.bt_offset + full;
        const int p = parents[li * parent_stride + tid];
        s_from[tid] = -1;
        if (p >= 0 && p < s.n_beams && p != tid) {
            const int from = last[p * s.stride], to = last[tid * s.stride];
            if (from > 0 && from < g.num_blocks && to > 0 && to < g.num_blocks && from != to) {
                s_from[tid] = static_cast<int64_t>(from) * g.sb * es;
                s_to[tid] = static_cast<int64_t>(to) * g.sb * es;
            }
        }
    }
    __syncthreads();
    // unit -> (K or V, outer, inner, unit of the row); tokens are the inner index of
    // head-major pages, heads of the others
    const int units = (g.v_off >= 0 ? 2 : 1) * rest * g.H * head_units;
    const int i = (static_cast<int>(item) - s.tile_begin) * kReorderThreads + tid;
    if (i >= units) return;
    const int per_plane = rest * g.H * head_units;
    const int v = i >= per_plane ? 1 : 0;
    int r = i - v * per_plane;
    const int row = static_cast<int>(inner.div(static_cast<uint32_t>(r)));       // head_units
    const int u = r - row * head_units;
    int token, head;
    if (token_inner) {
        head = row / rest;
        token = row - head * rest;
    } else {
        token = static_cast<int>(mid.div(static_cast<uint32_t>(row)));           // H
        head = row - token * g.H;
    }
    uint8_t* base = desc_at<uint8_t*>(d, layer_off)[l] +
                    (static_cast<int64_t>(token) * g.ss + static_cast<int64_t>(head) * g.sh + (v != 0 ? g.v_off : 0)) * es +
                    static_cast<int64_t>(u) * static_cast<int>(sizeof(U));
    U x[W];
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < s.n_beams && s_from[w] >= 0) x[w] = *reinterpret_cast<const U*>(base + s_from[w]);
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < s.n_beams && s_from[w] >= 0) *reinterpret_cast<U*>(base + s_to[w]) = x[w];
}

// The ids of full pages: a lane holds one place of all the lists of a request.
template <int W>
__global__ __launch_bounds__(kReorderThreads) void reorder_lists_kernel(DescArg d, int32_t* block_table,
                                                                        const int32_t* __restrict__ parents,
                                                                        int64_t parent_stride, int page_size) {
    __shared__ int s_from[kReorderBeams];
    const BeamLists s = desc_load(desc_at<BeamLists>(d, 0) + blockIdx.y);
    const int tid = static_cast<int>(threadIdx.x);
    if (tid < s.n_beams) {
        const int p = parents[blockIdx.y * parent_stride + tid];
        s_from[tid] = p >= 0 && p < s.n_beams && p != tid ? p : -1;
    }
    __syncthreads();
    const int at = static_cast<int>(blockIdx.x) * kReorderThreads + tid;
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

}  // namespace

void launch_select_beams(const SelectArgs& a, int kind, int regs, hipStream_t stream) {
    const int64_t units = static_cast<int64_t>(a.B) * a.W * a.splits;
    const unsigned blocks = static_cast<unsigned>((units + kSplitsPerBlock - 1) / kSplitsPerBlock);
#define DARIC_SS(K)                                                                                   \
    do {                                                                                              \
        if (regs == 16) DARIC_LAUNCH((select_split_kernel<K, 16>), blocks, kSplitThreads, 0, stream, a); \
        else DARIC_LAUNCH((select_split_kernel<K, 64>), blocks, kSplitThreads, 0, stream, a);         \
    } while (0)
    if (kind == kBF16) DARIC_SS(kBF16);
    else if (kind == kF16) DARIC_SS(kF16);
    else DARIC_SS(kF32);
#undef DARIC_SS
    check_launch("select_beams");
    const int per_lane = (a.W * a.splits + 63) / 64;
    DARIC_LAUNCH(select_join_kernel, static_cast<unsigned>(a.B), kJoinThreads, static_cast<size_t>(per_lane) * 64, stream, a, per_lane);
    check_launch("select_beams join");
}

void launch_reorder(const DescArg& d, int layer_off, int n_layers, const KVGeom& g, int es, int unit,
                    int32_t* block_table, const int32_t* parents, int64_t parent_stride, int n_lists, int most_beams,
                    int64_t most_pages, int64_t tiles, hipStream_t stream) {
    const int head_units = g.D * es / unit;
    const FastDiv inner(static_cast<uint32_t>(head_units)), mid(static_cast<uint32_t>(g.H));
    const int token_inner = g.ss < g.sh ? 1 : 0;
    for_layer_minor(n_layers, tiles, [&](const LayerMinor& lm, unsigned blocks) {
#define DARIC_RW(U, W) DARIC_LAUNCH((reorder_rows_kernel<U, W>), blocks, kReorderThreads, 0, stream, d, layer_off, lm, g, \
                                    es, block_table, parents, parent_stride, n_lists, inner, mid, token_inner, head_units)
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
    });
    if (most_pages == 0) return;
    const dim3 grid(static_cast<unsigned>((most_pages + kReorderThreads - 1) / kReorderThreads), static_cast<unsigned>(n_lists));
    if (most_beams <= 8) DARIC_LAUNCH((reorder_lists_kernel<8>), grid, kReorderThreads, 0, stream, d, block_table, parents, parent_stride, g.PS);
    else DARIC_LAUNCH((reorder_lists_kernel<32>), grid, kReorderThreads, 0, stream, d, block_table, parents, parent_stride, g.PS);
    check_launch("reorder_beams lists");
}

}  // namespace daric
