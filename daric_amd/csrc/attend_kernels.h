// Attention over the paged KV cache, and the weight its tokens receive.
//
// Attention of a row r (one head of one query) over the tokens j it sees:
//   t_j = c <q_r, K_j>,  c = scale * k_scale * log2(e)
//   lse = (m + log2 l) ln 2,  l = sum_j 2^(t_j - m)
//   out = v_scale / l * sum_j 2^(t_j - m) V_j
// with the running maximum m, the sum l and the weighted rows kept in fp32
// over one pass of the tokens. The products run on the matrix cores as
// S^T = K Q^T and O^T = V^T P^T in tiles of 16 (rows of q in the columns) by
// 32 tokens: S^T leaves a lane with 2 x 4 consecutive tokens of one row, which
// is what the second product wants of P^T if V's tokens are taken in the same
// order, so the weights never leave their lanes. A lane reads, of those 8
// tokens, one slice of head_dim / 16 values of V and pairs the tokens' values
// with byte permutes: K and V go from memory to the matrix cores without LDS.
//
// e4m3 codes become bf16 or fp16 (q's type) exactly; the scales of a head act
// on c and on the result. The weights P are rounded to q's type for the second
// product, by at most half a step of it each, where the output is rounded to the
// same type; l sums them unrounded. fp16 has that step above 2^-14 only, and
// nothing below 2^-25: its weights are scaled (WeightRange).
#pragma once

#include <cmath>

#include "attend.h"
#include "elem.h"
#include "kernels.h"
#include "launch.h"

namespace daric {
namespace attend {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// A word at any element of a 16-bit type: `out` may begin at an odd one.
typedef uint32_t word_any __attribute__((aligned(2)));

constexpr float kLn2 = 0.693147180559945309f;

template <int QK>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (QK == kBF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
#else
    (void)a; (void)b;
    return c;
#endif
}

// The running maximum m of a row is kept so that weights 2^(t - m) use what q's type
// holds: a score t that passes it by more than OVER makes m = t - START, so the
// heaviest token met so far weighs 2^START to 2^OVER. bf16 has fp32's range: a new
// maximum weighs 1, and weights up to 2^8 save most tiles the exchange. fp16 holds half
// steps from 2^-14 to 2^16: the heaviest weighs 2^14 to 2^15, so weights down to 2^-28
// of it (19 in powers of e) keep their half step and lighter ones lose at most 2^-39 of
// it. (With a heaviest weight of 1 a token 17 below it in powers of e weighed 2^-24 for
// 2^-24.5, and one 18 below nothing.) Scores past 2^20 are so coarse in fp32 that START
// could be lost in their rounding: their maxima weigh 1.
template <int QK>
struct WeightRange {
    static constexpr bool FP16 = QK == kF16;
    static constexpr float START = FP16 ? 14.0f : 0.0f, OVER = FP16 ? 15.0f : 8.0f;
    static __device__ __forceinline__ float below(float t) {
        return FP16 && fabsf(t) < 1048576.0f ? t - START : t;
    }
    // log(l 2^m), without the factor 2^START that m and l both hold in fp16.
    static __device__ __forceinline__ float log_sum(float m, float l) {
        return (FP16 ? m + START + log2f(l * 0x1p-14f) : m + log2f(l)) * kLn2;
    }
};

// Two e4m3 codes (the low or high half of w) as a word of q's type.
template <int QK, bool HI>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (QK == kBF16)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
#else
    return w;
#endif
}

template <int QK>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const float p[2] = {lo, hi};
    return Elem<QK>::pack_word(p);
}

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_perm(hi, lo, sel);
#else
    (void)hi; (void)sel;
    return lo;
#endif
}

__device__ __forceinline__ float exp2_hw(float x) {
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_exp2f(x);
#else
    return x;
#endif
}

template <bool NT, typename W>
__device__ __forceinline__ W load_word(const W* p) {
    if constexpr (NT) return __builtin_nontemporal_load(p);
    else return *p;
}

// N words from p: one load of up to 16 bytes each, or (VALUES) value by value
// of ES bytes, the values from `left` on zero. NT: read once, not to be kept.
template <int N, int ES, bool VALUES, bool NT = false>
__device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* p, int left) {
    if constexpr (VALUES) {
        constexpr int PW = 4 / ES;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i] = 0;
#pragma unroll
            for (int b = 0; b < PW; ++b) {
                if (i * PW + b < left) {
                    const uint32_t v = ES == 2 ? *reinterpret_cast<const uint16_t*>(p + (i * PW + b) * ES)
                                               : p[i * PW + b];
                    w[i] |= v << (b * ES * 8);
                }
            }
        }
    } else if constexpr (N == 1) {
        w[0] = load_word<NT>(reinterpret_cast<const uint32_t*>(p));
    } else if constexpr (N == 2) {
        const u32x2 v = load_word<NT>(reinterpret_cast<const u32x2*>(p));
        w[0] = v[0]; w[1] = v[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 v = load_word<NT>(reinterpret_cast<const u32x4*>(p + i * 4));
            w[i] = v[0]; w[i + 1] = v[1]; w[i + 2] = v[2]; w[i + 3] = v[3];
        }
    }
}

// Where a lane (n = lane % 16, g = lane / 16) stands:
//   K, A operand of S^T, half h of the tile: token 16 h + n, values
//     kdim(step, g) .. + 7 of each step of 32
//   Q, B operand of S^T: row n, the same values
//   S^T: row n, tokens 16 h + 4 g + i
//   V, A operand of O^T: tokens 16 h + 4 g + i, values E n .. E n + E - 1
//   O^T: row n, value E (4 g + i) + e of matrix e
// A 16-byte unit of e4m3 K holds two steps' values.
template <int CK>
__device__ __forceinline__ int kdim(int step, int g) {
    return CK == kE4M3 ? 64 * (step >> 1) + 16 * g + 8 * (step & 1) : 32 * step + 8 * g;
}

// Rows of K and V of one tile as they lie in memory.
template <int CK, int DP>
struct TileRows {
    static constexpr int ES = CK == kE4M3 ? 1 : 2;
    static constexpr int KU = DP * ES / 64;        // 16-byte units of K per lane and half
    static constexpr int E = DP / 16;              // values of V per lane and token
    static constexpr int VW = E * ES / 4;          // words of them
    uint32_t k[2][KU][4];
    uint32_t v[8][VW];
    uint32_t ok;                                   // tokens that are there
};

// Where a tile's rows lie. PAGED: each half of 16 tokens lies in one page (pages
// of a multiple of 16 tokens), whose id all lanes share. Otherwise a lane holds
// the row of one token.
template <bool PAGED> struct TileAt;
template <> struct TileAt<true> {
    int32_t id[2], slot[2];
    int t0;
};
template <> struct TileAt<false> {
    int64_t row;
    bool there;
};

// Reads the rows of one KV head. A page id of 0 (the null block) or out of range
// has no tokens: they read a row of block 0 and count for nothing.
template <int CK, int DP, int MODE, bool PAGED>
struct RowReader {
    using Rows = TileRows<CK, DP>;
    using At = TileAt<PAGED>;
    static constexpr int ES = Rows::ES;
    const uint8_t* head;       // K row of block 0, slot 0
    const int32_t* bt;         // the sequence's block list
    int64_t sb, ss, v_off;     // bytes
    FastDiv page;
    int PS, D, num_blocks, n_total, last_page;
    int n, g;

    __device__ __forceinline__ void init(const AttArgs& a, int64_t bt_offset, int total, int h, int lane) {
        sb = a.g.sb * ES; ss = a.g.ss * ES; v_off = a.g.v_off * ES;
        head = a.layer + a.g.sh * ES * h;
        bt = a.block_table + bt_offset;
        page = a.page;
        PS = a.g.PS; D = a.g.D; num_blocks = a.g.num_blocks;
        n_total = total;
        last_page = static_cast<int>(page.div(static_cast<uint32_t>(total - 1)));
        n = lane & 15; g = lane >> 4;
    }
    __device__ __forceinline__ bool is_page(int id) const { return id > 0 && id < num_blocks; }
    // Offset of a token's row, and whether the token is there.
    __device__ __forceinline__ int64_t row_of(int t, bool* there) const {
        const int p = min(static_cast<int>(page.div(static_cast<uint32_t>(t))), last_page);
        const int id = bt[p];
        *there = t < n_total && is_page(id);
        const int slot = *there ? t - p * PS : 0;
        return static_cast<int64_t>(*there ? id : 0) * sb + static_cast<int64_t>(slot) * ss;
    }
    // Tile of tokens t0 .. t0 + 31.
    __device__ __forceinline__ At locate(int t0) const {
        At a;
        if constexpr (PAGED) {
            a.t0 = t0;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int t = t0 + 16 * hh;
                const int p = min(static_cast<int>(page.div(static_cast<uint32_t>(t))), last_page);
                a.id[hh] = uniform_load(bt + p);
                a.slot[hh] = t < n_total ? t - p * PS : 0;
            }
        } else {
            a.row = row_of(t0 + (16 * (g & 1) + n), &a.there);
        }
        return a;
    }
    __device__ __forceinline__ void load_k(uint32_t (*k)[4], const uint8_t* p) const {
#pragma unroll
        for (int u = 0; u < Rows::KU; ++u) {
            const int d = CK == kE4M3 ? 64 * u + 16 * g : 32 * u + 8 * g;
            if constexpr (MODE == kAttWhole) {
                load_words<4, ES, false>(k[u], p + d * ES, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) k[u][i] = 0;
                if (d < D) load_words<4, ES, MODE == kAttValues>(k[u], p + d * ES, D - d);
            }
        }
    }
    __device__ __forceinline__ void load_v(uint32_t* w, const uint8_t* p) const {
        const int d = Rows::E * n;
        if constexpr (MODE == kAttWhole) {
            load_words<Rows::VW, ES, false, true>(w, p + d * ES, 0);
        } else {
#pragma unroll
            for (int i = 0; i < Rows::VW; ++i) w[i] = 0;
            // slices of 8 values at most, each there or not as a whole
            constexpr int STEP = MODE != kAttValues && Rows::E > 8 ? 8 * ES / 4 : Rows::VW;
#pragma unroll
            for (int i = 0; i < Rows::VW; i += STEP) {
                const int di = d + i * 4 / ES;
                if (di < D) load_words<STEP, ES, MODE == kAttValues, true>(w + i, p + di * ES, D - di);
            }
        }
    }
    template <bool WITH_V>
    __device__ __forceinline__ void load(Rows& r, const At& a) const {
        if constexpr (PAGED) {
            r.ok = 0;
            const uint32_t k_lane = static_cast<uint32_t>(n * static_cast<int>(ss));
            const uint32_t v_lane = static_cast<uint32_t>(4 * g * static_cast<int>(ss));
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const bool is = is_page(a.id[hh]);
                const int left = n_total - a.t0 - 16 * hh;
                if (is && left > 0) r.ok |= (left >= 16 ? 0xffffu : (1u << left) - 1u) << (16 * hh);
                const uint8_t* p = head + static_cast<int64_t>(is ? a.id[hh] : 0) * sb + static_cast<int64_t>(a.slot[hh]) * ss;
                load_k(r.k[hh], p + k_lane);
                if constexpr (WITH_V) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) load_v(r.v[4 * hh + i], p + v_off + i * ss + v_lane);
                }
            }
        } else {
            // lane L has the row of token L % 32; the others get it from there
            r.ok = static_cast<uint32_t>(__ballot(a.there));
            const int lo = static_cast<int>(a.row), hi = static_cast<int>(a.row >> 32);
            const auto from = [&](int t) {
                return head + static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(__shfl(hi, t, 64))) << 32) |
                                                   static_cast<uint32_t>(__shfl(lo, t, 64)));
            };
            load_k(r.k[0], from(n));
            load_k(r.k[1], from(16 + n));
            if constexpr (WITH_V) {
#pragma unroll
                for (int j = 0; j < 8; ++j) load_v(r.v[j], from(16 * (j >> 2) + 4 * g + (j & 3)) + v_off);
            }
        }
    }
};

// One K operand of S^T.
template <int CK, int QK, int DP>
__device__ __forceinline__ u32x4 k_operand(const TileRows<CK, DP>& r, int half, int step) {
    if constexpr (CK == kE4M3) {
        const uint32_t* w = r.k[half][step >> 1] + 2 * (step & 1);
        return u32x4{e4m3_pair<QK, false>(w[0]), e4m3_pair<QK, true>(w[0]), e4m3_pair<QK, false>(w[1]),
                     e4m3_pair<QK, true>(w[1])};
    } else {
        const uint32_t* w = r.k[half][step];
        return u32x4{w[0], w[1], w[2], w[3]};
    }
}

// V operands of values e and e + 1 (e even): the lane's 8 tokens in order.
template <int CK, int QK, int DP>
__device__ __forceinline__ void v_operands(const TileRows<CK, DP>& r, int e, u32x4* lo, u32x4* hi) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (CK == kE4M3) {
            const uint32_t x = perm(r.v[2 * i + 1][e >> 2], r.v[2 * i][e >> 2], e & 2 ? 0x07030602u : 0x05010400u);
            (*lo)[i] = e4m3_pair<QK, false>(x);
            (*hi)[i] = e4m3_pair<QK, true>(x);
        } else {
            (*lo)[i] = perm(r.v[2 * i + 1][e >> 1], r.v[2 * i][e >> 1], 0x05040100u);
            (*hi)[i] = perm(r.v[2 * i + 1][e >> 1], r.v[2 * i][e >> 1], 0x07060302u);
        }
    }
}

// The row of q that matrix column `n` of row tile `rt` holds: query R / G,
// head R % G of the KV head's group.
struct QRow {
    int i;        // query of the sequence, -1: none
    int head;     // in all
};
__device__ __forceinline__ QRow q_row(const AttArgs& a, int n_rows, int h, int R) {
    QRow r;
    const int i = static_cast<int>(a.group.div(static_cast<uint32_t>(R)));
    r.i = i < n_rows ? i : -1;
    r.head = h * a.G + (R - i * a.G);
    return r;
}

template <int CK, int DP, int MODE>
__device__ __forceinline__ void load_q(const AttArgs& a, const AttSeq& s, const QRow& r, int g, u32x4 (&q)[DP / 32]) {
#pragma unroll
    for (int st = 0; st < DP / 32; ++st) {
        uint32_t w[4] = {0, 0, 0, 0};
        const int d = kdim<CK>(st, g);
        if (r.i >= 0 && (MODE == kAttWhole || d < a.g.D)) {
            const uint8_t* p = a.q + (static_cast<int64_t>(s.row0 + r.i) * a.q_row + r.head * a.q_head + d) * 2;
            load_words<4, 2, MODE == kAttValues>(w, p, a.g.D - d);
        }
        q[st] = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// Bit b: the query sees token t0 + b, if it is there (32 tokens).
__device__ __forceinline__ uint32_t row_sees(const AttArgs& a, const AttSeq& s, int i, int t0) {
    if (i < 0) return 0;
    const int d0 = t0 - s.n_ctx;                       // draft of the first token
    if (d0 <= -32) return ~0u;
    if (d0 >= s.n_rows) return 0;                      // no such drafts: no mask word of them either
    if (a.mask == nullptr) {
        const int c = i - d0 + 1;
        return c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1u;
    }
    const uint64_t* w = a.mask + static_cast<int64_t>(s.row0 + i) * a.words;
    if (d0 < 0) return ((1u << -d0) - 1u) | static_cast<uint32_t>(w[0] << -d0);
    const int at = d0 >> 6, sh = d0 & 63;
    uint64_t v = w[at] >> sh;
    if (sh > 32 && at + 1 < a.words) v |= w[at + 1] << (64 - sh);
    return static_cast<uint32_t>(v);
}

// The work item of block b, of n items whose KV head is their lowest digit:
// workgroups go to the 8 XCDs in turn, and the heads of one part of a sequence
// read the same pages, so they go to one XCD, whose address translations then
// cover an eighth of the pages.
__device__ __forceinline__ int xcd_item(int b, int n, const FastDiv& heads) {
    const int H = static_cast<int>(heads.d);
    const int set = b / (8 * H), in = b - set * 8 * H;
    const int left = min(8, n / H - set * 8);            // parts of this set
    const int h = in / left, p = in - h * left;
    return (set * 8 + p) * H + h;
}

// V of a draft may hold infinities and NaN, and a row that does not see the draft
// must not get 0 times them. Where a tile behind the cached tokens holds such
// values, they are taken out of the product (drop_odd) and the rows that see them
// marked, in two bits per row and value of the head: a sum with them is +inf (1),
// -inf (2) or NaN (3), whatever else is in it (mark_odd; rare, so slow and small).
template <int CK, int N>
__device__ __forceinline__ bool drop_odd(uint32_t (&w)[N]) {
    constexpr uint32_t EXP = CK == kBF16 ? 0x7f80u : CK == kF16 ? 0x7c00u : 0x7fu;
    constexpr int BITS = CK == kE4M3 ? 8 : 16;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int b = 0; b < 32; b += BITS)
            if ((w[i] & (EXP << b)) == (EXP << b)) {
                odd = true;
                w[i] &= ~(((1u << BITS) - 1u) << b);
            }
    return odd;
}
// Marks the `rows` rows from R0 on (rows of the head) that see tokens t0 .. + n of
// a sequence; a wavefront's work. marks: [rows][words] of LDS.
template <int CK>
__device__ __forceinline__ void mark_odd(const AttArgs& a, const uint8_t* v_head, const int32_t* bt, int n_ctx,
                                                   int n_rows, int row0, int t0, int n, int R0, int rows,
                                                   uint32_t* marks, int words) {
    constexpr int ES = CK == kE4M3 ? 1 : 2;
    const int lane = static_cast<int>(threadIdx.x) & 63;
#pragma unroll 1
    for (int t = t0; t < min(t0 + n, n_ctx + n_rows); ++t) {
        const int p = t / a.g.PS, id = bt[p];
        if (id <= 0 || id >= a.g.num_blocks) continue;
        const uint8_t* v = v_head + (static_cast<int64_t>(id) * a.g.sb + static_cast<int64_t>(t - p * a.g.PS) * a.g.ss) * ES;
#pragma unroll 1
        for (int d = lane; d < a.g.D; d += 64) {
            float x;
            if constexpr (CK == kE4M3) x = e4m3_to_f32(v[d]);
            else if constexpr (CK == kBF16) x = bf16_to_f32(reinterpret_cast<const uint16_t*>(v)[d]);
            else x = f16_to_f32(reinterpret_cast<const uint16_t*>(v)[d]);
            if (fabsf(x) <= 3.402823466e38f) continue;
            const uint32_t mark = (x != x ? 3u : x > 0.0f ? 1u : 2u) << (2 * (d & 15));
#pragma unroll 1
            for (int R = 0; R < rows; ++R) {
                const int i = (R0 + R) / a.G, b = t - n_ctx;
                if (i >= n_rows) break;
                const bool sees = b < 0 || (a.mask == nullptr ? b <= i
                    : ((a.mask[static_cast<int64_t>(row0 + i) * a.words + (b >> 6)] >> (b & 63)) & 1u) != 0);
                if (sees) atomicOr(&marks[R * words + (d >> 4)], mark);
            }
        }
    }
}
// A sum with its mark.
__device__ __forceinline__ float with_mark(float x, uint32_t word, int d) {
    const uint32_t mark = (word >> (2 * (d & 15))) & 3u;
    const float inf = __builtin_huge_valf();
    return mark == 0 ? x : mark == 1 ? x + inf : mark == 2 ? x - inf : __builtin_nanf("");
}

// ------------------------------------------------------------------ attend
// One workgroup: one KV head, 16 rows of q and one part of a sequence's tokens,
// whose tiles its wavefronts take in turn; they join in LDS at the end.
// Bound by memory: K and V are read once, by whole rows of a head. V is read past the
// caches; K, of which an instruction takes half a line of each row, must find the
// other half there. MI355X, one row to a sequence: 32 sequences of 310 to 8191 tokens
// (bf16, 8 KV heads of 128, 414 MB read from HBM) 67 us, 6.2 TB/s, where a plain read of
// as much takes 62; with K past the caches too 81, with V through them 86. Two sequences
// of 131072 and 100001 tokens, e4m3, 474 MB from HBM: 88 us, 5.4 TB/s; head-major pages
// 76.
template <int CK, int QK, int DP, int MODE, bool PAGED>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attend_kernel(DescArg d, AttArgs a) {
    using Rows = TileRows<CK, DP>;
    constexpr int E = Rows::E, STEPS = DP / 32, WAVES = 4;
    constexpr int LD = DP + 4;                        // floats of a row in LDS: no two rows on one bank
    __shared__ float s_o[WAVES][kAttRows][LD];
    __shared__ float s_m[WAVES][kAttRows], s_l[WAVES][kAttRows];
    __shared__ uint32_t s_mark[kAttRows][DP / 16], s_marked;
    const DescPtr<AttSeq> seqs = desc_at<AttSeq>(d, 0);
    const int item = xcd_item(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x), a.heads);
    const int si = __builtin_amdgcn_readfirstlane(find_by_tile(seqs, a.n_seqs, item));
    const AttSeq s = desc_load(seqs + si);
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    // item of the sequence: (part, row tile, head), the head first
    const int local = item - s.tile_begin;
    const int pr = static_cast<int>(a.heads.div(static_cast<uint32_t>(local)));
    const int h = local - pr * a.g.H;
    const int row_tiles = (s.n_rows * a.G + kAttRows - 1) / kAttRows;
    const int part = pr / row_tiles, rt = pr - part * row_tiles;
    const int total = s.n_ctx + s.n_rows;
    const QRow row = q_row(a, s.n_rows, h, rt * kAttRows + n);
    // causal: nothing behind the last row's own token is seen
    const int last_i = min(s.n_rows - 1, static_cast<int>(a.group.div(static_cast<uint32_t>(rt * kAttRows + kAttRows - 1))));
    const int end = a.mask == nullptr ? s.n_ctx + last_i + 1 : total;
    // the sequence's tiles in equal parts
    const int tiles = (total + kAttTile - 1) / kAttTile;
    const int part_tiles = (tiles + s.n_parts - 1) / s.n_parts;
    const int tile_end = min((part + 1) * part_tiles, (end + kAttTile - 1) / kAttTile);

    RowReader<CK, DP, MODE, PAGED> rd;
    rd.init(a, s.bt_offset, total, h, lane);
    u32x4 q[STEPS];
    load_q<CK, DP, MODE>(a, s, row, g, q);
    const float c = a.scale_log2 * (a.k_scale != nullptr ? a.k_scale[h] : 1.0f);
    f32x4 acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = f32x4{0, 0, 0, 0};
    float m = -3.402823466e38f, l = 0.0f;
    if (tid < kAttRows * (DP / 16)) (&s_mark[0][0])[tid] = 0;
    if (tid == 0) s_marked = 0;
    __syncthreads();

    const auto tile_of = [&](Rows& r, int tile) {
        const int t0 = tile * kAttTile;
        f32x4 sc[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            sc[0] = mfma<QK>(k_operand<CK, QK, DP>(r, 0, st), q[st], sc[0]);
            sc[1] = mfma<QK>(k_operand<CK, QK, DP>(r, 1, st), q[st], sc[1]);
        }
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = sc[j >> 2][j & 3] * c;
        const bool drafts = t0 + kAttTile > s.n_ctx;
        uint32_t vis = r.ok;
        if (r.ok != ~0u || drafts) {
            vis = r.ok & row_sees(a, s, row.i, t0);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int b = 16 * (j >> 2) + 4 * g + (j & 3);
                if (!((vis >> b) & 1u)) t[j] = -__builtin_huge_valf();
                if (!((r.ok >> b) & 1u)) {
#pragma unroll
                    for (int w = 0; w < Rows::VW; ++w) r.v[j][w] = 0;
                }
            }
        }
        // A new maximum only where a score passes the old one by so much: most tiles
        // then skip the exchange.
        float top = t[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, t[j]);
        if (__builtin_expect(__ballot(top - m > WeightRange<QK>::OVER) != 0, 0)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float mn = fmaxf(m, WeightRange<QK>::below(top));
            const float al = exp2_hw(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] *= al;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = exp2_hw(t[j] - m);
            l += p[j];
        }
        if (drafts) {
            bool odd = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) odd |= drop_odd<CK>(r.v[j]);
            if (__builtin_expect(__ballot(odd) != 0, 0)) {
                mark_odd<CK>(a, rd.head + rd.v_off, rd.bt, s.n_ctx, s.n_rows, s.row0, t0, kAttTile, rt * kAttRows, kAttRows,
                             &s_mark[0][0], DP / 16);
                if (lane == 0) s_marked = 1;
            }
        }
        const u32x4 pb = {pack2<QK>(p[0], p[1]), pack2<QK>(p[2], p[3]), pack2<QK>(p[4], p[5]), pack2<QK>(p[6], p[7])};
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            u32x4 lo, hi;
            v_operands<CK, QK, DP>(r, e, &lo, &hi);
            acc[e] = mfma<QK>(lo, pb, acc[e]);
            acc[e + 1] = mfma<QK>(hi, pb, acc[e + 1]);
        }
    };

    // A wavefront's next tile is on its way while it works on one, and the pages
    // of the one after that are known (rows of 256 values leave no registers for
    // a second tile).
    constexpr bool AHEAD = DP < 256;
    int tile = part * part_tiles + wave;
    if (tile < tile_end) {
        Rows cur;
        rd.template load<true>(cur, rd.locate(tile * kAttTile));
        auto at = rd.locate(min(tile + WAVES, tile_end - 1) * kAttTile);
        for (;;) {
            const int next = tile + WAVES;
            Rows coming;
            if (AHEAD && next < tile_end) {
                rd.template load<true>(coming, at);
                at = rd.locate(min(next + WAVES, tile_end - 1) * kAttTile);
            }
            tile_of(cur, tile);
            if (next >= tile_end) break;
            if constexpr (AHEAD) {
                cur = coming;
            } else {
                rd.template load<true>(cur, at);
                at = rd.locate(min(next + WAVES, tile_end - 1) * kAttTile);
            }
            tile = next;
        }
    }

    // Join the wavefronts.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) {
        s_m[wave][n] = m;
        s_l[wave][n] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) s_o[wave][n][E * (4 * g + i) + e] = acc[e][i];
    __syncthreads();
    // lane: row tid / 16, values V8 * (tid % 16) ..
    const int rn = tid >> 4, dc = (tid & 15) * E;
    const QRow orow = q_row(a, s.n_rows, h, rt * kAttRows + rn);
    float mm = s_m[0][rn];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, s_m[w][rn]);
    float ll = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float al = exp2_hw(s_m[w][rn] - mm);
        ll += s_l[w][rn] * al;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += s_o[w][rn][dc + e] * al;
    }
    if (orow.i < 0) return;
    if (s_marked) {
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = with_mark(o[e], s_mark[rn][(dc + e) >> 4], dc + e);
    }
    if (s.n_parts > 1) {
        float* po = a.part + (static_cast<int64_t>(item) * kAttRows + rn) * DP;
#pragma unroll
        for (int e = 0; e < E; ++e) po[dc + e] = o[e];
        if ((tid & 15) == 0) {
            float* pm = a.part_ml + (static_cast<int64_t>(item) * kAttRows + rn) * 2;
            pm[0] = mm;
            pm[1] = ll;
        }
        return;
    }
    const int64_t at = static_cast<int64_t>(s.row0 + orow.i) * a.Hq + orow.head;
    const float inv = ll == 0.0f ? 0.0f : (a.v_scale != nullptr ? a.v_scale[h] : 1.0f) / ll;
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + at * a.g.D;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float x = ll == 0.0f ? 0.0f : o[e] * inv;
        if (dc + e < a.g.D) out[dc + e] = static_cast<uint16_t>(QK == kBF16 ? f32_to_bf16(x) : f32_to_f16(x));
    }
    if ((tid & 15) == 0) a.lse[at] = ll == 0.0f ? -__builtin_huge_valf() : WeightRange<QK>::log_sum(mm, ll);
}

// -------------------------------------------------------- attend, many rows
// One workgroup: one KV head, 16 NT rows of q to each of WAVES wavefronts and one
// part of a sequence's tokens, in steps of 16 to a wavefront. K and V are staged in LDS as the
// operands of the matrix instructions lie in registers, a wavefront's operand in
// 1 KiB, so that reads and writes of it touch every bank alike: e4m3 becomes q's
// type and V's tokens are paired once per workgroup, and a read feeds NT
// instructions. The next step's rows come from memory meanwhile, into the other
// half of the LDS.
// Bound by products, softmax and staging, of which the two wavefronts of a SIMD overlap
// only a part: the matrix cores are busy 36% of the time, the vector unit issues 40%.
// MI355X, 2048 rows of 32 heads behind 6144 tokens (bf16, 8 KV heads of 128, 240
// GFLOP): 262 us, 918 TFLOP/s, where a library product of 8192 x 8192 x 8192 reaches
// 1208 (the first launches after a pause take 303 to 310, at lower clocks). Of 328 us of
// an earlier form, in first launches, 254 were left without the staging, 270 without the
// softmax, 185 without both; 256 rows to a workgroup 312, 128 rows 365, 64 rows 505 (the
// last before the staging was spread over the step). e4m3 263, fp16 282; heads of 64
// 193 (625 TFLOP/s), of 256 1481 (325).
template <int CK, int QK, int DP, int MODE, bool PAGED, int WAVES, int NT>
__global__ __launch_bounds__(WAVES * 64, DP == 256 ? 1 : 2) void attend_rows_kernel(DescArg d, AttArgs a) {
    using Rows = TileRows<CK, DP>;
    constexpr int E = Rows::E, STEPS = DP / 32, ROWS = WAVES * 16 * NT, STEP = WAVES * 16;
    constexpr int K_AT = 0, V_AT = WAVES * STEPS * 64, UNITS = V_AT + WAVES / 2 * E * 64;    // 16-byte units of a step
    __shared__ u32x4 s_kv[2][UNITS];
    __shared__ uint32_t s_ok[2][WAVES];
    __shared__ uint32_t s_mark[ROWS][DP / 16], s_marked;
    const DescPtr<AttSeq> seqs = desc_at<AttSeq>(d, 0);
    const int item = a.by_head ? static_cast<int>(blockIdx.x)
                               : xcd_item(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x), a.heads);
    const int si = __builtin_amdgcn_readfirstlane(find_by_tile(seqs, a.n_seqs, item));
    const AttSeq s = desc_load(seqs + si);
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int local = item - s.tile_begin;
    const int pr = static_cast<int>(a.heads.div(static_cast<uint32_t>(local)));
    const int h = local - pr * a.g.H;
    const int row_tiles = (s.n_rows * a.G + ROWS - 1) / ROWS;
    const int part = pr / row_tiles, rt = pr - part * row_tiles;
    const int total = s.n_ctx + s.n_rows;
    const int R0 = rt * ROWS + wave * 16 * NT;         // the wavefront's first row
    const auto query = [&](int R) { return min(s.n_rows - 1, static_cast<int>(a.group.div(static_cast<uint32_t>(R)))); };
    // tokens that some row of the workgroup, of the wavefront sees, and that all
    // rows of the wavefront see
    const bool causal = a.mask == nullptr;
    const int end = causal ? s.n_ctx + query(rt * ROWS + ROWS - 1) + 1 : total;
    const int wave_end = R0 < s.n_rows * a.G ? (causal ? s.n_ctx + query(R0 + 16 * NT - 1) + 1 : total) : 0;
    const int wave_all = causal ? s.n_ctx + query(R0) + 1 : s.n_ctx;
    const int steps = (total + STEP - 1) / STEP;
    const int part_steps = (steps + s.n_parts - 1) / s.n_parts;
    const int step0 = part * part_steps;
    const int step_end = min(step0 + part_steps, (end + STEP - 1) / STEP);

    RowReader<CK, DP, MODE, false> rd;
    rd.init(a, s.bt_offset, total, h, lane);
    // The scores' factor c is made positive by q's sign, so that a score of -inf
    // is a masked one; with c = 0 all scores are 0, of a zero q.
    float c = a.scale_log2 * (a.k_scale != nullptr ? a.k_scale[h] : 1.0f);
    const uint32_t q_keep = c == 0.0f ? 0u : ~0u, q_flip = c < 0.0f ? 0x80008000u : 0u;
    c = c == 0.0f ? 1.0f : fabsf(c);
    u32x4 q[NT][STEPS];
    int qi[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const QRow row = q_row(a, s.n_rows, h, R0 + t * 16 + n);
        qi[t] = row.i;
        load_q<CK, DP, MODE>(a, s, row, g, q[t]);
#pragma unroll
        for (int st = 0; st < STEPS; ++st) q[t][st] = (q[t][st] & q_keep) ^ q_flip;
    }
    constexpr bool SCALED = WeightRange<QK>::FP16;     // scores are scaled before they are compared
    f32x4 acc[NT][E];
    float m[NT], l[NT], limit[NT];                     // limit: scores beyond it need a new maximum
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = limit[t] = -3.402823466e38f;
        l[t] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[t][e] = f32x4{0, 0, 0, 0};
    }

    // A wavefront stages 16 of a step's tokens: all in one page (PAGED), or lane n
    // with the page of token n. The page is known a step before its rows are asked for.
    const int sub = wave >> 1, half = wave & 1;
    uint32_t sk[Rows::KU][4], sv[4][Rows::VW];
    uint32_t there_k = 0;
    int page_id = 0;
    const auto locate = [&](int step) {
        const int t = step * STEP + 16 * wave + (PAGED ? 0 : n);
        const int p = min(static_cast<int>(rd.page.div(static_cast<uint32_t>(t))), rd.last_page);
        page_id = PAGED ? uniform_load(rd.bt + p) : rd.bt[p];
    };
    const auto fetch = [&](int step) {
        const int t = step * STEP + 16 * wave + (PAGED ? 0 : n);
        const bool there = t < total && rd.is_page(page_id);
        const int p = static_cast<int>(rd.page.div(static_cast<uint32_t>(t)));
        const uint32_t id = there ? static_cast<uint32_t>(page_id) : 0u;
        const uint32_t slot = there ? static_cast<uint32_t>(t - p * rd.PS) : 0u;
        const int64_t row = static_cast<int64_t>(id) * rd.sb + static_cast<int64_t>(slot) * rd.ss;
        if constexpr (PAGED) {
            there_k = !there ? 0u : total - t >= 16 ? 0xffffu : (1u << (total - t)) - 1u;
            const uint8_t* base = rd.head + row;
            rd.load_k(sk, base + static_cast<uint32_t>(n * static_cast<int>(rd.ss)));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                rd.load_v(sv[i], base + rd.v_off + i * rd.ss + static_cast<uint32_t>(4 * g * static_cast<int>(rd.ss)));
        } else {
            there_k = static_cast<uint32_t>(__ballot(there)) & 0xffffu;
            const int lo = static_cast<int>(row), hi = static_cast<int>(row >> 32);
            rd.load_k(sk, rd.head + row);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int from = 4 * g + i;
                const int64_t o = static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(__shfl(hi, from, 64))) << 32) |
                                                       static_cast<uint32_t>(__shfl(lo, from, 64)));
                rd.load_v(sv[i], rd.head + rd.v_off + o);
            }
        }
    };
    const auto stage = [&](int step, int buf) {
        const int t = step * STEP + 16 * wave;
        if (there_k != 0xffffu) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < Rows::VW; ++w) sv[i][w] = (there_k >> (4 * g + i)) & 1u ? sv[i][w] : 0u;
        }
        if (t + 16 > s.n_ctx) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= drop_odd<CK>(sv[i]);
            if (__builtin_expect(__ballot(odd) != 0, 0)) {
                mark_odd<CK>(a, rd.head + rd.v_off, rd.bt, s.n_ctx, s.n_rows, s.row0, t, 16, rt * ROWS, ROWS,
                             &s_mark[0][0], DP / 16);
                if (lane == 0) s_marked = 1;
            }
        }
        if (lane == 0) s_ok[buf][wave] = there_k;
        u32x4* ks = &s_kv[buf][K_AT + (sub * 2 + half) * STEPS * 64 + lane];
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            if constexpr (CK == kE4M3) {
                const uint32_t* w = sk[st >> 1] + 2 * (st & 1);
                ks[st * 64] = u32x4{e4m3_pair<QK, false>(w[0]), e4m3_pair<QK, true>(w[0]), e4m3_pair<QK, false>(w[1]),
                                    e4m3_pair<QK, true>(w[1])};
            } else {
                ks[st * 64] = u32x4{sk[st][0], sk[st][1], sk[st][2], sk[st][3]};
            }
        }
        u32x2* vs = reinterpret_cast<u32x2*>(&s_kv[buf][V_AT + sub * E * 64 + lane]) + half;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            u32x2 lo, hi;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (CK == kE4M3) {
                    const uint32_t x = perm(sv[2 * i + 1][e >> 2], sv[2 * i][e >> 2], e & 2 ? 0x07030602u : 0x05010400u);
                    lo[i] = e4m3_pair<QK, false>(x);
                    hi[i] = e4m3_pair<QK, true>(x);
                } else {
                    lo[i] = perm(sv[2 * i + 1][e >> 1], sv[2 * i][e >> 1], 0x05040100u);
                    hi[i] = perm(sv[2 * i + 1][e >> 1], sv[2 * i][e >> 1], 0x07060302u);
                }
            }
            vs[e * 128] = lo;
            vs[e * 128 + 128] = hi;
        }
    };

    // The scores of tile sb of a step, -inf where masked. K's operands are all asked
    // for at once.
    const auto scores = [&](f32x4 (&sc)[NT][2], int t0, int buf, int sb) {
        const u32x4* ks = &s_kv[buf][K_AT + sb * 2 * STEPS * 64 + lane];
        const uint32_t ok = __builtin_amdgcn_readfirstlane(s_ok[buf][2 * sb] | (s_ok[buf][2 * sb + 1] << 16));
        u32x4 kf[2 * STEPS];
#pragma unroll
        for (int i = 0; i < 2 * STEPS; ++i) kf[i] = ks[i * 64];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = f32x4{0, 0, 0, 0};
        __builtin_amdgcn_s_setprio(1);
        // 2 NT sums in turn: an instruction that waits for its own sum stalls
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int t = 0; t < NT; ++t) sc[t][hh] = mfma<QK>(kf[hh * STEPS + st], q[t][st], sc[t][hh]);
        __builtin_amdgcn_s_setprio(0);
        if (__builtin_expect(ok != ~0u || t0 + kAttTile > wave_all, 0)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t vis = ok & row_sees(a, s, qi[t], t0);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!((vis >> (16 * (j >> 2) + 4 * g + (j & 3))) & 1u)) sc[t][j >> 2][j & 3] = -__builtin_huge_valf();
            }
        }
        if constexpr (SCALED) {
#pragma unroll
            for (int t = 0; t < NT; ++t) sc[t][0] *= c, sc[t][1] *= c;
        }
    };
    const auto top_of = [&](const f32x4 (&sc)[NT][2], int t) {
        float top = sc[t][0][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, sc[t][j >> 2][j & 3]);
        return top;
    };
    // With bf16 weights the sums are never scaled: a scaling on a side way through the
    // loop moved them to other registers and back in every tile (38 of its 190
    // instructions). A row's maximum is that of the first tile in which it sees a token,
    // and weights up to 2^14 of it are as exact. A wavefront whose scores pass that takes
    // its rows' maxima in a second pass over the tokens and its sums in a third: 2048 rows
    // whose heaviest token, 16 powers of 2 above the rest, comes late take 623 us, 264
    // where it is the first or none is; eight trees of up to 61 drafts 137 and 72.
    // fp16 weights have no such range to spare (WeightRange): sums are scaled where a
    // score passes the maximum by 2^OVER, in one pass: 288 to 298 us wherever the heaviest
    // stands (276 without the scaling).
    constexpr float LOWEST = -3.402823466e38f;
    enum { kFirst, kMaxima, kLast, kDone };
    int pass = wave_end > 0 ? kFirst : kDone;
    bool failed = false;
    // Past 2^20 the product c times a score may be rounded by more than the weights'
    // range: there it is rounded for the score as it was for the maximum (c_in is 1).
    bool far = false;
    float c_in = c;
    // The rows in registers go to LDS, and the next ones are asked for, in the middle
    // of a step's tiles, by the two wavefronts of a SIMD at different tiles, so that
    // one of them feeds the matrix cores meanwhile.
    const int stage_at = WAVES == 8 && wave < 4 ? 1 : WAVES / 2 - 1;
    const auto stage_next = [&](int step, int buf) {
        if (step + 1 >= step_end) return;
        stage(step + 1, buf ^ 1);
        if (step + 2 >= step_end) return;
        fetch(step + 2);
        locate(min(step + 3, steps - 1));
    };
    const auto attend_tiles = [&](int step, int buf, int tiles) {
#pragma unroll 1
        for (int sb = 0; sb < WAVES / 2; ++sb) {
            if (sb == stage_at) stage_next(step, buf);
            if (sb >= tiles || failed) continue;
            const int t0 = step * STEP + sb * kAttTile;
            const u32x4* vs = &s_kv[buf][V_AT + sb * E * 64 + lane];
            f32x4 sc[NT][2];
            scores(sc, t0, buf, sb);
            bool over = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
                over |= SCALED ? top_of(sc, t) - m[t] > WeightRange<QK>::OVER : top_of(sc, t) > limit[t];
            if (SCALED && __builtin_expect(__ballot(over) != 0, 0)) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float top = top_of(sc, t);
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float mn = fmaxf(m[t], WeightRange<QK>::below(top));
                    const float al = exp2_hw(m[t] - mn);
                    m[t] = mn;
                    l[t] *= al;
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[t][e] *= al;
                }
            } else if (!SCALED && __builtin_expect(__ballot(over) != 0, 0)) {
                bool known = false;                    // a row with a maximum, and sums, already
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float top = top_of(sc, t);
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    if (top > limit[t]) {
                        known |= m[t] != LOWEST;
                        m[t] = fmaxf(m[t], top * c);
                        limit[t] = pass == kMaxima ? top : fmaxf((m[t] + 14.0f) / c, top);
                        far |= fabsf(m[t]) > 1048576.0f;
                    }
                }
                far = __ballot(far) != 0;
                c_in = far ? 1.0f : c;
                if (pass == kFirst && __ballot(known) != 0) {
                    failed = true;
                    continue;
                }
            }
            if (pass == kMaxima) continue;
            if (__builtin_expect(far, 0)) {
#pragma unroll
                for (int t = 0; t < NT; ++t) sc[t][0] *= c, sc[t][1] *= c;
            }
            constexpr int VF = E < 8 ? E : 8;          // V operands read at once
            u32x4 vf[VF];
#pragma unroll
            for (int e = 0; e < VF; ++e) vf[e] = vs[e * 64];
            __builtin_amdgcn_sched_barrier(0);
            u32x4 pb[NT];
            const auto softmax = [&](int t) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = sc[t][j >> 2][j & 3];
                    p[j] = exp2_hw(SCALED ? x - m[t] : fmaf(x, c_in, -m[t]));
                    l[t] += p[j];
                }
                pb[t] = u32x4{pack2<QK>(p[0], p[1]), pack2<QK>(p[2], p[3]), pack2<QK>(p[4], p[5]), pack2<QK>(p[6], p[7])};
            };
            softmax(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (t + 1 < NT) softmax(t + 1);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[t][e] = mfma<QK>(e < VF ? vf[e % VF] : vs[e * 64], pb[t], acc[t][e]);
                if (t + 1 < NT) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 5, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };

    for (int i = tid; i < ROWS * (DP / 16); i += WAVES * 64) (&s_mark[0][0])[i] = 0;
    if (tid == 0) s_marked = 0;
    __syncthreads();
    if (step0 < step_end) {
#pragma unroll 1
        for (;;) {
            if (pass != kDone) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    l[t] = 0.0f;
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[t][e] = f32x4{0, 0, 0, 0};
                }
            }
            locate(step0);
            fetch(step0);
            locate(min(step0 + 1, steps - 1));
            stage(step0, 0);
            if (step0 + 1 < step_end) {
                fetch(step0 + 1);
                locate(min(step0 + 2, steps - 1));
            }
            __syncthreads();
#pragma unroll 1
            for (int step = step0; step < step_end; ++step) {
                const int tiles = pass == kDone
                                      ? 0 : min(WAVES / 2, (wave_end - step * STEP + kAttTile - 1) / kAttTile);
                attend_tiles(step, (step - step0) & 1, tiles);
                __syncthreads();
            }
            pass = failed ? kMaxima : pass == kMaxima ? kLast : kDone;
            failed = false;
            if (__builtin_expect(__syncthreads_or(pass != kDone) == 0, 1)) break;
            if (pass == kLast) {
#pragma unroll
                for (int t = 0; t < NT; ++t) limit[t] = __builtin_huge_valf();
            }
        }
    }

    const float vsc = a.v_scale != nullptr ? a.v_scale[h] : 1.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        l[t] += __shfl_xor(l[t], 16, 64);
        l[t] += __shfl_xor(l[t], 32, 64);
        if (qi[t] < 0) continue;
        const int R = R0 + t * 16 + n;
        if (s_marked) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int dd = E * (4 * g + i) + e;
                    acc[t][e][i] = with_mark(acc[t][e][i], s_mark[wave * 16 * NT + t * 16 + n][dd >> 4], dd);
                }
        }
        if (s.n_parts > 1) {
            const int64_t at = static_cast<int64_t>(item) * ROWS + wave * 16 * NT + t * 16 + n;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) a.part[at * DP + E * (4 * g + i) + e] = acc[t][e][i];
            if (g == 0) {
                a.part_ml[at * 2] = m[t];
                a.part_ml[at * 2 + 1] = l[t];
            }
            continue;
        }
        const int64_t at = static_cast<int64_t>(s.row0 + qi[t]) * a.Hq + h * a.G + (R - qi[t] * a.G);
        const float inv = vsc / l[t];
        uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + at * a.g.D;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const int dd = E * (4 * g + i) + e;
                if (MODE != kAttWhole && dd >= a.g.D) continue;      // head_dim is even here
                const float x0 = l[t] == 0.0f ? 0.0f : acc[t][e][i] * inv, x1 = l[t] == 0.0f ? 0.0f : acc[t][e + 1][i] * inv;
                *reinterpret_cast<word_any*>(out + dd) = pack2<QK>(x0, x1);
            }
        if (g == 0) a.lse[at] = l[t] == 0.0f ? -__builtin_huge_valf() : WeightRange<QK>::log_sum(m[t], l[t]);
    }
}

// Joins the parts of the rows of q (one head of one query each), 32 lanes to a
// row and part in turn, PG parts of a row at once. The parts' maxima come first,
// a lane each, so that no load waits for another: with one lane walking all 61
// parts of a row the join of two long sequences took 94 us, as long as their
// attention.
template <int QK, int DP, int PG>
__global__ __launch_bounds__(256) void attend_join_kernel(DescArg d, AttArgs a, int n_rows) {
    constexpr int V = DP / 32, ROWS = 8 / PG;
    __shared__ float s_o[8][DP];
    __shared__ float s_l[8];
    const DescPtr<AttSeq> seqs = desc_at<AttSeq>(d, 0);
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, slot = tid >> 5;
    const int pg = slot % PG;
    const int r = static_cast<int>(blockIdx.x) * ROWS + slot / PG;
    int lo = 0, hi = a.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (seqs[mid].at <= r) lo = mid; else hi = mid - 1;
    }
    const int parts = r < n_rows ? seqs[lo].n_parts : 0;
    if (PG == 1 && parts <= 1) return;
    const int local = r - seqs[lo].at;
    const int i = local / a.Hq, head = local - i * a.Hq;
    const int h = static_cast<int>(a.group.div(static_cast<uint32_t>(head)));
    const int R = i * a.G + head - h * a.G;
    const int row_tiles = (seqs[lo].n_rows * a.G + a.tile_rows - 1) / a.tile_rows;
    const int rt = R / a.tile_rows;
    const int64_t first = (static_cast<int64_t>(seqs[lo].tile_begin) + rt * a.g.H + h) * a.tile_rows + (R - rt * a.tile_rows);
    const int64_t step = static_cast<int64_t>(row_tiles) * a.g.H * a.tile_rows;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first;
    float mm = -3.402823466e38f;
    for (int p = lane; p < parts; p += 32) mm = fmaxf(mm, ml[p * step].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor(mm, x, 64));
    float ll = 0.0f, o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = 0.0f;
    const float* po = a.part + first * DP + lane * V;
#pragma unroll 4
    for (int p = pg; p < parts; p += PG) {
        const float2 x = ml[p * step];
        const float al = exp2_hw(x.x - mm);
        ll += x.y * al;
        const float* src = po + p * step * DP;
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] += src[v] * al;
    }
    if constexpr (PG > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) s_o[slot][lane * V + v] = o[v];
        if (lane == 0) s_l[slot] = ll;
        __syncthreads();
        if (pg != 0 || parts <= 1) return;
#pragma unroll
        for (int x = 1; x < PG; ++x) {
            ll += s_l[slot + x];
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] += s_o[slot + x][lane * V + v];
        }
    }
    const int64_t at = static_cast<int64_t>(seqs[lo].row0 + i) * a.Hq + head;
    const float inv = (a.v_scale != nullptr ? a.v_scale[h] : 1.0f) / ll;
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + at * a.g.D;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float x = ll == 0.0f ? 0.0f : o[v] * inv;
        if (lane * V + v < a.g.D) out[lane * V + v] = static_cast<uint16_t>(QK == kBF16 ? f32_to_bf16(x) : f32_to_f16(x));
    }
    if (lane == 0) a.lse[at] = ll == 0.0f ? -__builtin_huge_valf() : WeightRange<QK>::log_sum(mm, ll);
}

// Sums 8 values over the 16 lanes of a group: a lane of n < 8 gets the sum of
// value sum_of(n). Each step exchanges half of what is left, 8 exchanges in all
// (32 where every value goes through every step).
__device__ __forceinline__ int sum_of(int n) { return 4 * (n & 1) + (n & 2) + ((n >> 2) & 1); }
template <int W>
__device__ __forceinline__ void sum_halves(float (&v)[8], int n) {
    const bool up = (n & (4 / W)) != 0;
#pragma unroll
    for (int k = 0; k < W; ++k) {
        const float lo = v[k], hi = v[k + W];
        v[k] = (up ? hi : lo) + __shfl_xor(up ? lo : hi, 4 / W, 64);
    }
}
__device__ __forceinline__ float sum_group(float (&v)[8], int n) {
    sum_halves<4>(v, n);
    sum_halves<2>(v, n);
    sum_halves<1>(v, n);
    return v[0] + __shfl_xor(v[0], 8, 64);
}

// ------------------------------------------------------------------- weigh
// One workgroup: one KV head, 128 tokens, 32 to a wavefront, whose K rows stay
// in registers while all rows of the sequence pass (a few, or any of odd layouts).
// Bound by memory, and by the wait for it (57% of the wavefronts' time): the batch of
// attend_kernel, 213 MB of K from HBM, 42 us, 5.1 TB/s (45 by weigh_rows_kernel, 53 with
// K past the caches). Each token's sum is one
// lane's, then 16 lanes', in a fixed order.
template <int CK, int QK, int DP, int MODE, bool PAGED>
__global__ __launch_bounds__(256) void weigh_kernel(DescArg d, AttArgs a) {
    using Rows = TileRows<CK, DP>;
    constexpr int STEPS = DP / 32;
    const DescPtr<AttSeq> seqs = desc_at<AttSeq>(d, 0);
    const int item = xcd_item(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x), a.heads);
    const int si = __builtin_amdgcn_readfirstlane(find_by_tile(seqs, a.n_seqs, item));
    const AttSeq s = desc_load(seqs + si);
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int local = item - s.tile_begin;
    const int tg = static_cast<int>(a.heads.div(static_cast<uint32_t>(local)));
    const int h = local - tg * a.g.H;
    const int total = s.n_ctx + s.n_rows;
    const int t0 = tg * kWeighTokens + wave * kAttTile;
    if (t0 >= total) return;
    RowReader<CK, DP, MODE, PAGED> rd;
    rd.init(a, s.bt_offset, total, h, lane);
    Rows r;
    rd.template load<false>(r, rd.locate(t0));
    const float c = a.scale_log2 * (a.k_scale != nullptr ? a.k_scale[h] : 1.0f);
    const bool edge = r.ok != ~0u || t0 + kAttTile > s.n_ctx;
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = 0.0f;
    const int rows = s.n_rows * a.G;
    for (int R0 = 0; R0 < rows; R0 += kAttRows) {
        const QRow row = q_row(a, s.n_rows, h, R0 + n);
        u32x4 q[STEPS];
        load_q<CK, DP, MODE>(a, s, row, g, q);
        const float lse = row.i >= 0 ? a.lse[static_cast<int64_t>(s.row0 + row.i) * a.Hq + row.head] * (1.0f / kLn2)
                                     : -__builtin_huge_valf();
        f32x4 sc[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            sc[0] = mfma<QK>(k_operand<CK, QK, DP>(r, 0, st), q[st], sc[0]);
            sc[1] = mfma<QK>(k_operand<CK, QK, DP>(r, 1, st), q[st], sc[1]);
        }
        // a row that saw nothing (lse -inf) gives no weight
        uint32_t vis = lse == -__builtin_huge_valf() ? 0u : r.ok;
        if (edge) vis &= row_sees(a, s, row.i, t0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = exp2_hw(fmaf(sc[j >> 2][j & 3], c, -lse));
            const int b = 16 * (j >> 2) + 4 * g + (j & 3);
            sum[j] += (vis >> b) & 1u ? x : 0.0f;
        }
    }
    const float mine = sum_group(sum, n);
    const int j = sum_of(n), t = t0 + 16 * (j >> 2) + 4 * g + (j & 3);
    if (n < 8 && t < total) {
        float* w = a.weights + h * a.columns + s.at + t;
        *w = a.add ? *w + mine : mine;
    }
}

// ------------------------------------------------------- weigh, many rows
// A wavefront's 64 tokens: K as operands, and the tokens' sums.
template <int CK, int QK, int DP, int MODE>
struct WeighTokens {
    using Rows = TileRows<CK, DP>;
    static constexpr int STEPS = DP / 32;
    u32x4 k[2][2][STEPS];
    uint32_t ok[2];
    float sum[2][8];
    float c;
    int t0, n, g;
    bool edge;

    __device__ __forceinline__ void init(const AttArgs& a, const AttSeq& s, int h, int first, int lane) {
        const int total = s.n_ctx + s.n_rows;
        RowReader<CK, DP, MODE, false> rd;
        rd.init(a, s.bt_offset, total, h, lane);
        t0 = first;
        n = lane & 15; g = lane >> 4;
        c = a.scale_log2 * (a.k_scale != nullptr ? a.k_scale[h] : 1.0f);
        edge = t0 + 2 * kAttTile > s.n_ctx;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            Rows r;
            rd.template load<false>(r, rd.locate(t0 + b * kAttTile));
            ok[b] = __builtin_amdgcn_readfirstlane(r.ok);
            edge = edge || ok[b] != ~0u;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int st = 0; st < STEPS; ++st) k[b][hh][st] = k_operand<CK, QK, DP>(r, hh, st);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[b][j] = 0.0f;
        }
    }
    // Adds the weights of the 16 rows from R on; lse: of row n, in powers of 2.
    __device__ __forceinline__ void add(const AttArgs& a, const AttSeq& s, const u32x4 (&q)[STEPS], float lse, int R) {
        f32x4 sc[2][2];
#pragma unroll
        for (int b = 0; b < 2; ++b) sc[b][0] = sc[b][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) sc[b][hh] = mfma<QK>(k[b][hh][st], q[st], sc[b][hh]);
        // a row that saw nothing, or is none, gives no weight
        const bool dead = lse == -__builtin_huge_valf();
        if (__builtin_expect(edge || __ballot(dead) != 0, 0)) {
            const int i = static_cast<int>(a.group.div(static_cast<uint32_t>(R + n)));
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint32_t vis = dead || i >= s.n_rows ? 0u : ok[b] & row_sees(a, s, i, t0 + b * kAttTile);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = exp2_hw(fmaf(sc[b][j >> 2][j & 3], c, -lse));
                    sum[b][j] += (vis >> (16 * (j >> 2) + 4 * g + (j & 3))) & 1u ? x : 0.0f;
                }
            }
        } else {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[b][j] += exp2_hw(fmaf(sc[b][j >> 2][j & 3], c, -lse));
        }
    }
};
template <int CK, int DP, int MODE>
__device__ __forceinline__ float load_row(const AttArgs& a, const AttSeq& s, int h, int R, int g, u32x4 (&q)[DP / 32]) {
    const QRow row = q_row(a, s.n_rows, h, R);
    load_q<CK, DP, MODE>(a, s, row, g, q);
    return row.i >= 0 ? a.lse[static_cast<int64_t>(s.row0 + row.i) * a.Hq + row.head] * (1.0f / kLn2) : -__builtin_huge_valf();
}

// One workgroup: one KV head, 256 tokens, 64 to a wavefront, whose K operands stay
// in registers while the rows pass through LDS as operands, 64 at a time, one
// matrix tile staged by each wavefront and read by all. Bound by neither unit alone: the
// vector unit issues 44% of the time (16 exponentials of a quarter of its rate per lane to
// 16 matrix instructions), the matrix cores are busy 25%, and the wavefronts wait 42% of
// theirs: each tile's exponentials follow its products. MI355X, the last 64 rows of 64
// heads against 32768 and 20064 tokens, e4m3, 55 GFLOP: 83 us, 667 TFLOP/s (204 us by
// weigh_kernel).
template <int CK, int QK, int DP, int MODE>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 3) void weigh_rows_kernel(DescArg d, AttArgs a) {
    constexpr int STEPS = DP / 32, WAVES = 4, STEP = WAVES * kAttRows;
    __shared__ u32x4 s_q[2][WAVES][STEPS][64];
    __shared__ float s_lse[2][WAVES][kAttRows];
    const DescPtr<AttSeq> seqs = desc_at<AttSeq>(d, 0);
    const int item = xcd_item(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x), a.heads);
    const int si = __builtin_amdgcn_readfirstlane(find_by_tile(seqs, a.n_seqs, item));
    const AttSeq s = desc_load(seqs + si);
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int local = item - s.tile_begin;
    const int tg = static_cast<int>(a.heads.div(static_cast<uint32_t>(local)));
    const int h = local - tg * a.g.H;
    const int first = tg * kWeighRowsTokens;
    WeighTokens<CK, QK, DP, MODE> w;
    w.init(a, s, h, first + wave * 2 * kAttTile, lane);
    const int rows = s.n_rows * a.G;
    u32x4 sq[STEPS];
    float sl = 0.0f;
    const auto stage = [&](int buf) {
#pragma unroll
        for (int st = 0; st < STEPS; ++st) s_q[buf][wave][st][lane] = sq[st];
        if (g == 0) s_lse[buf][wave][n] = sl;
    };
    // causal: the first tokens' rows come first
    const int R_first = a.mask == nullptr ? max(0, first - s.n_ctx) * a.G / STEP * STEP : 0;
    sl = load_row<CK, DP, MODE>(a, s, h, R_first + wave * kAttRows + n, g, sq);
    stage(0);
    __syncthreads();
#pragma unroll 1
    for (int R = R_first; R < rows; R += STEP) {
        const int buf = (R - R_first) / STEP & 1;
        if (R + STEP < rows) sl = load_row<CK, DP, MODE>(a, s, h, R + STEP + wave * kAttRows + n, g, sq);
        const int tiles = min(WAVES, (rows - R + kAttRows - 1) / kAttRows);
#pragma unroll 1
        for (int t = 0; t < tiles; ++t) {
            u32x4 q[STEPS];
#pragma unroll
            for (int st = 0; st < STEPS; ++st) q[st] = s_q[buf][t][st][lane];
            w.add(a, s, q, s_lse[buf][t][n], R + t * kAttRows);
        }
        if (R + STEP < rows) stage(buf ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const float mine = sum_group(w.sum[b], n);
        const int j = sum_of(n), t = w.t0 + b * kAttTile + 16 * (j >> 2) + 4 * g + (j & 3);
        if (n < 8 && t < s.n_ctx + s.n_rows) {
            float* o = a.weights + h * a.columns + s.at + t;
            *o = a.add ? *o + mine : mine;
        }
    }
}

// The same where the tokens are few: 64 to a workgroup, whose 8 wavefronts take the
// rows' tiles in turn from memory and join in LDS.
template <int CK, int QK, int DP, int MODE>
__global__ __launch_bounds__(512, 2) void weigh_split_kernel(DescArg d, AttArgs a) {
    constexpr int STEPS = DP / 32, WAVES = 8;
    __shared__ float s_sum[WAVES][2 * kAttTile];
    const DescPtr<AttSeq> seqs = desc_at<AttSeq>(d, 0);
    const int item = xcd_item(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x), a.heads);
    const int si = __builtin_amdgcn_readfirstlane(find_by_tile(seqs, a.n_seqs, item));
    const AttSeq s = desc_load(seqs + si);
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int local = item - s.tile_begin;
    const int tg = static_cast<int>(a.heads.div(static_cast<uint32_t>(local)));
    const int h = local - tg * a.g.H;
    const int first = tg * kWeighSplitTokens;
    WeighTokens<CK, QK, DP, MODE> w;
    w.init(a, s, h, first, lane);
    const int rows = s.n_rows * a.G;
    constexpr int STEP = WAVES * kAttRows;
    int R = (a.mask == nullptr ? max(0, first - s.n_ctx) * a.G / STEP * STEP : 0) + wave * kAttRows;
    if (R < rows) {
        u32x4 q[STEPS];
        float l = load_row<CK, DP, MODE>(a, s, h, R + n, g, q);
#pragma unroll 1
        for (;;) {
            u32x4 next[STEPS];
            float nl = 0.0f;
            if (R + STEP < rows) nl = load_row<CK, DP, MODE>(a, s, h, R + STEP + n, g, next);
            w.add(a, s, q, l, R);
            R += STEP;
            if (R >= rows) break;
            for (int st = 0; st < STEPS; ++st) q[st] = next[st];
            l = nl;
        }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const float mine = sum_group(w.sum[b], n);
        const int j = sum_of(n);
        if (n < 8) s_sum[wave][b * kAttTile + 16 * (j >> 2) + 4 * g + (j & 3)] = mine;
    }
    __syncthreads();
    if (tid < 2 * kAttTile && first + tid < s.n_ctx + s.n_rows) {
        float x = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) x += s_sum[v][tid];
        float* o = a.weights + h * a.columns + s.at + first + tid;
        *o = a.add ? *o + x : x;
    }
}

// Instances of the kernels for one pair of cache and query types.
template <typename F>
void for_forms(int dp, int mode, bool paged, F&& f) {
    using std::integral_constant;
    const auto with = [&](auto dpc) {
        if (mode == kAttValues) f(dpc, integral_constant<int, kAttValues>(), std::false_type());
        else if (mode == kAttPadded && paged) f(dpc, integral_constant<int, kAttPadded>(), std::true_type());
        else if (mode == kAttPadded) f(dpc, integral_constant<int, kAttPadded>(), std::false_type());
        else if (paged) f(dpc, integral_constant<int, kAttWhole>(), std::true_type());
        else f(dpc, integral_constant<int, kAttWhole>(), std::false_type());
    };
    if (dp == 64) with(integral_constant<int, 64>());
    else if (dp == 128) with(integral_constant<int, 128>());
    else with(integral_constant<int, 256>());
}

template <int CK, int QK>
void run_attend(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    if (p.row_tile > 0) {
        const auto with = [&](auto dp, auto mode, auto paged, auto waves, auto nt) {
            DARIC_LAUNCH((attend_rows_kernel<CK, QK, decltype(dp)::value, decltype(mode)::value, decltype(paged)::value,
                                             decltype(waves)::value, decltype(nt)::value>),
                         static_cast<unsigned>(p.items), decltype(waves)::value * 64, 0, stream, d, a);
        };
        // pages of other sizes: the padded form for whole heads too
        for_forms(p.dp, p.paged ? p.mode : static_cast<int>(kAttPadded), p.paged, [&](auto dp, auto mode, auto paged) {
            using std::integral_constant;
            if constexpr (decltype(mode)::value == kAttPadded || (decltype(mode)::value == kAttWhole && decltype(paged)::value)) {
                if (p.row_tile == 1) with(dp, mode, paged, integral_constant<int, 4>(), integral_constant<int, 1>());
                else if constexpr (decltype(dp)::value < 256) {
                    if (p.row_tile == 2) with(dp, mode, paged, integral_constant<int, 4>(), integral_constant<int, 2>());
                    else with(dp, mode, paged, integral_constant<int, 8>(), integral_constant<int, 2>());
                }
            }
        });
        check_launch("attend_pages");
        return;
    }
    for_forms(p.dp, p.mode, p.paged, [&](auto dp, auto mode, auto paged) {
        DARIC_LAUNCH((attend_kernel<CK, QK, decltype(dp)::value, decltype(mode)::value, decltype(paged)::value>),
                     static_cast<unsigned>(p.items), 256, 0, stream, d, a);
    });
    check_launch("attend_pages");
}

template <int CK, int QK>
void run_weigh(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    if (p.row_tile > 0) {
        for_forms(p.dp, p.mode, true, [&](auto dp, auto mode, auto) {
            if constexpr (decltype(mode)::value != kAttValues) {
                if (p.row_tile == 1)
                    DARIC_LAUNCH((weigh_rows_kernel<CK, QK, decltype(dp)::value, decltype(mode)::value>),
                                 static_cast<unsigned>(p.items), 256, 0, stream, d, a);
                else
                    DARIC_LAUNCH((weigh_split_kernel<CK, QK, decltype(dp)::value, decltype(mode)::value>),
                                 static_cast<unsigned>(p.items), 512, 0, stream, d, a);
            }
        });
        check_launch("weigh_tokens");
        return;
    }
    for_forms(p.dp, p.mode, p.paged, [&](auto dp, auto mode, auto paged) {
        DARIC_LAUNCH((weigh_kernel<CK, QK, decltype(dp)::value, decltype(mode)::value, decltype(paged)::value>),
                     static_cast<unsigned>(p.items), 256, 0, stream, d, a);
    });
    check_launch("weigh_tokens");
}

template <int QK>
void run_join(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    for_forms(p.dp, kAttWhole, true, [&](auto dp, auto, auto) {
        constexpr int DP = decltype(dp)::value;
        const int rows = static_cast<int>(p.join_rows);
        // many rows fill the chip by themselves (MI355X, 12000 rows in few parts: eight
        // parts of a row at once 27 us, one 10)
        if (p.max_parts <= 4 || rows >= 4096) DARIC_LAUNCH((attend_join_kernel<QK, DP, 1>), (rows + 7) / 8, 256, 0, stream, d, a, rows);
        else DARIC_LAUNCH((attend_join_kernel<QK, DP, 8>), rows, 256, 0, stream, d, a, rows);
    });
    check_launch("attend_pages join");
}

}  // namespace attend
}  // namespace daric
