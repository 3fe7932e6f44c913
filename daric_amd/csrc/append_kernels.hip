// New rows of a step (gfx950): rotation to their positions, and the append of K and
// V to the paged cache with it on the way.
//
// Pair i of row r turns by the angle p * f_i, p the row's position and f_i the
// fp32 frequency: (x1, x2) -> (x1 c - x2 s, x2 c + x1 s), c and s the cosine and sine
// times m. The angle's product and its reduction to an eighth of a turn are fp64,
// since positions are absolute: at position 10^6 an fp32 product is off by up to
// 0.03 rad, where in fp64 it is exact to 2^-53 of itself. What remains, at most
// pi / 4, goes through the power series of sine and cosine in fp32 (to y^9 and
// y^10: sine and cosine off by 2^-29 and 2^-33 at pi / 4). The rotation is fp32, rounded
// once to the type it is stored in; an e4m3 cache takes the correctly rounded
// quotient by the head's scale, saturating, as the row merge does.
//
// A workgroup takes `tile` rows of one sequence: a table of their cosines and sines
// in LDS, one computation for all of a row's heads, and then the rows' items. An
// item is two accesses of VEC values: the two halves of VEC pairs (neox), VEC
// neighbouring pairs (interleaved), or two runs of values that are only copied
// (the unrotated end of a head, V). The first items' loads are issued before the
// table is made.
//
// Bound by memory where rows are many, by latency (position, block table, angles,
// then the stores) where they are few. MI355X, bf16, traced medians: 16384 rows of 40
// heads of 128 rotated into a new tensor, 336 MB, in 54 us with the rows in the 256 MB
// cache behind the L2s (6.2 TB/s) and 70 us without (4.8; a copy of 1 GiB by torch runs
// at 5.15); 16303 rows of 32 + 8 + 8 heads appended, 401 MB, 65 us and 84; one row 5 us;
// 48 single rows of 64 + 8 + 8 heads into an e4m3 cache 7 us. Vector issue takes 25 of
// the 54 us.
// Odd halves cost width: rows of 80 with 20 rotated values go in 4-byte accesses,
// 77 MB in 32 us.
#include <hip/hip_runtime.h>

#include "append.h"
#include "elem.h"
#include "kernels.h"
#include "launch.h"

namespace daric {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 2;

// Cosine and sine of p * f, times m.
__device__ __forceinline__ void cos_sin(int64_t p, float f, float m, float* c, float* s) {
    constexpr double kQuarters = 0.63661977236758134308;      // 2 / pi
    const double x = static_cast<double>(p) * static_cast<double>(f) * kQuarters;
    const double n = __builtin_rint(x);
    const int quarter = static_cast<int>(n - 4.0 * __builtin_floor(n * 0.25));
    const float y = static_cast<float>((x - n) * 1.57079632679489661923);
    const float z = y * y;
    const float sn = y + y * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
    const float cs = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
    const float a = (quarter & 1) != 0 ? sn : cs, b = (quarter & 1) != 0 ? cs : sn;
    *c = ((quarter + 1) & 2) != 0 ? -a * m : a * m;
    *s = (quarter & 2) != 0 ? -b * m : b * m;
}

// VEC values of a type as the words that hold them.
template <int KIND, int VEC>
struct Values {
    static constexpr int kBytes = VEC * (KIND == kF32 ? 4 : KIND == kE4M3 ? 1 : 2);
    static constexpr int kWords = (kBytes + 3) / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const uint8_t* p) {
        if constexpr (kBytes == 16) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = x[i];
        } else if constexpr (kBytes == 8) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(p);
            w[0] = x[0];
            w[1] = x[1];
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    // PAST: past the caches (16-byte stores)
    template <bool PAST>
    __device__ __forceinline__ void store(uint8_t* p) const {
        if constexpr (kBytes == 16) {
            const u32x4 x = {w[0], w[1], w[2], w[3]};
            if constexpr (PAST) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p));
            else *reinterpret_cast<u32x4*>(p) = x;
        }
        else if constexpr (kBytes == 8) *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
        else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        else if constexpr (kBytes == 2) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
        else *p = static_cast<uint8_t>(w[0]);
    }
    __device__ __forceinline__ void unpack(float* x) const {
        if constexpr (KIND == kF32) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = u2f(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                float two[2];
                Elem<KIND>::unpack_word(w[i], two);
                x[2 * i] = two[0];
                if (2 * i + 1 < VEC) x[2 * i + 1] = two[1];
            }
        }
    }
    __device__ __forceinline__ void pack(const float* x) {
        if constexpr (KIND == kF32) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[i] = f2u(x[i]);
        } else {
            constexpr int EPW = Elem<KIND>::EPW;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                float some[EPW];
#pragma unroll
                for (int j = 0; j < EPW; ++j) some[j] = EPW * i + j < VEC ? x[EPW * i + j] : 0.0f;
                w[i] = Elem<KIND>::pack_word(some);
            }
        }
    }
};

__device__ __forceinline__ DescPtr<AppendSeq> sequences(const DescArg& d) { return desc_at<AppendSeq>(d, 0); }
__device__ __forceinline__ DescPtr<AppendSeq> sequences(const FewSeqs& d) { return (DescPtr<AppendSeq>)d.s; }

template <int FROM, int TO, int VEC, bool PAST, class Desc>
__global__ __launch_bounds__(kThreads) void append_kernel(Desc d, AppendArgs a) {
    extern __shared__ __align__(16) float s_turn[];      // cosines and sines, [tile][R / 2] each
    __shared__ int64_t s_slot[kThreads / 2];             // K element of each row's token, -1: nowhere
    using From = Values<FROM, VEC>;
    using To = Values<TO, VEC>;
    const int tid = static_cast<int>(threadIdx.x);
    const int block = static_cast<int>(blockIdx.x);
    const DescPtr<AppendSeq> seqs = sequences(d);
    const int si = a.one_tile ? block : find_by_tile(seqs, a.n_seqs, block);
    const AppendSeq s = desc_load(seqs + si);
    const int t0 = (block - s.tile_begin) * a.tile;
    const int nt = min(a.tile, s.n_rows - t0);
    const int64_t row0 = static_cast<int64_t>(s.row0) + t0;
    const int half = a.R >> 1;
    float* const s_cos = s_turn;
    float* const s_sin = s_turn + a.tile * half;
    const int n_items = nt * static_cast<int>(a.d_token.d);

    struct Item {
        From x, y;
        int tok, head, c;       // row of the tile, head of its tensor, item of the head's row
        int kind;               // 0: q, 1: K, 2: V
        bool second;            // the item has two accesses
    };
    // Offsets of an item's accesses in its head's row, in values.
    const auto places = [&](const Item& it, int* u, int* v) {
        const int rotated = it.kind == 2 ? 0 : half / VEC;
        if (it.c < rotated) {
            *u = a.is_neox ? it.c * VEC : 2 * it.c * VEC;
            *v = a.is_neox ? *u + half : *u + VEC;
        } else {
            const int n = (it.kind == 2 ? a.copy_items : a.rot_items) - rotated;
            const int first = it.kind == 2 ? 0 : a.R;
            *u = first + (it.c - rotated) * VEC;
            *v = *u + n * VEC;
        }
    };
    const auto fetch = [&](int i, Item& it) {
        it.tok = static_cast<int>(a.d_token.div(static_cast<uint32_t>(i)));
        int r = i - it.tok * static_cast<int>(a.d_token.d);
        it.kind = r < a.q_end ? 0 : r < a.k_end ? 1 : 2;
        r -= it.kind == 0 ? 0 : it.kind == 1 ? a.q_end : a.k_end;
        const int per = it.kind == 2 ? a.copy_items : a.rot_items;
        it.head = static_cast<int>((it.kind == 2 ? a.d_copy : a.d_rot).div(static_cast<uint32_t>(r)));
        it.c = r - it.head * per;
        int u, v;
        places(it, &u, &v);
        it.second = v < a.D;
        const HeadRows& t = it.kind == 0 ? a.q : it.kind == 1 ? a.k : a.v;
        const uint8_t* p = t.data + ((row0 + it.tok) * t.row + it.head * t.head) * (From::kBytes / VEC);
        it.x.load(p + u * (From::kBytes / VEC));
        if (it.second) it.y.load(p + v * (From::kBytes / VEC));
    };
    const auto finish = [&](Item& it) {
        int u, v;
        places(it, &u, &v);
        const bool turns = it.kind != 2 && it.c < half / VEC;
        float x[VEC], y[VEC];
        if (turns) {
            it.x.unpack(x);
            it.y.unpack(y);
            const float* cs = s_cos + it.tok * half + it.c * VEC;
            const float* sn = s_sin + it.tok * half + it.c * VEC;
            if (a.is_neox) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float p = x[i], q = y[i];
                    x[i] = p * cs[i] - q * sn[i];
                    y[i] = q * cs[i] + p * sn[i];
                }
            } else {
                // pair i is values 2 i and 2 i + 1 of the 2 VEC
                float w[2 * VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    w[i] = x[i];
                    w[VEC + i] = y[i];
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float p = w[2 * i], q = w[2 * i + 1];
                    w[2 * i] = p * cs[i] - q * sn[i];
                    w[2 * i + 1] = q * cs[i] + p * sn[i];
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    x[i] = w[i];
                    y[i] = w[VEC + i];
                }
            }
        }
        if (it.kind == 0) {
            if (a.in_place && !turns) return;
            if (turns) {
                it.x.pack(x);
                it.y.pack(y);
            }
            uint8_t* p = a.q_out + ((row0 + it.tok) * a.out_row + it.head * a.out_head) * (From::kBytes / VEC);
            it.x.template store<PAST>(p + u * (From::kBytes / VEC));
            if (it.second) it.y.template store<PAST>(p + v * (From::kBytes / VEC));
            return;
        }
        if constexpr (FROM != kF32) {
            const int64_t slot = s_slot[it.tok];
            if (slot < 0) return;
            uint8_t* p = a.layer + (slot + it.head * a.g.sh + (it.kind == 2 ? a.g.v_off : 0)) * (To::kBytes / VEC);
            To xo, yo;
            if constexpr (TO == kE4M3) {
                if (!turns) {
                    it.x.unpack(x);
                    it.y.unpack(y);
                }
                const float* scale = it.kind == 1 ? a.k_scale : a.v_scale;
                if (scale != nullptr) {
                    const QuantDiv qd = quant_div(scale[it.head]);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        x[i] = quant_quotient(qd, x[i]);
                        y[i] = quant_quotient(qd, y[i]);
                    }
                }
                xo.pack(x);
                yo.pack(y);
            } else {
                if (turns) {
                    it.x.pack(x);
                    it.y.pack(y);
                }
                xo = it.x;
                yo = it.y;
            }
            xo.template store<PAST>(p + u * (To::kBytes / VEC));
            if (it.second) yo.template store<PAST>(p + v * (To::kBytes / VEC));
        }
    };

    Item it[kUnroll];
    int i = tid;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        it[k] = Item{};
        if (i + k * kThreads < n_items) fetch(i + k * kThreads, it[k]);
    }
    for (int x = tid; x < nt * half; x += kThreads) {
        const int tok = static_cast<int>(a.d_half.div(static_cast<uint32_t>(x)));
        const int64_t p = a.positions != nullptr ? a.positions[row0 + tok] : static_cast<int64_t>(s.n_ctx) + t0 + tok;
        cos_sin(p, a.inv_freq[x - tok * half], a.m, s_cos + x, s_sin + x);
    }
    if (a.g.H > 0 && tid < nt) {
        const int token = s.n_ctx + t0 + tid;
        const int page = token / a.g.PS;
        const int id = a.block_table[s.bt_offset + page];
        s_slot[tid] = id > 0 && id < a.g.num_blocks
                          ? static_cast<int64_t>(id) * a.g.sb + static_cast<int64_t>(token - page * a.g.PS) * a.g.ss
                          : -1;
    }
    __syncthreads();
    while (true) {
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            if (i + k * kThreads < n_items) finish(it[k]);
        i += kUnroll * kThreads;
        if (i >= n_items) break;
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            if (i + k * kThreads < n_items) fetch(i + k * kThreads, it[k]);
    }
}

template <class Desc>
void launch(const Desc& d, const AppendArgs& a, int from, int to, int vec, bool past, int64_t tiles, hipStream_t stream) {
    const size_t lds = static_cast<size_t>(a.tile) * a.R * sizeof(float);
#define DARIC_AP(F, T, V, P) DARIC_LAUNCH((append_kernel<F, T, V, P, Desc>), static_cast<unsigned>(tiles), kThreads, lds, stream, d, a)
#define DARIC_AV(F, T)                    \
    do {                                  \
        if (vec == 8 && past) DARIC_AP(F, T, 8, true); \
        else if (vec == 8) DARIC_AP(F, T, 8, false);   \
        else if (vec == 4) DARIC_AP(F, T, 4, false);   \
        else if (vec == 2) DARIC_AP(F, T, 2, false);   \
        else DARIC_AP(F, T, 1, false);                 \
    } while (0)
    if (from == kF32) {
        if (vec == 4 && past) DARIC_AP(kF32, kF32, 4, true);
        else if (vec == 4) DARIC_AP(kF32, kF32, 4, false);
        else if (vec == 2) DARIC_AP(kF32, kF32, 2, false);
        else DARIC_AP(kF32, kF32, 1, false);
    } else if (to == kE4M3) {
        if (from == kBF16) DARIC_AV(kBF16, kE4M3);
        else DARIC_AV(kF16, kE4M3);
    } else if (from == kBF16) DARIC_AV(kBF16, kBF16);
    else DARIC_AV(kF16, kF16);
#undef DARIC_AV
#undef DARIC_AP
    check_launch("append_tokens");
}

}  // namespace

void launch_append(const FewSeqs& d, const AppendArgs& a, int from, int to, int vec, bool past, int64_t tiles, hipStream_t stream) {
    launch(d, a, from, to, vec, past, tiles, stream);
}
void launch_append(const DescArg& d, const AppendArgs& a, int from, int to, int vec, bool past, int64_t tiles, hipStream_t stream) {
    launch(d, a, from, to, vec, past, tiles, stream);
}

}  // namespace daric
