// Top-k of a run of fp32 keys by one workgroup (gfx950), shared by the recompute
// selection and the eviction.
#pragma once

#include <hip/hip_runtime.h>

#include "elem.h"
#include "kernels.h"

namespace daric {

// Rank of a key: the IEEE total order of its bits, NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float f) {
    uint32_t b = f2u(f);
    if ((b & 0x7fffffffu) > 0x7f800000u) b = 0x7fc00000u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Per-chunk top-k by a workgroup of T lanes: the k largest of n order keys, ties
// to the lower index, written in ascending index order to orow[0 .. k-1] (when
// not null) and, when s_sel is not null, to the LDS array s_sel (visible to the
// other lanes after the caller's next barrier).
//
// Bound by latency: a chain of passes with barriers between them, so the passes
// are few and each pass is short. Wavefront w takes the consecutive keys of
// slots [w * slots, (w + 1) * slots) of 64, slot by slot, and holds them in
// registers (KPT slots; KPT = 0: it reads them again in each pass, for chunks
// longer than any register file). Radix passes find the k-th largest key: three
// of 11, 11 and 10 bits, or for a single wavefront, which would spend itself on
// 2048 bins, four of 8. A pass whose digit holds exactly the keys still wanted
// is the last. Lanes add to the LDS histogram one by one, except where all keys
// of a wavefront share the digit (ties, zeros), which one lane adds. The last
// step needs one barrier: the wavefronts' counts give each its place in the
// output.
// Against 256 lanes with four 8-bit passes over keys in LDS (from 8192 tokens,
// in memory), MI355X, 15% of the tokens selected: one chunk of 500 tokens 6.0 ->
// 4.6 us, 16 of 5000 29.2 -> 9.5 us, one of 12000 78 -> 18 us, 6 of 30000 194 ->
// 36 us, 6144 of 512 31.2 -> 23.6 us; all keys equal 6-440 -> 6-94 us.
constexpr int kTopkWave = 256, kTopkGroup = 2048;   // longest chunks of one and of four wavefronts
template <int T>
struct TopkLds {
    static constexpr int kBits = T == 64 ? 8 : 11;
    static constexpr int kBins = 1 << kBits;
    static constexpr int kPerLane = kBins / T;
    // Bin x lies at (x % kPerLane) * T + x / kPerLane, so that the lanes, which
    // sum kPerLane neighbouring bins each, read consecutive words.
    static __device__ __forceinline__ uint32_t at(uint32_t x) {
        return (x % kPerLane) * T + x / kPerLane;
    }
    uint32_t hist[kBins];
    uint32_t wave_a[T / 64], wave_b[T / 64];
    uint32_t digit, above, count;
};

template <int T, int KPT, typename KeyAt>
__device__ __forceinline__ void chunk_topk(KeyAt key_at, int n, int k, int32_t* __restrict__ orow, int32_t* s_sel,
                                           TopkLds<T>& sm) {
    constexpr int W = T / 64;
    using Lds = TopkLds<T>;
    constexpr int BPT = Lds::kPerLane;
    constexpr int R = KPT > 0 ? KPT : 1;
    const int tid = static_cast<int>(threadIdx.x);
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Places past 2^31 - 1 occur where KPT is 0 only; unsigned places ran the
    // register forms 2% slower.
    const int slots = KPT > 0 ? (n + T - 1) / T : topk_slots(n, T);
    const int i0 = wave * slots * 64 + lane;
    uint32_t key[R];
    if constexpr (KPT > 0) {
#pragma unroll
        for (int s = 0; s < KPT; ++s) {
            key[s] = 0;
            if (s < slots && i0 + s * 64 < n) key[s] = key_at(i0 + s * 64);
        }
    }
    // f(slot, key, whether there is one) for the wavefront's slots
    const auto each = [&](auto&& f) {
        if constexpr (KPT > 0) {
#pragma unroll
            for (int s = 0; s < KPT; ++s)
                if (s < slots) f(s, key[s], i0 + s * 64 < n);
        } else {
            for (int s = 0; s < slots; ++s) {
                const uint32_t i = static_cast<uint32_t>(i0) + static_cast<uint32_t>(s) * 64;
                const bool in = i < static_cast<uint32_t>(n);
                f(s, in ? key_at(static_cast<int>(i)) : 0u, in);
            }
        }
    };
#pragma unroll
    for (int b = 0; b < BPT; ++b) sm.hist[b * T + tid] = 0;
    __syncthreads();

    uint32_t prefix = 0, mask = 0, krem = static_cast<uint32_t>(k);
    bool whole = k >= n;      // every key from `prefix` up is taken
    int left_bits = 32;
    while (left_bits > 0 && !whole) {
        const int width = min(left_bits, Lds::kBits);
        const int shift = left_bits - width;
        left_bits = shift;
        const uint32_t dmask = (1u << width) - 1u;
        each([&](int, uint32_t v, bool in) {
            const bool act = in && (v & mask) == prefix;
            const uint32_t dig = (v >> shift) & dmask;
            const unsigned long long some = __ballot(act);
            if (some == 0) return;
            const int lead = __ffsll(static_cast<long long>(some)) - 1;
            const uint32_t d0 = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(dig), lead));
            if (__ballot(act && dig != d0) == 0) {
                if (lane == lead) atomicAdd(&sm.hist[Lds::at(d0)], static_cast<uint32_t>(__popcll(some)));
            } else if (act) {
                atomicAdd(&sm.hist[Lds::at(dig)], 1u);
            }
        });
        __syncthreads();
        // Lane t sums bins [kBins - (t + 1) * BPT, kBins - t * BPT), highest first,
        // and leaves them empty for the next pass.
        uint32_t c[BPT], mine = 0;
#pragma unroll
        for (int b = 0; b < BPT; ++b) {
            const int at = (BPT - 1 - b) * T + (T - 1 - tid);
            c[b] = sm.hist[at];
            sm.hist[at] = 0;
            mine += c[b];
        }
        uint32_t incl = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        if constexpr (W > 1) {
            if (lane == 63) sm.wave_a[wave] = incl;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; ++w) incl += w < wave ? sm.wave_a[w] : 0u;
        }
        uint32_t above = incl - mine;          // keys with a larger digit
        if (above < krem && incl >= krem) {
#pragma unroll
            for (int b = 0; b < BPT; ++b) {
                if (above < krem && above + c[b] >= krem) {
                    sm.digit = static_cast<uint32_t>(Lds::kBins - 1 - tid * BPT - b);
                    sm.above = above;
                    sm.count = c[b];
                }
                above += c[b];
            }
        }
        __syncthreads();
        prefix |= sm.digit << shift;
        mask |= dmask << shift;
        krem -= sm.above;
        whole = sm.count == krem;
    }
    // Take every key with a larger prefix and, of those equal to it, all
    // (whole) or the first krem in index order.
    uint32_t n_gt = 0, n_eq = 0;
    const auto over = [&](uint32_t v, bool in) { return in && (whole ? v >= prefix : v > prefix); };
    each([&](int, uint32_t v, bool in) {
        n_gt += static_cast<uint32_t>(__popcll(__ballot(over(v, in))));
        n_eq += static_cast<uint32_t>(__popcll(__ballot(in && !whole && v == prefix)));
    });
    uint32_t gt = 0, eq = 0;                   // of the wavefronts before
    if constexpr (W > 1) {
        if (lane == 0) {
            sm.wave_a[wave] = n_gt;
            sm.wave_b[wave] = n_eq;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) {
            gt += w < wave ? sm.wave_a[w] : 0u;
            eq += w < wave ? sm.wave_b[w] : 0u;
        }
    }
    const unsigned long long below = (1ull << lane) - 1ull;
    each([&](int s, uint32_t v, bool in) {
        const bool g = over(v, in), e = in && !whole && v == prefix;
        const unsigned long long mg = __ballot(g), me = __ballot(e);
        const uint32_t eq_rank = eq + static_cast<uint32_t>(__popcll(me & below));
        const uint32_t pos = gt + static_cast<uint32_t>(__popcll(mg & below)) + min(eq_rank, krem);
        if ((g || (e && eq_rank < krem)) && pos < static_cast<uint32_t>(k)) {
            const int i = KPT > 0 ? i0 + s * 64 : static_cast<int>(static_cast<uint32_t>(i0) + static_cast<uint32_t>(s) * 64);
            if (orow != nullptr) orow[pos] = i;
            if (s_sel != nullptr) s_sel[pos] = i;
        }
        gt += static_cast<uint32_t>(__popcll(mg));
        eq += static_cast<uint32_t>(__popcll(me));
    });
}

}  // namespace daric
