// Eviction of the lightest tokens of a sequence from the paged cache (gfx950).
//
// Of a sequence's n tokens the first `first`, the last `recent` and the heaviest
// others stay, `keep` in all. A kept token that stands in one of the first
// `keep` slots stays there; the i-th of those slots whose token goes takes the
// i-th kept token from behind them. So every row that moves goes from a slot >=
// keep to one < keep: no row is both read and written, all move at once, and
// the order of the rest of the cache (K rows carry their positions) does not
// change. Moving every kept token up in order would move about all of them, each
// over a row that another still has to be read from.
//
// evict_plan_kernel, a workgroup per (layer, head, sequence): the top-k of the
// weights (topk.h), then the slots from its ascending indices alone.
// evict_move_kernel: tiles of slots, whose moving rows are gathered in LDS
// first, so that all lanes copy. Read and written past the caches (202 -> 180 us for
// an eviction of 8 sequences from 32 layers).
//
// The plan is bound by the latency of its passes (its wavefronts wait 59% of their time,
// vector issue 30%), the move by memory. MI355X, 8 sequences of 1100 to 2500 tokens cut to
// 1024 in 32 layers of 8 x 128 bf16: plan 41 us, rows 179 us for 962 MB of HBM read and
// written, 5.4 TB/s (a copy of 1 GiB by torch: 4.8); one sequence of 16384 cut to 2048 in
// 80 e4m3 layers: 61 us, and 112 for 598 MB, 5.3 TB/s.
#include "attend.h"
#include "kernels.h"
#include "launch.h"
#include "topk.h"

namespace daric {
namespace {

constexpr int kMoveSlots = 256;
constexpr int kMoveThreads = 256;
// Selected indices of a plan workgroup in LDS, beside the top-k's 8 KiB.
constexpr size_t kPlanLds = 48 * 1024;

// The selected indices stand in LDS (IN_LDS: as many as the call selects at most),
// or in the workspace `sel` where they do not fit.
template <int T, int KPT, bool IN_LDS>
__global__ __launch_bounds__(T) void evict_plan_kernel(DescArg d, float* __restrict__ weights, int64_t columns,
                                                       int n_seqs, int32_t* sel, int32_t* __restrict__ kept,
                                                       int kmax, int64_t rows0) {
    static_assert(T <= 256 || sizeof(TopkLds<T>) >= sizeof(TopkLds<256>), "the short forms' LDS fits");
    __shared__ __align__(16) uint8_t s_mem[sizeof(TopkLds<T>)];
    __shared__ int s_early;
    extern __shared__ int32_t s_ids[];
    const int64_t row = rows0 + blockIdx.y;                // (layer, head)
    const int si = static_cast<int>(blockIdx.x);
    const EvictSeq s = desc_load(desc_at<EvictSeq>(d, 0) + si);
    const int tid = static_cast<int>(threadIdx.x);
    float* w = weights + row * columns + s.col0;
    int32_t* o = kept + (row * n_seqs + si) * kmax;
    int32_t* const ids = IN_LDS ? s_ids : sel + (row * n_seqs + si) * kmax;
    const int n = s.n, keep = min(s.keep, n);
    for (int i = keep + tid; i < kmax; i += T) o[i] = -1;
    if (n <= s.keep) {
        for (int i = tid; i < n; i += T) o[i] = i;
        return;
    }
    const int mid = n - s.first - s.recent;                // tokens to choose from
    const int k = keep - s.first - s.recent;
    const auto form = [&](auto lanes, auto slots) {
        constexpr int N = decltype(lanes)::value;
        if (tid >= N) return;
        if (tid == 0) s_early = 0;
        const auto key_at = [&](int i) -> uint32_t { return order_key(w[s.first + i]); };
        if (k > 0)
            chunk_topk<N, decltype(slots)::value>(key_at, mid, k, IN_LDS ? nullptr : ids, IN_LDS ? ids : nullptr,
                                                  *reinterpret_cast<TopkLds<N>*>(s_mem));
        __syncthreads();
        // early: indices whose token stands in one of the `keep` slots
        const int edge = min(keep - s.first, mid);
        for (int b = tid; b < k; b += N)
            if (ids[b] < edge && (b + 1 == k || ids[b + 1] >= edge)) s_early = b + 1;
        __syncthreads();
        const int early = s_early;
        const int late = k - early;
        const int behind = max(keep, n - s.recent);        // first of the recent tokens that move
        for (int x = tid; x < early; x += N) o[s.first + ids[x]] = s.first + ids[x];
        // Free slot i is y = i + (selected indices before it): index x has ids[x] - x
        // free slots before it. A lane searches for its slot; the gap of each index
        // filled by the index's lane took 112 us instead of 88 (with 1024 lanes) where
        // one token in nine stays (640 rows of 16384 tokens).
        for (int i = tid; i < edge - early; i += N) {
            int lo = 0, hi = early;
            while (lo < hi) {
                const int at = (lo + hi) >> 1;
                if (ids[at] - at <= i) lo = at + 1; else hi = at;
            }
            const int src = i < late ? s.first + ids[early + i] : behind + (i - late);
            o[s.first + i + lo] = src;
            w[s.first + i + lo] = w[src];
        }
        for (int i = tid; i < s.first; i += N) o[i] = i;
        for (int i = n - s.recent + tid; i < keep; i += N) o[i] = i;
        __syncthreads();
        for (int i = keep + tid; i < n; i += N) w[i] = 0.0f;
    };
    using std::integral_constant;
    if (T > 64 && mid <= kTopkWave) form(integral_constant<int, 64>(), integral_constant<int, kTopkWave / 64>());
    else if (T > 256 && mid <= kTopkGroup) form(integral_constant<int, 256>(), integral_constant<int, kTopkGroup / 256>());
    else form(integral_constant<int, T>(), integral_constant<int, KPT>());
}

template <typename U>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(DescArg d, int layer_off, LayerMinor lm, KVGeom g,
                                                                  int es, const int32_t* __restrict__ block_table,
                                                                  const int32_t* __restrict__ kept, int kmax, int heads,
                                                                  int n_seqs, int slot_tiles, FastDiv page,
                                                                  FastDiv row_units, FastDiv head_units) {
    __shared__ int64_t s_src[kMoveSlots], s_dst[kMoveSlots];
    __shared__ int s_wave[kMoveThreads / 64];
    int l;
    int64_t item;
    lm.at(l, item);
    // item: (sequence, slot tile, head), the head first
    const int h = static_cast<int>(item % heads);
    const int st = static_cast<int>(item / heads);
    const int si = st / slot_tiles, tile = st - si * slot_tiles;
    const EvictSeq s = desc_load(desc_at<EvictSeq>(d, 0) + si);
    if (s.n <= s.keep || tile * kMoveSlots >= s.keep) return;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int32_t* bt = block_table + s.bt_offset;
    const int32_t* k_row = kept + ((static_cast<int64_t>(l) * heads + h) * n_seqs + si) * kmax;
    const int slot = tile * kMoveSlots + tid;
    bool moves = false;
    int64_t src = 0, dst = 0;
    if (slot < s.keep) {
        const int from = k_row[slot];
        if (from != slot) {
            const int ps = static_cast<int>(page.div(static_cast<uint32_t>(from)));
            const int pd = static_cast<int>(page.div(static_cast<uint32_t>(slot)));
            const int is = bt[ps], id = bt[pd];
            moves = is > 0 && is < g.num_blocks && id > 0 && id < g.num_blocks;
            src = static_cast<int64_t>(is) * g.sb + static_cast<int64_t>(from - ps * g.PS) * g.ss;
            dst = static_cast<int64_t>(id) * g.sb + static_cast<int64_t>(slot - pd * g.PS) * g.ss;
        }
    }
    const unsigned long long some = __ballot(moves);
    if (lane == 0) s_wave[wave] = __popcll(some);
    __syncthreads();
    int at = __popcll(some & ((1ull << lane) - 1)), count = 0;
#pragma unroll
    for (int w = 0; w < kMoveThreads / 64; ++w) {
        if (w < wave) at += s_wave[w];
        count += s_wave[w];
    }
    if (moves) {
        s_src[at] = src;
        s_dst[at] = dst;
    }
    __syncthreads();
    uint8_t* base = desc_at<uint8_t*>(d, layer_off)[l] + static_cast<int64_t>(h) * g.sh * es;
    const int per = static_cast<int>(row_units.d);          // units of a moving row, K and V, all its heads
    const auto offset = [&](int i, int64_t* from, int64_t* to) {
        const int m = static_cast<int>(row_units.div(static_cast<uint32_t>(i)));
        const int u = i - m * per;
        const int part = static_cast<int>(head_units.div(static_cast<uint32_t>(u)));   // (head, K or V)
        const int64_t o = (g.v_off >= 0 ? (part & 1) * g.v_off + (part >> 1) * g.sh : part * g.sh) * es +
                          static_cast<int64_t>(u - part * static_cast<int>(head_units.d)) * static_cast<int>(sizeof(U));
        *from = s_src[m] * es + o;
        *to = s_dst[m] * es + o;
    };
    constexpr int UNROLL = 4;
    const int units = count * per;
    int i = tid;
    for (; i + (UNROLL - 1) * kMoveThreads < units; i += UNROLL * kMoveThreads) {
        int64_t from[UNROLL], to[UNROLL];
        U v[UNROLL];
#pragma unroll
        for (int x = 0; x < UNROLL; ++x) offset(i + x * kMoveThreads, &from[x], &to[x]);
#pragma unroll
        for (int x = 0; x < UNROLL; ++x) v[x] = __builtin_nontemporal_load(reinterpret_cast<const U*>(base + from[x]));
#pragma unroll
        for (int x = 0; x < UNROLL; ++x) __builtin_nontemporal_store(v[x], reinterpret_cast<U*>(base + to[x]));
    }
    for (; i < units; i += kMoveThreads) {
        int64_t from, to;
        offset(i, &from, &to);
        *reinterpret_cast<U*>(base + to) = *reinterpret_cast<const U*>(base + from);
    }
}

}  // namespace

void launch_evict(const DescArg& d, int layer_off, int n_layers, const KVGeom& g, int es, int unit,
                  const int32_t* block_table, float* weights, int64_t columns, int heads, int n_seqs,
                  int max_tokens, int max_keep, int max_chosen, int32_t* sel, int32_t* kept, int kmax, hipStream_t stream) {
    constexpr int kMaxGridY = 65535;
    const int64_t rows = static_cast<int64_t>(n_layers) * heads;
    const int64_t groups = rows * n_seqs;
    for (int64_t r0 = 0; r0 < rows; r0 += kMaxGridY) {
        const dim3 grid(static_cast<unsigned>(n_seqs), static_cast<unsigned>(std::min<int64_t>(kMaxGridY, rows - r0)));
        const size_t lds = static_cast<size_t>(max_chosen) * sizeof(int32_t);
        const bool in_lds = lds <= kPlanLds;
#define DARIC_EP(TH, KPT)                                                                                          \
    do {                                                                                                           \
        if (in_lds) DARIC_LAUNCH((evict_plan_kernel<TH, KPT, true>), grid, TH, lds, stream, d, weights, columns,   \
                                 n_seqs, sel, kept, kmax, r0);                                                     \
        else DARIC_LAUNCH((evict_plan_kernel<TH, KPT, false>), grid, TH, 0, stream, d, weights, columns, n_seqs,   \
                          sel, kept, kmax, r0);                                                                    \
    } while (0)
        // As many lanes as the top-k takes (launch_topk), but that 512 take runs of up to
        // 16384 too where there are many: 640 of 16112 tokens 88 -> 61 us, two workgroups
        // of 1024 lanes to a CU leaving a second round a quarter full (MI355X).
        if (max_tokens <= kTopkWave) DARIC_EP(64, kTopkWave / 64);
        else if (max_tokens <= kTopkGroup) DARIC_EP(256, kTopkGroup / 256);
        else if (max_tokens <= 8192 && groups > 256) DARIC_EP(512, 16);
        else if (max_tokens <= 16384 && groups > 256) DARIC_EP(512, 32);
        else if (max_tokens <= 8192) DARIC_EP(1024, 8);
        else if (max_tokens <= 32768) DARIC_EP(1024, 32);
        else if (groups > 1024) DARIC_EP(512, 0);
        else DARIC_EP(1024, 0);
#undef DARIC_EP
        check_launch("evict_tokens plan");
    }
    if (max_keep == 0) return;
    const int slot_tiles = (max_keep + kMoveSlots - 1) / kMoveSlots;
    const int head_units = g.D * es / unit;
    const int row_units = head_units * (g.v_off >= 0 ? 2 : 1) * (heads > 1 ? 1 : g.H);
    for_layer_minor(n_layers, static_cast<int64_t>(n_seqs) * slot_tiles * heads, [&](const LayerMinor& lm, unsigned blocks) {
#define DARIC_EM(U) DARIC_LAUNCH((evict_move_kernel<U>), blocks, kMoveThreads, 0, stream, d, layer_off, lm, g, es, \
                                 block_table, kept, kmax, heads, n_seqs, slot_tiles, FastDiv(static_cast<uint32_t>(g.PS)), \
                                 FastDiv(static_cast<uint32_t>(row_units)), FastDiv(static_cast<uint32_t>(head_units)))
        if (unit == 16) DARIC_EM(u32x4);
        else if (unit == 8) DARIC_EM(u32x2);
        else if (unit == 4) DARIC_EM(uint32_t);
        else if (unit == 2) DARIC_EM(uint16_t);
        else DARIC_EM(uint8_t);
#undef DARIC_EM
        check_launch("evict_tokens");
    });
}

}  // namespace daric
