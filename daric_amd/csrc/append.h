// New rows of a step: their rotation to positions and their way into the paged
// cache. Descriptors shared by the host checks, the launcher and the kernels.
#pragma once

#include <hip/hip_runtime_api.h>

#include "jobs.h"

namespace daric {

// A sequence of an append: rows [row0, row0 + n_rows) become the tokens behind its
// n_ctx cached ones, in the pages from block_table[bt_offset] on.
struct alignas(16) AppendSeq {
    int64_t bt_offset;
    int32_t row0, n_rows, n_ctx;
    int32_t tile_begin;   // first workgroup of the sequence
    int32_t pad0, pad1;
};
static_assert(sizeof(AppendSeq) == 32, "AppendSeq layout");

// Few sequences, in an argument block of their own: a launch with DescArg's 2832 bytes takes
// the host 4.5 us, with 600 bytes in all 3.5 (MI355X host).
struct alignas(16) FewSeqs {
    static constexpr int kMost = 8;
    AppendSeq s[kMost];
};

// Rows of heads; strides in elements, the values of a head contiguous.
struct HeadRows {
    const uint8_t* data;
    int64_t row, head;
};

// Element kinds of the rows beside those of a cache (ElemKind).
constexpr int kF32 = 3;

struct AppendArgs {
    KVGeom g;                     // of the cache (H = 0: rows are rotated only)
    uint8_t* layer;
    const int32_t* block_table;
    HeadRows q, k, v;             // Hq, g.H and g.H heads; without V where g.v_off < 0
    uint8_t* q_out;
    int64_t out_row, out_head;
    const int64_t* positions;     // of row r, or null: its token's place in the sequence
    const float* inv_freq;        // [R / 2]
    const float* k_scale;         // [H] or null
    const float* v_scale;
    float m;                      // factor of cos and sin
    int32_t Hq, D, R, is_neox;
    int32_t n_seqs, tile;         // rows of a workgroup
    int32_t one_tile;             // every sequence is one tile: workgroup i takes sequence i
    int32_t in_place;             // q_out is q: what is not rotated stays
    // items of a row of q and K, and of V; of a token's q and K heads, and of all
    int32_t rot_items, copy_items;
    int32_t q_end, k_end;         // first item behind q's and behind K's
    FastDiv d_token, d_rot, d_copy, d_half;
};

// Values of the widest access that the rows' sizes allow (half: of a rotated half,
// rest: of the unrotated end; alignment is the caller's): 8, 4, 2 or 1.
inline int append_vec(int64_t half, int64_t rest, int most) {
    int v = most;
    while (v > 1 && (half % v != 0 || rest % v != 0)) v /= 2;
    return v;
}

// from: ElemKind of the rows or kF32; to: kE4M3 for an e4m3 cache, else `from`. past: 16-byte
// stores go past the caches.
void launch_append(const FewSeqs& d, const AppendArgs& a, int from, int to, int vec, bool past, int64_t tiles, hipStream_t stream);
void launch_append(const DescArg& d, const AppendArgs& a, int from, int to, int vec, bool past, int64_t tiles, hipStream_t stream);

}  // namespace daric
