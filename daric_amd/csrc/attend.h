// Attention over the paged cache: descriptors shared by the host checks, the
// launchers and the kernels.
#pragma once

#include <hip/hip_runtime_api.h>

#include "jobs.h"

namespace daric {

// Tokens of a tile: the inner dimension of one matrix instruction over V.
constexpr int kAttTile = 32;
// Query rows (a row is one head of one query) of a matrix tile.
constexpr int kAttRows = 16;

// A sequence of an attention call: rows [row0, row0 + n_rows) of q, whose own
// K and V stand behind n_ctx cached tokens in the pages from block_table
// [bt_offset] on.
struct alignas(16) AttSeq {
    int64_t bt_offset;
    int32_t row0, n_rows, n_ctx;
    int32_t tile_begin;   // first workgroup of the sequence
    int32_t n_parts;      // parts its tokens are cut into
    int32_t at;           // attend: first of its rows times heads in the join; weigh: first column of weights
};
static_assert(sizeof(AttSeq) == 32, "AttSeq layout");

struct AttArgs {
    KVGeom g;
    const uint8_t* layer;
    const int32_t* block_table;
    const uint8_t* q;          // rows of Hq heads, elements of 2 bytes
    int64_t q_row, q_head;     // strides in elements
    const uint64_t* mask;      // [T, words] or null: causal
    const float* k_scale;      // [H] or null
    const float* v_scale;
    uint8_t* out;              // [T, Hq, D]
    float* lse;                // [T, Hq]
    float* part;               // partial sums, [items][tile_rows][head_dim rounded up]
    float* part_ml;            // their maxima and sums, [items][tile_rows][2]
    float* weights;            // weigh: [H, columns]
    int64_t columns;
    float scale_log2;          // scale * log2(e)
    int32_t words;             // 64-bit words of a mask row
    int32_t G, Hq;             // query heads per KV head, in all
    int32_t n_seqs;
    int32_t tile_rows;         // rows of q of a workgroup
    int32_t by_head;           // many rows: head by head on the XCDs
    int32_t add;               // weigh: add to weights instead of setting them
    FastDiv group, page, heads;
};

// How the kernels read rows of the cache: whole units of a full head, whole
// units with the lanes past head_dim idle, or value by value (any alignment).
enum AttMode : int { kAttWhole = 0, kAttPadded = 1, kAttValues = 2 };

// How an attend call is cut: rows of a workgroup, tiles of a part.
struct AttPlan {
    int mode, dp;                  // head_dim rounded up to 64, 128 or 256
    bool paged;                    // pages hold whole halves of a tile
    int row_tile;                  // attend_rows_kernel: rows of a workgroup in 64s (1, 2, 4);
                                   // weigh_rows_kernel: 1, weigh_split_kernel: 2;
                                   // 0: attend_kernel, weigh_kernel
    int64_t items, join_rows;      // workgroups; rows times heads of all sequences
    int64_t max_parts;             // of a sequence: with more than one, a second kernel joins them
};

// Launchers by cache and query type. `d` holds the sequences.
#define DARIC_ATTEND_TYPES(name)                                                                                \
    void attend_##name(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream);               \
    void weigh_##name(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream);
DARIC_ATTEND_TYPES(bf16)
DARIC_ATTEND_TYPES(f16)
DARIC_ATTEND_TYPES(e4m3_bf16)
DARIC_ATTEND_TYPES(e4m3_f16)
#undef DARIC_ATTEND_TYPES
// The join of the parts, by query type.
void join_bf16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream);
void join_f16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream);
// Tokens of a weigh workgroup: of few rows, of many, of many rows and few tokens.
constexpr int kWeighTokens = 128, kWeighRowsTokens = 256, kWeighSplitTokens = 64;

// An eviction: the tokens [0, n) of a sequence, of which `keep` stay.
struct alignas(16) EvictSeq {
    int64_t bt_offset, col0;       // first column of weights
    int32_t n, keep, first, recent;
};
static_assert(sizeof(EvictSeq) == 32, "EvictSeq layout");
// d: the sequences, then (at layer_off) the layers' addresses. heads: H, or 1 where
// one selection serves all heads of a layer; unit: bytes of an access that all
// rows allow; max_tokens: the most tokens a selection chooses from, max_chosen the
// most it takes, max_keep the most slots of a sequence that loses tokens (0: none
// does).
void launch_evict(const DescArg& d, int layer_off, int n_layers, const KVGeom& g, int es, int unit,
                  const int32_t* block_table, float* weights, int64_t columns, int heads, int n_seqs,
                  int max_tokens, int max_keep, int max_chosen, int32_t* sel, int32_t* kept, int kmax, hipStream_t stream);

}  // namespace daric
