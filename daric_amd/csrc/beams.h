// Beam search: the choice of candidates and the reordering of the paged cache by
// it. Descriptors shared by the host checks, the launchers and the kernels.
#pragma once

#include <hip/hip_runtime_api.h>

#include "jobs.h"

namespace daric {

constexpr int kMaxCandidates = 64;     // of a request
constexpr int kMaxBeams = 64;          // of a request, in a choice
// Of a row of logits, for one wavefront. MI355X, 4, 8 and 16 KiB: 256 rows of 128000 bf16 33,
// 27 and 31 us, 4 rows 13.6, 13.7 and 13.6, 35 rows of 50021 fp32 14.1, 13.5 and 14.0.
constexpr int kSplitBytes = 8192;
constexpr int64_t kMaxSplits = 32768;  // of a request

// A candidate of a split of a row: its logit and its token (-1: none).
struct alignas(8) BeamCandidate {
    float x;
    int32_t token;
};

struct SelectArgs {
    const uint8_t* logits;         // [B, W, V], values contiguous
    int64_t batch, row;            // strides in values
    const float* scores;           // [B, W]
    const uint8_t* ended;          // [B, W] or null
    float* out_scores;             // [B, k]
    int32_t* parents;
    int32_t* tokens;
    BeamCandidate* part;           // [B * W][splits][k], best first
    float* part_ms;                // [B * W][splits][2]: maximum, sum of exp(x - maximum)
    int32_t W, k, splits, end_token;
    int32_t B;
    int32_t token_bits;            // of a token in a candidate's place: 26 for fp32 logits, else 32
    int64_t V;
    FastDiv d_splits, d_beams;     // by splits and by W
};

// kind: kBF16, kF16 or kF32 (append.h).
void launch_select_beams(const SelectArgs& a, int kind, hipStream_t stream);

// A request of a reorder: beam w's block list is block_table[bt_offset + w * stride ...].
struct alignas(16) BeamLists {
    int64_t bt_offset;
    int64_t stride;
    int32_t n_beams, n_tokens;
    int32_t tile_begin;    // first workgroup over its last pages' rows
    int32_t pad0;
};
static_assert(sizeof(BeamLists) == 32, "BeamLists layout");

constexpr int kReorderBeams = 32;      // of a request: their units are held in registers
constexpr int kReorderThreads = 256;

// The lists at byte 0 of d, the layers' addresses at layer_off. most_beams, most_pages:
// the largest n_beams and n_tokens / PS; tiles: workgroups of a layer's rows (unit
// bytes each lane, all beams of a request). parents: rows of parent_stride, one a request.
void launch_reorder(const DescArg& d, int layer_off, int n_layers, const KVGeom& g, int es, int unit,
                    int32_t* block_table, const int32_t* parents, int64_t parent_stride, int n_lists, int most_beams,
                    int64_t most_pages, int64_t tiles, hipStream_t stream);

}  // namespace daric
