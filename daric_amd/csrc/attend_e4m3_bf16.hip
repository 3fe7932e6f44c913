// Attention over e4m3 caches read by bf16 queries (a source file per pair of types: they build side by side).
#include "attend_kernels.h"

namespace daric {

void attend_e4m3_bf16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_attend<kE4M3, kBF16>(d, a, p, stream);
}
void weigh_e4m3_bf16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_weigh<kE4M3, kBF16>(d, a, p, stream);
}

}  // namespace daric
