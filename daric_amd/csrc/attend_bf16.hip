// Attention over bf16 caches (a source file per pair of types: they build side by side).
#include "attend_kernels.h"

namespace daric {

void attend_bf16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_attend<kBF16, kBF16>(d, a, p, stream);
}
void weigh_bf16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_weigh<kBF16, kBF16>(d, a, p, stream);
}
void join_bf16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_join<kBF16>(d, a, p, stream);
}

}  // namespace daric
