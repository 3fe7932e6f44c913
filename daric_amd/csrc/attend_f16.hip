// Attention over fp16 caches (a source file per pair of types: they build side by side).
#include "attend_kernels.h"

namespace daric {

void attend_f16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_attend<kF16, kF16>(d, a, p, stream);
}
void weigh_f16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_weigh<kF16, kF16>(d, a, p, stream);
}
void join_f16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_join<kF16>(d, a, p, stream);
}

}  // namespace daric
