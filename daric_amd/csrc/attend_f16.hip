// Attention over fp16 caches (a source file per pair of types: they build side by side).
#include "attend_kernels.h"

namespace daric {

void attend_f16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_attend<kF16, kF16>(d, a, p, stream);
}
void weigh_f16(const DescArg& d, const AttArgs& a, int mode, int dp, int64_t items, hipStream_t stream) {
    attend::run_weigh<kF16, kF16>(d, a, mode, dp, items, stream);
}
void join_f16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::for_forms(p.dp, kAttWhole, [&](auto dp, auto) {
        DARIC_LAUNCH((attend::attend_join_kernel<kF16, decltype(dp)::value>), static_cast<unsigned>(p.groups), 256, 0,
                     stream, d, a);
    });
    check_launch("attend_pages join");
}

}  // namespace daric
