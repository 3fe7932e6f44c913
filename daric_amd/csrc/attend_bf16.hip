// Attention over bf16 caches (a source file per pair of types: they build side by side).
#include "attend_kernels.h"

namespace daric {

void attend_bf16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::run_attend<kBF16, kBF16>(d, a, p, stream);
}
void weigh_bf16(const DescArg& d, const AttArgs& a, int mode, int dp, int64_t items, hipStream_t stream) {
    attend::run_weigh<kBF16, kBF16>(d, a, mode, dp, items, stream);
}
void join_bf16(const DescArg& d, const AttArgs& a, const AttPlan& p, hipStream_t stream) {
    attend::for_forms(p.dp, kAttWhole, [&](auto dp, auto) {
        DARIC_LAUNCH((attend::attend_join_kernel<kBF16, decltype(dp)::value>), static_cast<unsigned>(p.groups), 256, 0,
                     stream, d, a);
    });
    check_launch("attend_pages join");
}

}  // namespace daric
