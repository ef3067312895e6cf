// Instances of the gradients' passes: queries, approximate slopes.
#include "pam_attention_bwd.h"

namespace pamatt {
extern const Variant kDqApprox[] = {
    {1, 4, attention_dq_kernel<1, 4, true>},
    {1, 8, attention_dq_kernel<1, 8, true>},
    {2, 6, attention_dq_kernel<2, 6, true>},
    {2, 8, attention_dq_kernel<2, 8, true>},
    {4, 5, attention_dq_kernel<4, 5, true>},
    {4, 6, attention_dq_kernel<4, 6, true>},
    {4, 8, attention_dq_kernel<4, 8, true>},
    {4, 12, attention_dq_kernel<4, 12, true>},
    {4, 16, attention_dq_kernel<4, 16, true>},
    {0, 0, nullptr},
};
}  // namespace pamatt
