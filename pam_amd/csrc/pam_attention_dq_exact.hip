// Instances of the gradients' passes: queries, any slopes.
#include "pam_attention_bwd.h"

namespace pamatt {
extern const Variant kDqExact[] = {
    {1, 4, attention_dq_kernel<1, 4, false>},
    {1, 8, attention_dq_kernel<1, 8, false>},
    {2, 6, attention_dq_kernel<2, 6, false>},
    {2, 8, attention_dq_kernel<2, 8, false>},
    {4, 5, attention_dq_kernel<4, 5, false>},
    {4, 6, attention_dq_kernel<4, 6, false>},
    {4, 8, attention_dq_kernel<4, 8, false>},
    {4, 12, attention_dq_kernel<4, 12, false>},
    {4, 16, attention_dq_kernel<4, 16, false>},
    {0, 0, nullptr},
};
}  // namespace pamatt
