// Instances of the gradients' passes: queries, approximate slopes.
#include "pam_attention_bwd.h"

namespace pamatt {
extern const Variant kDqApprox[] = {
    dq_of<1, 4, true, true>(),
    dq_of<1, 8, true, true>(),
    dq_of<2, 6, true, true>(),
    dq_of<2, 8, true, true>(),
    dq_of<4, 5, true, true>(),
    dq_of<4, 6, true, true>(),
    dq_of<4, 8, true, true>(),
    dq_of<8, 6, true, true>(),
    dq_of<8, 8, true, true>(),
    dq_of<1, 4, false, true>(),
    dq_of<1, 8, false, true>(),
    dq_of<2, 8, false, true>(),
    dq_of<4, 8, false, true>(),
    dq_of<8, 8, false, true>(),
    {0, 0, false, nullptr},
};
}  // namespace pamatt
