// Instances of the gradients' passes: queries, exact slopes.
#include "pam_attention_bwd.h"

namespace pamatt {
extern const Variant kDqExact[] = {
    dq_of<1, 4, true, false>(),
    dq_of<1, 8, true, false>(),
    dq_of<2, 6, true, false>(),
    dq_of<2, 8, true, false>(),
    dq_of<4, 5, true, false>(),
    dq_of<4, 6, true, false>(),
    dq_of<4, 8, true, false>(),
    dq_of<8, 6, true, false>(),
    dq_of<8, 8, true, false>(),
    dq_of<1, 4, false, false>(),
    dq_of<1, 8, false, false>(),
    dq_of<2, 8, false, false>(),
    dq_of<4, 8, false, false>(),
    dq_of<8, 8, false, false>(),
    {0, 0, false, nullptr},
};
}  // namespace pamatt
