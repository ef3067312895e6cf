// Instances of the forward pass.
#include "pam_attention_fwd.h"

namespace pamatt {
extern const Variant kForward[] = {
    forward_of<1, 4, true>(),
    forward_of<1, 8, true>(),
    forward_of<1, 12, true>(),
    forward_of<1, 16, true>(),
    forward_of<2, 10, true>(),
    forward_of<2, 12, true>(),
    forward_of<2, 16, true>(),
    forward_of<4, 12, true>(),
    forward_of<4, 16, true>(),
    forward_of<1, 4, false>(),
    forward_of<1, 8, false>(),
    forward_of<1, 16, false>(),
    forward_of<2, 16, false>(),
    forward_of<4, 16, false>(),
    {0, 0, false, nullptr},
};
}  // namespace pamatt
