// Instances of the gradients' passes: keys and values, approximate slopes.
#include "pam_attention_bwd.h"

namespace pamatt {
extern const Variant kDkvApprox[] = {
    dkv_of<1, 4, true, true>(),
    dkv_of<1, 8, true, true>(),
    dkv_of<2, 6, true, true>(),
    dkv_of<2, 8, true, true>(),
    dkv_of<4, 5, true, true>(),
    dkv_of<4, 6, true, true>(),
    dkv_of<4, 8, true, true>(),
    dkv_of<8, 6, true, true>(),
    dkv_of<8, 8, true, true>(),
    dkv_of<1, 4, false, true>(),
    dkv_of<1, 8, false, true>(),
    dkv_of<2, 8, false, true>(),
    dkv_of<4, 8, false, true>(),
    dkv_of<8, 8, false, true>(),
    {0, 0, false, nullptr},
};
}  // namespace pamatt
