// Instances of the gradients' passes: keys and values, exact slopes.
#include "pam_attention_bwd.h"

namespace pamatt {
extern const Variant kDkvExact[] = {
    dkv_of<1, 4, true, false>(),
    dkv_of<1, 8, true, false>(),
    dkv_of<2, 6, true, false>(),
    dkv_of<2, 8, true, false>(),
    dkv_of<4, 5, true, false>(),
    dkv_of<4, 6, true, false>(),
    dkv_of<4, 8, true, false>(),
    dkv_of<8, 6, true, false>(),
    dkv_of<8, 8, true, false>(),
    dkv_of<1, 4, false, false>(),
    dkv_of<1, 8, false, false>(),
    dkv_of<2, 8, false, false>(),
    dkv_of<4, 8, false, false>(),
    dkv_of<8, 8, false, false>(),
    {0, 0, false, nullptr},
};
}  // namespace pamatt
