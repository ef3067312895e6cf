// Instances of the forward pass: heads of 65 to 128 values.
#include "pam_attention_fwd.h"

namespace pamatt {
extern const Variant kFwd2[] = {
    {2, 10, attention_kernel<2, 10>}, {2, 12, attention_kernel<2, 12>}, {2, 14, attention_kernel<2, 14>}, {2, 16, attention_kernel<2, 16>}, {0, 0, nullptr},
};
}  // namespace pamatt
