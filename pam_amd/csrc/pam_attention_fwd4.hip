// Instances of the forward pass: heads of more than 128 values.
#include "pam_attention_fwd.h"

namespace pamatt {
extern const Variant kFwd4[] = {
    {4, 10, attention_kernel<4, 10>}, {4, 12, attention_kernel<4, 12>}, {4, 16, attention_kernel<4, 16>}, {0, 0, nullptr},
};
}  // namespace pamatt
