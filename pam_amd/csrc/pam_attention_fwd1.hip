// Instances of the forward pass: heads of up to 64 values.
#include "pam_attention_fwd.h"

namespace pamatt {
extern const Variant kFwd1[] = {
    {1, 4, attention_kernel<1, 4>}, {1, 8, attention_kernel<1, 8>}, {1, 12, attention_kernel<1, 12>}, {1, 16, attention_kernel<1, 16>}, {0, 0, nullptr},
};
}  // namespace pamatt
