// The matrix kernels whose sums are chains of bounded length: sums that go out by WAY_LAYER (one file each: they compile side by side).
#include "pam_gemm_kernel.h"

template void pamgemm::launch_layer<32, pamgemm::WAY_LAYER, true>(int, unsigned, hipStream_t, const pamgemm::GemmArgs&);
