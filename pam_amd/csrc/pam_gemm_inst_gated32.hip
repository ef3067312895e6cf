// The matrix kernels with 32-deep k-tiles whose sums go out by WAY_GATED (one file per pair: they compile side by side).
#include "pam_gemm_kernel.h"

template void pamgemm::launch_layer<32, pamgemm::WAY_GATED>(int, unsigned, hipStream_t, const pamgemm::GemmArgs&);
