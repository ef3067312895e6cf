// The matrix kernels whose sums are chains of bounded length: plain products (one file each: they compile side by side).
#include "pam_gemm_kernel.h"

template void pamgemm::launch_gemm<32, pamgemm::MODE_PAM, true>(int, int, unsigned, hipStream_t, const pamgemm::GemmArgs&);
