// Products of a few rows with the epilogue of a linear_act or a gated layer (pam_thin.hip).
#pragma once
#include <hip/hip_runtime.h>

namespace pamthin {

struct Layer {
    const float* a; long a_sr;                    // [m][k], contiguous along k
    const float* w; long w_sr;                    // [rows][k], contiguous along k; gated: the gate's rows and as many others
    const float* bias;                            // one per row of w, or null
    const float* residual; long residual_sr;      // [m][n] or null
    float* z;                                     // [m][rows] or null
    float* y;                                     // [m][n]
    int m, n, k, activation;
    float off;
};

// Whether a product of these sizes and layouts is one for launch().
bool takes(long m, long rows, long k, long a_sc, long w_sc);
int launch(const char* what, const Layer& layer, bool gated, hipStream_t st);

}  // namespace pamthin
