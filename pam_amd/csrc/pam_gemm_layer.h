// The matrix kernel's products whose sums go out through an activation (pam_gemm.hip).
#pragma once
#include <stddef.h>

namespace pamgemm {

// Columns of the product that computes a gated layer of `hidden` outputs.
long gated_columns(long hidden);
// Scratch of a layer's product of that many columns.
size_t layer_workspace(long m, long n, long k);
// What pam_hip_linear_act_fwd and pam_hip_gated_linear_fwd compute; n: outputs of a row.
int layer_product(const char* what, bool gated, const float* a, long a_sr, long a_sc, const float* w, long w_sr, long w_sc, const float* bias,
                  const float* residual, long residual_sr, int activation, float* z, float* y, long m, long n, long k, float offset,
                  void* workspace, size_t workspace_bytes, void* stream);

}  // namespace pamgemm
