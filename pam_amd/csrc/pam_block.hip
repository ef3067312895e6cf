// The product with an activation and a residual, and the gated layer: entry points and the elementwise kernels.
#include <algorithm>

#include "pam_activation.h"
#include "pam_common.h"
#include "pam_thin.h"

using namespace pamdev;

namespace {

constexpr int kThreads = 256;

Activation activation_of(int kind, float offset) { return Activation{kind, offset, offset != 1.0f}; }
bool known(int activation) { return activation >= PAM_HIP_ACT_NONE && activation <= PAM_HIP_ACT_GELU; }
size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
unsigned groups_for(size_t values) { return (unsigned)std::min<size_t>((values + kThreads - 1) / kThreads, 1u << 20); }

// y = act(z) + residual, m rows of n
__global__ __launch_bounds__(kThreads) void act_kernel(const float* z, const float* __restrict__ residual, long residual_sr, float* y,
                                                      size_t total, long n, Activation act)
{
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (size_t)gridDim.x * kThreads) {
        const float v = act(z[i]);
        y[i] = residual ? v + residual[(long)(i / n) * residual_sr + (long)(i % n)] : v;
    }
}

// y = act(g) (*) u, z = [g | u]
__global__ __launch_bounds__(kThreads) void gate_kernel(const float* __restrict__ z, float* __restrict__ y, size_t total, long f, Activation act)
{
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (size_t)gridDim.x * kThreads) {
        const size_t at = i / f * (2 * f) + i % f;
        y[i] = pam_mul_off(act(z[at]), z[at + f], act.off, act.has_off);
    }
}

__global__ __launch_bounds__(kThreads) void act_bwd_kernel(const float* __restrict__ z, const float* __restrict__ dy, float* __restrict__ dz, size_t total,
                                                          Activation act, ApproxFlags flags)
{
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (size_t)gridDim.x * kThreads)
        dz[i] = activation_grad(act, z[i], dy[i], flags);
}

__global__ __launch_bounds__(kThreads) void gate_bwd_kernel(const float* __restrict__ z, const float* __restrict__ dy, float* __restrict__ dz, size_t total,
                                                           long f, Activation act, ApproxFlags flags)
{
    for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (size_t)gridDim.x * kThreads) {
        const size_t at = i / f * (2 * f) + i % f;
        const float g = z[at], u = z[at + f], d = dy[i], a = act(g);
        dz[at] = activation_grad(act, g, mul_grad(a, u, d, flags.a, act.off, act.has_off), flags);
        dz[at + f] = mul_grad(u, a, d, flags.b, act.off, act.has_off);
    }
}

int check_sizes(const char* what, long m, long n, long k, int activation)
{
    if (m < 0 || n < 0 || k < 0 || m > (1L << 30) || n > (1L << 30) || k > (1L << 30))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: size out of range", what);
    if (!known(activation)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: unknown activation %d", what, activation);
    return PAM_HIP_OK;
}

}  // namespace

extern "C" {

size_t pam_hip_linear_act_workspace_bytes(long m, long n, long k) { return pam_hip_gemm_workspace_bytes(1, m, n, k); }

int pam_hip_linear_act_fwd(const float* a, long a_sr, long a_sc, const float* w, long w_sr, long w_sc, const float* bias,
                           int activation, const float* residual, long residual_sr, float* z, float* y, long m, long n, long k,
                           float offset, void* workspace, size_t workspace_bytes, void* stream)
{
    int rc = check_sizes("linear_act_fwd", m, n, k, activation);
    if (rc != PAM_HIP_OK) return rc;
    if (m == 0 || n == 0) return PAM_HIP_OK;
    if (!y || (k > 0 && (!a || !w))) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "linear_act_fwd: null pointer");
    if (pamthin::takes(m, n, k, a_sc, w_sc))
        return pamthin::launch("linear_act_fwd", pamthin::Layer{a, a_sr, w, w_sr, bias, residual, residual_sr, z, y, (int)m, (int)n, (int)k, activation, offset}, false, (hipStream_t)stream);
    float* sums = z ? z : y;
    rc = pam_hip_pam_linear_fwd(a, a_sr, a_sc, w, w_sc, w_sr, bias, sums, n, 1, m, n, k, offset, workspace, workspace_bytes, stream);
    if (rc != PAM_HIP_OK || (!z && !residual && activation == PAM_HIP_ACT_NONE)) return rc;
    const size_t total = (size_t)m * n;
    hipLaunchKernelGGL(act_kernel, dim3(groups_for(total)), dim3(kThreads), 0, (hipStream_t)stream, sums, residual, residual_sr, y, total, n,
                       activation_of(activation, offset));
    return pamhost::check_launch("linear_act_fwd");
}

size_t pam_hip_gated_linear_workspace_bytes(long m, long f, long k)
{
    if (m <= 0 || f <= 0 || k < 0) return 0;
    return align256((size_t)m * 2 * f * sizeof(float)) + pam_hip_gemm_workspace_bytes(1, m, 2 * f, k);
}

int pam_hip_gated_linear_fwd(const float* a, long a_sr, long a_sc, const float* w, long w_sr, long w_sc, const float* bias,
                             int activation, float* z, float* y, long m, long f, long k, float offset,
                             void* workspace, size_t workspace_bytes, void* stream)
{
    int rc = check_sizes("gated_linear_fwd", m, 2 * f, k, activation);
    if (rc != PAM_HIP_OK) return rc;
    if (m == 0 || f == 0) return PAM_HIP_OK;
    if (!y || (k > 0 && (!a || !w))) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "gated_linear_fwd: null pointer");
    if (pamthin::takes(m, 2 * f, k, a_sc, w_sc))
        return pamthin::launch("gated_linear_fwd", pamthin::Layer{a, a_sr, w, w_sr, bias, nullptr, 0, z, y, (int)m, (int)f, (int)k, activation, offset}, true, (hipStream_t)stream);
    if (!workspace || workspace_bytes < pam_hip_gated_linear_workspace_bytes(m, f, k))
        return pamhost::fail(PAM_HIP_ERR_WORKSPACE, "gated_linear_fwd: workspace of %zu bytes needed", pam_hip_gated_linear_workspace_bytes(m, f, k));
    const size_t held = align256((size_t)m * 2 * f * sizeof(float));
    float* sums = z ? z : (float*)workspace;
    rc = pam_hip_pam_linear_fwd(a, a_sr, a_sc, w, w_sc, w_sr, bias, sums, 2 * f, 1, m, 2 * f, k, offset, (char*)workspace + held, workspace_bytes - held, stream);
    if (rc != PAM_HIP_OK) return rc;
    const size_t total = (size_t)m * f;
    hipLaunchKernelGGL(gate_kernel, dim3(groups_for(total)), dim3(kThreads), 0, (hipStream_t)stream, sums, y, total, f, activation_of(activation, offset));
    return pamhost::check_launch("gated_linear_fwd");
}

int pam_hip_act_bwd(const float* z, const float* dy, float* dz, size_t n, int activation, float offset, int approx_a, int approx_b,
                    int approx_exp, void* stream)
{
    if (!known(activation) || n > (size_t)1 << 41) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "act_bwd: unknown activation %d or size out of range", activation);
    if (n == 0) return PAM_HIP_OK;
    if (!z || !dy || !dz) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "act_bwd: null pointer");
    hipLaunchKernelGGL(act_bwd_kernel, dim3(groups_for(n)), dim3(kThreads), 0, (hipStream_t)stream, z, dy, dz, n, activation_of(activation, offset),
                       ApproxFlags{approx_a != 0, approx_b != 0, approx_exp != 0});
    return pamhost::check_launch("act_bwd");
}

int pam_hip_gated_bwd(const float* z, const float* dy, float* dz, long m, long f, int activation, float offset, int approx_a, int approx_b,
                      int approx_exp, void* stream)
{
    const int rc = check_sizes("gated_bwd", m, 2 * f, 0, activation);
    if (rc != PAM_HIP_OK) return rc;
    if (m == 0 || f == 0) return PAM_HIP_OK;
    if (!z || !dy || !dz) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "gated_bwd: null pointer");
    const size_t total = (size_t)m * f;
    hipLaunchKernelGGL(gate_bwd_kernel, dim3(groups_for(total)), dim3(kThreads), 0, (hipStream_t)stream, z, dy, dz, total, f,
                       activation_of(activation, offset), ApproxFlags{approx_a != 0, approx_b != 0, approx_exp != 0});
    return pamhost::check_launch("gated_bwd");
}

}  // extern "C"
