// The product with an activation and a residual, and the gated layer: entry points and the elementwise kernels.
#include <algorithm>

#include "pam_activation.h"
#include "pam_common.h"
#include "pam_gemm_layer.h"
#include "pam_thin.h"

using namespace pamdev;

namespace {

constexpr int kThreads = 256;

Activation activation_of(int kind, float offset) { return Activation{kind, offset, offset != 1.0f}; }
bool known(int activation) { return activation >= PAM_HIP_ACT_NONE && activation <= PAM_HIP_ACT_GELU; }
unsigned groups_for(size_t values) { return (unsigned)std::min<size_t>((values + kThreads - 1) / kThreads, 1u << 20); }

// The gradients for z: dz = [dg | du] of rows of f values (GATED), or of one row of all of them.
//
// Bound by memory, 12 bytes a value or 20 a gated one.  A lane takes four consecutive values (a row's last ones overlap the
// ones before, written alike).  With every value of the wavefront of ordinary size the chain is integer additions, and products with powers
// of two where a slope is exact (pam_activation.h); otherwise the checked functions compute it value by value.  4096 x 2048 gated values, 168 MB:
// 27 us approximate, 40 exact (checked value by value 66).
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

struct BwdArgs {
    const float* z; const float* dy; float* dz;
    long f;                                       // values of a row; GATED: of a half
    uint32_t per_row, units;                      // lanes' shares of a row, of all rows
    Activation act;
    ApproxFlags flags;
};

template <bool GATED>
__device__ __forceinline__ void bwd_value(const BwdArgs& a, float g, float u, float d, float& dg, float& du)
{
    if (GATED) {
        const float y = a.act(g);
        du = mul_grad(u, y, d, a.flags.b, a.act.off, a.act.has_off);
        d = mul_grad(y, u, d, a.flags.a, a.act.off, a.act.has_off);
    }
    dg = activation_grad(a.act, g, d, a.flags);
}

// APPROXIMATE: all slopes are.
template <bool GATED, bool APPROXIMATE>
__global__ __launch_bounds__(kThreads) void act_bwd_kernel(BwdArgs a)
{
    const uint32_t unit = blockIdx.x * kThreads + threadIdx.x;
    if (unit >= a.units) return;
    const uint32_t row = GATED ? unit / a.per_row : 0u, share = GATED ? unit - row * a.per_row : unit;
    const long column = min((long)share * 4, a.f - 4), at = (long)row * a.f + column, z_at = GATED ? at + (long)row * a.f : at;
    const v4f g = *reinterpret_cast<const v4f_any*>(a.z + z_at), d = *reinterpret_cast<const v4f_any*>(a.dy + at);
    const v4f u = GATED ? *reinterpret_cast<const v4f_any*>(a.z + z_at + a.f) : g;
    v4f dg, du;
    const bool sigmoid = a.act.kind >= PAM_HIP_ACT_SILU, relu = a.act.kind == PAM_HIP_ACT_RELU;
    const RawGrad<APPROXIMATE> ar(a.act.off);
    bool held = usual_sigmoid_offset(a.act.off);
    WindowAct gates;
    WindowActGrad grads;                          // (and the gated product's operands: two of them make 2^[-80, 80))
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool nothing = is_zero(d[i]);
        const RawSigmoid s(ar, g[i], a.act.scale());
        float y = g[i], to_gate = d[i];
        if (sigmoid) {
            if (!is_zero(g[i])) gates.see(g[i]);
            y = s.result(ar, g[i]);
        } else if (relu) y = g[i] <= 0.0f ? 0.0f : g[i];
        if (!APPROXIMATE) held = held && !(nothing || (GATED && is_zero(y)));      // (exact slopes of zeros: the checked functions')
        if (GATED) {
            if (!nothing) grads.see(d[i]);
            if (!sigmoid && !is_zero(y)) grads.see(y);
            grads.see(u[i]);                      // (a zero there is left to the checked functions)
            du[i] = APPROXIMATE ? mul_or_zero(ar, d[i], y) : ar.of_mul(u[i], y, d[i], a.flags.b);
            to_gate = nothing ? u2f(f2u(u[i]) & kSign) : ar.of_mul(y, u[i], d[i], a.flags.a);
        }
        if (sigmoid) {
            if (!nothing) grads.see(to_gate);
            dg[i] = nothing ? 0.0f : s.grad(ar, to_gate, a.act.scale(), a.flags);
        } else dg[i] = relu && g[i] <= 0.0f ? 0.0f : to_gate;
    }
    if (__ballot(!(held && grads.held() && gates.held())) != 0ull) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float dgi, dui = 0.0f;
            bwd_value<GATED>(a, g[i], u[i], d[i], dgi, dui);
            dg[i] = dgi; du[i] = dui;
        }
    }
    *reinterpret_cast<v4f_any*>(a.dz + z_at) = dg;
    if (GATED) *reinterpret_cast<v4f_any*>(a.dz + z_at + a.f) = du;
}

// ... of rows of fewer than four values
template <bool GATED>
__global__ __launch_bounds__(kThreads) void short_act_bwd_kernel(BwdArgs a, long rows)
{
    for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < rows * a.f; i += (long)gridDim.x * kThreads) {
        const long row = i / a.f, z_at = GATED ? i + row * a.f : i;
        float dg, du;
        bwd_value<GATED>(a, a.z[z_at], GATED ? a.z[z_at + a.f] : 0.0f, a.dy[i], dg, du);
        a.dz[z_at] = dg;
        if (GATED) a.dz[z_at + a.f] = du;
    }
}

template <bool GATED>
int launch_bwd(const char* what, BwdArgs a, long rows, hipStream_t st)
{
    if (a.f < 4) {
        hipLaunchKernelGGL((short_act_bwd_kernel<GATED>), dim3(groups_for((size_t)(rows * a.f))), dim3(kThreads), 0, st, a, rows);
        return pamhost::check_launch(what);
    }
    const auto launch = [&]() {
        const dim3 grid((a.units + kThreads - 1) / kThreads);
        if (a.flags.a && a.flags.b && a.flags.e) hipLaunchKernelGGL((act_bwd_kernel<GATED, true>), grid, dim3(kThreads), 0, st, a);
        else hipLaunchKernelGGL((act_bwd_kernel<GATED, false>), grid, dim3(kThreads), 0, st, a);
        return pamhost::check_launch(what);
    };
    // (a launch counts its units in 32 bits: more rows, or a longer one, are several launches)
    constexpr long kMost = 1L << 30;
    if (GATED) {
        a.per_row = (uint32_t)((a.f + 3) / 4);
        for (long first = 0; first < rows; ) {
            const long n = std::min(rows - first, std::max(1L, kMost / (long)a.per_row));
            a.units = (uint32_t)(n * a.per_row);
            const int rc = launch();
            if (rc != PAM_HIP_OK) return rc;
            first += n; a.z += n * 2 * a.f; a.dz += n * 2 * a.f; a.dy += n * a.f;
        }
        return PAM_HIP_OK;
    }
    for (long left = a.f; left > 0; ) {
        a.f = left - 4 * kMost < 4 ? left : 4 * kMost;                        // (a launch's row has at least four)
        if (a.f > 4 * kMost) a.f = 2 * kMost;
        a.per_row = a.units = (uint32_t)((a.f + 3) / 4);
        const int rc = launch();
        if (rc != PAM_HIP_OK) return rc;
        left -= a.f; a.z += a.f; a.dz += a.f; a.dy += a.f;
    }
    return PAM_HIP_OK;
}

int check_sizes(const char* what, long m, long n, long k, int activation)
{
    if (m < 0 || n < 0 || k < 0 || m > (1L << 30) || n > (1L << 30) || k > (1L << 30))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: size out of range", what);
    if (!known(activation)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: unknown activation %d", what, activation);
    return PAM_HIP_OK;
}

long both_halves(long f) { return f < 0 || f > (1L << 30) ? f : 2 * f; }      // (out of range as it is, not past a long)

}  // namespace

extern "C" {

size_t pam_hip_linear_act_workspace_bytes(long m, long n, long k) { return pamgemm::layer_workspace(m, n, k); }

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
    return pamgemm::layer_product("linear_act_fwd", false, a, a_sr, a_sc, w, w_sr, w_sc, bias, residual, residual_sr, activation, z, y, m, n, k, offset,
                                  workspace, workspace_bytes, stream);
}

size_t pam_hip_gated_linear_workspace_bytes(long m, long f, long k)
{
    return m <= 0 || f <= 0 ? 0 : pamgemm::layer_workspace(m, pamgemm::gated_columns(f), k);
}

int pam_hip_gated_linear_fwd(const float* a, long a_sr, long a_sc, const float* w, long w_sr, long w_sc, const float* bias,
                             int activation, float* z, float* y, long m, long f, long k, float offset,
                             void* workspace, size_t workspace_bytes, void* stream)
{
    int rc = check_sizes("gated_linear_fwd", m, both_halves(f), k, activation);
    if (rc != PAM_HIP_OK) return rc;
    if (m == 0 || f == 0) return PAM_HIP_OK;
    if (!y || (k > 0 && (!a || !w))) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "gated_linear_fwd: null pointer");
    if (pamthin::takes(m, 2 * f, k, a_sc, w_sc))
        return pamthin::launch("gated_linear_fwd", pamthin::Layer{a, a_sr, w, w_sr, bias, nullptr, 0, z, y, (int)m, (int)f, (int)k, activation, offset}, true, (hipStream_t)stream);
    return pamgemm::layer_product("gated_linear_fwd", true, a, a_sr, a_sc, w, w_sr, w_sc, bias, nullptr, 0, activation, z, y, m, f, k, offset,
                                  workspace, workspace_bytes, stream);
}

int pam_hip_act_bwd(const float* z, const float* dy, float* dz, size_t n, int activation, float offset, int approx_a, int approx_b,
                    int approx_exp, void* stream)
{
    if (!known(activation) || n > (size_t)1 << 41) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "act_bwd: unknown activation %d or size out of range", activation);
    if (n == 0) return PAM_HIP_OK;
    if (!z || !dy || !dz) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "act_bwd: null pointer");
    return launch_bwd<false>("act_bwd", BwdArgs{z, dy, dz, (long)n, 0, 0, activation_of(activation, offset), ApproxFlags{approx_a != 0, approx_b != 0, approx_exp != 0}},
                             1, (hipStream_t)stream);
}

int pam_hip_gated_bwd(const float* z, const float* dy, float* dz, long m, long f, int activation, float offset, int approx_a, int approx_b,
                      int approx_exp, void* stream)
{
    const int rc = check_sizes("gated_bwd", m, both_halves(f), 0, activation);
    if (rc != PAM_HIP_OK) return rc;
    if (m == 0 || f == 0) return PAM_HIP_OK;
    if (!z || !dy || !dz) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "gated_bwd: null pointer");
    return launch_bwd<true>("gated_bwd", BwdArgs{z, dy, dz, f, 0, 0, activation_of(activation, offset), ApproxFlags{approx_a != 0, approx_b != 0, approx_exp != 0}},
                            m, (hipStream_t)stream);
}

}  // extern "C"
