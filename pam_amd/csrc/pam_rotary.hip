// The rotation of queries' and keys' heads by their positions, after an optional norm of each head, and its gradient.
#include <algorithm>
#include <climits>

#include "../../include/pam_hip_extra.h"
#include "pam_activation.h"
#include "pam_common.h"

using namespace pamdev;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

struct RotaryArgs {
    pam_hip_heads part[2];
    float* terms[2];                              // backward: per-head terms of the weights' gradients, [rows of the part][dim]
    const float* cos; const float* sin; long table_rows;
    const long long* positions; long p_sb, p_st;
    long tokens, rows;
    int heads, dim, half, interleaved;            // heads: of both parts
    float eps, off; bool has_off;
    ApproxFlags flags;
};

// A head: its values, its outputs, the rows of the tables.
struct Head {
    int part; long row;                           // which tensor, which of its heads
    const float* x; const float* dy; const float* weight;
    float* y;
    const float* cos; const float* sin;           // null: no such position
};
__device__ __forceinline__ Head find_head(const RotaryArgs& a, long row)
{
    Head h;
    const long token = row / a.heads, b = token / a.tokens, t = token - b * a.tokens;
    long at = row - token * a.heads;
    h.part = at >= a.part[0].heads ? 1 : 0;
    const pam_hip_heads& p = a.part[h.part];
    if (h.part) at -= a.part[0].heads;
    h.row = token * p.heads + at;
    h.x = p.x + b * p.x_sb + t * p.x_st + at * p.x_sh;
    h.dy = p.dy ? p.dy + b * p.dy_sb + t * p.dy_st + at * p.dy_sh : nullptr;
    h.weight = p.weight;
    h.y = p.y + h.row * a.dim;
    const long long pos = a.positions ? a.positions[b * a.p_sb + t * a.p_st] : t;
    const bool there = pos >= 0 && pos < a.table_rows;
    h.cos = there ? a.cos + pos * a.half : nullptr;
    h.sin = there ? a.sin + pos * a.half : nullptr;
    return h;
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s, 64);
    return v;
}

// mean(x (*) x) + eps and its root, over the wavefront
struct Root { float sum, variance, root; };
__device__ __forceinline__ Root head_root(const RotaryArgs& a, const float* x, int lane)
{
    float sum = 0.0f;
    for (int i = lane; i < a.dim; i += 64) sum += pam_mul_off(x[i], x[i], a.off, a.has_off);
    Root r;
    r.sum = wave_sum(sum);
    r.variance = pad_div_off(r.sum, (float)a.dim, a.off, a.has_off) + a.eps;
    r.root = pow_half(r.variance, a.off, a.has_off);
    return r;
}
__device__ __forceinline__ float normed(const RotaryArgs& a, float x, float root) { return pad_div_off(x, root, a.off, a.has_off); }

__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a)
{
    const long row = (long)blockIdx.x * kWaves + threadIdx.x / 64;
    const int lane = threadIdx.x % 64;
    if (row >= a.rows) return;
    const Head h = find_head(a, row);
    const float root = h.weight ? head_root(a, h.x, lane).root : 1.0f;
    auto value = [&](int i) { return h.weight ? pam_mul_off(normed(a, h.x[i], root), h.weight[i], a.off, a.has_off) : h.x[i]; };
    for (int p = lane; p < a.half; p += 64) {
        const int i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + a.half;
        const float z1 = value(i), z2 = value(j);
        const float c = h.cos ? h.cos[p] : u2f(kQNaN), s = h.sin ? h.sin[p] : u2f(kQNaN);
        h.y[i] = pam_mul_off(z1, c, a.off, a.has_off) - pam_mul_off(z2, s, a.off, a.has_off);
        h.y[j] = pam_mul_off(z2, c, a.off, a.has_off) + pam_mul_off(z1, s, a.off, a.has_off);
    }
    for (int i = 2 * a.half + lane; i < a.dim; i += 64) h.y[i] = value(i);
}

// The gradient: dz from dy by the rotation's products, then through weight, quotient, root, mean and square.
__global__ __launch_bounds__(kThreads) void rotary_bwd_kernel(RotaryArgs a)
{
    const long row = (long)blockIdx.x * kWaves + threadIdx.x / 64;
    const int lane = threadIdx.x % 64;
    if (row >= a.rows) return;
    const Head h = find_head(a, row);
    const float off = a.off;
    const bool has_off = a.has_off, norm = h.weight != nullptr;
    const ApproxFlags f = a.flags;
    const Root r = norm ? head_root(a, h.x, lane) : Root{0.0f, 0.0f, 1.0f};
    float* terms = a.terms[h.part] ? a.terms[h.part] + h.row * a.dim : nullptr;
    auto n_of = [&](int i) { return normed(a, h.x[i], r.root); };
    auto z_of = [&](int i) { return norm ? pam_mul_off(n_of(i), h.weight[i], off, has_off) : h.x[i]; };
    // calls to(i, dz of value i) for the lane's values
    auto walk = [&](auto to) {
        for (int p = lane; p < a.half; p += 64) {
            const int i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + a.half;
            const float z1 = z_of(i), z2 = z_of(j), d1 = h.dy[i], d2 = h.dy[j];
            const float c = h.cos ? h.cos[p] : u2f(kQNaN), s = h.sin ? h.sin[p] : u2f(kQNaN);
            to(i, mul_grad(z1, c, d1, f.a, off, has_off) + mul_grad(z1, s, d2, f.a, off, has_off));
            to(j, mul_grad(z2, c, d2, f.a, off, has_off) + mul_grad(z2, s, -d1, f.a, off, has_off));
        }
        for (int i = 2 * a.half + lane; i < a.dim; i += 64) to(i, h.dy[i]);
    };
    if (!norm) {
        walk([&](int i, float dz) { h.y[i] = dz; });
        return;
    }
    float droot = 0.0f;
    walk([&](int i, float dz) {
        const float n = n_of(i);
        if (terms) terms[i] = mul_grad(h.weight[i], n, dz, f.b, off, has_off);
        droot += div_grad_b(h.x[i], r.root, mul_grad(n, h.weight[i], dz, f.a, off, has_off), f.b, off, has_off);
    });
    droot = wave_sum(droot);
    // pow(v, 0.5) = 2^(log2(v) (*) 0.5), zero where v is zero; then the mean's quotient
    const float l = log2_entry(r.variance, off, has_off), t = pam_mul_off(l, 0.5f, off, has_off);
    const float dt = exp2_grad(t, exp2_entry(t, off, has_off), r.variance == 0.0f ? 0.0f : droot, f.e, off, has_off);
    const float dl = mul_grad(l, 0.5f, dt, f.a, off, has_off);
    const float dv = f.e ? pad_div_off(pad_div_off(dl, r.variance, off, has_off), kActLn2, off, has_off) : log2_entry_bwd(r.variance, dl, off, has_off);
    const float dsquare = div_grad_a(r.sum, (float)a.dim, dv, f.a, off, has_off);
    walk([&](int i, float dz) {
        const float x = h.x[i], n = n_of(i);
        const float through = div_grad_a(x, r.root, mul_grad(n, h.weight[i], dz, f.a, off, has_off), f.a, off, has_off);
        h.y[i] = through + (mul_grad(x, x, dsquare, f.a, off, has_off) + mul_grad(x, x, dsquare, f.b, off, has_off));
    });
}

int fill(const char* what, RotaryArgs& a, const pam_hip_heads* parts, int count, const float* cos, const float* sin, long table_rows,
         const long long* positions, long p_sb, long p_st, long batch, long tokens, long dim, long rotated, int interleaved, float eps, float offset,
         bool backward)
{
    if (count < 1 || count > 2 || !parts) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: one or two tensors", what);
    if (batch < 0 || tokens < 0 || dim < 0 || rotated < 0 || table_rows < 0 || parts[0].heads < 0 || (count > 1 && parts[1].heads < 0))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: negative size", what);
    if (rotated % 2 != 0 || rotated > dim) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the rotated part is an even number of a head's values", what);
    const long heads = parts[0].heads + (count > 1 ? parts[1].heads : 0);
    if (batch > (1L << 30) || tokens > (1L << 30) || dim > (1L << 20) || heads > (1L << 20) || (batch && tokens && heads > (1L << 40) / batch / tokens))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: size out of range", what);
    a.rows = batch * tokens * heads;
    for (int i = 0; i < 2; ++i) {
        a.part[i] = i < count ? parts[i] : pam_hip_heads{};
        a.terms[i] = nullptr;
        if (a.rows && dim && a.part[i].heads && (!a.part[i].x || !a.part[i].y || (backward && !a.part[i].dy)))
            return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: null pointer", what);
    }
    if (a.rows && rotated && (!cos || !sin) && table_rows > 0) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: null pointer", what);
    a.cos = cos; a.sin = sin; a.table_rows = table_rows; a.positions = positions; a.p_sb = p_sb; a.p_st = p_st;
    a.tokens = tokens; a.heads = (int)heads; a.dim = (int)dim; a.half = (int)(rotated / 2); a.interleaved = interleaved != 0;
    a.eps = eps; a.off = offset; a.has_off = offset != 1.0f;
    a.flags = ApproxFlags{false, false, false};
    if ((a.rows + kWaves - 1) / kWaves > INT_MAX) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: too many heads", what);
    return PAM_HIP_OK;
}

}  // namespace

extern "C" {

int pam_hip_rotary_fwd(const pam_hip_heads* parts, int count, const float* cos, const float* sin, long table_rows, const long long* positions,
                       long positions_sb, long positions_st, long batch, long tokens, long dim, long rotated, int interleaved, float eps,
                       float offset, void* stream)
{
    RotaryArgs a;
    const int rc = fill("rotary_fwd", a, parts, count, cos, sin, table_rows, positions, positions_sb, positions_st, batch, tokens, dim, rotated, interleaved, eps, offset, false);
    if (rc != PAM_HIP_OK || a.rows == 0 || dim == 0) return rc;
    hipLaunchKernelGGL(rotary_kernel, dim3((unsigned)((a.rows + kWaves - 1) / kWaves)), dim3(kThreads), 0, (hipStream_t)stream, a);
    return pamhost::check_launch("rotary_fwd");
}

static size_t terms_floats(const pam_hip_heads& p, long batch, long tokens, long dim) { return p.dweight ? (size_t)(batch * tokens * p.heads) * dim : 0; }

size_t pam_hip_rotary_bwd_workspace_bytes(const pam_hip_heads* parts, int count, long batch, long tokens, long dim)
{
    size_t bytes = 0;
    for (int i = 0; parts && i < count && i < 2; ++i) {
        const long rows = batch * tokens * parts[i].heads;
        if (parts[i].dweight) bytes += ((terms_floats(parts[i], batch, tokens, dim) * 4 + 255) & ~(size_t)255) + ((pam_hip_column_sums_workspace_bytes(rows, dim, 1) + 255) & ~(size_t)255);
    }
    return bytes;
}

int pam_hip_rotary_bwd(const pam_hip_heads* parts, int count, const float* cos, const float* sin, long table_rows, const long long* positions,
                       long positions_sb, long positions_st, long batch, long tokens, long dim, long rotated, int interleaved, float eps,
                       float offset, int approx_a, int approx_b, int approx_exp, void* workspace, size_t workspace_bytes, void* stream)
{
    RotaryArgs a;
    int rc = fill("rotary_bwd", a, parts, count, cos, sin, table_rows, positions, positions_sb, positions_st, batch, tokens, dim, rotated, interleaved, eps, offset, true);
    if (rc != PAM_HIP_OK || dim == 0) return rc;
    a.flags = ApproxFlags{approx_a != 0, approx_b != 0, approx_exp != 0};
    const size_t need = pam_hip_rotary_bwd_workspace_bytes(parts, count, batch, tokens, dim);
    if (need && (!workspace || workspace_bytes < need)) return pamhost::fail(PAM_HIP_ERR_WORKSPACE, "rotary_bwd: workspace of %zu bytes needed", need);
    char* at = (char*)workspace;
    for (int i = 0; i < count; ++i)
        if (parts[i].dweight) {
            a.terms[i] = (float*)at;
            at += (terms_floats(parts[i], batch, tokens, dim) * 4 + 255) & ~(size_t)255;
        }
    if (a.rows) {
        hipLaunchKernelGGL(rotary_bwd_kernel, dim3((unsigned)((a.rows + kWaves - 1) / kWaves)), dim3(kThreads), 0, (hipStream_t)stream, a);
        rc = pamhost::check_launch("rotary_bwd");
    }
    for (int i = 0; i < count && rc == PAM_HIP_OK; ++i)
        if (parts[i].dweight) {
            const long rows = batch * tokens * parts[i].heads;
            const size_t bytes = pam_hip_column_sums_workspace_bytes(rows, dim, 1);
            rc = pam_hip_column_sums(a.terms[i], dim, parts[i].dweight, nullptr, 0, nullptr, rows, dim, bytes ? at : nullptr, bytes, stream);
            at += (bytes + 255) & ~(size_t)255;
        }
    return rc;
}

}  // extern "C"
