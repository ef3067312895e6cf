// Activations in PAM arithmetic and their gradients, as the chain of primitives computes them.
//   relu(x);  silu, gelu: y = x (/) u, u = 1 + e, e = 2^t, t = min(x (*) c, 64), c = -log2 e or -1.702 log2 e
// `off` is the offset of every PAM operation (pam/native.py:59-60, 168-169).
#pragma once
#include "../../include/pam_hip_block.h"
#include "pam_device.h"

namespace pamdev {

constexpr float kActCap = 64.0f;
constexpr float kSiluScale = (float)(-1.4426950408889634), kGeluScale = (float)(-1.702 * 1.4426950408889634);
constexpr float kActLn2 = (float)0.6931471805599453;

struct Activation {
    int kind;                    // PAM_HIP_ACT_*
    float off; bool has_off;
    __device__ __forceinline__ float scale() const { return kind == PAM_HIP_ACT_SILU ? kSiluScale : kGeluScale; }
    __device__ __forceinline__ float operator()(float x) const
    {
        if (kind == PAM_HIP_ACT_NONE) return x;
        if (kind == PAM_HIP_ACT_RELU) return x <= 0.0f ? 0.0f : x;              // (NaN stays)
        const float t = pam_mul_off(x, scale(), off, has_off);
        return pad_div_off(x, 1.0f + exp2_entry(t > kActCap ? kActCap : t, off, has_off), off, has_off);
    }
};

// Which gradients are the approximate ones: of first and second operands of products and quotients, of exp2.
struct ApproxFlags { bool a, b, e; };

// The gradient for A of A (*) B and for B, and those of A (/) B, as the autograd functions of the primitives compute them
// (pam/cuda_bindings.py:43-57, 78-97).
__device__ __forceinline__ float mul_grad(float own, float other, float d, bool approx, float off, bool has_off)
{ return approx ? pam_mul_off(d, other, off, has_off) : pam_mul_bwd(own, other, d, off, has_off); }
__device__ __forceinline__ float div_grad_a(float a, float b, float d, bool approx, float off, bool has_off)
{
    const float inv = pad_div_off(1.0f, b, off, has_off);
    return approx ? pam_mul_off(inv, d, off, has_off) : pam_mul_bwd(a, inv, d, 1.0f, false);
}
__device__ __forceinline__ float div_grad_b(float a, float b, float d, bool approx, float off, bool has_off)
{
    return approx ? -pam_mul_off(pad_div_off(pad_div_off(a, b, off, has_off), b, off, has_off), d, off, has_off)
                  : pad_div_bwd(a, b, d, off, has_off);
}
// ... of 2^t
__device__ __forceinline__ float exp2_grad(float t, float e, float d, bool approx, float off, bool has_off)
{ return approx ? pam_mul_off(pam_mul_off(e, kActLn2, off, has_off), d, off, has_off) : exp2_entry_bwd(t, d, off, has_off); }

// The gradient for x of act(x), d that of the result.
__device__ __forceinline__ float activation_grad(const Activation& act, float x, float d, const ApproxFlags& f)
{
    if (act.kind == PAM_HIP_ACT_NONE) return d;
    if (act.kind == PAM_HIP_ACT_RELU) return x <= 0.0f ? 0.0f : d;
    const float c = act.scale(), off = act.off;
    const bool has_off = act.has_off;
    const float t = pam_mul_off(x, c, off, has_off), tc = t > kActCap ? kActCap : t;
    const float e = exp2_entry(tc, off, has_off), u = 1.0f + e;
    const float du = div_grad_b(x, u, d, f.b, off, has_off);
    const float dt = t <= kActCap ? exp2_grad(tc, e, du, f.e, off, has_off) : 0.0f;      // (the bound passes no gradient)
    return div_grad_a(x, u, d, f.a, off, has_off) + mul_grad(x, c, dt, f.a, off, has_off);
}

}  // namespace pamdev
