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

// ---------------------------------------------------------------- the usual case

// The primitives as single integer additions: with signs and exponents in place a (*) b is bits(a) + bits(b) - bias, a (/) b is
// bits(a) - bits(b) + bias, and an offset, one more product or quotient of the result, is one more constant in either.  That holds while operands and results are normal numbers, which the
// callers make sure of by windows on what goes in: exponents of [first, last) per kind of value, chosen so that no result of
// a chain leaves the normal range, whatever the values in them.
struct Raw {
    uint32_t mul_add, div_add;
    __device__ __forceinline__ explicit Raw(float off) : mul_add(f2u(off) - 2u * kBias), div_add(2u * kBias - f2u(off)) {}
    __device__ __forceinline__ float mul(float a, float b) const { return u2f(f2u(a) + f2u(b) + mul_add); }
    __device__ __forceinline__ float div(float a, float b) const { return u2f(f2u(a) - f2u(b) + div_add); }
    // 2^t for |t| <= 126, t (*) 1 (*) offset first as the base-2 entry point has it
    __device__ __forceinline__ float exp2(float t) const
    {
        const float x = mul(t, 1.0f), whole = floorf(x);
        return u2f((uint32_t)((int)whole + 127) << 23) * ((1.0f + x) - whole);
    }
};
// The gradients of the primitives by additions and, where a slope is exact, a product with a power of two (the formulas of
// pam_mul_bwd, pad_div_bwd and the base-2 entry points for normal numbers).  APPROXIMATE: all are approximate; otherwise `approx` says.
template <bool APPROXIMATE>
struct RawGrad : Raw {
    uint32_t off_add;                             // bits(b (*) offset) - bits(b)
    __device__ __forceinline__ explicit RawGrad(float off) : Raw(off), off_add(f2u(off) - kBias) {}
    __device__ __forceinline__ static float slope(uint32_t other, float own) { return u2f((other + (f2u(own) & kMant)) & ~kMant); }
    __device__ __forceinline__ float of_mul(float own, float other, float d, bool approx) const
    {
        const float a = mul(d, other);
        return APPROXIMATE || approx ? a : d * slope(f2u(other) + off_add, own);
    }
    __device__ __forceinline__ float of_dividend(float a, float inverse, float d, bool approx) const       // inverse: 1 (/) b
    {
        const float v = mul(inverse, d);
        return APPROXIMATE || approx ? v : d * slope(f2u(inverse), a);
    }
    __device__ __forceinline__ float of_divisor(float quotient, float b, float d, bool approx) const       // b positive
    {
        const float a = mul(div(quotient, b), d);
        return -(APPROXIMATE || approx ? a : d * u2f((f2u(quotient) & ~kMant) - (f2u(b) & kExpo) + kBias));
    }
    __device__ __forceinline__ float of_exp2(float t, float e, float d, bool approx) const
    {
        const float a = mul(mul(e, kActLn2), d);
        return APPROXIMATE || approx ? a : u2f(f2u(e) & ~kMant) * d * slope(off_add + kBias, t);
    }
    __device__ __forceinline__ float of_log2(float v, float d, bool approx) const                          // v positive
    {
        const float a = div(div(d, v), kActLn2), log = (float)((int)f2u(v) - (int)kBias) * 0x1p-23f;
        return APPROXIMATE || approx ? a : d * slope(f2u(div(1.0f, 1.0f)), log) * u2f((254u << 23) - (f2u(v) & kExpo));
    }
};
template <int FIRST, int LAST>                    // magnitudes 2^FIRST <= |v| < 2^LAST: one shift-add and a max per value
struct Window {
    uint32_t most = 0;
    __device__ __forceinline__ void see(float v) { most = max(most, (f2u(v) << 1) - ((uint32_t)(FIRST + 127) << 24)); }
    __device__ __forceinline__ bool held() const { return most < ((uint32_t)(LAST - FIRST) << 24); }
};
// offsets that the windows allow for: at most a factor of 2^0.6 on each of a chain's results
__device__ __forceinline__ bool usual_offset(float off) { return off > 0.75f && off < 1.5f; }

__device__ __forceinline__ bool is_zero(float v) { return (f2u(v) << 1) == 0u; }
// a (*) b by addition, zeros by the definition (the sign of the other operand)
__device__ __forceinline__ float mul_or_zero(const Raw& ar, float a, float b)
{
    const bool za = is_zero(a), zb = is_zero(b);
    const uint32_t sign = ((za ? 0u : f2u(a)) ^ (zb ? 0u : f2u(b))) & kSign;
    return za || zb ? u2f(sign) : ar.mul(a, b);
}

// silu and gelu of zero and 2^-40 <= |x| < 16 by additions, with the offsets of usual_sigmoid_offset: t (*) offset lies within 44.3 of zero, u in
// [1, 2^44.4), x (/) u in 2^[-41, 4).  For the gradient d, |d| in 2^[-40, 40), the smallest result is x (/) u (/) u (*) d at x = -16: above
// 2^-125 with the largest offset, its own factors counted, and 2^-115 without one.  A zero x stands as 2^-40 (2^t is 1 there),
// which leaves the gradient what it is.
__device__ __forceinline__ bool usual_sigmoid_offset(float off) { return off > 0.9f && off < 1.06f; }
typedef Window<-40, 4> WindowAct;
typedef Window<-40, 40> WindowActGrad;
struct RawSigmoid {
    float x, t, e, u;
    __device__ __forceinline__ RawSigmoid(const Raw& ar, float value, float scale)
    {
        x = is_zero(value) ? 0x1p-40f : value;
        t = ar.mul(x, scale);
        e = ar.exp2(t);
        u = 1.0f + e;
    }
    __device__ __forceinline__ float result(const Raw& ar, float value) const { return is_zero(value) ? 0.0f : ar.div(x, u); }
    template <bool APPROXIMATE>
    __device__ __forceinline__ float grad(const RawGrad<APPROXIMATE>& ar, float d, float scale, const ApproxFlags& f) const        // d not zero
    {
        const float du = ar.of_divisor(ar.div(x, u), u, d, f.b), dt = ar.of_exp2(t, e, du, f.e);
        return ar.of_dividend(x, ar.div(1.0f, u), d, f.a) + ar.of_mul(x, scale, dt, f.a);
    }
};

// act(v) of a lane's values: by additions where all of the wavefront's are ordinary, else by the checked function, called.  Four at a time, in a
// loop that turns the array around, so that the code is there once (sixteen values written out: the same time, four times the code).
__device__ __noinline__ float any_activation(float x, int kind, float off) { return Activation{kind, off, off != 1.0f}(x); }
template <int N>
__device__ __forceinline__ void turn(float (&v)[N], int by)
{
    float w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = v[(i + by) % N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = w[i];
}
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int kind, float off)
{
    if (kind == PAM_HIP_ACT_NONE) return;
    if (kind == PAM_HIP_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] <= 0.0f ? 0.0f : v[i];
        return;
    }
    constexpr int kWide = N < 4 ? N : 4;
    const float scale = kind == PAM_HIP_ACT_SILU ? kSiluScale : kGeluScale;
    const Raw ar(off);
#pragma unroll 1
    for (int part = 0; part < N; part += kWide) {
        WindowAct seen;
        float y[kWide];
#pragma unroll
        for (int i = 0; i < kWide; ++i) {
            if (!is_zero(v[i])) seen.see(v[i]);
            y[i] = RawSigmoid(ar, v[i], scale).result(ar, v[i]);
        }
        if (__ballot(!seen.held() || !usual_sigmoid_offset(off)) != 0ull) {
#pragma unroll
            for (int i = 0; i < kWide; ++i) y[i] = v[i];
#pragma unroll 1
            for (int i = 0; i < kWide; ++i) {
                y[0] = any_activation(y[0], kind, off);
                turn(y, 1);
            }
        }
#pragma unroll
        for (int i = 0; i < kWide; ++i) v[i] = y[i];
        turn(v, kWide);
    }
}

}  // namespace pamdev
