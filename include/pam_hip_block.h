/*
 * pam_hip_block.h -- entry points of libpam_hip.so for the operators of a decoder block and its training step: a product with
 * an activation and a residual, the gated layer, the rotation of queries and keys, the clipping of gradients.  The reference
 * has no counterparts; each is a composition of the primitives of pam_hip.h.  Conventions as in pam_hip.h.  Results share no memory
 * with each other or with what is read, unless it is said that they may.
 */
#ifndef PAM_HIP_BLOCK_H
#define PAM_HIP_BLOCK_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Activations.  silu and gelu are x (/) (1 + 2^t), t = min(x (*) c, 64), with c = -log2 e and -1.702 log2 e: x times the
 * logistic function of x or 1.702 x as one quotient.  (Without the bound 2^t would overflow for x below -88, and the quotient by
 * an infinity is NaN in this arithmetic; x (/) 2^64 is nothing beside the sums it goes to.) */
enum { PAM_HIP_ACT_NONE = 0, PAM_HIP_ACT_RELU = 1, PAM_HIP_ACT_SILU = 2, PAM_HIP_ACT_GELU = 3 };

/* y[m][n] = act(a[m][k] (x) w[n][k]^T + bias[n]) + residual[m][n].  y and z are contiguous; bias and residual may be NULL;
 * residual's rows are contiguous, residual_sr apart.  z, if not NULL, receives what the activation is applied to (a backward pass
 * reads it).  The offset goes to every PAM operation, as in the chain of primitives: folded into w for the products.
 * Sums: up to 24 rows of a, with a and w contiguous along k, are added up lane by lane along k; otherwise as pam_hip_pam_matmul_fwd
 * adds them, in chains of at most 1024 terms (pam_hip_layer_grad).  The order depends on the sizes and strides, never on values. */
size_t pam_hip_linear_act_workspace_bytes(long m, long n, long k);
int pam_hip_linear_act_fwd(const float *a, long a_sr, long a_sc, const float *w, long w_sr, long w_sc, const float *bias,
                           int activation, const float *residual, long residual_sr, float *z, float *y, long m, long n, long k,
                           float offset, void *workspace, size_t workspace_bytes, void *stream);

/* y[m][f] = act(g) (*) u with [g | u] = a[m][k] (x) w[2 f][k]^T + bias[2 f]: w's first f rows are the gate's.
 * z, if not NULL, receives [g | u], m rows of 2 f. */
size_t pam_hip_gated_linear_workspace_bytes(long m, long f, long k);
int pam_hip_gated_linear_fwd(const float *a, long a_sr, long a_sc, const float *w, long w_sr, long w_sc, const float *bias,
                             int activation, float *z, float *y, long m, long f, long k, float offset,
                             void *workspace, size_t workspace_bytes, void *stream);

/* Gradients for z of the two above from the gradient of y (without the residual, whose gradient is dy itself): the chain of the
 * primitives' gradients.  approx_a / approx_b select the approximate gradient for first / second operands of products and
 * quotients, approx_exp the one of exp2.  All contiguous: n values; m rows of 2 f, f and 2 f values. */
int pam_hip_act_bwd(const float *z, const float *dy, float *dz, size_t n, int activation, float offset,
                    int approx_a, int approx_b, int approx_exp, void *stream);
int pam_hip_gated_bwd(const float *z, const float *dy, float *dz, long m, long f, int activation, float offset,
                      int approx_a, int approx_b, int approx_exp, void *stream);

/* The products of the layers' gradients, dX = dZ (x) W and dW^T = X^T (x) dZ: pam_hip_pam_matmul_fwd (kind 0, the approximate gradient,
 * mo not read) or pam_hip_pam_matmul_bwd (kind 1: l is the upstream gradient, 2: r is), with the sums held to chains of
 * 1024 terms, as in the two forward products above: a chunk of pam_hip_gemm_plan (or all of k, without a workspace) that is longer is
 * added up in equal chains of whole 32 terms, at most 1024, each from +0, whose sums are added in ascending order from +0.  The
 * workspaces of all three are those of the plain products. */
size_t pam_hip_layer_grad_workspace_bytes(long m, long n, long k);
int pam_hip_layer_grad(const float *l, long l_sr, long l_sc, const float *r, long r_sr, long r_sc, const float *mo, long mo_sr, long mo_sc,
                       float *dm, long dm_sr, long dm_sc, long m, long n, long k, int kind, float offset,
                       void *workspace, size_t workspace_bytes, void *stream);

/* The rotation of heads by their positions, after an optional norm of each head.
 *   n = x (/) pow(mean(x (*) x) + eps, 0.5),  z = n (*) weight            (weight NULL: z = x)
 *   y1 = z1 (*) cos - z2 (*) sin,  y2 = z2 (*) cos + z1 (*) sin            for the pairs of the first `rotated` values of a head:
 * values i and i + rotated / 2, or with `interleaved` 2 i and 2 i + 1; the other values are z's.  cos and sin:
 * [table_rows][rotated / 2].  positions: one row number per token, [batch][tokens] with the given strides, or NULL: token t is at
 * row t.  A position outside the table makes the rotated values NaN.
 * One launch takes one or two tensors of [batch][tokens][heads][dim] (queries and keys), whose heads are contiguous and whose
 * other strides are free; y and dx are contiguous. */
typedef struct {
    const float *x; long x_sb, x_st, x_sh;
    const float *dy; long dy_sb, dy_st, dy_sh;     /* backward only */
    const float *weight;                           /* [dim] or NULL */
    float *y;                                      /* forward: y; backward: dx */
    float *dweight;                                /* backward: [dim] or NULL */
    long heads;
} pam_hip_heads;
int pam_hip_rotary_fwd(const pam_hip_heads *parts, int count, const float *cos, const float *sin, long table_rows,
                       const long long *positions, long positions_sb, long positions_st, long batch, long tokens, long dim,
                       long rotated, int interleaved, float eps, float offset, void *stream);
size_t pam_hip_rotary_bwd_workspace_bytes(const pam_hip_heads *parts, int count, long batch, long tokens, long dim, long rotated);
int pam_hip_rotary_bwd(const pam_hip_heads *parts, int count, const float *cos, const float *sin, long table_rows,
                       const long long *positions, long positions_sb, long positions_st, long batch, long tokens, long dim,
                       long rotated, int interleaved, float eps, float offset, int approx_a, int approx_b, int approx_exp,
                       void *workspace, size_t workspace_bytes, void *stream);

/* norm[0] = pow(sum of g (*) g over all tensors, 0.5); out = g (*) scale with scale = min(1, max_norm (/) (norm + eps)).  in and
 * out of a tensor may be the same memory, and then nothing is written where the scale is 1; otherwise tensors must not overlap.  A
 * max_norm of infinity scales by 1.  out NULL for all tensors: only the norm.  A norm that is NaN makes every value NaN. */
typedef struct { const float *in; float *out; size_t n; } pam_hip_clip_tensor;
size_t pam_hip_clip_workspace_bytes(const pam_hip_clip_tensor *tensors, long count);
int pam_hip_clip_many(const pam_hip_clip_tensor *tensors, long count, float max_norm, float eps, float *norm, float offset,
                      void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* PAM_HIP_BLOCK_H */
