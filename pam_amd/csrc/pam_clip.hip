// The global norm of many gradients and their scaling to a bound.
#include <algorithm>

#include "../../include/pam_hip_block.h"
#include "pam_common.h"
#include "pam_device.h"

using namespace pamdev;

namespace {

constexpr int kThreads = 256;
constexpr unsigned kChunk = 8 * kThreads;         // values of a work-group

// The table of tensors travels in the kernel's arguments; a work-group takes kChunk consecutive values of one tensor and finds which by
// a binary search over the tensors' first work-groups on the scalar unit.
constexpr int kTensors = 96;
struct ClipTable {
    const float* in[kTensors]; float* out[kTensors];
    unsigned n[kTensors], first[kTensors];        // first: work-group; past the last tensor: all ones
    float* partial;                               // one sum per work-group
    const float* scale;
    float off; bool has_off;
};
static_assert(sizeof(ClipTable) <= 4096, "kernel arguments");
typedef const __attribute__((address_space(4))) ClipTable* Table;

struct Share { const float* in; float* out; unsigned count; };
__device__ __forceinline__ Share find_share(const Table t)
{
    int at = 0;
#pragma unroll
    for (int half = 64; half >= 1; half >>= 1)
        if (at + half < kTensors && t->first[at + half] <= blockIdx.x) at += half;
    const unsigned begin = (blockIdx.x - t->first[at]) * kChunk;
    float* out = t->out[at];
    return Share{t->in[at] + begin, out ? out + begin : nullptr, min(t->n[at] - begin, kChunk)};
}

template <class T>
__device__ __forceinline__ T group_sum(T v)
{
    __shared__ T waves[kThreads / 64];
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s, 64);
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = v;
    __syncthreads();
    return (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

__global__ __launch_bounds__(kThreads) void square_sums_kernel(ClipTable)
{
    const Table t = (Table)__builtin_amdgcn_kernarg_segment_ptr();
    const Share s = find_share(t);
    const float off = t->off; const bool has_off = t->has_off;
    float sum = 0.0f;
    for (unsigned i = threadIdx.x; i < s.count; i += kThreads) sum += pam_mul_off(s.in[i], s.in[i], off, has_off);
    sum = group_sum(sum);
    if (threadIdx.x == 0) t->partial[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const float* __restrict__ partial, long count, float max_norm, float eps, float off, bool has_off,
                                                       float* __restrict__ norm, float* __restrict__ scale)
{
    double sum = 0.0;
    for (long i = threadIdx.x; i < count; i += kThreads) sum += (double)partial[i];
    const float total = (float)group_sum(sum);
    if (threadIdx.x != 0) return;
    const float length = pow_half(total, off, has_off);
    norm[0] = length;
    if (f2u(max_norm) == kExpo) { scale[0] = 1.0f; return; }
    const float q = pad_div_off(max_norm, length + eps, off, has_off);
    scale[0] = q > 1.0f ? 1.0f : q;                                       // (NaN stays)
}

__global__ __launch_bounds__(kThreads) void scale_kernel(ClipTable)
{
    const Table t = (Table)__builtin_amdgcn_kernarg_segment_ptr();
    const Share s = find_share(t);
    const float off = t->off, scale = t->scale[0]; const bool has_off = t->has_off;
    const bool keep = scale == 1.0f;
    if (keep && s.in == s.out) return;
    for (unsigned i = threadIdx.x; i < s.count; i += kThreads) s.out[i] = keep ? s.in[i] : pam_mul_off(s.in[i], scale, off, has_off);
}

size_t chunks(size_t n) { return (n + kChunk - 1) / kChunk; }

// Calls launch(table, work-groups, work-groups before it) for tables of up to kTensors tensors.
template <class F>
int each_table(const pam_hip_clip_tensor* tensors, long count, ClipTable& table, F launch)
{
    constexpr size_t kPart = (size_t)1 << 31;     // (a longer tensor enters the table in parts: counts are 32-bit ones)
    static_assert(kPart % kChunk == 0, "parts are whole chunks");
    int held = 0;
    size_t groups = 0, before = 0;
    auto flush = [&]() -> int {
        if (held == 0) return PAM_HIP_OK;
        for (int i = held; i < kTensors; ++i) table.first[i] = ~0u;
        launch((unsigned)groups, before);
        before += groups; held = 0; groups = 0;
        return pamhost::check_launch("clip_many");
    };
    for (long i = 0; i < count; ++i)
        for (size_t at = 0; at < tensors[i].n; at += kPart) {
            const size_t n = std::min(kPart, tensors[i].n - at), need = chunks(n);
            if (held == kTensors || groups + need > ((size_t)1 << 30)) { const int rc = flush(); if (rc != PAM_HIP_OK) return rc; }
            table.in[held] = tensors[i].in + at; table.out[held] = tensors[i].out ? tensors[i].out + at : nullptr;
            table.n[held] = (unsigned)n; table.first[held] = (unsigned)groups;
            ++held; groups += need;
        }
    return flush();
}

size_t partials(const pam_hip_clip_tensor* tensors, long count)
{
    size_t n = 0;
    for (long i = 0; i < count; ++i) n += chunks(tensors[i].n);           // (parts are whole chunks)
    return n;
}

}  // namespace

extern "C" {

size_t pam_hip_clip_workspace_bytes(const pam_hip_clip_tensor* tensors, long count)
{
    if (!tensors || count <= 0) return 256;
    return ((partials(tensors, count) * sizeof(float) + 255) & ~(size_t)255) + 256;
}

int pam_hip_clip_many(const pam_hip_clip_tensor* tensors, long count, float max_norm, float eps, float* norm, float offset, void* workspace,
                      size_t workspace_bytes, void* stream)
{
    if (count < 0 || (count > 0 && !tensors) || !norm) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "clip_many: null pointer or negative count");
    bool wanted = false;
    for (long i = 0; i < count; ++i) {
        if (tensors[i].n == 0) continue;
        if (!tensors[i].in) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "clip_many: null pointer");
        if (tensors[i].n > (size_t)1 << 41) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "clip_many: more than 2^41 values");
        wanted = wanted || tensors[i].out;
    }
    for (long i = 0; wanted && i < count; ++i)
        if (tensors[i].n && !tensors[i].out) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "clip_many: some tensors without an output");
    const size_t need = pam_hip_clip_workspace_bytes(tensors, count);
    if (!workspace || workspace_bytes < need) return pamhost::fail(PAM_HIP_ERR_WORKSPACE, "clip_many: workspace of %zu bytes needed", need);
    const hipStream_t st = (hipStream_t)stream;
    float* scale = (float*)workspace;
    float* partial = scale + 64;
    ClipTable table;
    table.scale = scale; table.off = offset; table.has_off = offset != 1.0f;
    int rc = each_table(tensors, count, table, [&](unsigned groups, size_t before) {
        table.partial = partial + before;
        hipLaunchKernelGGL(square_sums_kernel, dim3(groups), dim3(kThreads), 0, st, table);
    });
    if (rc != PAM_HIP_OK) return rc;
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, partial, (long)partials(tensors, count), max_norm, eps, offset, offset != 1.0f, norm, scale);
    rc = pamhost::check_launch("clip_many");
    if (rc != PAM_HIP_OK || !wanted) return rc;
    return each_table(tensors, count, table, [&](unsigned groups, size_t) { hipLaunchKernelGGL(scale_kernel, dim3(groups), dim3(kThreads), 0, st, table); });
}

}  // extern "C"
