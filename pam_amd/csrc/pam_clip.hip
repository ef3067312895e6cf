// The global norm of many gradients and their scaling to a bound.
//
// Bound by memory: a pass over the values for the sum of squares, and one that reads and writes them.  253 tensors of 36.7 M values, 147 MB
// in all: 71 us (at the rate of a large copy 56 if the second pass found every value in a cache, 84 if none).  The tables of tensors travel in the kernels' arguments, 254 tensors or 167 with outputs
// at a time (no copy to wait for); a work-group takes kChunk consecutive values of one tensor and finds which by comparing all of the
// tensors' first work-groups with its own number at once (a binary search is eight waits for memory one after the other, 3 us more).  Loads are 128 bits at any float's address, a lane's all in flight.
// Sums: a lane's sixteen squares in a tree, then wavefronts and work-group in float32, work-groups' sums in float64.  The order is
// that of the table.
// g (*) g and g (*) scale are one integer addition each where a wavefront's values are zeros or in the window of ordinary sizes;
// otherwise the checked product.
#include <algorithm>

#include "../../include/pam_hip_block.h"
#include "pam_activation.h"
#include "pam_common.h"

using namespace pamdev;

namespace {

constexpr int kThreads = 256, kQuads = 4;
constexpr unsigned kChunk = 4 * kQuads * kThreads;          // values of a work-group
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

struct Options { float off; bool has_off; };
// What becomes of the work-groups' sums: the norm and the scale.
struct Bound {
    const float* partial; long count;
    float max_norm, eps;
    float* norm;
    Options o;
};
// n, first: values, first work-group of a tensor; past the last one all ones
constexpr int kReadTensors = 254, kScaleTensors = 167;      // as many as 4 KB hold
struct ReadTable {
    static constexpr int kTensors = kReadTensors;
    const float* in[kTensors];
    unsigned n[kTensors], first[kTensors];
    float* partial;                               // one sum per work-group
    Options o;
};
struct ScaleTable {
    static constexpr int kTensors = kScaleTensors;
    const float* in[kTensors]; float* out[kTensors];
    unsigned n[kTensors], first[kTensors];
    const float* scale;
    Bound b;
};
static_assert(sizeof(ReadTable) <= 4096 && sizeof(ScaleTable) <= 4096, "kernel arguments");

// The tensor of the work-group: its index, and where the work-group begins in it.
struct Share { int at; unsigned begin, count; };
template <class Table>
__device__ __forceinline__ Share find_share(const __attribute__((address_space(4))) Table* t)
{
    const int lane = threadIdx.x % 64;
    int at = -1;                                  // the last tensor that begins at or before the work-group
#pragma unroll
    for (int i = 0; i < Table::kTensors; i += 64)
        at += __popcll(__ballot(i + lane < Table::kTensors && t->first[min(i + lane, Table::kTensors - 1)] <= blockIdx.x));
    const unsigned begin = (blockIdx.x - t->first[at]) * kChunk;
    return Share{at, begin, min(t->n[at] - begin, kChunk)};
}

template <int THREADS, class T>
__device__ __forceinline__ T group_sum(T v)
{
    __shared__ T waves[THREADS / 64];
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s, 64);
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = v;
    __syncthreads();
    T total = waves[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) total += waves[w];
    return total;
}

// normal, in [2^-63, 2^63): squares and products with a scale in [2^-60, 1] are normal
typedef Window<-63, 63> WindowValue;
__device__ __forceinline__ void see(WindowValue& window, const v4f& v)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) window.see(is_zero(v[i]) ? 1.0f : v[i]);
}

// Quad q of a work-group's share; values past its end are zeros.  LAST: nobody reads it again.
template <bool LAST>
__device__ __forceinline__ v4f load_quad(const float* in, unsigned count, unsigned q)
{
    const unsigned i = 4 * q;
    if (i + 4 <= count) {
        const v4f_any* at = reinterpret_cast<const v4f_any*>(in + i);
        return LAST ? __builtin_nontemporal_load(at) : *at;
    }
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i < count) v[0] = in[i];
    if (i + 1 < count) v[1] = in[i + 1];
    if (i + 2 < count) v[2] = in[i + 2];
    return v;
}

__global__ __launch_bounds__(kThreads) void square_sums_kernel(ReadTable)
{
    const auto t = (const __attribute__((address_space(4))) ReadTable*)__builtin_amdgcn_kernarg_segment_ptr();
    const Share s = find_share(t);
    const float* in = t->in[s.at] + s.begin;
    const Options o{t->o.off, t->o.has_off};
    v4f v[kQuads];
#pragma unroll
    for (int u = 0; u < kQuads; ++u) v[u] = load_quad<false>(in, s.count, threadIdx.x + u * kThreads);
    WindowValue window;
#pragma unroll
    for (int u = 0; u < kQuads; ++u) see(window, v[u]);
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (__ballot(!window.held() || !usual_offset(o.off)) == 0ull) {
        const uint32_t add = f2u(o.off) - 2u * kBias;              // (the sign shifts out)
#pragma unroll
        for (int u = 0; u < kQuads; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += is_zero(v[u][i]) ? 0.0f : u2f((f2u(v[u][i]) << 1) + add);
    } else {
#pragma unroll 1
        for (int u = 0; u < kQuads; ++u) {
            const v4f w = u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : v[3];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += pam_mul_off(w[i], w[i], o.off, o.has_off);
        }
    }
    const float total = group_sum<kThreads>((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (threadIdx.x == 0) t->partial[blockIdx.x] = total;
}

template <int THREADS>
__device__ __forceinline__ float norm_of(const Bound& b)
{
    double sum = 0.0;
#pragma unroll 8
    for (long i = threadIdx.x; i < b.count; i += THREADS) sum += (double)b.partial[i];
    return pow_half((float)group_sum<THREADS>(sum), b.o.off, b.o.has_off);
}
__device__ __forceinline__ float scale_of(const Bound& b, float norm)
{
    if (f2u(b.max_norm) == kExpo) return 1.0f;
    const float q = pad_div_off(b.max_norm, norm + b.eps, b.o.off, b.o.has_off);
    return q > 1.0f ? 1.0f : q;                                           // (NaN stays)
}

constexpr long kFewSums = 1024;                   // up to as many, every work-group of the second pass adds them up itself, a launch less
template <int THREADS>
__global__ __launch_bounds__(THREADS) void norm_kernel(Bound b, float* __restrict__ scale)
{
    const float norm = norm_of<THREADS>(b);
    if (threadIdx.x != 0) return;
    b.norm[0] = norm;
    scale[0] = scale_of(b, norm);
}

template <bool FEW>
__global__ __launch_bounds__(kThreads) void scale_kernel(ScaleTable)
{
    const auto t = (const __attribute__((address_space(4))) ScaleTable*)__builtin_amdgcn_kernarg_segment_ptr();
    const Share s = find_share(t);
    const float* in = t->in[s.at] + s.begin;
    float* out = t->out[s.at] + s.begin;
    const Options o{t->b.o.off, t->b.o.has_off};
    float scale;
    if constexpr (FEW) {
        const Bound b{t->b.partial, t->b.count, t->b.max_norm, t->b.eps, t->b.norm, o};
        const float norm = norm_of<kThreads>(b);
        if (blockIdx.x == 0 && threadIdx.x == 0) b.norm[0] = norm;
        scale = scale_of(b, norm);
    } else scale = t->scale[0];
    const bool keep = scale == 1.0f;
    if (keep && in == out) return;
    v4f v[kQuads];
#pragma unroll
    for (int u = 0; u < kQuads; ++u) v[u] = load_quad<true>(in, s.count, threadIdx.x + u * kThreads);
    if (!keep) {
        WindowValue window;
#pragma unroll
        for (int u = 0; u < kQuads; ++u) see(window, v[u]);
        if (__ballot(!window.held() || !(scale >= 0x1p-60f && scale <= 1.0f) || !usual_offset(o.off)) == 0ull) {
            const Raw ar(o.off);
#pragma unroll
            for (int u = 0; u < kQuads; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[u][i] = is_zero(v[u][i]) ? 0.0f : ar.mul(v[u][i], scale);
        } else {
#pragma unroll
            for (int u = 0; u < kQuads; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[u][i] = pam_mul_off(v[u][i], scale, o.off, o.has_off);
        }
    }
#pragma unroll
    for (int u = 0; u < kQuads; ++u) {
        const unsigned i = 4 * (threadIdx.x + u * kThreads);
        // (past the caches: stores that stay there push out what the first pass left, 94 us instead of 78)
        if (i + 4 <= s.count) __builtin_nontemporal_store(v[u], reinterpret_cast<v4f_any*>(out + i));
        else {
            if (i < s.count) out[i] = v[u][0];
            if (i + 1 < s.count) out[i + 1] = v[u][1];
            if (i + 2 < s.count) out[i + 2] = v[u][2];
        }
    }
}

size_t chunks(size_t n) { return (n + kChunk - 1) / kChunk; }
void set_out(ReadTable&, int, float*) {}
void set_out(ScaleTable& t, int i, float* out) { t.out[i] = out; }

// Calls launch(work-groups, work-groups before them) for tables of as many tensors as one holds.
template <class Table, class F>
int each_table(const pam_hip_clip_tensor* tensors, long count, Table& table, F launch)
{
    constexpr size_t kPart = (size_t)1 << 31;     // (a longer tensor enters the table in parts: counts are 32-bit ones)
    static_assert(kPart % kChunk == 0, "parts are whole chunks");
    constexpr size_t kMostGroups = (size_t)1 << 23;          // (a launch counts its work-items in 32 bits)
    int held = 0;
    size_t groups = 0, before = 0;
    auto flush = [&]() -> int {
        if (held == 0) return PAM_HIP_OK;
        for (int i = held; i < Table::kTensors; ++i) table.first[i] = ~0u;
        launch((unsigned)groups, before);
        before += groups; held = 0; groups = 0;
        return pamhost::check_launch("clip_many");
    };
    for (long i = 0; i < count; ++i)
        for (size_t at = 0; at < tensors[i].n; at += kPart) {
            const size_t n = std::min(kPart, tensors[i].n - at), need = chunks(n);
            if (held == Table::kTensors || groups + need > kMostGroups) { const int rc = flush(); if (rc != PAM_HIP_OK) return rc; }
            table.in[held] = tensors[i].in + at;
            set_out(table, held, tensors[i].out ? tensors[i].out + at : nullptr);
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
    const Options options{offset, offset != 1.0f};
    ReadTable read;
    read.o = options;
    int rc = each_table(tensors, count, read, [&](unsigned groups, size_t before) {
        read.partial = partial + before;
        hipLaunchKernelGGL(square_sums_kernel, dim3(groups), dim3(kThreads), 0, st, read);
    });
    if (rc != PAM_HIP_OK) return rc;
    const Bound bound{partial, (long)partials(tensors, count), max_norm, eps, norm, options};
    const bool few = bound.count <= kFewSums;
    if (!few || !wanted || bound.count == 0) {
        if (few) hipLaunchKernelGGL(norm_kernel<kThreads>, dim3(1), dim3(kThreads), 0, st, bound, scale);
        else hipLaunchKernelGGL(norm_kernel<1024>, dim3(1), dim3(1024), 0, st, bound, scale);
        rc = pamhost::check_launch("clip_many");
        if (rc != PAM_HIP_OK || !wanted) return rc;
    }
    ScaleTable table;
    table.scale = scale; table.b = bound;
    return each_table(tensors, count, table, [&](unsigned groups, size_t) {
        if (few) hipLaunchKernelGGL(scale_kernel<true>, dim3(groups), dim3(kThreads), 0, st, table);
        else hipLaunchKernelGGL(scale_kernel<false>, dim3(groups), dim3(kThreads), 0, st, table);
    });
}

}  // extern "C"
