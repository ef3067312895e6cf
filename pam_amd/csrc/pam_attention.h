// Attention in PAM arithmetic, every product of a score and of a result made and added up where it is used.
//
//   a_ij = sum_d (q_id (*) scale) (*) k_jd,  x_ij = capped a_ij less slope (*) |i - j|,  t_ij = x_ij (*) log2 e,
//   e_ij = 2^t_ij,  l_i = sum_j e_ij,  n_id = sum_j e_ij (*) v_jd,  y_id = n_id (/) l_i        over the keys j that row i sees
//
// In this arithmetic a product or a quotient by a power of two is exact, and 2^(t - M) is 2^-M 2^t for a whole number M: one
// pass over the keys with a running whole M (raised where a t is more than kLag above it) gives the definition's result, whatever
// M has been on the way.  (The softmax of the primitives subtracts the largest of all rows' scores, which is no whole number, and moves the
// result with it.)
//
// A wavefront's lanes own rows (queries; in the pass for dk and dv, keys), with a row's values in the lane's registers, and the
// other side streams by.  A product takes two instructions on 64 lanes, an integer addition that reads the streamed value from another lane
// of the 16 (a data-parallel primitive of the addition itself: row_newbcast) and a float addition: no LDS, no barriers, and a wavefront alone in its
// work-group's progress.  A streamed row is one 128-bit load per lane, the same for the four sixteens of the wavefront.
// Rows of more than 64 values (32 in the backward passes, which hold three or four of them per lane) are cut into NS slices of
// at most 16 quads, each of which has its own sixteens of the wavefront, 64 / NS rows; a score's slices are added by lane swaps.
// Values read through scalar registers instead of lanes waited for the scalar cache: 2.2 T products/s where this has 6.4 (8 heads of 4096 x 4096 x 64, one
// wavefront on every second SIMD).
//
// The integer addition is the product while no exponent leaves the normal range.  Streamed values have to be in 2^[-40, 40), a lane's in 2^[-86, 80); a
// lane's zero stands as 2^-86, which adds less to a sum than its rounding.  A streamed row that is all zeros is left out by selects; a
// streamed block with anything else in it, or a wavefront with anything else in its rows, takes the full definition (`careful`).
#pragma once
#include "pam_activation.h"
#include "pam_common.h"
#include "../../include/pam_hip_attention.h"

namespace pamatt {
using namespace pamdev;

constexpr int kThreads = 256, kWaves = 4;
constexpr int kBlock = 8;                         // streamed rows at a time (four: 18.8 T products/s where eight have 20.9)
constexpr int kSpan = 64;                         // streamed rows per word of visibility
constexpr int kLink = 1024;                       // terms of a chain of sums; chains are added up in memory
constexpr float kLag = 8.0f;
constexpr float kLog2e = (float)1.4426950408889634, kTurn = (float)(2.0 * 1.4426950408889634);
constexpr float kLeast = -62.0f;                  // weights below 2^-62 of the largest so far are none

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

struct Tokens { const float* p; long sb, st, sh; };          // [batch][tokens][heads][dim], heads contiguous

struct Args {
    Tokens q, k, v;
    int batch, tokens, keys, heads, kv_heads, group, dim, values;      // dim: whole quads, of which `values` values count
    int rows;                                     // of one batch entry and key head: tokens x group, a token's heads behind each other
    int first;                                    // the position of the first query
    int causal, window;                           // window: 0 none
    const long long* prefix; const long long* documents;
    const float* slopes;
    float scale, cap, off;                        // cap: 0 none
    int tiles, chunks, chunk;                     // a unit is a tile of lanes' rows and a chunk (a multiple of kSpan) of the streamed ones
    // forward
    float* y;                                     // [batch][tokens][heads][dim]
    float2* stats;                                // l and M, [batch][kv_heads][rows], or null
    float* partial; float2* partial_stats;        // [batch][kv_heads][chunks][rows][dim], [...][rows]; or null: chunks is 1
    // backward
    const float4* records;                        // [batch][kv_heads][rows]: M (+inf: the row sees nothing), dl, largest exponent of dn, slope
    const float* qs; const float* dn;             // [batch][kv_heads][rows][dim]
    float* out0; float* out1;                     // [batch][kv_heads][chunks][lanes' rows][dim]: dq, or dk and dv
    ApproxFlags flags;
};

// ---------------------------------------------------------------- lanes

template <int N> __device__ __forceinline__ uint32_t from_lane(float x)          // the value that lane N of each sixteen has
{ return (uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(x), 0x150 + N, 0xf, 0xf, true); }

// f(constant<0>) ... f(constant<N - 1>)
template <int N> struct Index { static constexpr int value = N; };
template <int N, int END, class F> __device__ __forceinline__ void each(F&& f)
{
    if constexpr (N < END) { f(Index<N>{}); each<N + 1, END>(f); }
}

template <int NS> __device__ __forceinline__ float over_slices(float v)          // the slices' sum, in all of them
{
    typedef unsigned int u2 __attribute__((ext_vector_type(2)));
    if constexpr (NS == 4) { const u2 r = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false); v = u2f(r.x) + u2f(r.y); }
    if constexpr (NS >= 2) { const u2 r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false); v = u2f(r.x) + u2f(r.y); }
    return v;
}

constexpr uint32_t kStreamBase = (uint32_t)(127 - 40) << 24, kStreamSpan = 80u << 24;      // 2^[-40, 40) of bits << 1
constexpr uint32_t kLaneBase = (uint32_t)(127 - 86) << 24, kLaneSpan = 166u << 24;         // 2^[-86, 80)
constexpr uint32_t kStandIn = (uint32_t)(127 - 86) << 23;

template <int NS, int W4>
struct Place {                                    // what a lane has to do with
    int lane, row_in_wave, slice, at;             // at: the first value of its quad in a streamed row
    bool streams;                                 // it holds a part of streamed rows
    uint64_t streaming;                           // the lanes that do
    __device__ __forceinline__ explicit Place(int values)
    {
        constexpr int kRows = 64 / NS;
        lane = threadIdx.x % 64; row_in_wave = lane % kRows; slice = lane / kRows;
        at = slice * 4 * W4 + lane % 16 * 4;
        streams = lane % 16 < W4 && at < values;
        if (!streams) at = 0;
        streaming = __ballot(streams);
    }
};

// (comparisons with it are made where they are used, instead of kept from the beginning of a kernel to its end)
__device__ __forceinline__ int anew(int v) { asm volatile("" : "+v"(v)); return v; }

// Behind a row's values streamed rows have what `shift` makes ones of, and lanes' rows what makes + 0 of that.
__device__ __forceinline__ uint32_t stream_pad(uint32_t shift) { return kBias - shift; }
__device__ __forceinline__ uint32_t lane_pad(uint32_t shift) { return shift - kBias; }

// A lane's row: bits(value) + scale + add, zeros stood in for (unscaled).  scale: of a factor in 2^[-41, 41].  Returns false if a value,
// scaled, is out of the window.
template <int W4>
__device__ __forceinline__ bool load_lane(const float* row, int first, int dim, int values, uint32_t scale, uint32_t add, uint32_t pad, uint32_t (&out)[4 * W4])
{
    uint32_t most = 0u;
    first = anew(first);
#pragma unroll
    for (int n = 0; n < W4; ++n) {
        const v4f x = *reinterpret_cast<const v4f_any*>(row + min(first + 4 * n, dim - 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = (f2u(x[i]) << 1) == 0u ? kStandIn : f2u(x[i]) + scale;
            const bool there = first + 4 * n + i < values;
            most = max(most, there ? (b << 1) - kLaneBase : 0u);
            out[4 * n + i] = there ? b + add : pad;
        }
    }
    return most < kLaneSpan;
}

// The quad that a lane holds of a streamed row.
struct Stream {
    const float* p; long st;                      // uniform
    uint32_t at; int last, values; bool streams, whole;      // whole: all lanes below W4 have four values
    // the rows j ... j + 7, past the end the last one again
    __device__ __forceinline__ void rows(int j, v4f (&r)[kBlock]) const
    {
#pragma unroll
        for (int i = 0; i < kBlock; ++i) r[i] = *reinterpret_cast<const v4f_any*>(p + (long)min(j + i, last) * st + at);
    }
    __device__ __forceinline__ void pad(uint32_t shift, v4f (&r)[kBlock]) const      // (where they are used)
    {
        if (whole) return;
        const float one = u2f(stream_pad(shift));
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const bool there = streams && (int)at + d < values;
#pragma unroll
            for (int i = 0; i < kBlock; ++i) r[i][d] = there ? r[i][d] : one;
        }
    }
};
template <int NS, int W4>
__device__ __forceinline__ Stream stream_of(const Place<NS, W4>& here, const float* p, long st, int values, int count)
{ return Stream{p, st, (uint32_t)here.at, count - 1, values, here.streams, values == 4 * W4 * NS}; }

template <int N, class T> __device__ __forceinline__ void turned(T (&v)[N])      // all one place down, the first to the end
{
    const T first = v[0];
#pragma unroll
    for (int i = 0; i + 1 < N; ++i) v[i] = v[i + 1];
    v[N - 1] = first;
}

// What is the matter with a block of streamed rows: `zero`, the rows that are all zeros (they become ones, and their products are to
// be left out), `careful`, something else is.
struct Verdict { uint32_t zero; bool careful; };
__device__ __forceinline__ Verdict judge(uint64_t streaming, uint32_t shift, v4f (&r)[kBlock])
{
    uint32_t most = 0u;
#pragma unroll
    for (int j = 0; j < kBlock; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = max(most, ((f2u(r[j][i]) + shift) << 1) - kStreamBase);
    Verdict v{0u, false};
    if (__builtin_expect((__ballot(most >= kStreamSpan) & streaming) == 0ull, 1)) return v;
#pragma unroll 1
    for (int j = 0; j < kBlock; ++j) {
        bool all = true, odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            all = all && (f2u(r[0][i]) << 1) == 0u;
            odd = odd || ((f2u(r[0][i]) + shift) << 1) - kStreamBase >= kStreamSpan;
        }
        if ((__ballot(!all) & streaming) == 0ull) {
            v.zero |= 1u << j;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[0][i] = u2f(stream_pad(shift));
        } else if ((__ballot(odd) & streaming) != 0ull) v.careful = true;
        turned(r);
    }
    return v;
}

// sum over d of a lane's values with a streamed row's: `mine` as load_lane left them with add = bits(offset) - 2 bias
template <int W4> __device__ __forceinline__ float dot(const v4f& row, const uint32_t (&mine)[4 * W4])
{
    float sum = 0.0f;
    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += u2f(from_lane<decltype(n)::value>(row[i]) + mine[4 * n.value + i]);
    });
    return sum;
}
// out_d += f * (weight (*) a streamed row's d), weight as above; f is 0 or 1
template <int W4> __device__ __forceinline__ void add_row(const v4f& row, uint32_t weight, float f, float (&out)[4 * W4])
{
    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[4 * n.value + i] = __builtin_fmaf(u2f(from_lane<decltype(n)::value>(row[i]) + weight), f, out[4 * n.value + i]);
    });
}

// The same by the full definition, what turns `mine` back into a value's bits being `raw`.  One row's code each, in loops that turn the arrays
// around.
struct Full { float off; bool has_off; uint32_t raw, pad; };
__device__ __forceinline__ float full_product(const Full& f, uint32_t a, uint32_t b)
{
    const float c = pam_general(a, b);
    return f.has_off ? pam_general(f2u(c), f2u(f.off)) : c;
}
template <int W4> __device__ __forceinline__ float careful_dot(const Full& f, const v4f& row, const uint32_t (&mine)[4 * W4])
{
    float sum = 0.0f;
    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = (uint32_t)anew((int)mine[4 * n.value + i]);      // (taken apart here and not, for all rows, before the loop)
            sum += full_product(f, m == f.pad ? 0u : m + f.raw, from_lane<decltype(n)::value>(row[i]));
            __builtin_amdgcn_sched_barrier(0);    // (rare code: side by side the products took registers from the usual loops)
        }
    });
    return sum;
}
template <int W4> __device__ __forceinline__ void careful_add_row(const Full& f, const v4f& row, float weight, bool counts, float scale, float (&out)[4 * W4])
{
    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = full_product(f, f2u(weight), from_lane<decltype(n)::value>(row[i])) * scale;
            out[4 * n.value + i] += counts ? c : 0.0f;
            __builtin_amdgcn_sched_barrier(0);
        }
    });
}

// A block's scores (their slices added up).
template <int NS, int W4>
__device__ __forceinline__ void block_dots(const Full& f, bool careful, uint32_t zero, float scale, v4f (&r)[kBlock], const uint32_t (&mine)[4 * W4], float (&sum)[kBlock])
{
    if (__builtin_expect(careful, 0)) {
#pragma unroll 1
        for (int j = 0; j < kBlock; ++j) {
            sum[0] = careful_dot<W4>(f, r[0], mine) * scale;
            turned(r); turned(sum);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kBlock; ++j) sum[j] = dot<W4>(r[j], mine);
    }
#pragma unroll
    for (int j = 0; j < kBlock; ++j) sum[j] = over_slices<NS>(sum[j]);
    if (__builtin_expect(zero != 0u, 0)) {
#pragma unroll
        for (int j = 0; j < kBlock; ++j) sum[j] = (zero >> j) & 1u ? 0.0f : sum[j];
    }
}
// out += the block's weights times its rows; a weight that does not count is anything.  add: as in load_lane.
template <int W4>
__device__ __forceinline__ void block_add(const Full& f, bool careful, uint32_t zero, float scale, v4f (&r)[kBlock], float (&weight)[kBlock], uint32_t add, uint32_t counts,
                                          float (&out)[4 * W4])
{
    counts &= ~zero;
    if (__builtin_expect(careful, 0)) {
#pragma unroll 1
        for (int j = 0; j < kBlock; ++j) {
            careful_add_row<W4>(f, r[0], weight[0], (counts >> j) & 1u, scale, out);
            turned(r); turned(weight);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < kBlock; ++j) {
        const bool in = (counts >> j) & 1u;
        add_row<W4>(r[j], in ? f2u(weight[j]) + add : 0u, in ? 1.0f : 0.0f, out);
    }
}

// ---------------------------------------------------------------- which streamed rows a lane's row goes with

// Lanes' rows go with the streamed rows [low, high) and [0, before), where the documents agree.
struct Sight {
    int low, high, before;
    int first, last;                              // uniform: of all lanes
    const long long* of_streamed; int per;        // documents: row j of the streamed ones is of of_streamed[j / per], or null
    long long mine;                               // the lane's
    bool with_documents;
    __device__ __forceinline__ void close()
    {
        int a = before > 0 ? 0 : low < high ? low : 0x7fffffff, b = max(before, low < high ? high : 0);
#pragma unroll
        for (int s = 1; s < 64; s *= 2) { a = min(a, __shfl_xor(a, s, 64)); b = max(b, __shfl_xor(b, s, 64)); }
        first = __builtin_amdgcn_readfirstlane(a); last = __builtin_amdgcn_readfirstlane(b);
    }
    static __device__ __forceinline__ uint64_t bits_of(int from, int to)
    {
        from = max(from, 0); to = min(to, kSpan);
        return to > from ? (~0ull >> (64 - (to - from))) << from : 0ull;
    }
    // ... of the rows j0 ... j0 + 63
    __device__ __forceinline__ uint64_t span(int j0) const
    {
        uint64_t see = bits_of(low - j0, min(high, 0x7fffffff) - j0) | bits_of(-1, before - j0);
        if (with_documents && __ballot(see != 0ull) != 0ull) {
            const int j = j0 + (int)threadIdx.x % 64;
            const long long theirs = j < last ? of_streamed[j / per] : -1;
            const int lo = (int)theirs, hi = (int)(theirs >> 32);
            uint64_t same = 0ull;
            // (one document in all 64 of the one side and the other: the usual case)
            const long long one = ((long long)__builtin_amdgcn_readfirstlane(hi) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane(lo);
            if (__ballot(theirs != one) == 0ull) same = mine == one ? ~0ull : 0ull;
            else
#pragma unroll 4
                for (int i = 0; i < 64; ++i) {
                    const long long at = ((long long)__builtin_amdgcn_readlane(hi, i) << 32) | (uint32_t)__builtin_amdgcn_readlane(lo, i);
                    same |= (uint64_t)(at == mine) << i;
                }
            see &= mine < 0 ? 0ull : same;
        }
        return see;
    }
};

// ---------------------------------------------------------------- from a score to its exponent

// x (*) a positive constant, whose bits less the bias (offset counted) are `add`.  Underflow is zero; NaN and infinities are not numbers afterwards.
__device__ __forceinline__ float times(float x, uint32_t add)
{
    const int m = (int)(min(f2u(x) & ~kSign, kExpo + 1u) + add);
    return u2f((uint32_t)max(m, 0) | (f2u(x) & kSign));
}
// a (*) b of any finite numbers whose product is below 2^128; an underflow (a zero's, too) is zero or next to nothing
__device__ __forceinline__ float times_any(float a, float b, uint32_t off_add)
{
    const int m = (int)((f2u(a) & ~kSign) - kBias + (f2u(b) & ~kSign) + off_add);
    return u2f((uint32_t)max(m, 0) | ((f2u(a) ^ f2u(b)) & kSign));
}

struct Scoring {
    float cap, off;
    bool slopes;
    uint32_t off_add, log2e_add, mul_add;         // mul_add: of a product of two lanes' values
    __device__ __forceinline__ explicit Scoring(const Args& a) : cap(a.cap), off(a.off), slopes(a.slopes != nullptr), off_add(f2u(a.off) - kBias),
        log2e_add(f2u(kLog2e) - kBias + f2u(a.off) - kBias), mul_add(f2u(a.off) - 2u * kBias) {}

    // the cap's quantities for a score's magnitude: w = 2^-(u (*) 2 log2 e), th = (1 - w) (/) (1 + w), with u = |a| (/) cap held in 2^[-40, 6]
    // (th of less is nothing in 32 bits, and of more 1)
    struct Cap { float u, power, w, th; };
    __device__ __forceinline__ Cap capping(float a) const
    {
        const Raw ar(off);
        Cap c;
        c.u = fminf(fmaxf(fabsf(a), 0x1p-60f), 0x1p40f);
        c.u = fminf(fmaxf(ar.div(c.u, cap), 0x1p-40f), 64.0f);
        c.power = fminf(ar.mul(c.u, kTurn), 64.0f);
        c.w = u2f((uint32_t)((int)kBias - (int)rintf(c.power * 0x1p23f)));
        const float n = 1.0f - c.w;
        c.th = n > 0.0f ? ar.div(n, 1.0f + c.w) : 0.0f;
        return c;
    }
    __device__ __forceinline__ float capped(float a) const
    {
        const Cap c = capping(a);
        const float x = c.th > 0.0f ? u2f(f2u(c.th) + f2u(cap) + mul_add) : 0.0f;
        return fabsf(a) < 0x1p127f ? __builtin_copysignf(x, a) : u2f(kQNaN);
    }
    // slope: of magnitude below 2^91
    __device__ __forceinline__ float biased(float x, float slope, int distance) const
    {
        const float far = (float)(distance < 0 ? -distance : distance);
        return x - (far > 0.0f ? times_any(slope, far, off_add) : 0.0f);
    }
    __device__ __forceinline__ float exponent(float a, float slope, int distance) const
    {
        float x = cap != 0.0f ? capped(a) : a;
        if (slopes) x = biased(x, slope, distance);
        return times(x, log2e_add);
    }
};
// (2^-60 per place is no bias in 32 bits over 2^30 places, 2^90 leaves nothing beside the nearest key)
__device__ __forceinline__ float held_slope(float s) { return fabsf(s) < 0x1p-60f ? 0.0f : fabsf(s) > 0x1p90f ? __builtin_copysignf(0x1p90f, s) : s; }
__device__ __forceinline__ bool finite(float s) { return fabsf(s) < u2f(kExpo); }

// 2^u for kLeast <= u < 64, rounded once
__device__ __forceinline__ float power_of_two(float u) { return u2f((uint32_t)((int)rintf(u * 0x1p23f) + (int)kBias)); }
// 2^(from - to), not below 2^-126 (that times a sum is nothing); from - to at most 127
__device__ __forceinline__ float scale_between(float from, float to) { return u2f((uint32_t)((int)fmaxf(from - to, -126.0f) + 127) << 23); }

constexpr float kNothing = -3.0e38f;              // M of a row that has seen nothing yet

}  // namespace pamatt
