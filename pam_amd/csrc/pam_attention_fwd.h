// The forward pass of pam_attention.h: a wavefront's 64 / NS rows over a chunk of the keys.
#pragma once
#include "pam_attention.h"

namespace pamatt {

// A lane's row in memory: each of its quads as put(n, quad) leaves it.
template <int W4, class Put>
__device__ __forceinline__ void row_in_memory(float* at, int first, int dim, bool exists, Put put)
{
    first = anew(first);
#pragma unroll
    for (int n = 0; n < W4; ++n) {
        const int d = first + 4 * n;
        if (exists && d < dim) {
            v4f x = *reinterpret_cast<const v4f_any*>(at + d);
            put(n, x);
            *reinterpret_cast<v4f_any*>(at + d) = x;
        }
    }
}
template <int W4>
__device__ __forceinline__ void store_row(float* at, int first, int dim, bool exists, const float (&out)[4 * W4])
{
    first = anew(first);
#pragma unroll
    for (int n = 0; n < W4; ++n) {
        const int d = first + 4 * n;
        if (exists && d < dim) *reinterpret_cast<v4f_any*>(at + d) = v4f{out[4 * n], out[4 * n + 1], out[4 * n + 2], out[4 * n + 3]};
    }
}

// sums (/) l: the integer subtraction where the sums are ordinary numbers or zeros
template <int N>
__device__ __forceinline__ void over_total(float (&out)[N], float l, float off)
{
    uint32_t most = 0u;
#pragma unroll
    for (int d = 0; d < N; ++d) most = max(most, (f2u(out[d]) << 1) == 0u ? 0u : (f2u(out[d]) << 1) - (uint32_t)((127 - 60) << 24));
    if (__ballot(most >= (140u << 24) || !(l < 0x1p40f)) == 0ull) {
        const uint32_t add = 2u * kBias - f2u(off) - f2u(l);
#pragma unroll
        for (int d = 0; d < N; ++d) out[d] = (f2u(out[d]) << 1) == 0u ? out[d] : u2f(f2u(out[d]) + add);
        return;
    }
#pragma unroll 1
    for (int d = 0; d < N; ++d) {
        out[0] = pad_div_off(out[0], l, off, off != 1.0f);
        turned(out);
    }
}

// A unit of a launch: the tile of rows, the chunk, the batch entry and key head.  Consecutive work-groups take different heads, so that
// a head's keys stay with few of the XCDs' caches, and the last tiles, which see most keys where the order is causal, come first.
struct Unit { int head, b, kv, tile, chunk; };
__device__ __forceinline__ Unit unit_of(const Args& a)
{
    Unit u;
    const uint32_t heads = (uint32_t)(a.batch * a.kv_heads), at = blockIdx.x / heads;
    u.head = (int)(blockIdx.x - at * heads);
    u.b = u.head / a.kv_heads; u.kv = u.head - u.b * a.kv_heads;
    u.tile = a.tiles - 1 - (int)(at / (uint32_t)a.chunks); u.chunk = (int)(at % (uint32_t)a.chunks);
    return u;
}

// What a query's row sees: its keys.
__device__ __forceinline__ Sight sight_of_row(const Args& a, int b, int row)
{
    const int pos = a.first + row / a.group;
    Sight s;
    s.low = a.window ? max(0, pos - a.window + 1) : 0;
    s.high = min(a.causal ? pos + 1 : a.window ? (int)min((long)pos + a.window, (long)a.keys) : a.keys, a.keys);
    s.before = a.prefix ? (int)max(0ll, min(a.prefix[b], (long long)a.keys)) : 0;
    s.with_documents = a.documents != nullptr;
    s.of_streamed = a.documents ? a.documents + (long)b * a.keys : nullptr; s.per = 1;
    s.mine = a.documents && pos >= 0 ? s.of_streamed[pos] : 0;
    s.close();
    return s;
}

template <int NS, int W4>
__global__ __launch_bounds__(kThreads, 2) void attention_kernel(Args a)
{
    constexpr int kRows = 64 / NS, W = 4 * W4;
    const Place<NS, W4> here(a.values);
    const Unit u = unit_of(a);
    const int row0 = (u.tile * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64)) * kRows;
    if (row0 >= a.rows) return;                   // (no barriers below)
    const int mine = row0 + here.row_in_wave, row = min(mine, a.rows - 1);
    const bool exists = mine < a.rows;
    const int token = row / a.group, head = u.kv * a.group + row % a.group, pos = a.first + token, first = here.slice * W;
    const Scoring scoring(a);
    const Full full{a.off, a.off != 1.0f, 0u - scoring.mul_add, lane_pad(0u)};
    uint32_t q[W];
    bool odd = false;
    {
        // (q (*) scale first, by the full definition where it takes that)
        const float* from = a.q.p + (long)u.b * a.q.sb + (long)token * a.q.st + (long)head * a.q.sh;
        const uint32_t scale_add = f2u(a.scale) - kBias + scoring.off_add;
        odd = !load_lane<W4>(from, first, a.dim, a.values, scale_add, scoring.mul_add, lane_pad(0u), q);
        if (__ballot(odd) != 0ull) {
#pragma unroll 1
            for (int d = 0; d < W; ++d) {
                if (first + d < a.values) q[0] = f2u(pam_mul_off(from[first + d], a.scale, a.off, full.has_off)) + scoring.mul_add;
                turned(q);
            }
        }
    }
    const bool careful_lanes = __ballot(odd) != 0ull;
    float slope = 0.0f, wrong = 0.0f;             // wrong: becomes NaN with the first number that is none
    if (scoring.slopes) { slope = held_slope(a.slopes[head]); wrong = finite(a.slopes[head]) ? 0.0f : u2f(kQNaN); }
    const Sight sight = sight_of_row(a, u.b, row);
    const Stream keys = stream_of(here, a.k.p + (long)u.b * a.k.sb + (long)u.kv * a.k.sh, a.k.st, a.values, a.keys);
    const Stream values = stream_of(here, a.v.p + (long)u.b * a.v.sb + (long)u.kv * a.v.sh, a.v.st, a.values, a.keys);

    float out[W], l = 0.0f, l_before = 0.0f, M = kNothing, M_folded = kNothing;
    bool some = false, folded = false;
#pragma unroll
    for (int d = 0; d < W; ++d) out[d] = 0.0f;
    const long stat = ((long)u.head * a.chunks + u.chunk) * a.rows + row;
    float* const to = a.partial ? a.partial + stat * a.dim : a.y + (((long)u.b * a.tokens + token) * a.heads + head) * a.dim;
    int terms = 0;
    const int begin = max(sight.first / kSpan * kSpan, u.chunk * a.chunk), end = min(min(sight.last, a.keys), (u.chunk + 1) * a.chunk);
#pragma unroll 1
    for (int j0 = begin; j0 < end; j0 += kSpan) {
        const uint64_t see = sight.span(j0);
        if (__ballot(see != 0ull) == 0ull) continue;
        some = some || see != 0ull;
        const bool all = __ballot(see != ~0ull) == 0ull;
        if (terms >= kLink) {                     // the chain of sums so far joins those before it, in memory
            const float f = scale_between(M_folded, M);
            row_in_memory<W4>(to, first, a.dim, exists, [&](int n, v4f& x) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { x[i] = (folded ? x[i] * f : 0.0f) + out[4 * n + i]; }
            });
#pragma unroll
            for (int d = 0; d < W; ++d) out[d] = 0.0f;
            l_before += l; l = 0.0f;
            M_folded = M; folded = true; terms = 0;
        }
        terms += kSpan;
        v4f kr[kBlock], vr[kBlock];
        keys.rows(j0, kr);
#pragma unroll 1
        for (int i0 = 0; i0 < kSpan; i0 += kBlock) {
            const uint32_t sees = (uint32_t)(see >> i0) & 0xffu;
            if (!all && __ballot(sees != 0u) == 0ull) {
                keys.rows(j0 + i0 + kBlock, kr);
                continue;
            }
            values.rows(j0 + i0, vr);
            keys.pad(0u, kr);
            const Verdict kv = judge(here.streaming, 0u, kr);
            float t[kBlock];
            block_dots<NS, W4>(full, careful_lanes || kv.careful, kv.zero, 1.0f, kr, q, t);
            keys.rows(j0 + i0 + kBlock, kr);          // (the next block's; past the end the last key again)
            float most = kNothing;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) t[j] = scoring.exponent(t[j], slope, pos - (j0 + i0 + j));
            if (all)
#pragma unroll
                for (int j = 0; j < kBlock; ++j) most = fmaxf(most, t[j]);
            else
#pragma unroll
                for (int j = 0; j < kBlock; ++j) most = fmaxf(most, (sees >> j) & 1u ? t[j] : kNothing);
            if (__ballot(most > M + kLag) != 0ull) {
                const float raised = most > M + kLag ? floorf(most) : M, f = scale_between(M, raised);
                l *= f; l_before *= f;
#pragma unroll
                for (int d = 0; d < W; ++d) out[d] *= f;
                M = raised;
            }
            uint32_t counts = 0u;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                float power = t[j] - M;
                if (!all) power = (sees >> j) & 1u ? power : 2.0f * kLeast;
                wrong = __builtin_fmaf(power, 0.0f, wrong);
                const bool in = power >= kLeast;
                t[j] = power_of_two(fmaxf(power, kLeast));
                sum += in ? t[j] : 0.0f;
                counts |= in ? 1u << j : 0u;
            }
            l += sum;
            values.pad(0u, vr);
            const Verdict vv = judge(here.streaming, 0u, vr);
            block_add<W4>(full, vv.careful, vv.zero, 1.0f, vr, t, scoring.mul_add, counts, out);
        }
    }
    if (folded) {
        const float f = scale_between(M_folded, M);
        row_in_memory<W4>(to, first, a.dim, exists, [&](int n, v4f& x) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[4 * n + i] += x[i] * f;
        });
        l += l_before;
    }
    // (a row all of whose scores are no numbers has seen something all the same)
    l = some ? l + wrong : 0.0f;
    M = some ? (M == kNothing ? 0.0f : M) : kNothing;
    if (a.partial) {
        if (exists && here.slice == 0) a.partial_stats[stat] = make_float2(l, M);
        if (__ballot(some) != 0ull) store_row<W4>(to, first, a.dim, exists, out);
        return;
    }
    if (a.stats && exists && here.slice == 0) a.stats[((long)u.b * a.tokens + token) * a.heads + head] = make_float2(l, M);
    over_total(out, some ? l : 1.0f, a.off);
    store_row<W4>(to, first, a.dim, exists, out);
}

typedef void (*Kernel)(Args);
struct Variant { int slices, quads; Kernel kernel; };

}  // namespace pamatt
