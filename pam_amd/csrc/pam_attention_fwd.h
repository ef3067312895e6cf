// The forward pass of pam_attention.h: tiles of 64 rows over a chunk of the keys, a wavefront for each slice.
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

// A unit of a launch, a work-group: the tiles of 64 rows, the chunk, the batch entry and key head.  Consecutive work-groups take different heads, so that
// a head's keys stay with few of the XCDs' caches, and the last tiles, which see most keys where the order is causal, come first.  Work-groups go
// to the XCDs in turn, and a tile begins with another chunk than the one before: else an XCD had the same chunks of all of them, seen by all rows or by few.
struct Unit { int head, b, kv, tile, chunk; };
__device__ __forceinline__ Unit unit_of(const Args& a)
{
    Unit u;
    const uint32_t heads = (uint32_t)(a.batch * a.kv_heads), at = blockIdx.x / heads, tile = at / (uint32_t)a.chunks;
    u.head = (int)(blockIdx.x - at * heads);
    u.b = u.head / a.kv_heads; u.kv = u.head - u.b * a.kv_heads;
    u.tile = a.tiles - 1 - (int)tile; u.chunk = (int)((at + tile) % (uint32_t)a.chunks);
    return u;
}
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64); }

// The streamed rows of a unit's chunk: from row `origin` or its span on.
struct Chunk { int begin, end; };
__device__ __forceinline__ Chunk chunk_of(const Args& a, const Unit& u, int origin, int streamed)
{
    const long from = (a.windows ? origin / kSpan * kSpan : 0) + (long)u.chunk * a.chunk;
    return Chunk{(int)min(from, (long)streamed), (int)min(from + a.chunk, (long)streamed)};
}
// ... of the keys, where the tiles of queries begin with row row0
__device__ __forceinline__ Chunk chunk_of_keys(const Args& a, const Unit& u, int row0) { return chunk_of(a, u, max(0, a.first + row0 / a.group - a.window + 1), a.keys); }

// The launch's arguments as from memory: what the careful loops need is found again there, instead of in registers since the beginning.
__device__ __forceinline__ Args arguments_again()
{
    auto at = (const __attribute__((address_space(4))) Args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    return *(const Args*)at;
}
template <int NS> __device__ __forceinline__ int row_of_lane(const Unit& u, int rows) { return min((u.tile * kTiles<NS> + wave_of() / NS) * 64 + (int)threadIdx.x % 64, rows - 1); }
template <int NS> __device__ __forceinline__ const float* query_of_lane(const Args& a)
{
    const Unit u = unit_of(a);
    const int row = row_of_lane<NS>(u, a.rows);
    return a.q.p + (long)u.b * a.q.sb + (long)(row / a.group) * a.q.st + (long)(u.kv * a.group + row % a.group) * a.q.sh;
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

template <int NS, int W4, bool WHOLE>
__global__ __launch_bounds__(64 * kWaveCount<NS>, W4 > 8 ? 2 : 3) void attention_kernel(Args a)
{
    constexpr int W = 4 * W4;
    __shared__ Slices<NS, kBlock> slices;
    const Unit u = unit_of(a);
    const int wave = wave_of(), slice = wave % NS, row0 = (u.tile * kTiles<NS> + wave / NS) * 64, mine = row0 + (int)threadIdx.x % 64, row = min(mine, a.rows - 1), first = slice * W;
    const bool exists = mine < a.rows;
    const int token = row / a.group, head = u.kv * a.group + row % a.group, pos = a.first + token;
    Sight sight = sight_of_row(a, u.b, row);
    sight.close_team<NS>();
    const long stat = ((long)u.head * a.chunks + u.chunk) * a.rows + row;
    float* const to = a.partial ? a.partial + stat * a.dim : a.y + (((long)u.b * a.tokens + token) * a.heads + head) * a.dim;
    const Chunk chunk = chunk_of_keys(a, u, u.tile * kTiles<NS> * 64);
    const int begin = max(sight.first / kSpan * kSpan, chunk.begin), end = min(sight.last, chunk.end);
    if (a.partial && !any_seen<NS>(sight, begin, end)) {
        if (exists && slice == 0) a.partial_stats[stat] = make_float2(0.0f, kNothing);
        return;
    }
    const Scoring scoring(a);
    const Full full{a.off, a.off != 1.0f};
    uint32_t q[W];
    bool careful = in_team<NS>(load_lane<W4>(query_of_lane<NS>(a), first, a.dim, a.values, f2u(a.scale) - kBias + scoring.off_add, scoring.mul_add, q, Form::plain()).odd);       // (of q (*) scale)
    float slope = 0.0f, wrong = 0.0f;             // wrong: becomes NaN with the first number that is none
    if (scoring.slopes) { slope = held_slope(a.slopes[head]); wrong = finite(a.slopes[head]) ? 0.0f : u2f(kQNaN); }
    const Stream<WHOLE> keys(a.k.p + (long)u.b * a.k.sb + (long)u.kv * a.k.sh, a.k.st, a.keys, slice * W4, a.dim / 4);
    const Stream<WHOLE> values(a.v.p + (long)u.b * a.v.sb + (long)u.kv * a.v.sh, a.v.st, a.keys, slice * W4, a.dim / 4);
    float out[W], l, l_before, M, M_folded;
    bool some, folded;
    int terms, turn = 0;
    // scores to weights, M raised where one is far above it; returns which ones count
    const auto weigh = [&](float (&t)[kBlock], uint32_t sees, bool all, int j1) __attribute__((always_inline)) {
        float most = kNothing;
#pragma unroll
        for (int j = 0; j < kBlock; ++j) t[j] = scoring.exponent(t[j], slope, pos - (j1 + j));
        // (not from its distance to M: of scores near both ends of the range that may be an infinity, and counts for nothing)
        const auto met = [&](float exponent) __attribute__((always_inline)) { most = fmaxf(most, exponent); wrong = __builtin_fmaf(exponent, 0.0f, wrong); };
        if (all)
#pragma unroll
            for (int j = 0; j < kBlock; ++j) met(t[j]);
        else
#pragma unroll
            for (int j = 0; j < kBlock; ++j) met((sees >> j) & 1u ? t[j] : kNothing);
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
            const bool in = power >= kLeast;
            t[j] = power_of_two(fmaxf(power, kLeast));
            sum += in ? t[j] : 0.0f;
            counts |= in ? 1u << j : 0u;
        }
        l += sum;
        return counts;
    };
    // all blocks of the chunk; false: one of them did not want to
    const auto run = [&](auto&& start, auto&& block) __attribute__((always_inline)) {
        l = l_before = 0.0f; M = M_folded = kNothing;
        some = folded = false; terms = 0;
#pragma unroll
        for (int d = 0; d < W; ++d) out[d] = 0.0f;
#pragma unroll 1
        for (int j0 = begin; j0 < end; j0 += kSpan) {
            const uint64_t see = sight.span(j0);
            if (!in_team<NS>(see != 0ull)) continue;
            some = some || see != 0ull;
            const bool all = __ballot(see != ~0ull) == 0ull;
            if (terms >= kLink) {                 // the chain of sums so far joins those before it, in memory
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
            start(j0);
#pragma unroll 1
            for (int i0 = 0; i0 < kSpan; i0 += kBlock)
                if (!block(j0 + i0, (uint32_t)(see >> i0) & 0xffu, all)) return false;
        }
        return true;
    };
    if (!careful) {
        Pipe<W4, WHOLE> pipe;
        Look<W4, WHOLE> look_k, look_v;
        careful = !run([&](int j0) __attribute__((always_inline)) { pipe.request(keys, j0); look_k.load(keys, j0); look_v.load(values, j0); },
            [&](int j1, uint32_t sees, bool all) __attribute__((always_inline)) {
                float t[kBlock];
                if (!all && __ballot(sees != 0u) == 0ull) {
                    pipe.request(keys, j1 + kBlock); look_k.load(keys, j1 + kBlock); look_v.load(values, j1 + kBlock);
                    const bool wild = slices.add_up(turn, wave, t, false);
                    turn ^= 1;
                    return !wild;
                }
                const Verdict kv = judge(look_k, keys, a.values, 0u), vv = judge(look_v, values, a.values, 0u);
                look_k.load(keys, j1 + kBlock);      // (the next block's; past the end the last key again)
                look_v.load(values, j1 + kBlock);
                block_dots<W4, WHOLE>(pipe, keys, j1, values, j1, kv.zeros, NoLaneZeros{}, q, t);
                const bool wild = slices.add_up(turn, wave, t, kv.wild || vv.wild);
                turn ^= 1;
                if (__builtin_expect(wild, 0)) return false;
                const uint32_t counts = weigh(t, sees, all, j1);
                block_add<W4, WHOLE>(pipe, values, j1, keys, j1 + kBlock, vv.zeros, t, scoring.mul_add, counts, out);
                return true;
            });
    }
    if (__builtin_expect(careful, 0)) {
        const Args g = arguments_again();
        const float* const from = query_of_lane<NS>(g);
        load_plain<W4>(first, g.values, q, [&](int d) __attribute__((always_inline)) { return pam_mul_off(from[d], g.scale, g.off, g.off != 1.0f); });
        run([](int) {}, [&](int j1, uint32_t sees, bool all) __attribute__((always_inline)) {
            float t[kBlock];
            if (!all && __ballot(sees != 0u) == 0ull) {
                slices.add_up(turn, wave, t, false);
                turn ^= 1;
                return true;
            }
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
                t[0] = careful_dot<W4>(full, keys.template across<W4>(j1 + j), q);
                turned(t);
            }
            slices.add_up(turn, wave, t, false);
            turn ^= 1;
            const uint32_t counts = weigh(t, sees, all, j1);
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
                careful_add_row<W4>(full, values.template across<W4>(j1 + j), t[0], (counts >> j) & 1u, 1.0f, out);
                turned(t);
            }
            return true;
        });
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
        if (exists && slice == 0) a.partial_stats[stat] = make_float2(l, M);
        if (__ballot(some) != 0ull) store_row<W4>(to, first, a.dim, exists, out);
        return;
    }
    if (a.stats && exists && slice == 0) a.stats[((long)u.b * a.tokens + token) * a.heads + head] = make_float2(l, M);
    over_total(out, some ? l : 1.0f, a.off);
    store_row<W4>(to, first, a.dim, exists, out);
}

typedef void (*Kernel)(Args);
struct Variant { int slices, quads; bool whole; Kernel kernel; };      // whole: for rows of just these quads

template <int NS, int W4, bool WHOLE> constexpr Variant forward_of() { return Variant{NS, W4, WHOLE, attention_kernel<NS, W4, WHOLE>}; }

}  // namespace pamatt
