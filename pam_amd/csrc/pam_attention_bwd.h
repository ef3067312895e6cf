// The gradients of pam_attention.h.  With the rows' quantities
//   dn_id = dy_id (*) (1 (/) l_i),  dl_i = -sum_d (y_id (/) l_i) (*) dy_id
// of a kernel before (attention_rows_kernel),
//   de_ij = sum_d dn_id (*) v_jd + dl_i,   dx_ij = e_ij (*) de_ij,   da_ij through the cap,
//   dqs_id = sum_j da_ij (*) k_jd,   dk_jd = sum_i da_ij (*) qs_id,   dv_jd = sum_i e_ij (*) dn_id
// for approximate gradients; an exact one weighs the gradient by the slope of the other factor's piece instead.  (All slopes exact and no offset, or all
// approximate, have usual loops; mixed slopes and exact ones with an offset take the full definition throughout: 31 and 44 ms where 4.4 are below.)  Two kernels: in the first lanes own
// queries and keys stream by (a, de and dq: three products), in the second lanes own keys and queries stream by (a, de, dk and dv: four).
// Scores and weights are computed again in both; kept, they would be 8 bytes a pair, as long to read as two of the products of 64 values.
// 4096 causal tokens, 8 heads of 64 over 2: 0.93 ms for dq (13.8 T products/s), 1.70 for dk and dv (10), exact 1.7 and 2.1; three wavefronts on a SIMD are 6 % better than two for the
// first, and 30 % worse for the second, whose four slices of 32 then do not fit the registers.
// All that is linear in dy is scaled by a power of two: in the first kernel a query's largest |dn| to [1, 2), in the second the largest of a chunk's.  The full definition
// scales up only, so that nothing is lost beside a large value.
#pragma once
#include "pam_attention_fwd.h"

namespace pamatt {

// The gradient for a of e = 2^(x(a) (*) log2 e) from that of e.
template <bool APPROXIMATE>
struct PairGrad {
    const Scoring& s; ApproxFlags f;
    __device__ __forceinline__ bool a_approx() const { return APPROXIMATE || f.a; }
    __device__ __forceinline__ bool b_approx() const { return APPROXIMATE || f.b; }
    __device__ __forceinline__ bool e_approx() const { return APPROXIMATE || f.e; }
    __device__ __forceinline__ static float slope(uint32_t other, float own) { return u2f((other + (f2u(own) & kMant)) & ~kMant); }
    // own (*) other, for own; other positive
    __device__ __forceinline__ float of_mul(float own, float other, float d) const
    { return a_approx() ? times_any(d, other, s.off_add) : d * slope(f2u(other) + s.off_add, own); }
    // (integer additions know no NaN; through a cap a gradient of 2^90 counts as one, whose products on the way are below 2^127)
    __device__ __forceinline__ float checked(float a, float score, float e, float de) const
    {
        const float d = (*this)(a, score, e, de);
        return fabsf(de) < (s.cap == 0.0f ? u2f(kExpo) : 0x1p90f) && e == e ? d : u2f(kQNaN);
    }
    __device__ __forceinline__ float operator()(float a, float score, float e, float de) const
    {
        float d;
        if (e_approx()) d = times_any(e, de, s.off_add);
        else d = u2f(f2u(e) & ~kMant) * de * slope(f2u(kLog2e) + s.off_add, score);
        if (s.cap == 0.0f) return d;
        // x = th (*) cap, th = n (/) m, n = 1 - w, m = 1 + w, w = 2^-power, power = u (*) kTurn, u = |a| (/) cap
        const Raw ar(s.off);
        const Scoring::Cap c = s.capping(a);
        const float m = 1.0f + c.w, n = 1.0f - c.w, inverse = ar.div(1.0f, m), by_cap = ar.div(1.0f, s.cap);
        const float dth = of_mul(c.th, s.cap, d);
        const float dn = a_approx() ? times_any(dth, inverse, s.off_add) : dth * slope(f2u(inverse), n);
        const float over = c.th > 0.0f ? ar.div(c.th, m) : 0.0f;
        const float dm = b_approx() ? times_any(dth, over, s.off_add) : dth * u2f(c.th > 0.0f ? (f2u(c.th) & ~kMant) - (f2u(m) & kExpo) + kBias : 0u);
        const float dw = -(dm + dn);
        const float dpower = -(e_approx() ? times_any(times_any(c.w, kActLn2, s.off_add), dw, s.off_add) : u2f((f2u(c.w) & ~kMant)) * dw);
        const float du = of_mul(c.u, kTurn, dpower);
        return a_approx() ? times_any(du, by_cap, s.off_add) : du * slope(f2u(by_cap), a);
    }
};

// What `delta` times own (*) other gives own by the slope of the piece that it is in.
__device__ __forceinline__ float exact_term(const Full& f, float own, float other, float delta)
{ return pam_mul_bwd(own, other, delta, f.off, f.has_off); }

// The usual way's sums of slopes are kept times the own factor's power until the end.
constexpr uint32_t kPower = ~kMant;
__device__ __forceinline__ float over_power(float sum, uint32_t own) { return sum * u2f((2u * kBias - (own & kExpo)) | (own & kSign)); }

// The slopes of a row that lanes hold a quad each of, by the full definition.
template <int W4, class F> __device__ __forceinline__ void each_of_row(const v4f& row, F&& f)
{
    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f(4 * n.value + i, u2f(from_lane<decltype(n)::value>(row[i])));
            __builtin_amdgcn_sched_barrier(0);
        }
    });
}

// All blocks of a chunk of streamed rows, sums joined in memory after kLink of them; false: one block did not want to.  met: a row of the team saw one.
template <int NS, int W4, int SUMS, class Start, class Block>
__device__ __forceinline__ bool all_blocks(const Sight& sight, int begin, int end, float* const (&to)[SUMS], int first, int dim, bool exists, float (&out)[SUMS][4 * W4], bool& met,
                                           Start&& start, Block&& block)
{
    met = false;
    bool folded = false;
    int terms = 0;
#pragma unroll
    for (int n = 0; n < SUMS; ++n)
#pragma unroll
        for (int d = 0; d < 4 * W4; ++d) out[n][d] = 0.0f;
    const auto with_memory = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < SUMS; ++n)
            row_in_memory<W4>(to[n], first, dim, exists, [&](int quad, v4f& x) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { float in_memory = x[i]; f(in_memory, out[n][4 * quad + i]); x[i] = in_memory; }
            });
    };
#pragma unroll 1
    for (int j0 = begin; j0 < end; j0 += kSpan) {
        const uint64_t see = sight.span(j0);
        if (!in_team<NS>(see != 0ull)) continue;
        met = true;
        const bool all = __ballot(see != ~0ull) == 0ull;
        if (terms >= kLink) {
            with_memory([&](float& in_memory, float& sum) __attribute__((always_inline)) { in_memory = (folded ? in_memory : 0.0f) + sum; sum = 0.0f; });
            folded = true; terms = 0;
        }
        terms += kSpan;
        start(j0);
#pragma unroll 1
        for (int i0 = 0; i0 < kSpan; i0 += kBlock)
            if (!block(j0 + i0, (uint32_t)(see >> i0) & 0xffu, all)) return false;
    }
    if (folded) with_memory([&](float& in_memory, float& sum) __attribute__((always_inline)) { sum += in_memory; });
    return true;
}

// Whether a tile saw anything of its chunk is kept for those who put the chunks together: a tile that did not writes nothing, and is not read.
template <int NS> __device__ __forceinline__ bool met_anything(const Args& a, const Unit& u, int wave, bool met)
{
    if (threadIdx.x % 64 == 0 && wave % NS == 0)
        a.met[((long)u.head * a.chunks + u.chunk) * a.tiles * kTiles<NS> + u.tile * kTiles<NS> + wave / NS] = met;
    return met;
}

// How lanes hold what they own.  behind: the slices have places behind a head's values.  Exact slopes are taken with the lane's value, whose zero has to be a power of
// two that keeps the product where sums have all their bits: the window's end.  (Those of e (*) v with v in the lane: weights of 2^-62 leave it 2^-64.)
constexpr int kZero = -86, kZeroOfSlopes = 30, kBehindWeights = -64;
__device__ __forceinline__ Form form_of(bool approximate, bool behind)
{ return Form{behind ? kZero + 28 : kZero, approximate ? 80 : kZeroOfSlopes, bits_of_power(approximate ? kZero : kZeroOfSlopes), bits_of_power(kZero)}; }
__device__ __forceinline__ Form form_of_weighted(bool behind) { return Form{behind ? kBehindWeights + 28 : kBehindWeights, kZeroOfSlopes, bits_of_power(kZeroOfSlopes), bits_of_power(kBehindWeights)}; }

// Sums of up to 256 products of which a lane's zeros have made some 2^-86 times a streamed value below `above`: as good as rounded if they are at least this, and zero where the
// lane has nothing else.
constexpr float kLeastSum = 0x1p-54f;             // 2^8 2^-86 2^24
__device__ __forceinline__ void without_zeros(bool zeros, bool numbers, float (&sum)[kBlock])
{
    if (__builtin_expect(zeros, 0))
#pragma unroll
        for (int j = 0; j < kBlock; ++j) sum[j] = numbers ? sum[j] : 0.0f;
}
__device__ __forceinline__ bool too_small(bool zeros, const float (&sum)[kBlock], uint32_t counts, float above)
{
    bool found = false;
    if (__builtin_expect(zeros, 0))
#pragma unroll
        for (int j = 0; j < kBlock; ++j) found = found || ((counts >> j) & 1u && sum[j] != 0.0f && fabsf(sum[j]) < kLeastSum * above);
    return found;
}

// Pairs' gradients below 2^-86 (|dn| is 1, streamed values are at least 2^-40): those of at least 2^-116 are lifted to where products are in range, the others are none.
__device__ __forceinline__ bool lift(float (&da)[kBlock], uint32_t& counts, uint32_t& small)
{
    small &= counts;
    if (__builtin_expect(__ballot(small != 0u) == 0ull, 1)) return false;
#pragma unroll
    for (int j = 0; j < kBlock; ++j) {
        const bool lifted = (small >> j) & 1u;
        da[j] = lifted ? da[j] * (float)(1 << kLift) : da[j];
        if (lifted && fabsf(da[j]) < 0x1p-86f) { counts &= ~(1u << j); small &= ~(1u << j); }
    }
    return __ballot(small != 0u) != 0ull;
}

template <int NS, int W4, bool WHOLE, bool APPROXIMATE>
__global__ __launch_bounds__(64 * kWaveCount<NS>, 3) void attention_dq_kernel(Args a)
{
    constexpr int W = 4 * W4, N = 4 * Pipe<W4, WHOLE>::kQuads;
    __shared__ Slices<NS, kBlock> slices_s, slices_de;
    const Unit u = unit_of(a);
    const int wave = wave_of(), slice = wave % NS, row0 = (u.tile * kTiles<NS> + wave / NS) * 64, mine = row0 + (int)threadIdx.x % 64, row = min(mine, a.rows - 1), first = slice * W;
    const bool exists = mine < a.rows;
    const int pos = a.first + row / a.group;
    Sight sight = sight_of_row(a, u.b, row);
    sight.close_team<NS>();
    const Chunk chunk = chunk_of_keys(a, u, u.tile * kTiles<NS> * 64);
    const int begin = max(sight.first / kSpan * kSpan, chunk.begin), end = min(sight.last, chunk.end);
    if (!a.whole && !any_seen<NS>(sight, begin, end)) { met_anything<NS>(a, u, wave, false); return; }
    const Scoring scoring(a);
    const PairGrad<APPROXIMATE> pair{scoring, a.flags};
    const uint32_t dn_add = APPROXIMATE ? scoring.mul_add : 0u;
    const Full full{a.off, a.off != 1.0f};
    const float4 record = a.records[(long)u.head * a.rows + row];
    const float M = record.x, slope = record.w;
    float unit = u2f((uint32_t)(127 - (int)record.z) << 23), dl = record.y * unit;
    uint32_t q[W], dn[W];
    const long at = ((long)u.head * a.rows + row) * a.dim;
    // (what the exact slopes of e (*) v weigh is a factor, and may be zero)
    const bool behind = a.values < NS * W;
    Form q_form = form_of(APPROXIMATE, behind);
    if (a.values % 4 != 0) q_form.ones = a.values % 4;
    const Form dn_form = APPROXIMATE ? q_form : Form{-86, 80, 0u, 0u};
    const Held of_q = load_lane<W4>(a.qs + at, first, a.dim, a.values, 0u, scoring.mul_add, q, q_form);
    const Held of_dn = load_lane<W4>(a.dn + at, first, a.dim, a.values, 0u, dn_add, dn, dn_form, unit);
    const bool counts_at_all = M != u2f(kExpo);
    bool odd = of_q.odd || of_dn.odd;
    const bool zeros = in_team<NS>((APPROXIMATE ? of_dn.zeros : of_q.zeros) && counts_at_all);
    const LaneZeros<kZeroOfSlopes, kZero> q_zeros{zeros, scoring.mul_add};
    odd = odd || !finite(dl);
    // (all slopes, and no offset: what the usual way of the other kernel has)
    const bool unusual = !APPROXIMATE && (a.flags.a || a.flags.b || a.flags.e || a.off != 1.0f);
    bool careful = in_team<NS>(odd && counts_at_all) || unusual;
    const Stream<WHOLE> keys(a.k.p + (long)u.b * a.k.sb + (long)u.kv * a.k.sh, a.k.st, a.keys, slice * W4, a.dim / 4);
    const Stream<WHOLE> values(a.v.p + (long)u.b * a.v.sb + (long)u.kv * a.v.sh, a.v.st, a.keys, slice * W4, a.dim / 4);
    float out[1][W];
    const int head = u.kv * a.group + row % a.group;
    float* const to[1] = {a.out0 + (a.whole ? ((long)u.b * a.tokens + row / a.group) * a.heads + head : ((long)u.head * a.chunks + u.chunk) * a.rows + row) * a.dim};
    int turn = 0;
    // weights from scores, and which ones count (what is no number does)
    const auto weigh = [&](const float (&s)[kBlock], float (&e)[kBlock], uint32_t sees, bool all, int j1, bool& wrong) __attribute__((always_inline)) {
        uint32_t counts = 0u;
#pragma unroll
        for (int j = 0; j < kBlock; ++j) {
            float power = scoring.exponent(s[j], slope, pos - (j1 + j)) - M;
            if (!all) power = (sees >> j) & 1u ? power : 2.0f * kLeast;
            wrong = wrong || power != power;
            counts |= power < kLeast ? 0u : 1u << j;
            e[j] = power_of_two(fminf(fmaxf(power, kLeast), 60.0f));
            e[j] = power != power ? power : e[j];
        }
        return counts;
    };
    bool gave_up = false;                         // (what all of a tile's slices find behind the sums goes with the next ones)
    bool met = false;
    const auto skip = [&](float (&s)[kBlock], float (&de)[kBlock]) __attribute__((always_inline)) {      // (no row of the tile sees the block: its barriers)
        const bool wild = slices_s.add_up(turn, wave, s, gave_up);
        if (wild) { turn ^= 1; return false; }
        slices_de.add_up(turn, wave, de, false);
        turn ^= 1;
        return true;
    };
    const auto score_gradient = [&](float s, float e, float de, int far) __attribute__((always_inline)) {
        float x = s;
        if (!APPROXIMATE && !a.flags.e) {                          // (the score as log2 e multiplies it)
            x = scoring.cap != 0.0f ? scoring.capped(x) : x;
            if (scoring.slopes) x = scoring.biased(x, slope, far);
        }
        return pair.checked(s, x, e, de + dl);
    };
    if (!careful) {
        Pipe<W4, WHOLE> pipe;
        Look<W4, WHOLE> look_k, look_v;
        careful = !all_blocks<NS, W4, 1>(sight, begin, end, to, first, a.dim, exists, out, met,
            [&](int j0) __attribute__((always_inline)) { pipe.request(keys, j0); look_k.load(keys, j0); look_v.load(values, j0); },
            [&](int j1, uint32_t sees, bool all) __attribute__((always_inline)) {
                float s[kBlock], de[kBlock], e[kBlock];
                if (!all && __ballot(sees != 0u) == 0ull) {
                    pipe.request(keys, j1 + kBlock); look_k.load(keys, j1 + kBlock); look_v.load(values, j1 + kBlock);
                    return skip(s, de);
                }
                const Verdict kv = judge(look_k, keys, a.values, 0u), vv = judge(look_v, values, a.values, 0u);
                float above = 0.0f;
                if (APPROXIMATE && zeros) above = above_all(look_v);
                look_k.load(keys, j1 + kBlock);
                look_v.load(values, j1 + kBlock);
                bool wrong = false;
                if constexpr (APPROXIMATE) block_dots<W4, WHOLE>(pipe, keys, j1, values, j1, kv.zeros, NoLaneZeros{}, q, s);
                else block_dots<W4, WHOLE>(pipe, keys, j1, values, j1, kv.zeros, q_zeros, q, s);
                bool wild = slices_s.add_up(turn, wave, s, gave_up || kv.wild || vv.wild);
                if (__builtin_expect(wild, 0)) { turn ^= 1; return false; }      // (others may be reading that buffer)
                uint32_t counts = weigh(s, e, sees, all, j1, wrong);
                if constexpr (APPROXIMATE) {
                    block_dots<W4, WHOLE>(pipe, values, j1, keys, j1, vv.zeros, NoLaneZeros{}, dn, de);
                    without_zeros(zeros, of_dn.numbers, de);
                } else {
#pragma unroll
                    for (int j = 0; j < kBlock; ++j) de[j] = 0.0f;
                    uint32_t left = counts;
                    if (__builtin_expect(vv.zeros, 0))
                        pipe.rolled(values, j1, keys, j1, [&](int h, int d, const Piece& x) __attribute__((always_inline)) {
                            dot_power_piece_with_zeros<N>(x, f2u(e[0]) + scoring.mul_add, left & 1u ? kPower : 0u, dn + d, de[0]);
                            if (h == Pipe<W4, WHOLE>::kPieces - 1) { turned(e); turned(de); left >>= 1; }
                        });
                    else
                        pipe.block(values, j1, keys, j1, [&](int j, int d, const Piece& x) __attribute__((always_inline)) {
                            dot_power_piece<N>(x, f2u(e[j]) + scoring.mul_add, counts >> j & 1u ? kPower : 0u, dn + d, de[j]);
                        });
#pragma unroll
                    for (int j = 0; j < kBlock; ++j) de[j] = over_power(de[j], f2u(e[j]));
                }
                slices_de.add_up(turn, wave, de, false);
                turn ^= 1;
                if (APPROXIMATE) wrong = wrong || too_small(zeros, de, counts, above);
                uint32_t small = 0u;
#pragma unroll
                for (int j = 0; j < kBlock; ++j) {
                    de[j] = score_gradient(s[j], e[j], de[j], pos - (j1 + j));
                    if (APPROXIMATE) {
                        wrong = wrong || ((counts >> j) & 1u && !(fabsf(de[j]) < 0x1p80f));
                        small |= fabsf(de[j]) < 0x1p-86f ? 1u << j : 0u;
                    }
                }
                gave_up = gave_up || __ballot(wrong) != 0ull;
                if (NS == 1 && __builtin_expect(gave_up, 0)) return false;
                if constexpr (APPROXIMATE) {
                    const bool some_small = lift(de, counts, small);
                    block_add<W4, WHOLE>(pipe, keys, j1, keys, j1 + kBlock, kv.zeros, de, scoring.mul_add, counts, out[0], some_small, small);
                }
                else block_add_power<W4, WHOLE>(pipe, keys, j1, keys, j1 + kBlock, kv.zeros, kPower, de, counts, q, out[0]);
                return true;
            });
        careful = careful || in_team<NS>(gave_up);
        if (!APPROXIMATE)
#pragma unroll
            for (int d = 0; d < W; ++d) out[0][d] = over_power(out[0][d], q[d] - scoring.mul_add);
    }
    gave_up = false;
    if (__builtin_expect(careful, 0)) {
        const Args g = arguments_again();
        const Unit w = unit_of(g);
        const long of = (long)w.head * g.rows + row_of_lane<NS>(w, g.rows), from = of * g.dim;
        unit = fmaxf(unit, 1.0f); dl = g.records[of].y * unit;
        load_plain<W4>(first, g.values, q, [&](int d) __attribute__((always_inline)) { return g.qs[from + d]; });
        load_plain<W4>(first, g.values, dn, [&](int d) __attribute__((always_inline)) { return g.dn[from + d] * unit; });
        all_blocks<NS, W4, 1>(sight, begin, end, to, first, a.dim, exists, out, met, [](int) {}, [&](int j1, uint32_t sees, bool all) __attribute__((always_inline)) {
            float s[kBlock], de[kBlock], e[kBlock];
            if (!all && __ballot(sees != 0u) == 0ull) { skip(s, de); return true; }
            bool wrong = false;
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
                s[0] = careful_dot<W4>(full, keys.template across<W4>(j1 + j), q);
                turned(s);
            }
            slices_s.add_up(turn, wave, s, false);
            const uint32_t counts = weigh(s, e, sees, all, j1, wrong);
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
                const v4f row = values.template across<W4>(j1 + j);
                if (APPROXIMATE || a.flags.a) de[0] = careful_dot<W4>(full, row, dn);
                else {
                    de[0] = 0.0f;
                    each_of_row<W4>(row, [&](int d, float x) __attribute__((always_inline)) { de[0] += exact_term(full, e[0], x, u2f(plain(dn[d]))); });
                }
                turned(de); turned(e);
            }
            slices_de.add_up(turn, wave, de, false);
            turn ^= 1;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) de[j] = de[j] + dl == 0.0f ? 0.0f : score_gradient(s[j], e[j], de[j], pos - (j1 + j));      // (the usual loop leaves out what a zero makes)
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
                const v4f row = keys.template across<W4>(j1 + j);
                const bool in = (counts >> j) & 1u;
                if (APPROXIMATE || a.flags.a) careful_add_row<W4>(full, row, de[0], in, 1.0f, out[0]);
                else
                    each_of_row<W4>(row, [&](int d, float x) __attribute__((always_inline)) {
                        const float term = exact_term(full, u2f(plain(q[d])), x, de[0]);
                        out[0][d] += in ? term : 0.0f;
                    });
                turned(de);
            }
            return true;
        });
    }
    if (!a.whole && !met_anything<NS>(a, u, wave, met)) return;
    const float back = 1.0f / unit;
#pragma unroll
    for (int d = 0; d < W; ++d) out[0][d] *= back;
    if (a.whole) {                                // (else where the chunks are put together)
        const float* const from = a.q.p + (long)u.b * a.q.sb + (long)(row / a.group) * a.q.st + (long)head * a.q.sh;
#pragma unroll 1
        for (int d = 0; d < W; ++d) {
            if (first + d < a.values) out[0][0] = mul_grad(from[first + d], a.scale, out[0][0], a.flags.a, a.off, a.off != 1.0f);
            turned(out[0]);
        }
    }
    store_row<W4>(to[0], first, a.dim, exists, out[0]);
}

// What a key's lane sees: the rows of its head's queries.
__device__ __forceinline__ int row_of_token(const Args& a, long token) { return (int)max(0l, min(token * a.group, (long)a.rows)); }
__device__ __forceinline__ int first_row_of_key(const Args& a, int key)
{
    const long at = (long)key - a.first;
    return a.causal ? row_of_token(a, at) : a.window ? row_of_token(a, at - a.window + 1) : 0;
}
__device__ __forceinline__ Sight sight_of_key(const Args& a, int b, int key)
{
    Sight s;
    s.low = first_row_of_key(a, key);
    s.high = a.window ? row_of_token(a, (long)key - a.first + a.window) : a.rows;
    s.before = a.prefix && key < a.prefix[b] ? a.rows : 0;
    s.with_documents = a.documents != nullptr;
    s.of_streamed = a.documents ? a.documents + (long)b * a.keys + a.first : nullptr; s.per = a.group;
    s.mine = a.documents ? a.documents[(long)b * a.keys + key] : 0;
    s.close();
    return s;
}

// A unit's keys: the first ones have most queries where the order is causal.
__device__ __forceinline__ Unit unit_of_keys(const Args& a)
{
    Unit u = unit_of(a);
    u.tile = a.tiles - 1 - u.tile;
    return u;
}
template <int NS> __device__ __forceinline__ const float* key_of_lane(const Args& a, const Tokens& t)
{
    const Unit u = unit_of_keys(a);
    return t.p + (long)u.b * t.sb + (long)row_of_lane<NS>(u, a.keys) * t.st + (long)u.kv * t.sh;
}

template <int NS, int W4, bool WHOLE, bool APPROXIMATE>
__global__ __launch_bounds__(64 * kWaveCount<NS>, 2) void attention_dkv_kernel(Args a)
{
    constexpr int W = 4 * W4, N = 4 * Pipe<W4, WHOLE>::kQuads;
    __shared__ Slices<NS, kBlock> slices_s, slices_de;
    const Unit u = unit_of_keys(a);
    const int wave = wave_of(), slice = wave % NS, lane = (int)threadIdx.x % 64, key0 = (u.tile * kTiles<NS> + wave / NS) * 64, mine = key0 + lane, key = min(mine, a.keys - 1), first = slice * W;
    const bool exists = mine < a.keys;
    const Chunk chunk = chunk_of(a, u, first_row_of_key(a, u.tile * kTiles<NS> * 64), a.rows);
    Sight sight = sight_of_key(a, u.b, key);
    sight.close_team<NS>();
    const int begin = max(sight.first / kSpan * kSpan, chunk.begin), end = min(sight.last, chunk.end);
    if (!a.whole && !any_seen<NS>(sight, begin, end)) { met_anything<NS>(a, u, wave, false); return; }
    const Scoring scoring(a);
    const PairGrad<APPROXIMATE> pair{scoring, a.flags};
    typedef const __attribute__((address_space(4))) float4* Records;
    const float4* const all_records = a.records + (long)u.head * a.rows;
    const auto record = [&](int r) __attribute__((always_inline)) { const Records from = (Records)(all_records + min(r, a.rows - 1)); return make_float4(from->x, from->y, from->z, from->w); };
    // the largest |dn| of the chunk's rows is scaled to [1, 2)
    int most = -86;
    for (int r = chunk.begin + lane; r < chunk.end; r += 64) most = max(most, (int)all_records[r].z);
#pragma unroll
    for (int s = 1; s < 64; s *= 2) most = max(most, __shfl_xor(most, s, 64));
    most = APPROXIMATE ? __builtin_amdgcn_readfirstlane(most) : 0;
    const uint32_t shift = 0u - ((uint32_t)most << 23);
    float unit = u2f((uint32_t)(127 - most) << 23);
    const Full full{a.off, a.off != 1.0f};
    uint32_t k[W], v[W];
    const bool behind = a.values < NS * W;
    const Form k_form = form_of(APPROXIMATE, behind), v_form = APPROXIMATE ? k_form : form_of_weighted(behind);
    const Held of_k = load_lane<W4>(key_of_lane<NS>(a, a.k), first, a.dim, a.values, 0u, scoring.mul_add, k, k_form);
    const Held of_v = load_lane<W4>(key_of_lane<NS>(a, a.v), first, a.dim, a.values, 0u, scoring.mul_add + shift, v, v_form);
    const bool zeros = in_team<NS>(of_v.zeros), odd = of_k.odd || of_v.odd || (APPROXIMATE && zeros && most >= 60);      // (else streamed values are below 2)
    const LaneZeros<kZeroOfSlopes, kZero> k_zeros{APPROXIMATE ? 0 : in_team<NS>(of_k.zeros), scoring.mul_add};
    const LaneZeros<kZeroOfSlopes, kBehindWeights> v_zeros{zeros, scoring.mul_add};
    const bool unusual = !APPROXIMATE && (a.flags.a || a.flags.b || a.flags.e || a.off != 1.0f);
    bool careful = in_team<NS>(odd) || unusual;
    const Stream<WHOLE> queries(a.qs + (long)u.head * a.rows * a.dim, a.dim, a.rows, slice * W4, a.dim / 4);
    const Stream<WHOLE> grads(a.dn + (long)u.head * a.rows * a.dim, a.dim, a.rows, slice * W4, a.dim / 4);
    float out[2][W];                              // dk, dv
    const long at = (a.whole ? ((long)u.b * a.keys + key) * a.kv_heads + u.kv : ((long)u.head * a.chunks + u.chunk) * a.keys + key) * a.dim;
    float* const to[2] = {a.out0 + at, a.out1 + at};
    int turn = 0;
    const auto weigh = [&](const float (&s)[kBlock], float (&e)[kBlock], uint32_t sees, bool all, int r1, bool& wrong) __attribute__((always_inline)) {
        uint32_t counts = 0u;
#pragma unroll
        for (int j = 0; j < kBlock; ++j) {
            const float4 of = record(r1 + j);
            float power = scoring.exponent(s[j], of.w, a.first + (r1 + j) / a.group - key) - of.x;
            if (!all) power = (sees >> j) & 1u ? power : 2.0f * kLeast;
            wrong = wrong || power != power;
            counts |= power < kLeast ? 0u : 1u << j;
            e[j] = power_of_two(fminf(fmaxf(power, kLeast), 60.0f));
            e[j] = power != power ? power : e[j];
        }
        return counts;
    };
    bool gave_up = false;                         // (what all of a tile's slices find behind the sums goes with the next ones)
    bool met = false;
    const auto skip = [&](float (&s)[kBlock], float (&de)[kBlock]) __attribute__((always_inline)) {      // (no row of the tile sees the block: its barriers)
        const bool wild = slices_s.add_up(turn, wave, s, gave_up);
        if (wild) { turn ^= 1; return false; }
        slices_de.add_up(turn, wave, de, false);
        turn ^= 1;
        return true;
    };
    const auto score_gradient = [&](float s, float e, float de, int r) __attribute__((always_inline)) {
        const float4 of = record(r);
        float x = s;
        if (!APPROXIMATE && !a.flags.e) {
            x = scoring.cap != 0.0f ? scoring.capped(x) : x;
            if (scoring.slopes) x = scoring.biased(x, of.w, a.first + r / a.group - key);
        }
        return pair.checked(s, x, e, de + of.y * unit);
    };
    if (!careful) {
        Pipe<W4, WHOLE> pipe;
        Look<W4, WHOLE> look_q, look_n;
        careful = !all_blocks<NS, W4, 2>(sight, begin, end, to, first, a.dim, exists, out, met,
            [&](int r0) __attribute__((always_inline)) { pipe.request(queries, r0); look_q.load(queries, r0); look_n.load(grads, r0); },
            [&](int r1, uint32_t sees, bool all) __attribute__((always_inline)) {
                float s[kBlock], de[kBlock], e[kBlock];
                if (!all && __ballot(sees != 0u) == 0ull) {
                    pipe.request(queries, r1 + kBlock); look_q.load(queries, r1 + kBlock); look_n.load(grads, r1 + kBlock);
                    return skip(s, de);
                }
                const Verdict qv = judge(look_q, queries, a.values, 0u);
                Verdict nv{false, false};
                if (APPROXIMATE) nv = judge(look_n, grads, a.values, shift);
                else nv.wild = !all_finite(look_n, grads, a.values);
                look_q.load(queries, r1 + kBlock);
                look_n.load(grads, r1 + kBlock);
                bool wrong = false;
                if constexpr (APPROXIMATE) block_dots<W4, WHOLE>(pipe, queries, r1, grads, r1, qv.zeros, NoLaneZeros{}, k, s);
                else block_dots<W4, WHOLE>(pipe, queries, r1, grads, r1, qv.zeros, k_zeros, k, s);
                const bool wild = slices_s.add_up(turn, wave, s, gave_up || qv.wild || nv.wild);
                if (__builtin_expect(wild, 0)) { turn ^= 1; return false; }      // (others may be reading that buffer)
                uint32_t counts = weigh(s, e, sees, all, r1, wrong);
                if constexpr (APPROXIMATE) {
                    block_dots<W4, WHOLE>(pipe, grads, r1, grads, r1, nv.zeros, NoLaneZeros{}, v, de);
                    without_zeros(zeros, of_v.numbers, de);
                } else {
#pragma unroll
                    for (int j = 0; j < kBlock; ++j) de[j] = 0.0f;
                    uint32_t left = counts;
                    if (__builtin_expect(v_zeros.any, 0)) {
                        const Zeros codes = v_zeros.codes();
                        pipe.rolled(grads, r1, grads, r1, [&](int h, int d, const Piece& x) __attribute__((always_inline)) {
                            dot_lane_power_piece_with_zeros<N>(x, f2u(e[0]), left & 1u ? kPower : 0u, v + d, codes, de[0]);
                            if (h == Pipe<W4, WHOLE>::kPieces - 1) { turned(e); turned(de); left >>= 1; }
                        });
                    } else
                        pipe.block(grads, r1, grads, r1, [&](int j, int d, const Piece& x) __attribute__((always_inline)) {
                            dot_lane_power_piece<N>(x, f2u(e[j]), counts >> j & 1u ? kPower : 0u, v + d, de[j]);
                        });
#pragma unroll
                    for (int j = 0; j < kBlock; ++j) de[j] = over_power(de[j], f2u(e[j]));
                }
                slices_de.add_up(turn, wave, de, false);
                turn ^= 1;
                if (APPROXIMATE) wrong = wrong || too_small(zeros, de, counts, 2.0f);
                const uint32_t counts_e = counts;
                uint32_t small = 0u;
#pragma unroll
                for (int j = 0; j < kBlock; ++j) {
                    de[j] = score_gradient(s[j], e[j], de[j], r1 + j);
                    if (APPROXIMATE) {
                        wrong = wrong || ((counts >> j) & 1u && !(fabsf(de[j]) < 0x1p80f));
                        small |= fabsf(de[j]) < 0x1p-86f ? 1u << j : 0u;
                    }
                }
                gave_up = gave_up || __ballot(wrong) != 0ull;
                if (NS == 1 && __builtin_expect(gave_up, 0)) return false;
                // dv: e (*) dn, dk: da (*) qs
                if constexpr (APPROXIMATE) {
                    block_add<W4, WHOLE>(pipe, grads, r1, queries, r1, nv.zeros, e, scoring.mul_add + shift, counts_e, out[1]);
                    const bool some_small = lift(de, counts, small);
                    block_add<W4, WHOLE>(pipe, queries, r1, queries, r1 + kBlock, qv.zeros, de, scoring.mul_add, counts, out[0], some_small, small);
                } else {
                    pipe.block(grads, r1, queries, r1, [&](int j, int d, const Piece& x) __attribute__((always_inline)) {
                        add_lane_power_piece<N>(x, f2u(e[j]), counts_e >> j & 1u ? kPower : 0u, v + d, out[1] + d);
                    });
                    block_add_power<W4, WHOLE>(pipe, queries, r1, queries, r1 + kBlock, qv.zeros, kPower, de, counts, k, out[0]);
                }
                return true;
            });
        careful = careful || in_team<NS>(gave_up);
        if (!APPROXIMATE)
#pragma unroll
            for (int d = 0; d < W; ++d) { out[0][d] = over_power(out[0][d], k[d] - scoring.mul_add); out[1][d] = over_power(out[1][d], v[d] - scoring.mul_add - shift); }
    }
    gave_up = false;
    if (__builtin_expect(careful, 0)) {
        const Args g = arguments_again();
        unit = fmaxf(unit, 1.0f);
        const float* const of_k = key_of_lane<NS>(g, g.k); const float* const of_v = key_of_lane<NS>(g, g.v);
        load_plain<W4>(first, g.values, k, [&](int d) __attribute__((always_inline)) { return of_k[d]; });
        load_plain<W4>(first, g.values, v, [&](int d) __attribute__((always_inline)) { return of_v[d]; });
        all_blocks<NS, W4, 2>(sight, begin, end, to, first, a.dim, exists, out, met, [](int) {}, [&](int r1, uint32_t sees, bool all) __attribute__((always_inline)) {
            float s[kBlock], de[kBlock], e[kBlock];
            if (!all && __ballot(sees != 0u) == 0ull) { skip(s, de); return true; }
            bool wrong = false;
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
                s[0] = careful_dot<W4>(full, queries.template across<W4>(r1 + j), k);
                turned(s);
            }
            slices_s.add_up(turn, wave, s, false);
            const uint32_t counts = weigh(s, e, sees, all, r1, wrong);
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
                const v4f row = grads.template across<W4>(r1 + j);
                const bool in = (counts >> j) & 1u;
                if (APPROXIMATE || a.flags.a) de[0] = careful_dot<W4>(full, row, v) * unit;
                else {
                    de[0] = 0.0f;
                    each_of_row<W4>(row, [&](int d, float x) __attribute__((always_inline)) { de[0] += exact_term(full, e[0], u2f(plain(v[d])), x * unit); });
                }
                if (APPROXIMATE || a.flags.b) careful_add_row<W4>(full, row, e[0], in, unit, out[1]);
                else
                    each_of_row<W4>(row, [&](int d, float x) __attribute__((always_inline)) {
                        const float term = exact_term(full, u2f(plain(v[d])), e[0], x * unit);
                        out[1][d] += in ? term : 0.0f;
                    });
                turned(de); turned(e);
            }
            slices_de.add_up(turn, wave, de, false);
            turn ^= 1;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) de[j] = de[j] + record(r1 + j).y * unit == 0.0f ? 0.0f : score_gradient(s[j], e[j], de[j], r1 + j);
#pragma unroll 1
            for (int j = 0; j < kBlock; ++j) {
                const v4f row = queries.template across<W4>(r1 + j);
                const bool in = (counts >> j) & 1u;
                if (APPROXIMATE || a.flags.b) careful_add_row<W4>(full, row, de[0], in, 1.0f, out[0]);
                else
                    each_of_row<W4>(row, [&](int d, float x) __attribute__((always_inline)) {
                        const float term = exact_term(full, u2f(plain(k[d])), x, de[0]);
                        out[0][d] += in ? term : 0.0f;
                    });
                turned(de);
            }
            return true;
        });
    }
    if (!a.whole && !met_anything<NS>(a, u, wave, met)) return;
    const float back = 1.0f / unit;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int d = 0; d < W; ++d) out[n][d] *= back;
        store_row<W4>(to[n], first, a.dim, exists, out[n]);
    }
}

template <int NS, int W4, bool WHOLE, bool APPROXIMATE> constexpr Variant dq_of() { return Variant{NS, W4, WHOLE, attention_dq_kernel<NS, W4, WHOLE, APPROXIMATE>}; }
template <int NS, int W4, bool WHOLE, bool APPROXIMATE> constexpr Variant dkv_of() { return Variant{NS, W4, WHOLE, attention_dkv_kernel<NS, W4, WHOLE, APPROXIMATE>}; }

}  // namespace pamatt
