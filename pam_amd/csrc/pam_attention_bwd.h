// The gradients of pam_attention.h.  With the rows' quantities
//   dn_id = dy_id (*) (1 (/) l_i),  dl_i = -sum_d (y_id (/) l_i) (*) dy_id
// of a kernel before (attention_rows_kernel),
//   de_ij = sum_d dn_id (*) v_jd + dl_i,   dx_ij = e_ij (*) de_ij,   da_ij through the cap,
//   dqs_id = sum_j da_ij (*) k_jd,   dk_jd = sum_i da_ij (*) qs_id,   dv_jd = sum_i e_ij (*) dn_id
// for approximate gradients; an exact one weighs the gradient by the slope of the other factor's piece instead.  Two kernels: in the first lanes own
// queries and keys stream by (a, de and dq: three products), in the second lanes own keys and queries stream by (a, de, dk and dv: four).
// Scores and weights are computed again in both; kept, they would be 8 bytes a pair, as long to read as two of the products of 64 values.
// All that is linear in dy is scaled by a power of two: in the first kernel a query's largest |dn| to [1, 2), in the second the largest of a chunk's.
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
    // (integer additions know no NaN; gradients of 2^110 beside a row's largest |dn| count as one)
    __device__ __forceinline__ float checked(float a, float score, float e, float de) const
    {
        const float d = (*this)(a, score, e, de);
        return fabsf(de) < 0x1p110f && e == e ? d : u2f(kQNaN);
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

template <int NS, int W4, bool APPROXIMATE>
__global__ __launch_bounds__(kThreads, W4 > 12 ? 1 : 2) void attention_dq_kernel(Args a)
{
    constexpr int kRows = 64 / NS, W = 4 * W4;
    const Place<NS, W4> here(a.values);
    const Unit u = unit_of(a);
    const int row0 = (u.tile * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64)) * kRows;
    if (row0 >= a.rows) return;
    const int mine = row0 + here.row_in_wave, row = min(mine, a.rows - 1), first = here.slice * W;
    const bool exists = mine < a.rows;
    const int pos = a.first + row / a.group;
    const Scoring scoring(a);
    const PairGrad<APPROXIMATE> pair{scoring, a.flags};
    const Full full{a.off, a.off != 1.0f, 0u - scoring.mul_add, lane_pad(0u)};
    const float4 record = a.records[(long)u.head * a.rows + row];
    const float M = record.x, unit = u2f((uint32_t)(127 - (int)record.z) << 23), dl = record.y * unit, slope = record.w;
    uint32_t q[W], dn[W];
    const long at = ((long)u.head * a.rows + row) * a.dim;
    bool odd = !load_lane<W4>(a.qs + at, first, a.dim, a.values, 0u, scoring.mul_add, lane_pad(0u), q);
    odd = !load_lane<W4>(a.dn + at, first, a.dim, a.values, 0u - ((uint32_t)(int)record.z << 23), scoring.mul_add, lane_pad(0u), dn) || odd;
    odd = odd || !finite(dl);
    const bool careful_lanes = __ballot(odd && M != u2f(kExpo)) != 0ull;
    Sight sight = sight_of_row(a, u.b, row);
    const Stream keys = stream_of(here, a.k.p + (long)u.b * a.k.sb + (long)u.kv * a.k.sh, a.k.st, a.values, a.keys);
    const Stream values = stream_of(here, a.v.p + (long)u.b * a.v.sb + (long)u.kv * a.v.sh, a.v.st, a.values, a.keys);
    float out[W];
#pragma unroll
    for (int d = 0; d < W; ++d) out[d] = 0.0f;
    float* const to = a.out0 + (((long)u.head * a.chunks + u.chunk) * a.rows + row) * a.dim;
    bool folded = false;
    int terms = 0;
    const int begin = max(sight.first / kSpan * kSpan, u.chunk * a.chunk), end = min(min(sight.last, a.keys), (u.chunk + 1) * a.chunk);
#pragma unroll 1
    for (int j0 = begin; j0 < end; j0 += kSpan) {
        const uint64_t see = sight.span(j0);
        if (__ballot(see != 0ull) == 0ull) continue;
        const bool all = __ballot(see != ~0ull) == 0ull;
        if (terms >= kLink) {
            row_in_memory<W4>(to, first, a.dim, exists, [&](int n, v4f& x) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = (folded ? x[i] : 0.0f) + out[4 * n + i];
            });
#pragma unroll
            for (int d = 0; d < W; ++d) out[d] = 0.0f;
            folded = true; terms = 0;
        }
        terms += kSpan;
        v4f kr[kBlock], vr[kBlock];
#pragma unroll 1
        for (int i0 = 0; i0 < kSpan; i0 += kBlock) {
            const uint32_t sees = (uint32_t)(see >> i0) & 0xffu;
            if (!all && __ballot(sees != 0u) == 0ull) continue;
            keys.rows(j0 + i0, kr);
            values.rows(j0 + i0, vr);
            keys.pad(0u, kr);
            const Verdict kv = judge(here.streaming, 0u, kr);
            float s[kBlock], de[kBlock], e[kBlock];
            block_dots<NS, W4>(full, careful_lanes || kv.careful, kv.zero, 1.0f, kr, q, s);
            uint32_t counts = 0u;
            bool wrong = false;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                float power = scoring.exponent(s[j], slope, pos - (j0 + i0 + j)) - M;
                if (!all) power = (sees >> j) & 1u ? power : 2.0f * kLeast;
                wrong = wrong || power != power;
                counts |= power < kLeast ? 0u : 1u << j;          // (what is no number counts)
                e[j] = power_of_two(fminf(fmaxf(power, kLeast), 60.0f));
                e[j] = power != power ? power : e[j];
            }
            values.pad(0u, vr);
            const Verdict vv = judge(here.streaming, 0u, vr);
            if (APPROXIMATE || a.flags.a) {
                block_dots<NS, W4>(full, careful_lanes || vv.careful, vv.zero, 1.0f, vr, dn, de);
            } else {
#pragma unroll 1
                for (int j = 0; j < kBlock; ++j) {
                    float sum = 0.0f;
                    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t m = (uint32_t)anew((int)dn[4 * n.value + i]);
                            const bool is_zero = m - scoring.mul_add == kStandIn;
                            const float term = exact_term(full, e[0], u2f(from_lane<decltype(n)::value>(vr[0][i])), m == full.pad || is_zero ? 0.0f : u2f(m + full.raw));
                            sum += term;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    });
                    de[0] = (vv.zero >> j) & 1u ? 0.0f : over_slices<NS>(sum);
                    turned(vr); turned(e); turned(de);
                }
            }
            const bool small = careful_lanes || vv.careful;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                float x = s[j];
                if (!APPROXIMATE && !a.flags.e) {                  // (the score as log2 e multiplies it)
                    x = scoring.cap != 0.0f ? scoring.capped(x) : x;
                    if (scoring.slopes) x = scoring.biased(x, slope, pos - (j0 + i0 + j));
                }
                de[j] = pair.checked(s[j], x, e[j], de[j] + dl);
                // (less than 2^-86 is nothing beside |dn| of 1 and values of at least 2^-40; with smaller ones it may be all there is)
                const bool tiny = fabsf(de[j]) < 0x1p-86f;
                wrong = wrong || ((counts >> j) & 1u && (!(fabsf(de[j]) < 0x1p80f) || (small && tiny)));
                counts &= tiny && !small ? ~(1u << j) : ~0u;
            }
            const bool careful = careful_lanes || kv.careful || __ballot(wrong) != 0ull;
            if (APPROXIMATE || a.flags.a) {
                block_add<W4>(full, careful, kv.zero, 1.0f, kr, de, scoring.mul_add, counts, out);
            } else {
#pragma unroll 1
                for (int j = 0; j < kBlock; ++j) {
                    const bool in = ((counts & ~kv.zero) >> j) & 1u;
                    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t m = (uint32_t)anew((int)q[4 * n.value + i]);
                            const float term = exact_term(full, m == full.pad ? 1.0f : u2f(m + full.raw), u2f(from_lane<decltype(n)::value>(kr[0][i])), de[0]);
                            out[4 * n.value + i] += in ? term : 0.0f;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    });
                    turned(kr); turned(de);
                }
            }
        }
    }
    if (folded)
        row_in_memory<W4>(to, first, a.dim, exists, [&](int n, v4f& x) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[4 * n + i] += x[i];
        });
    const float back = 1.0f / unit;
#pragma unroll
    for (int d = 0; d < W; ++d) out[d] *= back;
    store_row<W4>(to, first, a.dim, exists, out);
}

// What a key's lane sees: the rows of its head's queries.
__device__ __forceinline__ Sight sight_of_key(const Args& a, int b, int key)
{
    const long at = (long)key - a.first, g = a.group, rows = a.rows;
    const auto held = [&](long tokens) { return (int)max(0l, min(tokens * g, rows)); };
    Sight s;
    s.low = a.causal ? held(at) : a.window ? held(at - a.window + 1) : 0;
    s.high = a.window ? held(at + a.window) : a.rows;
    s.before = a.prefix && key < a.prefix[b] ? a.rows : 0;
    s.with_documents = a.documents != nullptr;
    s.of_streamed = a.documents ? a.documents + (long)b * a.keys + a.first : nullptr; s.per = a.group;
    s.mine = a.documents ? a.documents[(long)b * a.keys + key] : 0;
    s.close();
    return s;
}

template <int NS, int W4, bool APPROXIMATE>
__global__ __launch_bounds__(kThreads, W4 > 8 ? 1 : 2) void attention_dkv_kernel(Args a)
{
    constexpr int kRows = 64 / NS, W = 4 * W4;
    const Place<NS, W4> here(a.values);
    Unit u = unit_of(a);
    u.tile = a.tiles - 1 - u.tile;                // (the first keys have most queries where the order is causal)
    const int key0 = (u.tile * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64)) * kRows;
    if (key0 >= a.keys) return;
    const int mine = key0 + here.row_in_wave, key = min(mine, a.keys - 1), first = here.slice * W;
    const bool exists = mine < a.keys;
    const Scoring scoring(a);
    const PairGrad<APPROXIMATE> pair{scoring, a.flags};
    typedef const __attribute__((address_space(4))) float4* Records;
    const float4* const all_records = a.records + (long)u.head * a.rows;
    const int chunk_begin = u.chunk * a.chunk, chunk_end = min(a.rows, chunk_begin + a.chunk);
    // the largest |dn| of the chunk's rows is scaled to [1, 2)
    int most = -86;
    for (int r = chunk_begin + here.lane; r < chunk_end; r += 64) most = max(most, (int)all_records[r].z);
#pragma unroll
    for (int s = 1; s < 64; s *= 2) most = max(most, __shfl_xor(most, s, 64));
    most = __builtin_amdgcn_readfirstlane(most);
    const uint32_t shift = 0u - ((uint32_t)most << 23);
    const float unit = u2f((uint32_t)(127 - most) << 23);
    const Full full_q{a.off, a.off != 1.0f, 0u - scoring.mul_add, lane_pad(0u)}, full_n{a.off, a.off != 1.0f, 0u - scoring.mul_add - shift, lane_pad(shift)};
    uint32_t k[W], v[W];
    bool odd = !load_lane<W4>(a.k.p + (long)u.b * a.k.sb + (long)key * a.k.st + (long)u.kv * a.k.sh, first, a.dim, a.values, 0u, scoring.mul_add, lane_pad(0u), k);
    odd = !load_lane<W4>(a.v.p + (long)u.b * a.v.sb + (long)key * a.v.st + (long)u.kv * a.v.sh, first, a.dim, a.values, 0u, scoring.mul_add + shift, lane_pad(shift), v) || odd;
    const bool careful_lanes = __ballot(odd) != 0ull;
    Sight sight = sight_of_key(a, u.b, key);
    const Stream queries = stream_of(here, a.qs + (long)u.head * a.rows * a.dim, a.dim, a.values, a.rows);
    const Stream grads = stream_of(here, a.dn + (long)u.head * a.rows * a.dim, a.dim, a.values, a.rows);
    float dk[W], dv[W];
#pragma unroll
    for (int d = 0; d < W; ++d) dk[d] = dv[d] = 0.0f;
    const long to = (((long)u.head * a.chunks + u.chunk) * a.keys + key) * a.dim;
    bool folded = false;
    int terms = 0;
    const int begin = max(sight.first / kSpan * kSpan, chunk_begin), end = min(min(sight.last, a.rows), chunk_begin + a.chunk);
#pragma unroll 1
    for (int r0 = begin; r0 < end; r0 += kSpan) {
        const uint64_t see = sight.span(r0);
        if (__ballot(see != 0ull) == 0ull) continue;
        const bool all = __ballot(see != ~0ull) == 0ull;
        if (terms >= kLink) {
            row_in_memory<W4>(a.out0 + to, first, a.dim, exists, [&](int n, v4f& x) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = (folded ? x[i] : 0.0f) + dk[4 * n + i];
            });
            row_in_memory<W4>(a.out1 + to, first, a.dim, exists, [&](int n, v4f& x) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = (folded ? x[i] : 0.0f) + dv[4 * n + i];
            });
#pragma unroll
            for (int d = 0; d < W; ++d) dk[d] = dv[d] = 0.0f;
            folded = true; terms = 0;
        }
        terms += kSpan;
        v4f qr[kBlock], nr[kBlock];
#pragma unroll 1
        for (int i0 = 0; i0 < kSpan; i0 += kBlock) {
            const uint32_t sees = (uint32_t)(see >> i0) & 0xffu;
            if (!all && __ballot(sees != 0u) == 0ull) continue;
            queries.rows(r0 + i0, qr);
            grads.rows(r0 + i0, nr);
            float4 record[kBlock];
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                const Records from = (Records)(all_records + min(r0 + i0 + j, a.rows - 1));
                record[j] = make_float4(from->x, from->y, from->z, from->w);
            }
            queries.pad(0u, qr);
            const Verdict qv = judge(here.streaming, 0u, qr);
            float s[kBlock], de[kBlock], e[kBlock];
            block_dots<NS, W4>(full_q, careful_lanes || qv.careful, qv.zero, 1.0f, qr, k, s);
            uint32_t counts = 0u;
            bool wrong = false;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                const int pos = a.first + (r0 + i0 + j) / a.group;
                float power = scoring.exponent(s[j], record[j].w, pos - key) - record[j].x;
                if (!all) power = (sees >> j) & 1u ? power : 2.0f * kLeast;
                wrong = wrong || power != power;
                counts |= power < kLeast ? 0u : 1u << j;
                e[j] = power_of_two(fminf(fmaxf(power, kLeast), 60.0f));
                e[j] = power != power ? power : e[j];
            }
            grads.pad(shift, nr);
            const Verdict nv = judge(here.streaming, shift, nr);
            const bool weights_wrong = __ballot(wrong) != 0ull;
            if (APPROXIMATE || a.flags.a) {
                block_dots<NS, W4>(full_n, careful_lanes || nv.careful, nv.zero, unit, nr, v, de);
            } else {
#pragma unroll 1
                for (int j = 0; j < kBlock; ++j) {
                    float sum = 0.0f;
                    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t m = (uint32_t)anew((int)v[4 * n.value + i]);
                            const float other = m == full_n.pad || m - scoring.mul_add - shift == kStandIn ? 0.0f : u2f(m + full_n.raw);
                            sum += exact_term(full_n, e[0], other, u2f(from_lane<decltype(n)::value>(nr[0][i])) * unit);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    });
                    de[0] = (nv.zero >> j) & 1u ? 0.0f : over_slices<NS>(sum);
                    turned(nr); turned(e); turned(de);
                }
            }
            // dv: e (*) dn
            if (APPROXIMATE || a.flags.b) {
                block_add<W4>(full_n, careful_lanes || nv.careful || weights_wrong, nv.zero, unit, nr, e, scoring.mul_add + shift, counts, dv);
            } else {
#pragma unroll 1
                for (int j = 0; j < kBlock; ++j) {
                    const bool in = ((counts & ~nv.zero) >> j) & 1u;
                    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t m = (uint32_t)anew((int)v[4 * n.value + i]);
                            const float own = m == full_n.pad ? 1.0f : u2f(m + full_n.raw);
                            const float term = exact_term(full_n, own, e[0], u2f(from_lane<decltype(n)::value>(nr[0][i])) * unit);
                            dv[4 * n.value + i] += in ? term : 0.0f;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    });
                    turned(nr); turned(e);
                }
            }
            const bool small = careful_lanes || nv.careful;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                float x = s[j];
                if (!APPROXIMATE && !a.flags.e) {
                    x = scoring.cap != 0.0f ? scoring.capped(x) : x;
                    if (scoring.slopes) x = scoring.biased(x, record[j].w, a.first + (r0 + i0 + j) / a.group - key);
                }
                de[j] = pair.checked(s[j], x, e[j], de[j] + record[j].y * unit);
                // (less than 2^-86 is nothing beside |dn| of 1 and values of at least 2^-40; with smaller ones it may be all there is)
                const bool tiny = fabsf(de[j]) < 0x1p-86f;
                wrong = wrong || ((counts >> j) & 1u && (!(fabsf(de[j]) < 0x1p80f) || (small && tiny)));
                counts &= tiny && !small ? ~(1u << j) : ~0u;
            }
            // dk: da (*) qs
            if (APPROXIMATE || a.flags.b) {
                block_add<W4>(full_q, careful_lanes || qv.careful || __ballot(wrong) != 0ull, qv.zero, 1.0f, qr, de, scoring.mul_add, counts, dk);
            } else {
#pragma unroll 1
                for (int j = 0; j < kBlock; ++j) {
                    const bool in = ((counts & ~qv.zero) >> j) & 1u;
                    each<0, W4>([&](auto n) __attribute__((always_inline)) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t m = (uint32_t)anew((int)k[4 * n.value + i]);
                            const float own = m == full_q.pad ? 1.0f : u2f(m + full_q.raw);
                            const float term = exact_term(full_q, own, u2f(from_lane<decltype(n)::value>(qr[0][i])), de[0]);
                            dk[4 * n.value + i] += in ? term : 0.0f;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    });
                    turned(qr); turned(de);
                }
            }
        }
    }
    if (folded) {
        row_in_memory<W4>(a.out0 + to, first, a.dim, exists, [&](int n, v4f& x) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) dk[4 * n + i] += x[i];
        });
        row_in_memory<W4>(a.out1 + to, first, a.dim, exists, [&](int n, v4f& x) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) dv[4 * n + i] += x[i];
        });
    }
    const float back = 1.0f / unit;
#pragma unroll
    for (int d = 0; d < W; ++d) { dk[d] *= back; dv[d] *= back; }
    store_row<W4>(a.out0 + to, first, a.dim, exists, dk);
    store_row<W4>(a.out1 + to, first, a.dim, exists, dv);
}

}  // namespace pamatt
