// The rotation of queries' and keys' heads by their positions, after an optional norm of each head, and its gradient.
//
// Bound by memory: 8 bytes a value forward, 12 backward.  4 x 4096 tokens of 16 + 4 heads of 128, normed: forward 65 us (5.2 TB/s, what a
// large copy reaches), forward and gradients with both weights' 180 us (160 at that rate).  A head is taken by a group of 2 ... 64 lanes, one unit each: four
// pairs of a rotated part (two 128-bit loads, `rotated / 2` apart or side by side) or four values of the rest, so that a
// pair's two values meet in one lane and the only exchange is the norm's sum over the group.  cos and sin are read per head; the heads of a
// token follow each other, so that all but the first find them in the cache next to the compute unit.  A work-group stays with
// one of the two tensors.  The backward pass runs as many work-groups as are resident, each over a share of the heads, and keeps
// the weight's gradient of its columns in registers; one row of sums per work-group is left to the column sums (one term per value
// written and read back instead made the pass a third longer in bytes).
// The chain of primitives is computed as one integer addition each (Raw), behind tests that what goes in is of ordinary size; a
// wavefront that meets a zero, an infinity or an extreme exponent computes its heads by the checked functions, with the same results.
// Heads that do not come in fours, or of more than 64 units, take a wavefront each by the checked functions.
#include <algorithm>

#include "../../include/pam_hip_extra.h"
#include "pam_activation.h"
#include "pam_common.h"

using namespace pamdev;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

struct PartArgs {
    const float* x; long x_sb, x_st, x_sh;
    const float* dy; long dy_sb, dy_st, dy_sh;
    const float* weight;
    float* y;
    float* sums;                                  // backward: [work-groups of the part][dim] of the weight's gradient, or null
    uint32_t rows, heads;                         // heads of all tokens (at most 2^30), of one
    int groups;                                   // work-groups of the part
};
struct RotaryArgs {
    PartArgs part[2];
    const float* cos; const float* sin; long table_rows;
    const long long* positions; long p_sb, p_st;
    uint32_t tokens;
    int dim, half, interleaved, lanes;            // lanes: of a group
    int first_group;                              // of the launch, of all work-groups (see launch())
    float eps, off; bool has_off;
    ApproxFlags flags;
};

// Windows of pam_activation.h on what goes into a chain of integer additions (Raw).
// With x in 2^[-20, 20), its root in 2^[-14, 21), w in 2^[-10, 10), dz in 2^[-44, 20): x / root in 2^[-42, 35), x / root / root in
// 2^[-64, 50), dz w in 2^[-55, 31), their product in 2^[-120, 82); the offset, between 3/4 and 3/2, is in at most five factors of it.  Heads
// without a norm: x or dy in 2^[-60, 60), times a table's value.
template <class W> __device__ __forceinline__ void see(W& window, const v4f& v) { window.see(v[0]); window.see(v[1]); window.see(v[2]); window.see(v[3]); }
typedef Window<-20, 20> WindowX;
typedef Window<-14, 21> WindowRoot;
typedef Window<-10, 10> WindowW;
typedef Window<-44, 20> WindowGrad;
typedef Window<-40, 4> WindowTable;
typedef Window<-60, 60> WindowPlain;
typedef Window<-80, 60> WindowSquare;             // the gradient for x (*) x: times x it is in 2^[-101, 81)
typedef Window<-50, 50> WindowRootGrad;           // between it and the root's there are the root, v in 2^[-28, 42) and the count
typedef Window<-24, 8> WindowLog;                 // log2 v: not zero

// A head: its values, the rows of the tables.
struct Head {
    const float* x; const float* dy; float* y;
    const float* cos; const float* sin;           // null: no such position
};
__device__ __forceinline__ Head find_head(const RotaryArgs& a, const PartArgs& p, uint32_t row)
{
    Head h;
    const uint32_t token = row / p.heads, at = row - token * p.heads, b = token / a.tokens, t = token - b * a.tokens;
    h.x = p.x + (long)b * p.x_sb + (long)t * p.x_st + (long)at * p.x_sh;
    h.dy = p.dy ? p.dy + (long)b * p.dy_sb + (long)t * p.dy_st + (long)at * p.dy_sh : nullptr;
    h.y = p.y + (long)row * a.dim;
    const long long pos = a.positions ? a.positions[(long)b * a.p_sb + (long)t * a.p_st] : (long long)t;
    const bool there = pos >= 0 && pos < a.table_rows;
    h.cos = there ? a.cos + pos * a.half : nullptr;
    h.sin = there ? a.sin + pos * a.half : nullptr;
    return h;
}

__device__ __forceinline__ float group_sum(float v, int lanes)
{
    for (int s = lanes / 2; s >= 1; s >>= 1) v += __shfl_xor(v, s, 64);
    return v;
}

// mean(x (*) x) + eps and its root, from the sum
struct Root { float sum, variance, root; };
__device__ __forceinline__ Root root_of(const RotaryArgs& a, float sum)
{
    Root r;
    r.sum = sum;
    r.variance = pad_div_off(sum, (float)a.dim, a.off, a.has_off) + a.eps;
    r.root = pow_half(r.variance, a.off, a.has_off);
    return r;
}
// The gradient for every x (*) x from that of the root: pow(v, 0.5) = 2^(log2(v) (*) 0.5), zero where v is zero; then the mean's quotient.
__device__ __forceinline__ float square_grad(const RotaryArgs& a, const ApproxFlags& f, const Root& r, float droot)
{
    const float off = a.off; const bool has_off = a.has_off;
    const float l = log2_entry(r.variance, off, has_off), t = pam_mul_off(l, 0.5f, off, has_off);
    const float dt = exp2_grad(t, exp2_entry(t, off, has_off), r.variance == 0.0f ? 0.0f : droot, f.e, off, has_off);
    const float dl = mul_grad(l, 0.5f, dt, f.a, off, has_off);
    const float dv = f.e ? pad_div_off(pad_div_off(dl, r.variance, off, has_off), kActLn2, off, has_off) : log2_entry_bwd(r.variance, dl, off, has_off);
    return div_grad_a(r.sum, (float)a.dim, dv, f.a, off, has_off);
}

// ---------------------------------------------------------------- value by value, by the checked functions

// The lane's part of a head: pair(q) for its pairs, rest(i) for its values behind the rotated part.  GROUPED: those of its unit (below),
// otherwise every `lanes`th.  Sums over them are kept in two parts as the groups' are (Sums), so that a head has the same sums, bit for bit,
// whichever way its wavefront takes.
template <bool GROUPED, class Pair, class Rest>
__device__ __forceinline__ void each_value(const RotaryArgs& a, int lane, int lanes, Pair pair, Rest rest)
{
    const int turning = a.half / 4, behind = 2 * a.half + (GROUPED ? 4 * (lane - turning) : lane);
    if (!GROUPED || lane < turning) {
        const int end = GROUPED ? 4 * lane + 4 : a.half;
#pragma unroll 1
        for (int q = GROUPED ? 4 * lane : lane; q < end; q += GROUPED ? 1 : lanes) pair(q);
    }
    if (!GROUPED || lane >= turning) {
        const int end = GROUPED ? min(behind + 4, a.dim) : a.dim;
#pragma unroll 1
        for (int i = behind; i < end; i += GROUPED ? 1 : lanes) rest(i);
    }
}
struct Sums {
    float part[2] = {0.0f, 0.0f};
    __device__ __forceinline__ void add(bool second, float v) { if (second) part[1] += v; else part[0] += v; }
    __device__ __forceinline__ float total(int lanes) const { return group_sum(part[0] + part[1], lanes); }
};
// Where a pair's values are, and the part of a sum that they are in: a unit's vectors hold firsts and seconds, or two pairs each.
struct Pair {
    int i, j; bool part_i, part_j;
    __device__ __forceinline__ Pair(const RotaryArgs& a, int q)
        : i(a.interleaved ? 2 * q : q), j(a.interleaved ? 2 * q + 1 : q + a.half), part_i(a.interleaved && (q & 2)), part_j(!a.interleaved || (q & 2)) {}
};

template <bool GROUPED>
__device__ __forceinline__ Root head_root(const RotaryArgs& a, const float* x, int lane, int lanes)
{
    Sums sum;
    auto square = [&](bool second, float v) { sum.add(second, pam_mul_off(v, v, a.off, a.has_off)); };
    each_value<GROUPED>(a, lane, lanes,
        [&](int q) { const Pair p(a, q); square(p.part_i, x[p.i]); square(p.part_j, x[p.j]); },
        [&](int i) { square(false, x[i]); });
    return root_of(a, sum.total(lanes));
}

template <bool GROUPED>
__device__ __forceinline__ void forward_by_value(const RotaryArgs& a, const float* weight, const Head& h, int lane, int lanes, bool store)
{
    const float root = weight ? head_root<GROUPED>(a, h.x, lane, lanes).root : 1.0f;
    if (!store) return;
    auto value = [&](int i) { return weight ? pam_mul_off(pad_div_off(h.x[i], root, a.off, a.has_off), weight[i], a.off, a.has_off) : h.x[i]; };
    each_value<GROUPED>(a, lane, lanes,
        [&](int q) {
            const Pair p(a, q);
            const float z1 = value(p.i), z2 = value(p.j);
            const float c = h.cos ? h.cos[q] : u2f(kQNaN), s = h.sin ? h.sin[q] : u2f(kQNaN);
            h.y[p.i] = pam_mul_off(z1, c, a.off, a.has_off) - pam_mul_off(z2, s, a.off, a.has_off);
            h.y[p.j] = pam_mul_off(z2, c, a.off, a.has_off) + pam_mul_off(z1, s, a.off, a.has_off);
        },
        [&](int i) { h.y[i] = value(i); });
}

// term(i, t): the weight's gradient gets t at value i from this head.  APPROXIMATE: all slopes are.
template <bool GROUPED, bool APPROXIMATE, class Term>
__device__ __forceinline__ void backward_by_value(const RotaryArgs& a, const float* weight, const Head& h, int lane, int lanes, bool store, Term term)
{
    const float off = a.off;
    const bool has_off = a.has_off, norm = weight != nullptr;
    const ApproxFlags f = APPROXIMATE ? ApproxFlags{true, true, true} : a.flags;
    const Root r = norm ? head_root<GROUPED>(a, h.x, lane, lanes) : Root{0.0f, 0.0f, 1.0f};
    Sums droot;
    float dsquare = 0.0f;
    // first the weight's gradient and the root's, then x's (one loop over both, so that the code is there once)
#pragma unroll 1
    for (int round = norm ? 0 : 1; round < 2; ++round) {
        auto take = [&](int i, bool second, float x, float n, float dz) {
            const float dn = norm ? mul_grad(n, weight[i], dz, f.a, off, has_off) : dz;
            if (round == 0) {
                if (store) term(i, mul_grad(weight[i], n, dz, f.b, off, has_off));
                droot.add(second, div_grad_b(x, r.root, dn, f.b, off, has_off));
            } else if (store) {
                h.y[i] = norm ? div_grad_a(x, r.root, dn, f.a, off, has_off) + (mul_grad(x, x, dsquare, f.a, off, has_off) + mul_grad(x, x, dsquare, f.b, off, has_off)) : dn;
            }
        };
        each_value<GROUPED>(a, lane, lanes,
            [&](int q) {
                const Pair p(a, q);
                const float x1 = h.x[p.i], x2 = h.x[p.j], d1 = h.dy[p.i], d2 = h.dy[p.j];
                const float n1 = norm ? pad_div_off(x1, r.root, off, has_off) : x1, n2 = norm ? pad_div_off(x2, r.root, off, has_off) : x2;
                const float z1 = norm ? pam_mul_off(n1, weight[p.i], off, has_off) : x1, z2 = norm ? pam_mul_off(n2, weight[p.j], off, has_off) : x2;
                const float c = h.cos ? h.cos[q] : u2f(kQNaN), s = h.sin ? h.sin[q] : u2f(kQNaN);
                take(p.i, p.part_i, x1, n1, mul_grad(z1, c, d1, f.a, off, has_off) + mul_grad(z1, s, d2, f.a, off, has_off));
                take(p.j, p.part_j, x2, n2, mul_grad(z2, c, d2, f.a, off, has_off) + mul_grad(z2, s, -d1, f.a, off, has_off));
            },
            [&](int i) {
                const float x = h.x[i];
                take(i, false, x, norm ? pad_div_off(x, r.root, off, has_off) : x, h.dy[i]);
            });
        if (round == 0) dsquare = square_grad(a, f, r, droot.total(lanes));
    }
}

// ---------------------------------------------------------------- a group of lanes per head

// What a lane has of a head: four pairs, or four values that are not rotated (in u[0]), or nothing.
struct Unit {
    bool there, rotates;
    int first, second;                            // where its vectors begin
    int table;                                    // ... in the tables' rows
    __device__ __forceinline__ Unit(const RotaryArgs& a, int unit)
    {
        const int turning = a.half / 4, rest = (a.dim - 2 * a.half) / 4;
        there = unit < turning + rest;
        rotates = unit < turning;
        table = min(unit, max(turning - 1, 0)) * 4;
        first = rotates ? (a.interleaved ? 2 : 1) * table : 2 * a.half + (there ? unit - turning : 0) * 4;
        second = rotates ? (a.interleaved ? first + 4 : first + a.half) : first;
        if (!there) first = second = 0;
    }
};
template <bool INTERLEAVED> __device__ __forceinline__ void to_pairs(const v4f (&u)[2], float (&z1)[4], float (&z2)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        z1[i] = INTERLEAVED ? u[i / 2][2 * (i % 2)] : u[0][i];
        z2[i] = INTERLEAVED ? u[i / 2][2 * (i % 2) + 1] : u[1][i];
    }
}
template <bool INTERLEAVED> __device__ __forceinline__ void from_pairs(const float (&z1)[4], const float (&z2)[4], v4f (&u)[2])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (INTERLEAVED) { u[i / 2][2 * (i % 2)] = z1[i]; u[i / 2][2 * (i % 2) + 1] = z2[i]; }
        else { u[0][i] = z1[i]; u[1][i] = z2[i]; }
    }
}
__device__ __forceinline__ void load_unit(const float* base, const Unit& at, v4f (&u)[2])
{
    u[0] = *reinterpret_cast<const v4f_any*>(base + at.first);
    u[1] = *reinterpret_cast<const v4f_any*>(base + at.second);
}
__device__ __forceinline__ void store_unit(float* base, const Unit& at, const v4f (&u)[2])
{
    if (at.there) __builtin_nontemporal_store(u[0], reinterpret_cast<v4f_any*>(base + at.first));
    if (at.rotates) __builtin_nontemporal_store(u[1], reinterpret_cast<v4f_any*>(base + at.second));
}
__device__ __forceinline__ void load_table(const Head& h, const Unit& at, bool any, v4f& c, v4f& s)
{
    const float nan = u2f(kQNaN);
    c = s = v4f{nan, nan, nan, nan};
    if (any && h.cos) { c = *reinterpret_cast<const v4f_any*>(h.cos + at.table); s = *reinterpret_cast<const v4f_any*>(h.sin + at.table); }
}

__device__ __forceinline__ float square_sum(const Raw& ar, const RotaryArgs& a, const Unit& at, const v4f (&x)[2])
{
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[v] += ar.mul(x[v][i], x[v][i]);
    return group_sum((at.there ? sum[0] : 0.0f) + (at.rotates ? sum[1] : 0.0f), a.lanes);
}

// root_of and square_grad as integer additions; `held`: all in their windows.
struct RawRoot { float sum, variance, log, half, root; bool held; };
__device__ __forceinline__ RawRoot raw_root_of(const Raw& ar, const RotaryArgs& a, float sum)
{
    RawRoot r;
    r.sum = sum;
    r.variance = ar.div(sum, (float)a.dim) + a.eps;
    r.log = ar.div((float)((int)f2u(r.variance) - (int)kBias) * 0x1p-23f, 1.0f);
    r.half = ar.mul(r.log, 0.5f);
    r.root = ar.exp2(r.half);
    WindowLog log;
    WindowRoot root;
    WindowPlain variance;
    log.see(r.log); root.see(r.root); variance.see(r.variance);
    r.held = log.held() && root.held() && variance.held() && r.variance > 0.0f;
    return r;
}
template <bool APPROXIMATE>
__device__ __forceinline__ float raw_square_grad(const RawGrad<APPROXIMATE>& ar, const RotaryArgs& a, const RawRoot& r, float droot)
{
    const ApproxFlags f = a.flags;
    const float dl = ar.of_mul(r.log, 0.5f, ar.of_exp2(r.half, r.root, droot, f.e), f.a);
    return ar.of_dividend(r.sum, ar.div(1.0f, (float)a.dim), ar.of_log2(r.variance, dl, f.e), f.a);
}

// The token at position 0 has sines of zero.  Its products with them are left out; the tests see one in their place.
__device__ __forceinline__ bool stands_still(v4f& s)
{
    const bool still = ((f2u(s[0]) | f2u(s[1]) | f2u(s[2]) | f2u(s[3])) << 1) == 0u;
    if (still) s = v4f{1.0f, 1.0f, 1.0f, 1.0f};
    return still;
}

// Whether `here` is true in all lanes of the group.
__device__ __forceinline__ bool in_group(bool here, int lanes)
{
    const uint64_t group = (lanes == 64 ? ~0ull : (1ull << lanes) - 1ull) << (threadIdx.x % 64 & ~(lanes - 1));
    return (__ballot(here) & group) == group;
}
__device__ __forceinline__ bool all_zero(const v4f (&u)[2])
{
    uint32_t any = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) any |= f2u(u[i / 4][i % 4]);
    return (any << 1) == 0u;
}

// What a lane knows of the head's weight: its values, and whether they are in their window.
struct Weight { v4f w[2]; bool norm, held; };
__device__ __forceinline__ Weight load_weight(const float* weight, const Unit& at)
{
    Weight r{{}, weight != nullptr, true};
    if (!r.norm) return r;
    load_unit(weight, at, r.w);
    WindowW window;
    see(window, r.w[0]); see(window, r.w[1]);
    r.held = window.held();
    return r;
}
// y of a lane's unit; false if a value of the wavefront is outside its window, and y is then not computed.
template <bool INTERLEAVED>
__device__ __forceinline__ bool forward_head(const RotaryArgs& a, const Unit& at, const v4f (&x)[2], const Weight& w, const v4f& c, v4f s, v4f (&y)[2])
{
    const Raw ar(a.off);
    const bool still = stands_still(s);
    WindowTable tables;
    if (at.rotates) { see(tables, c); see(tables, s); }
    bool held = usual_offset(a.off) && tables.held() && w.held;
    y[0] = x[0]; y[1] = x[1];
    if (w.norm) {
        WindowX seen;
        see(seen, x[0]); see(seen, x[1]);
        const RawRoot r = raw_root_of(ar, a, square_sum(ar, a, at, x));
        held = held && seen.held() && r.held;
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[v][i] = ar.mul(ar.div(x[v][i], r.root), w.w[v][i]);
    } else if (at.rotates) {
        WindowPlain seen;
        see(seen, x[0]); see(seen, x[1]);
        held = held && seen.held();
    }
    if (at.rotates) {
        float z1[4], z2[4], y1[4], y2[4];
        to_pairs<INTERLEAVED>(y, z1, z2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y1[i] = ar.mul(z1[i], c[i]) - (still ? 0.0f : ar.mul(z2[i], s[i]));
            y2[i] = ar.mul(z2[i], c[i]) + (still ? 0.0f : ar.mul(z1[i], s[i]));
        }
        from_pairs<INTERLEAVED>(y1, y2, y);
    }
    return __ballot(!held) == 0ull;
}

template <bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a)
{
    const int block = a.first_group + (int)blockIdx.x;
    const bool other = block >= a.part[0].groups;
    const PartArgs& p = other ? a.part[1] : a.part[0];
    const int lanes = a.lanes;
    const Unit at(a, threadIdx.x & (lanes - 1));
    // (lanes of heads past the end go along with the last head, for the sums over a group, and store nothing)
    const uint32_t mine = (uint32_t)(block - (other ? a.part[0].groups : 0)) * (kThreads / lanes) + threadIdx.x / lanes;
    const Head h = find_head(a, p, min(mine, p.rows - 1));
    v4f x[2], c, s, y[2];
    load_unit(h.x, at, x);
    const Weight w = load_weight(p.weight, at);
    load_table(h, at, a.half > 0, c, s);
    if (!forward_head<INTERLEAVED>(a, at, x, w, c, s, y)) forward_by_value<true>(a, p.weight, h, threadIdx.x & (lanes - 1), lanes, mine < p.rows);
    else if (mine < p.rows) store_unit(h.y, at, y);
}

// The gradient; APPROXIMATE: all slopes are, so that z is not needed.  term: the weight's gradient.  False as above.
template <bool INTERLEAVED, bool APPROXIMATE>
__device__ __forceinline__ bool backward_head(const RotaryArgs& a, const Unit& at, const v4f (&x)[2], v4f (&d)[2], const Weight& w, const v4f& c, v4f s,
                                              v4f (&dx)[2], v4f (&term)[2])
{
    const RawGrad<APPROXIMATE> ar(a.off);
    const ApproxFlags f = a.flags;
    // (a token that the loss leaves out: behind a norm the gradients of such a head are zeros, the tests see ones in their place)
    const bool nothing = w.norm && in_group(all_zero(d), a.lanes);
    if (nothing) d[0] = d[1] = v4f{1.0f, 1.0f, 1.0f, 1.0f};
    const bool still = stands_still(s);
    bool held = usual_offset(a.off) && w.held;
    RawRoot r{};
    v4f z[2] = {x[0], x[1]};
    if (w.norm) {
        WindowX seen;
        see(seen, x[0]); see(seen, x[1]);
        r = raw_root_of(ar, a, square_sum(ar, a, at, x));
        held = held && seen.held() && r.held;
        if (!APPROXIMATE)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) z[v][i] = ar.mul(ar.div(x[v][i], r.root), w.w[v][i]);
    }
    dx[0] = d[0]; dx[1] = d[1];
    if (at.rotates) {
        WindowTable tables;
        WindowPlain seen;
        see(tables, c); see(tables, s); see(seen, d[0]); see(seen, d[1]);
        if (!APPROXIMATE && !w.norm) { see(seen, x[0]); see(seen, x[1]); }
        held = held && tables.held() && seen.held();
        float d1[4], d2[4], z1[4], z2[4], o1[4], o2[4];
        to_pairs<INTERLEAVED>(d, d1, d2);
        to_pairs<INTERLEAVED>(z, z1, z2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o1[i] = ar.of_mul(z1[i], c[i], d1[i], f.a) + (still ? 0.0f : ar.of_mul(z1[i], s[i], d2[i], f.a));
            o2[i] = ar.of_mul(z2[i], c[i], d2[i], f.a) - (still ? 0.0f : ar.of_mul(z2[i], s[i], d1[i], f.a));
        }
        from_pairs<INTERLEAVED>(o1, o2, dx);
    }
    if (w.norm) {
        WindowGrad grads;
        see(grads, dx[0]); see(grads, dx[1]);
        float through[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float n = ar.div(x[v][i], r.root), dz = dx[v][i];
                dx[v][i] = ar.of_mul(n, w.w[v][i], dz, f.a);
                term[v][i] = ar.of_mul(w.w[v][i], n, dz, f.b);
                through[v] += ar.of_divisor(n, r.root, dx[v][i], f.b);
            }
        const float droot = group_sum((at.there ? through[0] : 0.0f) + (at.rotates ? through[1] : 0.0f), a.lanes);
        const float dsquare = raw_square_grad(ar, a, r, droot), inverse = ar.div(1.0f, r.root);
        WindowSquare squares;
        WindowRootGrad root_grads;
        squares.see(dsquare); root_grads.see(droot);
        held = held && grads.held() && squares.held() && root_grads.held();
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float q = ar.of_mul(x[v][i], x[v][i], dsquare, f.a), q2 = APPROXIMATE ? q : ar.of_mul(x[v][i], x[v][i], dsquare, f.b);
                dx[v][i] = nothing ? 0.0f : ar.of_dividend(x[v][i], inverse, dx[v][i], f.a) + (q + q2);
                term[v][i] = nothing ? 0.0f : term[v][i];
            }
    }
    return __ballot(!held) == 0ull;
}

// LDS accesses of a wavefront's lanes to each other's values stay in order.
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wavefront notes the heads that it could not do by raw additions and computes them behind a run of kRun turns, where the
// registers of the usual path are free.  (Within its loop the checked functions' many cases cost that path 137 registers and scalar
// spills, three wavefronts per SIMD; called as a function, the callee's registers counted.)
constexpr int kRun = 32;

template <bool INTERLEAVED, bool APPROXIMATE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void rotary_bwd_kernel(RotaryArgs a)
{
    __shared__ float held[kThreads * 8];          // the weight's gradient of every group: at most 8 values a lane
    const bool other = (int)blockIdx.x >= a.part[0].groups;
    const PartArgs& p = other ? a.part[1] : a.part[0];
    const int lanes = a.lanes, lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = kThreads / lanes;
    const int work_group = (int)blockIdx.x - (other ? a.part[0].groups : 0);
    const uint32_t rows = p.rows, step = (uint32_t)(p.groups * groups), first = (uint32_t)(work_group * groups + group);
    const int turns = (int)((rows - (uint32_t)(work_group * groups) + step - 1) / step);
    float* mine = held + group * a.dim;
    for (int i = lane; i < a.dim; i += lanes) mine[i] = 0.0f;
    wave_fence();
    auto head = [&](int turn) __attribute__((always_inline)) {
        return find_head(a, p, min(first + turn * step, rows - 1));      // (past the end: along with the last head, and nothing stored)
    };
#pragma unroll 1
    for (int run = 0; run < turns; run += kRun) {
        const int end = min(run + kRun, turns);
        uint32_t odd = 0u;
        {
            const Unit at(a, lane);
            const Weight w = load_weight(p.weight, at);
            v4f sum[2] = {};
#pragma unroll 1
            for (int turn = run; turn < end; ++turn) {
                const Head h = head(turn);
                v4f x[2] = {}, d[2], c, s, dx[2], term[2] = {};
                load_unit(h.dy, at, d);
                if (w.norm || !APPROXIMATE) load_unit(h.x, at, x);
                load_table(h, at, a.half > 0, c, s);
                if (!backward_head<INTERLEAVED, APPROXIMATE>(a, at, x, d, w, c, s, dx, term)) { odd |= 1u << (turn - run); continue; }
                if (first + turn * step < rows) {
                    store_unit(h.y, at, dx);
                    sum[0] += term[0]; sum[1] += term[1];
                }
            }
            if (p.sums) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (at.there) mine[at.first + i] += sum[0][i];
                    if (at.rotates) mine[at.second + i] += sum[1][i];
                }
                wave_fence();                     // (below, a value of the head may be another lane's than here)
            }
        }
        odd = __builtin_amdgcn_readfirstlane(odd);
#pragma unroll 1
        for (int turn = run; turn < end; ++turn)
            if ((odd >> (turn - run)) & 1u)
                backward_by_value<true, APPROXIMATE>(a, p.weight, head(turn), lane, lanes, first + turn * step < rows, [&](int i, float t) { mine[i] += t; });
        wave_fence();
    }
    if (!p.sums) return;
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += kThreads) {
        float total = held[i];
        for (int g = 1; g < groups; ++g) total += held[g * a.dim + i];
        p.sums[(long)work_group * a.dim + i] = total;
    }
}

// ---------------------------------------------------------------- a wavefront per head: any size

template <bool BACKWARD>
__global__ __launch_bounds__(kThreads) void any_rotary_kernel(RotaryArgs a)
{
    const int block = a.first_group + (int)blockIdx.x;
    const bool other = block >= a.part[0].groups;
    const PartArgs& p = other ? a.part[1] : a.part[0];
    const uint32_t row = (uint32_t)(block - (other ? a.part[0].groups : 0)) * kWaves + threadIdx.x / 64;
    const int lane = threadIdx.x % 64;
    if (row >= p.rows) return;
    const Head h = find_head(a, p, row);
    float* terms = p.sums ? p.sums + (long)row * a.dim : nullptr;      // (one row per head)
    if (BACKWARD) backward_by_value<false, false>(a, p.weight, h, lane, 64, true, [&](int i, float t) { if (terms) terms[i] = t; });
    else forward_by_value<false>(a, p.weight, h, lane, 64, true);
}

// ---------------------------------------------------------------- host

// Lanes of a group: the power of two that holds a head's units; 0: the head takes the kernels for any size.
int lanes_for(long dim, long rotated)
{
    if (rotated % 8 != 0 || dim % 4 != 0) return 0;
    const long units = rotated / 8 + (dim - rotated) / 4;
    if (units > 64) return 0;
    int lanes = 2;
    while (lanes < units) lanes *= 2;
    return lanes;
}
constexpr long kBackwardGroups = 1024;            // work-groups of a backward launch: the four per compute unit that are resident
// work-groups of a part of `rows` heads, of `all` heads in the launch
long backward_groups(long rows, long all, int lanes)
{
    const long whole = (rows + kThreads / lanes - 1) / (kThreads / lanes);
    return all == 0 ? 0 : std::min(whole, std::max(1L, (long)((double)kBackwardGroups * (double)rows / (double)all)));
}

int fill(const char* what, RotaryArgs& a, const pam_hip_heads* parts, int count, const float* cos, const float* sin, long table_rows,
         const long long* positions, long p_sb, long p_st, long batch, long tokens, long dim, long rotated, int interleaved, float eps, float offset,
         bool backward)
{
    if (count < 1 || count > 2 || !parts) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: one or two tensors", what);
    if (batch < 0 || tokens < 0 || dim < 0 || rotated < 0 || table_rows < 0 || parts[0].heads < 0 || (count > 1 && parts[1].heads < 0))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: negative size", what);
    if (rotated % 2 != 0 || rotated > dim) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the rotated part is an even number of a head's values", what);
    const long heads = parts[0].heads + (count > 1 ? parts[1].heads : 0);
    if (batch > (1L << 30) || tokens > (1L << 30) || dim > (1L << 20) || heads > (1L << 20) || (batch && tokens && heads > (1L << 30) / batch / tokens))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: size out of range", what);
    for (int i = 0; i < 2; ++i) {
        const pam_hip_heads h = i < count ? parts[i] : pam_hip_heads{};
        a.part[i] = PartArgs{h.x, h.x_sb, h.x_st, h.x_sh, backward ? h.dy : nullptr, h.dy_sb, h.dy_st, h.dy_sh, h.weight, h.y, nullptr, (uint32_t)(batch * tokens * h.heads), (uint32_t)h.heads, 0};
        if (backward && h.dweight && !h.weight) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the gradient of a weight that is not there", what);
        if (a.part[i].rows && dim && (!h.x || !h.y || (backward && !h.dy))) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: null pointer", what);
    }
    if (a.part[0].rows + a.part[1].rows && rotated && (!cos || !sin) && table_rows > 0) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: null pointer", what);
    a.cos = cos; a.sin = sin; a.table_rows = table_rows; a.positions = positions; a.p_sb = p_sb; a.p_st = p_st;
    a.tokens = (uint32_t)tokens; a.dim = (int)dim; a.half = (int)(rotated / 2); a.interleaved = interleaved != 0;
    a.lanes = lanes_for(dim, rotated);
    a.eps = eps; a.off = offset; a.has_off = offset != 1.0f;
    a.flags = ApproxFlags{false, false, false};
    return PAM_HIP_OK;
}

// Launches a kernel over the parts' work-groups (at most 2^28 and two).  A launch counts its work-items in 32 bits, so that more than 2^24
// work-groups are several launches.
template <class Kernel>
int launch(const char* what, RotaryArgs& a, Kernel kernel, void* stream)
{
    constexpr long kMost = 1L << 23;
    const long groups = (long)a.part[0].groups + a.part[1].groups;
    for (long first = 0; first < groups; first += kMost) {
        a.first_group = (int)first;
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(kMost, groups - first)), dim3(kThreads), 0, (hipStream_t)stream, a);
        const int rc = pamhost::check_launch(what);
        if (rc != PAM_HIP_OK) return rc;
    }
    return PAM_HIP_OK;
}
void whole_groups(RotaryArgs& a, int per_group) { for (PartArgs& p : a.part) p.groups = (int)((p.rows + per_group - 1) / per_group); }

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// Rows of sums that the backward pass leaves of a part: one per work-group, or per head.
long sum_rows(const pam_hip_heads* parts, int count, int i, long batch, long tokens, long dim, long rotated)
{
    const long rows = batch * tokens * parts[i].heads, all = batch * tokens * (parts[0].heads + (count > 1 ? parts[1].heads : 0));
    const int lanes = lanes_for(dim, rotated);
    return lanes ? backward_groups(rows, all, lanes) : rows;
}

}  // namespace

extern "C" {

int pam_hip_rotary_fwd(const pam_hip_heads* parts, int count, const float* cos, const float* sin, long table_rows, const long long* positions,
                       long positions_sb, long positions_st, long batch, long tokens, long dim, long rotated, int interleaved, float eps,
                       float offset, void* stream)
{
    RotaryArgs a;
    const int rc = fill("rotary_fwd", a, parts, count, cos, sin, table_rows, positions, positions_sb, positions_st, batch, tokens, dim, rotated, interleaved, eps, offset, false);
    if (rc != PAM_HIP_OK || dim == 0) return rc;
    whole_groups(a, a.lanes ? kThreads / a.lanes : kWaves);
    return launch("rotary_fwd", a, !a.lanes ? any_rotary_kernel<false> : interleaved ? rotary_kernel<true> : rotary_kernel<false>, stream);
}

size_t pam_hip_rotary_bwd_workspace_bytes(const pam_hip_heads* parts, int count, long batch, long tokens, long dim, long rotated)
{
    size_t bytes = 0;
    for (int i = 0; parts && batch > 0 && tokens > 0 && i < count && i < 2; ++i)
        if (parts[i].dweight) {
            const long rows = sum_rows(parts, count, i, batch, tokens, dim, rotated);
            bytes += align256((size_t)rows * dim * sizeof(float)) + align256(pam_hip_column_sums_workspace_bytes(rows, dim, 1));
        }
    return bytes;
}

int pam_hip_rotary_bwd(const pam_hip_heads* parts, int count, const float* cos, const float* sin, long table_rows, const long long* positions,
                       long positions_sb, long positions_st, long batch, long tokens, long dim, long rotated, int interleaved, float eps,
                       float offset, int approx_a, int approx_b, int approx_exp, void* workspace, size_t workspace_bytes, void* stream)
{
    RotaryArgs a;
    int rc = fill("rotary_bwd", a, parts, count, cos, sin, table_rows, positions, positions_sb, positions_st, batch, tokens, dim, rotated, interleaved, eps, offset, true);
    if (rc != PAM_HIP_OK || dim == 0) return rc;
    a.flags = ApproxFlags{approx_a != 0, approx_b != 0, approx_exp != 0};
    const size_t need = pam_hip_rotary_bwd_workspace_bytes(parts, count, batch, tokens, dim, rotated);
    if (need && (!workspace || workspace_bytes < need)) return pamhost::fail(PAM_HIP_ERR_WORKSPACE, "rotary_bwd: workspace of %zu bytes needed", need);
    char* at = (char*)workspace;
    long rows[2] = {0, 0};
    for (int i = 0; i < count; ++i)
        if (parts[i].dweight) {
            rows[i] = sum_rows(parts, count, i, batch, tokens, dim, rotated);
            a.part[i].sums = (float*)at;
            at += align256((size_t)rows[i] * dim * sizeof(float));
        }
    if (a.lanes) {
        const long all = (long)a.part[0].rows + a.part[1].rows;
        for (PartArgs& p : a.part) p.groups = (int)backward_groups(p.rows, all, a.lanes);
        const bool approximate = a.flags.a && a.flags.b && a.flags.e;
        rc = launch("rotary_bwd", a, interleaved ? (approximate ? rotary_bwd_kernel<true, true> : rotary_bwd_kernel<true, false>)
                                                 : (approximate ? rotary_bwd_kernel<false, true> : rotary_bwd_kernel<false, false>), stream);
    } else {
        whole_groups(a, kWaves);
        rc = launch("rotary_bwd", a, any_rotary_kernel<true>, stream);
    }
    for (int i = 0; i < count && rc == PAM_HIP_OK; ++i)
        if (parts[i].dweight) {
            const size_t bytes = pam_hip_column_sums_workspace_bytes(rows[i], dim, 1);
            rc = pam_hip_column_sums(a.part[i].sums, dim, parts[i].dweight, nullptr, 0, nullptr, rows[i], dim, bytes ? at : nullptr, bytes, stream);
            at += align256(bytes);
        }
    return rc;
}

}  // extern "C"
