// Attention's entry points, and the small kernels beside pam_attention_fwd.h and pam_attention_bwd.h: the rows' quantities that the gradients
// start from, and the chunks' sums put together.
#include <algorithm>
#include <cmath>

#include "pam_attention.h"

namespace pamatt {

typedef void (*Kernel)(Args);
struct Variant { int slices, quads; bool whole; Kernel kernel; };
extern const Variant kForward[], kDqApprox[], kDqExact[], kDkvApprox[], kDkvExact[];

}  // namespace pamatt

using namespace pamatt;

namespace {

// The chunks of a row: weights scaled to the largest M, sums added in ascending order.  A thread has a quad of a row.
__global__ __launch_bounds__(kThreads) void attention_join_kernel(Args a)
{
    const long quads = a.dim / 4, id = (long)blockIdx.x * kThreads + threadIdx.x, all = (long)a.batch * a.kv_heads * a.rows * quads;
    if (id >= all) return;
    const long at = id / quads, head = at / a.rows, row = at - head * a.rows;
    const int d = (int)(id - at * quads) * 4;
    float M = kNothing;
    for (int c = 0; c < a.chunks; ++c) M = fmaxf(M, a.partial_stats[(head * a.chunks + c) * a.rows + row].y);
    float l = 0.0f;
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < a.chunks; ++c) {
        const long from = (head * a.chunks + c) * a.rows + row;
        const float2 s = a.partial_stats[from];
        if (s.y == kNothing) continue;
        const float f = scale_between(s.y, M);
        const v4f x = *reinterpret_cast<const v4f*>(a.partial + from * a.dim + d);
        l += s.x * f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += x[i] * f;
    }
    const int b = (int)(head / a.kv_heads), kv = (int)(head - (long)b * a.kv_heads);
    const long to = ((long)b * a.tokens + row / a.group) * a.heads + kv * a.group + row % a.group;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = M == kNothing ? 0.0f : pad_div_off(sum[i], l, a.off, a.off != 1.0f);
    *reinterpret_cast<v4f_any*>(a.y + to * a.dim + d) = sum;
    if (a.stats && d == 0) a.stats[to] = make_float2(l, M);
}

// A query's head: qs, dn and its record (see pam_attention_bwd.h).  Sixteen lanes have one.  dl's terms are added up in the order in which the passes
// add up dn (*) v, each slice's of `width` values from the first to the last, so that the two cancel to nothing where a row sees a single key.
struct RowArgs { Args a; const float* y; Tokens dy; const float2* stats; float4* records; float* qs; float* dn; int slices, width; };
__global__ __launch_bounds__(kThreads) void attention_rows_kernel(RowArgs r)
{
    __shared__ float terms[kThreads / 16][256 + 1];
    const Args& a = r.a;
    const long all = (long)a.batch * a.tokens * a.heads, mine = (long)blockIdx.x * (kThreads / 16) + threadIdx.x / 16, id = min(mine, all - 1);
    const int lane = threadIdx.x % 16, last = a.values - 1;
    const long token = id / a.heads, b = token / a.tokens, t = token - b * a.tokens;
    const int head = (int)(id - token * a.heads), kv = head / a.group;
    const long row = t * a.group + head % a.group, to = (b * a.kv_heads + kv) * a.rows + row;
    const float off = a.off;
    const bool has_off = off != 1.0f;
    const float2 stats = r.stats[id];
    const float* const q = a.q.p + b * a.q.sb + t * a.q.st + (long)head * a.q.sh;
    const float* const dy = r.dy.p + b * r.dy.sb + t * r.dy.st + (long)head * r.dy.sh;
    const float* const y = r.y + id * a.dim;
    const bool sees = stats.y != kNothing;
    const float l = sees ? stats.x : 1.0f;
    const bool whole = fabsf(l) < u2f(kExpo);
    float dl = 0.0f;
    uint32_t most = 0u;
    for (int d = lane; d < a.dim; d += 16) {
        const bool there = d < a.values;
        const float g = dy[min(d, last)], out = y[min(d, last)];
        // (the sums that y was the quotient of: the same bits as far as they matter to a slope)
        const float sums = whole ? pam_mul(has_off ? pam_mul(out, off) : out, l) : l;
        const float dn = div_grad_a(sums, l, g, a.flags.a, off, has_off);
        r.qs[to * a.dim + d] = pam_mul_off(q[min(d, last)], a.scale, off, has_off);          // (behind the values the last one again)
        r.dn[to * a.dim + d] = dn;
        if (!there) continue;
        terms[threadIdx.x / 16][d] = a.flags.b ? -pam_mul_off(pad_div_off(out, l, off, has_off), g, off, has_off) : -(u2f(f2u(out) & ~kMant) / u2f(f2u(l) & kExpo)) * g;
        most = max(most, f2u(dn) & ~kSign);
    }
    // (all sixteen lanes are there: a work-group past the end repeats the last row)
    for (int s = 8; s >= 1; s /= 2) most = max(most, (uint32_t)__shfl_xor((int)most, s, 16));
    __syncthreads();
    if (lane < r.slices) {
        const int end = min(a.values, (lane + 1) * r.width);
#pragma unroll 8
        for (int d = lane * r.width; d < end; ++d) dl += terms[threadIdx.x / 16][d];
    }
    for (int s = 1; s < 8; s *= 2) dl += __shfl_xor(dl, s, 16);
    if (lane != 0 || mine >= all) return;
    // a query without a gradient counts as one that sees nothing: it has none to give
    const bool none = !sees || (most == 0u && dl == 0.0f);
    const int exponent = max(-86, min(60, (int)(most >> 23) - 127));
    r.records[to] = make_float4(none ? u2f(kExpo) : stats.y, none ? 0.0f : dl, none ? -86.0f : (float)exponent, a.slopes ? held_slope(a.slopes[head]) : 0.0f);
}

// dq from the chunks' sums, through q (*) scale; or dk and dv (the second half of the launch): nothing behind the sums.
struct SumArgs { Args a; const float* parts[2]; float* out[2]; int of_keys; long tiles; };          // tiles: of 64 rows
__global__ __launch_bounds__(kThreads) void attention_sum_kernel(SumArgs s)
{
    const Args& a = s.a;
    const long quads = a.dim / 4, lanes = s.of_keys ? a.keys : a.rows, all = (long)a.batch * a.kv_heads * lanes * quads;
    long id = (long)blockIdx.x * kThreads + threadIdx.x;
    const int which = id >= all;
    if (which) id -= all;
    if (id >= all || (which && !s.of_keys)) return;
    const float* const parts = which ? s.parts[1] : s.parts[0];
    const long at = id / quads, head = at / lanes, row = at - head * lanes, b = head / a.kv_heads, kv = head - b * a.kv_heads;
    const int d = (int)(id - at * quads) * 4;
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int c = 0; c < a.chunks; ++c)
        if (a.met[(head * a.chunks + c) * s.tiles + row / 64]) sum += *reinterpret_cast<const v4f*>(parts + ((head * a.chunks + c) * lanes + row) * a.dim + d);
    long to;
    if (s.of_keys) to = (b * a.keys + row) * a.kv_heads + kv;
    else {
        const long t = row / a.group, h = kv * a.group + row % a.group;
        const float* const q = a.q.p + b * a.q.sb + t * a.q.st + h * a.q.sh;
        to = (b * a.tokens + t) * a.heads + h;
        const bool has_off = a.off != 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) if (d + i < a.values) sum[i] = mul_grad(q[d + i], a.scale, sum[i], a.flags.a, a.off, has_off);
    }
    *reinterpret_cast<v4f_any*>((which ? s.out[1] : s.out[0]) + to * a.dim + d) = sum;
}

// ---------------------------------------------------------------- host

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// Of the kernels' instances the one whose slices have just a row's quads, or else the first one wide enough of those that may have more.  (All lists
// are the same, so that all passes add up a row's products in one order.)
const Variant& variant_for(const Variant* list, long dim)
{
    for (const Variant* v = list; v->slices; ++v)
        if (v->whole ? 4L * v->slices * v->quads == dim : 4L * v->slices * v->quads >= dim) return *v;
    return list[0];                               // (no call: rows have up to 256 values)
}

// How the streamed rows are cut.  All units of a launch run at once or in a few turns of `slots` of them, so that a last turn of a few units costs as
// much as a full one: among the cuts that fill one, two, ... turns the one is taken whose turns times the spans that a unit works on are least.  (4096 causal tokens, 8 heads over 2:
// chunks of 256 keys, two turns and a bit, 0.70 ms; the cut taken 0.55.)  Which spans a tile sees is what the order and the window say; prefixes and documents are on the device.
// A chunk is at least two spans (documents leave a tile little of what the order does, but chunks of one span cost 307 us where three took 267, 210 since units
// that see nothing end early: 2 x 2048 tokens, heads of 128), what a unit does besides its spans counts as a fifth of one.
// Of a window the chunks are counted from where a tile's begins, so that there are as many as one window has and no more scratch than that, however long the rows are.
struct Plan { int tiles, chunks, chunk; };
long tiles_of(int slices) { return slices >= 4 ? 1 : 4 / slices; }              // of a work-group (kTiles)
template <class Range>                            // range(first, last row of a tile, low, high): the streamed rows that those see; range.reach(rows of a tile): of any tile at most
Plan plan_for(long heads, long lanes, int slices, long streamed, int waves_per_simd, const Range& range)
{
    const long per_tile = 64 * tiles_of(slices), tiles = (lanes + per_tile - 1) / per_tile, samples = std::min(tiles, 32L);
    const bool windows = range.a.windows;
    long spans = std::max(1L, (streamed + kSpan - 1) / kSpan);
    if (windows) spans = std::min(spans, (range.reach(per_tile) + kSpan - 2) / kSpan + 1);
    const long slots = 256L * 4 * waves_per_simd / (slices * tiles_of(slices));
    long low[32], high[32], total = 0, longest = 0;      // of tiles evenly spread, in spans
    for (long n = 0; n < samples; ++n) {
        const long tile = (2 * n + 1) * tiles / (2 * samples);
        long from = 0, to = streamed;
        range(tile * per_tile, std::min(lanes, (tile + 1) * per_tile) - 1, from, to);
        low[n] = std::max(0L, from) / kSpan; high[n] = std::max(low[n], (std::min(to, streamed) + kSpan - 1) / kSpan);
        if (windows) { high[n] -= low[n]; low[n] = 0; }
        total += high[n] - low[n]; longest = std::max(longest, high[n] - low[n]);
    }
    const double each = samples ? (double)heads * tiles / samples : 0.0;
    double best = 0.0;
    long chosen = spans;
    for (int turns = 1; turns <= 6; ++turns) {
        long size = std::max(2L, (long)(each * total / (turns * slots)));
        double units = 0.0;
        for (int tries = 0; tries < 12; ++tries, size += 1 + size / 16) {
            size = std::min(size, std::max(2L, spans));
            units = 0.0;
            for (long n = 0; n < samples; ++n) units += high[n] == low[n] ? 0.0 : (double)((high[n] - 1) / size - low[n] / size + 1);
            units *= each;
            if (units <= turns * slots || size >= spans) break;
        }
        size = std::min(size, spans);
        const double cost = std::ceil(units / slots) * (std::min(size, windows ? longest : spans) + 0.2);
        if (turns == 1 || cost < best * 0.97) { best = cost; chosen = size; }
        if (size <= 2) break;
    }
    return Plan{(int)tiles, (int)((spans + chosen - 1) / chosen), (int)(chosen * kSpan)};
}

int check(const char* what, const pam_hip_attention_shape* s, Args& a)
{
    if (!s) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: null pointer", what);
    if (s->batch < 0 || s->tokens < 0 || s->keys < 0 || s->heads < 0 || s->kv_heads < 0 || s->window < 0)
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: negative size", what);
    if (s->dim < 4 || s->dim > 256 || s->dim % 4 != 0 || s->values < 1 || s->values > s->dim || s->values <= s->dim - 4)
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: heads of %ld values in rows of %ld: up to 256, in rows of the next multiple of four", what, s->values, s->dim);
    if (s->kv_heads == 0 ? s->heads != 0 : s->heads % s->kv_heads != 0)
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: %ld heads do not share %ld", what, s->heads, s->kv_heads);
    if (s->batch > (1L << 20) || s->heads > (1L << 16) || s->tokens > (1L << 28) || s->keys > (1L << 28) || s->batch * s->kv_heads > (1L << 20)
        || (s->kv_heads && s->heads / s->kv_heads * s->tokens > (1L << 30)) || s->batch * s->tokens * s->heads > (1L << 32))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: size out of range", what);
    if (!(s->scale > 0x1p-40f && s->scale < 0x1p40f)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the scale lies between 2^-40 and 2^40", what);
    if (s->cap != 0.0f && !(s->cap > 0x1p-20f && s->cap < 0x1p20f)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the cap lies between 2^-20 and 2^20", what);
    if (!(s->offset > 0.75f && s->offset < 1.5f)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the offset lies between 0.75 and 1.5", what);
    if (s->documents && s->tokens > s->keys) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: more queries than keys, whose documents are given", what);
    a.batch = (int)s->batch; a.tokens = (int)s->tokens; a.keys = (int)s->keys; a.heads = (int)s->heads; a.kv_heads = (int)s->kv_heads;
    a.group = s->kv_heads ? (int)(s->heads / s->kv_heads) : 1; a.dim = (int)s->dim; a.values = (int)s->values;
    a.rows = a.tokens * a.group; a.first = a.keys - a.tokens; a.causal = s->causal != 0; a.window = (int)std::min(s->window, 1L << 29);
    a.prefix = s->prefix; a.documents = s->documents; a.slopes = s->slopes; a.scale = s->scale; a.cap = s->cap; a.off = s->offset;
    a.windows = a.window != 0 && !a.prefix;
    return PAM_HIP_OK;
}
Tokens tokens_of(const pam_hip_tokens* t) { return Tokens{t->p, t->sb, t->st, t->sh}; }
long heads_of(const Args& a) { return (long)a.batch * a.kv_heads; }

// A launch counts its work-items in 32 bits.
int launch(const char* what, const Variant& v, const Args& a, hipStream_t st)
{
    const long groups = heads_of(a) * a.tiles * a.chunks;
    if (groups > (1L << 23)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: size out of range", what);
    hipLaunchKernelGGL(v.kernel, dim3((unsigned)groups), dim3(64 * v.slices * tiles_of(v.slices)), 0, st, a);
    return pamhost::check_launch(what);
}
int groups_for(const char* what, long items, unsigned& groups)
{
    const long n = (items + kThreads - 1) / kThreads;
    if (n > (1L << 23)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: size out of range", what);
    groups = (unsigned)n;
    return PAM_HIP_OK;
}

// What a tile of queries' rows, or of keys, sees.
struct OfRows {
    const Args& a;
    void operator()(long from, long to, long& low, long& high) const
    {
        const long first = a.first + from / a.group, last = a.first + to / a.group;
        if (a.windows) low = first - a.window + 1;
        if (a.causal) high = last + 1;
        else if (a.window) high = last + a.window;
    }
    long reach(long rows) const { return (rows + a.group - 2) / a.group + (a.causal ? 1L : 2L) * a.window; }
};
struct OfKeys {
    const Args& a;
    void operator()(long from, long to, long& low, long& high) const
    {
        if (a.prefix) return;
        if (a.causal) low = (from - a.first) * a.group;
        else if (a.window) low = (from - a.window + 1 - a.first) * a.group;
        if (a.window) high = (to + a.window - a.first) * a.group;
    }
    long reach(long keys) const { return (keys - 1 + (a.causal ? 1L : 2L) * a.window) * a.group; }
};
Plan forward_plan(const Args& a)
{
    const Variant& v = variant_for(kForward, a.dim);
    return plan_for(heads_of(a), a.rows, v.slices, a.keys, v.quads > 8 ? 2 : 3, OfRows{a});
}
Plan dq_plan(const Args& a) { return plan_for(heads_of(a), a.rows, variant_for(kDqApprox, a.dim).slices, a.keys, 3, OfRows{a}); }
Plan dkv_plan(const Args& a) { return plan_for(heads_of(a), a.keys, variant_for(kDkvApprox, a.dim).slices, a.rows, 2, OfKeys{a}); }

struct BackwardSpace { size_t records, qs, dn, dq, dk, dv, met_q, met_kv, bytes; };
BackwardSpace backward_space(const Args& a, bool want_q, bool want_kv)
{
    BackwardSpace s{};
    const size_t rows = (size_t)heads_of(a) * a.rows, keys = (size_t)heads_of(a) * a.keys, row = (size_t)a.dim * sizeof(float);
    size_t at = 0;
    const auto take = [&](size_t n) { const size_t from = at; at += align256(n); return from; };
    s.records = take(rows * sizeof(float4)); s.qs = take(rows * row); s.dn = take(rows * row);
    // (a pass of one chunk writes its gradients itself)
    const Plan of_q = want_q ? dq_plan(a) : Plan{0, 1, 0}, of_kv = want_kv ? dkv_plan(a) : Plan{0, 1, 0};
    const auto flags = [&](const Plan& p) { return (size_t)heads_of(a) * p.chunks * p.tiles * tiles_of(variant_for(kDqApprox, a.dim).slices); };
    if (of_q.chunks > 1) { s.dq = take(rows * row * of_q.chunks); s.met_q = take(flags(of_q)); }
    if (of_kv.chunks > 1) { s.dk = take(keys * row * of_kv.chunks); s.dv = take(keys * row * of_kv.chunks); s.met_kv = take(flags(of_kv)); }
    s.bytes = at;
    return s;
}

}  // namespace

extern "C" {

size_t pam_hip_attention_workspace_bytes(const pam_hip_attention_shape* shape)
{
    Args a{};
    if (check("attention", shape, a) != PAM_HIP_OK || a.keys == 0) return 0;
    const Plan p = forward_plan(a);
    if (p.chunks == 1) return 0;
    const size_t rows = (size_t)heads_of(a) * a.rows * p.chunks;
    return align256(rows * sizeof(float2)) + align256(rows * a.dim * sizeof(float));
}

int pam_hip_attention_fwd(const pam_hip_attention_shape* shape, const pam_hip_tokens* q, const pam_hip_tokens* k, const pam_hip_tokens* v,
                          float* y, float* stats, void* workspace, size_t workspace_bytes, void* stream)
{
    Args a{};
    int rc = check("attention_fwd", shape, a);
    if (rc != PAM_HIP_OK || a.batch == 0 || a.kv_heads == 0 || a.rows == 0) return rc;
    if (!q || !k || !v || !q->p || !y || (a.keys && (!k->p || !v->p))) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "attention_fwd: null pointer");
    const size_t need = pam_hip_attention_workspace_bytes(shape);
    if (need && (!workspace || workspace_bytes < need)) return pamhost::fail(PAM_HIP_ERR_WORKSPACE, "attention_fwd: workspace of %zu bytes needed", need);
    a.q = tokens_of(q); a.k = tokens_of(k); a.v = tokens_of(v);
    a.y = y; a.stats = reinterpret_cast<float2*>(stats);
    const hipStream_t st = (hipStream_t)stream;
    const Plan p = forward_plan(a);
    a.tiles = p.tiles; a.chunks = p.chunks; a.chunk = p.chunk;
    if (need) {
        a.partial_stats = (float2*)workspace;
        a.partial = (float*)((char*)workspace + align256((size_t)heads_of(a) * a.rows * p.chunks * sizeof(float2)));
    }
    unsigned groups = 0;
    rc = groups_for("attention_fwd", heads_of(a) * a.rows * (a.dim / 4), groups);
    if (rc == PAM_HIP_OK) rc = launch("attention_fwd", variant_for(kForward, a.dim), a, st);
    if (rc != PAM_HIP_OK || !need) return rc;
    hipLaunchKernelGGL(attention_join_kernel, dim3(groups), dim3(kThreads), 0, st, a);
    return pamhost::check_launch("attention_fwd");
}

size_t pam_hip_attention_bwd_workspace_bytes(const pam_hip_attention_shape* shape, int want_q, int want_kv)
{
    Args a{};
    if (check("attention_bwd", shape, a) != PAM_HIP_OK) return 0;
    return backward_space(a, want_q != 0, want_kv != 0).bytes;
}

int pam_hip_attention_bwd(const pam_hip_attention_shape* shape, const pam_hip_tokens* q, const pam_hip_tokens* k, const pam_hip_tokens* v,
                          const float* y, const float* stats, const pam_hip_tokens* dy, float* dq, float* dk, float* dv,
                          int approx_a, int approx_b, int approx_exp, void* workspace, size_t workspace_bytes, void* stream)
{
    Args a{};
    int rc = check("attention_bwd", shape, a);
    if (rc != PAM_HIP_OK || a.batch == 0 || a.kv_heads == 0) return rc;
    const bool want_kv = dk != nullptr;
    if ((dk == nullptr) != (dv == nullptr)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "attention_bwd: the gradients of keys and values come together");
    if (!q || !k || !v || !dy || (a.rows && (!q->p || !y || !stats || !dy->p)) || (a.keys && (!k->p || !v->p)))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "attention_bwd: null pointer");
    const BackwardSpace space = backward_space(a, dq != nullptr, want_kv);
    if (space.bytes && (!workspace || workspace_bytes < space.bytes)) return pamhost::fail(PAM_HIP_ERR_WORKSPACE, "attention_bwd: workspace of %zu bytes needed", space.bytes);
    char* const ws = (char*)workspace;
    a.q = tokens_of(q); a.k = tokens_of(k); a.v = tokens_of(v);
    a.flags = ApproxFlags{approx_a != 0, approx_b != 0, approx_exp != 0};
    const bool approximate = approx_a && approx_b && approx_exp;
    a.records = (const float4*)(ws + space.records); a.qs = (const float*)(ws + space.qs); a.dn = (const float*)(ws + space.dn);
    const hipStream_t st = (hipStream_t)stream;
    unsigned groups = 0, row_groups = 0, key_groups = 0;
    if ((rc = groups_for("attention_bwd", heads_of(a) * a.rows * 16, groups)) || (rc = groups_for("attention_bwd", heads_of(a) * a.rows * (a.dim / 4), row_groups))
        || (rc = groups_for("attention_bwd", 2 * heads_of(a) * a.keys * (a.dim / 4), key_groups))) return rc;
    if (a.rows) {
        const Variant& v = variant_for(kDqApprox, a.dim);
        const RowArgs r{a, y, tokens_of(dy), reinterpret_cast<const float2*>(stats), (float4*)(ws + space.records), (float*)(ws + space.qs), (float*)(ws + space.dn), v.slices, 4 * v.quads};
        hipLaunchKernelGGL(attention_rows_kernel, dim3(groups), dim3(kThreads), 0, st, r);
        if ((rc = pamhost::check_launch("attention_bwd"))) return rc;
    }
    const auto pass = [&](const Variant* list, const Plan& p, float* part0, float* part1, float* out0, float* out1, size_t met, int of_keys, unsigned sum_groups) {
        Args d = a;
        d.tiles = p.tiles; d.chunks = p.chunks; d.chunk = p.chunk; d.whole = p.chunks == 1; d.met = (unsigned char*)ws + met;
        d.out0 = d.whole ? out0 : part0; d.out1 = d.whole ? out1 : part1;
        const int failed = launch("attention_bwd", variant_for(list, a.dim), d, st);
        if (failed || d.whole) return failed;
        hipLaunchKernelGGL(attention_sum_kernel, dim3(sum_groups), dim3(kThreads), 0, st, SumArgs{d, {part0, part1}, {out0, out1}, of_keys, (long)p.tiles * tiles_of(variant_for(list, a.dim).slices)});
        return pamhost::check_launch("attention_bwd");
    };
    if (dq && a.rows && (rc = pass(approximate ? kDqApprox : kDqExact, dq_plan(a), (float*)(ws + space.dq), nullptr, dq, nullptr, space.met_q, 0, row_groups))) return rc;
    if (want_kv && a.keys
        && (rc = pass(approximate ? kDkvApprox : kDkvExact, dkv_plan(a), (float*)(ws + space.dk), (float*)(ws + space.dv), dk, dv, space.met_kv, 1, key_groups))) return rc;
    return PAM_HIP_OK;
}

}  // extern "C"
