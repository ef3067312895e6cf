// Attention of a few new tokens over a paged cache (pam_attention.h has the formulas), for single tokens while decoding.
//
// Bound by reading the cache once, or, where many rows share it, by the products.  A wavefront takes 64 keys at a time.  For the scores a lane owns a key, 32 of
// its values in registers while the queries' rows come by in scalar registers (pam_attention.h): two instructions a product and no sums over
// lanes, so that the keys are read once for up to 12 rows.  Then a lane per key makes the weights, and for the results a group of L lanes
// owns a key's row of values, a quad each (4 ... 64 lanes), and reads the rows' weights from LDS.  Every sequence's keys are cut into as
// many parts as there are work-groups for it, by its own length; four wavefronts of a work-group take 64 keys in turn, their sums are put
// together through LDS, and the parts' by a second kernel.  Scaling by powers of two is exact, so that none of this moves a result beyond the
// order of its sums.
// 16 sequences of up to 4000 tokens, 16 heads of 128 over 4: 42 us for 134 MB (3.2 TB/s; 2040 spans are one for every wavefront, whose waits for memory follow
// each other), the join 6; one sequence of 100000, five tokens, 8 heads over 2: 170 us for 1.02 G products, 6 T/s: two sets of twelve rows for twenty, a
// query's piece used for one key of every lane, and with a bias by distance most spans' weights are none, which takes a factor for every product (159 us without).
// Heads that are no whole quads take a kernel in which groups of lanes own keys for the scores, too.
#include <algorithm>

#include "pam_attention.h"

using namespace pamatt;

namespace {

constexpr int kSteps = 4;                         // keys' rows in flight, of every lane
constexpr int kMostParts = 512, kMostRows = 12;
typedef void (*Kernel)(struct CacheArgs);

struct CacheArgs {
    Tokens q;
    const float* k; const float* v; long c_sp, c_st, c_sh;      // pages, places in one, heads
    const int* table; const long long* lengths; const long long* counts;
    const float* slopes;
    float* y;
    float* partial; float2* partial_stats;        // [kv_heads][batch x parts][rows][quads of values], [...]: l, M; or null: parts is 1
    int batch, tokens, heads, kv_heads, group, values, rows;
    int page, pages, per_sequence, window, capacity;      // per_sequence: entries of the table; capacity: the places that they make
    int lanes, parts, sets, rows_each;            // parts: on average, of a sequence
    float scale, cap, off;
};

struct RowPlace { int token, head; };
__device__ __forceinline__ RowPlace place_of(const CacheArgs& a, int kv, int row) { return RowPlace{row / a.group, kv * a.group + row % a.group}; }

// The sum over a group of lanes, in all of them.
template <int CTRL> __device__ __forceinline__ float across(float v) { return u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), CTRL, 0xf, 0xf, true)); }
template <int N> __device__ __forceinline__ void group_sums(float (&v)[N], int lanes)
{
    typedef unsigned int u2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += across<0xb1>(v[i]);                       // lane ^ 1
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += across<0x4e>(v[i]);                       // lane ^ 2
    if (lanes >= 8)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += across<0x141>(v[i]);                  // the other four of eight
    if (lanes >= 16)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += across<0x140>(v[i]);                  // the other eight of sixteen
    if (lanes >= 32)
#pragma unroll
        for (int i = 0; i < N; ++i) { const u2 r = __builtin_amdgcn_permlane16_swap(f2u(v[i]), f2u(v[i]), false, false); v[i] = u2f(r.x) + u2f(r.y); }
    if (lanes >= 64)
#pragma unroll
        for (int i = 0; i < N; ++i) { const u2 r = __builtin_amdgcn_permlane32_swap(f2u(v[i]), f2u(v[i]), false, false); v[i] = u2f(r.x) + u2f(r.y); }
}

// LDS accesses of a wavefront's lanes to each other's values stay in order.
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The lane's quads of kSteps keys' rows, ones behind a head's values.
struct Lane { int first, values; bool streams; uint64_t streaming; };
__device__ __forceinline__ void load_rows(const float* base, const long (&at)[kSteps], const Lane& here, v4f (&r)[kSteps])
{
    if (here.values % 4 == 0) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) r[i] = *reinterpret_cast<const v4f_any*>(base + at[i] + here.first);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int d = 0; d < 4; ++d) r[i][d] = here.streams ? r[i][d] : 1.0f;
        return;
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const bool there = here.streams && here.first + d < here.values;
            const float x = base[at[i] + (there ? here.first + d : 0)];
            r[i][d] = there ? x : 1.0f;
        }
}
__device__ __forceinline__ bool ordinary(const v4f (&r)[kSteps])
{
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int d = 0; d < 4; ++d) most = max(most, (f2u(r[i][d]) << 1) - kStreamBase);
    return __ballot(most >= kStreamSpan) == 0ull;
}

// Which spans of a sequence the rows row0 ... row0 + count - 1 see.
struct Spans {
    int length, given, begin, end;                // keys; the first one's span is where the count begins
    __device__ __forceinline__ Spans(const CacheArgs& a, int b, int row0, int count)
    {
        length = (int)max(0ll, min(a.lengths[b], 1ll << 30));
        given = a.counts ? (int)max(0ll, min(a.counts[b], (long long)a.tokens)) : a.tokens;
        const int last_token = min((row0 + count - 1) / a.group, given - 1), first_token = row0 / a.group;
        const bool any = first_token <= last_token;
        // (no key behind the table's last place is looked for, however long a sequence says it is: a row that would see one is no number)
        end = any ? min(length + last_token + 1, a.capacity) : 0;
        begin = any && a.window ? min(max(0, length + first_token - a.window + 1), end) : 0;
    }
    __device__ __forceinline__ int count() const { return (end + kSpan - 1) / kSpan - begin / kSpan; }
};
// How the parts of a key head's work-groups (batch x parts) go to the sequences: up to 64 sequences share them by their lengths, so that each part has
// the same number of spans for every wavefront; more have a fixed number each.  (16 sequences of 4000 tokens and less, 512 work-groups: 48 us
// with a fixed number.)
struct Cut { int b, first, parts, each; };        // of sequence b: its first part, how many, the spans in one
__device__ __forceinline__ Cut cut_of(const CacheArgs& a, int row0, int count, bool by_part, int which)          // by_part: of the sequence that has part `which`
{
    Cut c;
    if (a.batch > 64 || a.parts == 1) {
        c.b = by_part ? which / a.parts : which; c.first = c.b * a.parts; c.parts = a.parts;
        c.each = (Spans(a, c.b, row0, count).count() + a.parts - 1) / a.parts;
        return c;
    }
    const int lane = threadIdx.x % 64, all = a.batch * a.parts;
    const int spans = lane < a.batch ? Spans(a, lane, row0, count).count() : 0;
    const auto sum = [](int v) { for (int s = 1; s < 64; s *= 2) v += __shfl_xor(v, s, 64); return v; };
    int each = max(kWaves, (sum(spans) / all + kWaves - 1) / kWaves * kWaves), parts = 0;
    for (;; each += max(kWaves, each / 8 / kWaves * kWaves)) {                   // (ends: parts <= sum / each + batch, and there are at least twice batch)
        parts = lane < a.batch ? max(1, (spans + each - 1) / each) : 0;
        if (__builtin_amdgcn_readfirstlane(sum(parts)) <= all) break;
    }
    int upto = parts;
    for (int s = 1; s < 64; s *= 2) { const int x = __shfl_up(upto, s, 64); upto += lane >= s ? x : 0; }
    c.b = __builtin_amdgcn_readfirstlane(by_part ? (int)__popcll(__ballot(lane < a.batch && upto <= which)) : which);
    c.parts = __shfl(parts, min(c.b, 63), 64);
    c.first = __builtin_amdgcn_readfirstlane(__shfl(upto, min(c.b, 63), 64) - c.parts);
    c.parts = __builtin_amdgcn_readfirstlane(c.parts);
    c.each = __builtin_amdgcn_readfirstlane(each);
    return c;
}
// What a kernel's work-group is there for.
struct Share {
    int row0, here_rows, slot, b, kv, length, given, begin, end;                 // slot: where its sums go
    __device__ __forceinline__ Share(const CacheArgs& a, int rows_each)
    {
        // (work-groups go to the eight XCDs in turn: those that read the same keys for other rows are eight apart, on one of them)
        const int x = (int)blockIdx.x, all = a.batch * a.parts;
        slot = x / (8 * a.sets) * 8 + x % 8;
        row0 = x / 8 % a.sets * rows_each;
        here_rows = 0;
        kv = slot / all;
        if (kv >= a.kv_heads) return;
        const int count = min(rows_each, a.rows - row0);
        const Cut cut = cut_of(a, row0, count, true, slot - kv * all);
        b = cut.b;
        if (b >= a.batch) return;                 // (more parts than the sequences need)
        here_rows = count;
        const Spans of(a, b, row0, count);
        length = of.length; given = of.given;
        begin = (of.begin / kSpan + (slot - kv * all - cut.first) * cut.each) * kSpan; end = min(of.end, begin + cut.each * kSpan);
    }
};
// Where a key's row lies, and whether it does.
struct KeyPlace { long at; bool there; };
__device__ __forceinline__ KeyPlace key_place(const CacheArgs& a, const int* table, int j, bool exists)
{
    KeyPlace p{0, exists};
    if (exists) {
        const int of = table[j / a.page];
        p.there = of >= 0 && of < a.pages;
        p.at = p.there ? (long)of * a.c_sp + (long)(j % a.page) * a.c_st : 0;
    }
    return p;
}

// The wavefronts' sums (each lane's quad of `acc`, over groups of L lanes) and what they are over, put together and written.
template <int ROWS>
__device__ __forceinline__ void finish(const CacheArgs& a, const Share& me, float (&acc)[ROWS][4], float (&l)[ROWS], const float (&M_of)[ROWS], uint32_t saw,
                                       float (&sums)[ROWS][256 + 4], float2 (&stats)[kWaves][ROWS])
{
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), L = a.lanes;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        for (int s = L; s < 64; s *= 2)
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[r][d] += __shfl_xor(acc[r][d], s, 64);
        for (int s = 1; s < 64; s *= 2) l[r] += __shfl_xor(l[r], s, 64);
        const int token = (me.row0 + min(r, me.here_rows - 1)) / a.group;
        const bool beyond = token < me.given && me.length + token >= a.capacity, some = beyond || __ballot((saw >> r) & 1u) != 0ull;
        l[r] = beyond ? u2f(kQNaN) : l[r];
        const float M = some && M_of[r] == kNothing ? 0.0f : M_of[r];            // (seen, and no number)
        if (lane == 0) stats[wave][r] = make_float2(some ? l[r] : 0.0f, some ? M : kNothing);
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
        if (w == wave && lane < L)
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                float most = kNothing;
#pragma unroll
                for (int o = 0; o < kWaves; ++o) most = fmaxf(most, stats[o][r].y);
                const bool mine = stats[w][r].y != kNothing;
                const float f = mine ? scale_between(stats[w][r].y, most) : 0.0f;
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const float x = mine ? acc[r][d] * f : 0.0f;
                    sums[r][lane * 4 + d] = w == 0 ? x : sums[r][lane * 4 + d] + x;
                }
            }
        __syncthreads();
    }
    const int quads = (a.values + 3) / 4;
    for (int i = threadIdx.x; i < me.here_rows * quads; i += kThreads) {
        const int r = i / quads, d = i % quads * 4;
        float most = kNothing, total = 0.0f;
        const v4f sum = {sums[r][d], sums[r][d + 1], sums[r][d + 2], sums[r][d + 3]};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = fmaxf(most, stats[w][r].y);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float2 s = stats[w][r];
            total += s.y == kNothing ? 0.0f : s.x * scale_between(s.y, most);
        }
        const RowPlace at = place_of(a, me.kv, me.row0 + r);
        if (a.partial) {
            const long to = (long)me.slot * a.rows + me.row0 + r;
            *reinterpret_cast<v4f*>(a.partial + to * quads * 4 + d) = sum;
            if (d == 0) a.partial_stats[to] = make_float2(total, most);
        } else {
            float* const to = a.y + (((long)me.b * a.tokens + at.token) * a.heads + at.head) * a.values + d;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (d + c < a.values) to[c] = most == kNothing ? 0.0f : pad_div_off(sum[c], total, a.off, a.off != 1.0f);
        }
    }
}

// ---------------------------------------------------------------- heads of any size

template <int ROWS>
__global__ __launch_bounds__(kThreads, 4) void cached_attention_kernel(CacheArgs a)
{
    __shared__ float scores[kWaves][kSpan][ROWS];                                // of a wavefront's keys, then their weights
    __shared__ float sums[ROWS][256 + 4];
    __shared__ float2 stats[kWaves][ROWS];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), L = a.lanes, keys_a_step = 64 / L;
    const Share me(a, ROWS);
    if (me.here_rows <= 0) return;
    const int row0 = me.row0, here_rows = me.here_rows, b = me.b, kv = me.kv, length = me.length, given = me.given, begin = me.begin, end = me.end;
    const bool has_off = a.off != 1.0f;
    const uint32_t off_add = f2u(a.off) - kBias, mul_add = f2u(a.off) - 2u * kBias;
    Args scoring_args{};
    scoring_args.cap = a.cap; scoring_args.off = a.off; scoring_args.slopes = a.slopes;
    const Scoring scoring(scoring_args);
    const Full full{a.off, has_off};

    Lane here;
    here.first = lane % L * 4; here.values = a.values;
    here.streams = here.first < a.values;
    if (!here.streams) here.first = 0;
    here.streaming = __ballot(here.streams);
    uint32_t q[ROWS][4];
    float acc[ROWS][4], l[ROWS], M[ROWS];
    bool odd = false;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const RowPlace at = place_of(a, kv, row0 + min(r, here_rows - 1));
        const float* const from = a.q.p + (long)b * a.q.sb + (long)at.token * a.q.st + (long)at.head * a.q.sh;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const bool there = here.streams && here.first + d < a.values;
            const float v = from[there ? here.first + d : 0];
            const uint32_t scaled = (f2u(v) << 1) == 0u ? kStandIn : f2u(v) + (f2u(a.scale) - kBias + off_add);
            const bool out = there && (scaled << 1) - kLaneBase >= kLaneSpan;
            odd = odd || out;
            q[r][d] = there ? scaled + mul_add : lane_pad(0u);
            acc[r][d] = 0.0f;
        }
        l[r] = 0.0f; M[r] = kNothing;
    }
    const bool careful_rows = __ballot(odd) != 0ull;
    const int* const table = a.table + (long)b * a.per_sequence;
    const float* const k = a.k + (long)kv * a.c_sh;
    const float* const v = a.v + (long)kv * a.c_sh;
    uint32_t saw = 0u;                            // a bit for every row

#pragma unroll 1
    for (int j0 = begin + wave * kSpan; j0 < end; j0 += kWaves * kSpan) {
        // a lane per key: where its row lies
        const int j = j0 + lane;
        const bool exists = j < end;
        const KeyPlace place = key_place(a, table, j, exists);
        const bool there = place.there;
        const long at = place.at;
        const auto row_at = [&](int step, long (&out)[kSteps]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int from = (step + i) * keys_a_step + lane / L;
                out[i] = (long)(((uint64_t)(uint32_t)__shfl((int)(at >> 32), from, 64) << 32) | (uint32_t)__shfl((int)at, from, 64));
            }
        };
        v4f rows[kSteps];
        long where[kSteps];
        // scores
#pragma unroll 1
        for (int step = 0; step < L; step += kSteps) {
            row_at(step, where);
            load_rows(k, where, here, rows);
            const bool careful = careful_rows || !ordinary(rows);
#pragma unroll
            for (int i0 = 0; i0 < kSteps; i0 += (ROWS > 8 ? 1 : 2)) {
                constexpr int kTwo = ROWS > 8 ? 1 : 2;
                float s[kTwo * ROWS];
#pragma unroll
                for (int i = 0; i < kTwo; ++i)
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        float sum = 0.0f;
#pragma unroll
                        for (int d = 0; d < 4; ++d) sum += u2f(f2u(rows[i0 + i][d]) + q[r][d]);
                        s[i * ROWS + r] = sum;
                    }
                if (__builtin_expect(careful, 0)) {
#pragma unroll 1
                    for (int n = 0; n < kTwo * ROWS; ++n) {
                        // (the query from memory again, as it is: q has something else in a zero's place; the key's values by selects, so that the array stays in registers)
                        const RowPlace place_of_row = place_of(a, kv, row0 + min(n % ROWS, here_rows - 1));
                        const float* const from = a.q.p + (long)b * a.q.sb + (long)place_of_row.token * a.q.st + (long)place_of_row.head * a.q.sh;
                        float sum = 0.0f;
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            const bool there = here.streams && here.first + d < a.values;
                            uint32_t theirs = f2u(rows[i0][d]);
#pragma unroll
                            for (int i = 1; i < kTwo; ++i) theirs = n / ROWS == i ? f2u(rows[i0 + i][d]) : theirs;
                            const float mine = pam_mul_off(from[there ? here.first + d : 0], a.scale, a.off, has_off);
                            sum += full_product(full, there ? f2u(mine) : 0u, theirs);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        s[0] = sum;
                        turned(s);
                    }
                }
                group_sums(s, L);
                if (lane % L == 0)
#pragma unroll
                    for (int i = 0; i < kTwo; ++i)
#pragma unroll
                        for (int r = 0; r < ROWS; ++r) scores[wave][(step + i0 + i) * keys_a_step + lane / L][r] = s[i * ROWS + r];
            }
        }
        wave_fence();
        // weights: a lane per key
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int token = (row0 + min(r, here_rows - 1)) / a.group;
            const int pos = length + token;
            const bool sees = exists && token < given && j <= pos && (a.window == 0 || j > pos - a.window);
            const float slope = a.slopes ? a.slopes[place_of(a, kv, row0 + min(r, here_rows - 1)).head] : 0.0f;
            float t = scoring.exponent(scores[wave][lane][r], held_slope(slope), pos - j);
            t = there && finite(slope) ? t : u2f(kQNaN);
            float most = sees ? t : kNothing;
            most = most != most ? kNothing : most;
#pragma unroll
            for (int s = 1; s < 64; s *= 2) most = fmaxf(most, __shfl_xor(most, s, 64));
            if (most > M[r] + kLag) {              // (the same in all lanes)
                const float raised = u2f((uint32_t)__builtin_amdgcn_readfirstlane((int)f2u(floorf(most)))), f = scale_between(M[r], raised);
                l[r] *= f;
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[r][d] *= f;
                M[r] = raised;
            }
            const float power = sees ? t - M[r] : 2.0f * kLeast;
            saw |= sees ? 1u << r : 0u;
            const bool in = power >= kLeast;
            const float e = power_of_two(fmaxf(power, kLeast));
            l[r] += in ? e : sees ? t * 0.0f : 0.0f;      // (what is no number makes none of the sum)
            scores[wave][lane][r] = in ? e : 0.0f;
            __builtin_amdgcn_sched_barrier(0);    // (row by row: all of them side by side take the registers of the loops around)
        }
        wave_fence();
        // values
#pragma unroll 1
        for (int step = 0; step < L; step += kSteps) {
            row_at(step, where);
            load_rows(v, where, here, rows);
            const bool careful = !ordinary(rows);
            if (__builtin_expect(careful, 0)) {
#pragma unroll 1
                for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        const float e = scores[wave][(step + i) * keys_a_step + lane / L][r];
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            const float c = full_product(full, f2u(e), f2u(rows[0][d]));
                            acc[r][d] += e > 0.0f ? c : 0.0f;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                    turned(rows);
                }
                continue;
            }
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    const float e = scores[wave][(step + i) * keys_a_step + lane / L][r];
                    const uint32_t weight = e > 0.0f ? f2u(e) + mul_add : 0u;
                    const float one = e > 0.0f ? 1.0f : 0.0f;
#pragma unroll
                    for (int d = 0; d < 4; ++d) acc[r][d] = __builtin_fmaf(u2f(f2u(rows[i][d]) + weight), one, acc[r][d]);
                }
        }
        wave_fence();                             // (the next span's scores go where these weights are)
    }

    finish<ROWS>(a, me, acc, l, M, saw, sums, stats);
}

// ---------------------------------------------------------------- heads of whole quads

// Work-groups that a compute unit has at once, what the registers leave room for.  (The next span's keys asked for before this one's values are added up, in two:
// 16 sequences of up to 4000 tokens 47 us where three take 42; keys read a line by eight lanes and passed on through LDS 49.)
constexpr int groups_at_once(int rows) { return rows <= 4 ? 3 : 2; }
constexpr int kSlice = 8;                         // quads of a key in a lane's registers

// Rows of queries, one after the other: a token's heads of this key head, then the next token's; the last one again behind the last.
struct Queries {
    const char* first; long step, wrap; int group, head0, count;                 // uniform
    __device__ __forceinline__ Queries(const CacheArgs& a, const Share& me)
    {
        const RowPlace at = place_of(a, me.kv, me.row0);
        first = (const char*)(a.q.p + (long)me.b * a.q.sb + (long)at.token * a.q.st + (long)at.head * a.q.sh);
        step = a.q.sh * (long)sizeof(float); wrap = (a.q.st - (a.group - 1) * a.q.sh) * (long)sizeof(float);
        group = a.group; head0 = me.row0 % a.group; count = me.here_rows;
    }
    __device__ __forceinline__ const char* after(const char* at, int& head, int r) const          // row r + 1, at being row r and `head` its head
    {
        const bool over = head + 1 == group;
        const long by = over ? wrap : step;
        head = over ? 0 : head + 1;
        return at + (r + 1 < count ? by : 0l);
    }
};

template <int ROWS, bool WHOLE>
__global__ __launch_bounds__(kThreads, groups_at_once(ROWS)) void cached_rows_kernel(CacheArgs a)
{
    constexpr int kAhead = ROWS <= 4 ? 8 : 4;     // rows of values that a lane has on their way
    constexpr int kPad = ROWS < 4 ? ROWS : (ROWS + 3) / 4 * 4;
    __shared__ float weights[kWaves][kSpan][kPad];                               // a key's, of all rows: bits(weight) + mul_add
    __shared__ float sums[ROWS][256 + 4];
    __shared__ float2 stats[kWaves][ROWS];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), L = a.lanes, keys_a_step = 64 / L, quads = a.values / 4;
    const Share me(a, ROWS);
    if (me.here_rows <= 0) return;
    const bool has_off = a.off != 1.0f;
    Args scoring_args{};
    scoring_args.cap = a.cap; scoring_args.off = a.off; scoring_args.slopes = a.slopes;
    const Scoring scoring(scoring_args);
    const Full full{a.off, has_off};
    const uint32_t scale_add = f2u(a.scale) - kBias + scoring.off_add, key_add = scale_add + scoring.mul_add, mul_add = scoring.mul_add, none = kStandIn + mul_add;
    const Queries queries(a, me);
    const int* const table = a.table + (long)me.b * a.per_sequence;
    const float* const k = a.k + (long)me.kv * a.c_sh;
    const float* const v = a.v + (long)me.kv * a.c_sh;
    // the first span's keys are on their way before anything waits
    const auto load_keys = [&](long at, int slice, v4f (&x)[kSlice]) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < kSlice; ++n) x[n] = *reinterpret_cast<const v4f_any*>(k + at + 4 * (WHOLE ? slice * kSlice + n : min(slice * kSlice + n, quads - 1)));
    };
    const auto place_of_span = [&](int j0) __attribute__((always_inline)) { return key_place(a, table, max(0, min(j0 + lane, me.end - 1)), me.begin < me.end); };      // (behind the last key that one again)
    KeyPlace place = place_of_span(me.begin + wave * kSpan);
    v4f next[kSlice];
    load_keys(place.at, 0, next);
    // the queries, scaled, have to be in the streamed values' window; zeros are left out by factors
    bool q_zeros = false, q_wild = false;
    for (int i = threadIdx.x; i < me.here_rows * quads; i += kThreads) {
        const RowPlace at = place_of(a, me.kv, me.row0 + i / quads);
        const v4f x = *reinterpret_cast<const v4f_any*>(a.q.p + (long)me.b * a.q.sb + (long)at.token * a.q.st + (long)at.head * a.q.sh + i % quads * 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const bool zero = (f2u(x[c]) << 1) == 0u;
            q_zeros = q_zeros || zero;
            q_wild = q_wild || (!zero && ((f2u(x[c]) + scale_add) << 1) - kStreamBase >= kStreamSpan);
        }
    }
    q_zeros = __syncthreads_or(q_zeros) != 0; q_wild = __syncthreads_or(q_wild) != 0;

    float acc[ROWS][4], l[ROWS], M[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        l[r] = 0.0f; M[r] = kNothing;
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[r][d] = 0.0f;
    }
    const int own = min(lane % L, quads - 1) * 4;                                // of a row of values
    const bool streams = lane % L < quads;
    uint32_t saw = 0u;                            // a bit for every row

#pragma unroll 1
    for (int j0 = me.begin + wave * kSpan; j0 < me.end; j0 += kWaves * kSpan) {
        const int j = j0 + lane;
        const bool exists = j < me.end;
        const auto row_at = [&](int step, long (&out)[kAhead]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int from = (step + i) * keys_a_step + lane / L;
                out[i] = (long)(((uint64_t)(uint32_t)__shfl((int)(place.at >> 32), from, 64) << 32) | (uint32_t)__shfl((int)place.at, from, 64));
            }
        };
        const auto load_values = [&](int step, v4f (&x)[kAhead]) __attribute__((always_inline)) {
            long where[kAhead];
            row_at(min(step, L - kAhead), where);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) x[i] = *reinterpret_cast<const v4f_any*>(v + where[i] + own);
        };
        // scores
        float s[ROWS];
        bool left_out = false;                    // a key that a row does not see, or one whose weight is none
#pragma unroll
        for (int r = 0; r < ROWS; ++r) s[r] = 0.0f;
        const int slices = (quads + kSlice - 1) / kSlice;
        uint32_t odd = 0u;
#pragma unroll 1
        for (int slice = 0; slice < slices; ++slice) {
            uint32_t mine[4 * kSlice];
#pragma unroll
            for (int n = 0; n < kSlice; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t x = f2u(next[n][c]);
                    x = (x << 1) == 0u || (!WHOLE && slice * kSlice + n >= quads) ? kStandIn : x;
                    odd = max(odd, (x << 1) - kLaneBase);
                    mine[4 * n + c] = x + key_add;
                }
            if (slice + 1 < slices) load_keys(place.at, slice + 1, next);
            const Stream<WHOLE> layout(nullptr, 0, 1, WHOLE ? 0 : slice * kSlice, quads);
            const char* row = queries.first + (WHOLE ? slice * kSlice * 16l : 0l);
            int head = queries.head0;
            Piece now = piece_of<4, WHOLE>(layout, (const float*)row, 0);
            if (__builtin_expect(!q_zeros, 1)) {
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    const char* const after = queries.after(row, head, r);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        asm volatile("" ::"s"(now.a));
                        __builtin_amdgcn_sched_barrier(0);
                        const Piece later = h == 0 ? piece_of<4, WHOLE>(layout, (const float*)row, 4) : piece_of<4, WHOLE>(layout, (const float*)after, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        dot_piece<16>(now, mine + 16 * h, s[r]);
                        __builtin_amdgcn_sched_barrier(0);
                        now = later;
                    }
                    row = after;
                }
            } else {
#pragma unroll 1
                for (int r = 0; r < ROWS; ++r) {
                    dot_piece_with_zeros<16, false>(now, mine, Zeros{}, s[0]);
                    now = piece_of<4, WHOLE>(layout, (const float*)row, 4);
                    dot_piece_with_zeros<16, false>(now, mine + 16, Zeros{}, s[0]);
                    row = queries.after(row, head, r);
                    now = piece_of<4, WHOLE>(layout, (const float*)row, 0);
                    turned(s);
                }
            }
        }
        if (__builtin_expect(q_wild || __ballot(odd >= kLaneSpan) != 0ull, 0)) {
            // the full definition
            const char* row = queries.first;
            int head = queries.head0;
#pragma unroll 1
            for (int r = 0; r < ROWS; ++r) {
                s[0] = 0.0f;
#pragma unroll 1
                for (int d = 0; d < a.values; ++d) {
                    const float query = reinterpret_cast<const float*>(row)[d];
                    s[0] += full_product(full, f2u(pam_mul_off(query, a.scale, a.off, has_off)), f2u(k[place.at + d]));
                }
                row = queries.after(row, head, r);
                turned(s);
            }
        }
        v4f rows[kAhead];
        load_values(0, rows);
        const KeyPlace after = place_of_span(j0 + kWaves * kSpan);               // (the table is read while the values are)
        // weights: a lane per key
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int token = (me.row0 + min(r, me.here_rows - 1)) / a.group, pos = me.length + token;
            const bool sees = exists && token < me.given && j <= pos && (a.window == 0 || j > pos - a.window);
            const float slope = a.slopes ? a.slopes[place_of(a, me.kv, me.row0 + min(r, me.here_rows - 1)).head] : 0.0f;
            float t = scoring.exponent(s[r], held_slope(slope), pos - j);
            t = place.there && finite(slope) ? t : u2f(kQNaN);
            float most = sees ? t : kNothing;
            most = most != most ? kNothing : most;
            if (__ballot(most > M[r] + kLag) != 0ull) {
#pragma unroll
                for (int n = 1; n < 64; n *= 2) most = fmaxf(most, __shfl_xor(most, n, 64));
                const float raised = u2f((uint32_t)__builtin_amdgcn_readfirstlane((int)f2u(floorf(most)))), f = scale_between(M[r], raised);
                l[r] *= f;
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[r][d] *= f;
                M[r] = raised;
            }
            const float power = sees ? t - M[r] : 2.0f * kLeast;
            saw |= sees ? 1u << r : 0u;
            const bool in = power >= kLeast;
            const float e = power_of_two(fmaxf(power, kLeast));
            l[r] += in ? e : sees ? t * 0.0f : 0.0f;      // (what is no number makes none of the sum)
            // (one that does not count stands as 2^-86, which no weight is; a factor leaves its products out, since a value that is not seen may be of any size)
            weights[wave][lane][r] = u2f((in ? f2u(e) : kStandIn) + mul_add);
            left_out = left_out || !in;
            __builtin_amdgcn_sched_barrier(0);    // (row by row: all of them side by side take the registers of the loops around)
        }
        wave_fence();
        const bool factors = __ballot(left_out) != 0ull;
        // values
#pragma unroll 1
        for (int step = 0; step < L; step += kAhead) {
            v4f later[kAhead];
            load_values(step + kAhead, later);
            uint32_t most = 0u;
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
                for (int d = 0; d < 4; ++d) most = max(most, (f2u(rows[i][d]) << 1) - kStreamBase);
            if (__builtin_expect((__ballot(most >= kStreamSpan && streams)) != 0ull, 0)) {
                // zeros are left out by factors, anything else takes the full definition
                bool odd_value = false;
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
#pragma unroll
                    for (int d = 0; d < 4; ++d) odd_value = odd_value || ((f2u(rows[i][d]) << 1) != 0u && (f2u(rows[i][d]) << 1) - kStreamBase >= kStreamSpan);
                const bool wild = __ballot(odd_value && streams) != 0ull;
#pragma unroll 1
                for (int i = 0; i < kAhead; ++i) {
                    const float* const of = weights[wave][(step + i) * keys_a_step + lane / L];
                    if (!wild) {
                        v4f x = rows[0], f;
#pragma unroll
                        for (int d = 0; d < 4; ++d) { f[d] = (f2u(x[d]) << 1) == 0u ? 0.0f : 1.0f; x[d] = (f2u(x[d]) << 1) == 0u ? 1.0f : x[d]; }
#pragma unroll
                        for (int r = 0; r < ROWS; ++r)
#pragma unroll
                            for (int d = 0; d < 4; ++d) acc[r][d] = __builtin_fmaf(u2f(f2u(x[d]) + f2u(of[r])), f2u(of[r]) == none ? 0.0f : f[d], acc[r][d]);
                    } else {
#pragma unroll 1
                        for (int r = 0; r < ROWS; ++r) {
                            const uint32_t weight = f2u(of[r]) - mul_add;
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                const float c = full_product(full, weight, f2u(rows[0][d]));
#pragma unroll
                                for (int n = 0; n < ROWS; ++n) acc[n][d] += n == r && weight != kStandIn ? c : 0.0f;
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                    }
                    turned(rows);
                }
            } else if (factors) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const float* const of = weights[wave][(step + i) * keys_a_step + lane / L];
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        const float one = f2u(of[r]) == none ? 0.0f : 1.0f;
#pragma unroll
                        for (int d = 0; d < 4; ++d) acc[r][d] = __builtin_fmaf(u2f(f2u(rows[i][d]) + f2u(of[r])), one, acc[r][d]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const float* const of = weights[wave][(step + i) * keys_a_step + lane / L];
#pragma unroll
                    for (int r = 0; r < ROWS; ++r)
#pragma unroll
                        for (int d = 0; d < 4; ++d) acc[r][d] += u2f(f2u(rows[i][d]) + f2u(of[r]));
                }
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) rows[i] = later[i];
        }
        wave_fence();                             // (the next span's weights go where these are)
        place = after;
        load_keys(place.at, 0, next);
    }
    if (!streams)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[r][d] = 0.0f;
    finish<ROWS>(a, me, acc, l, M, saw, sums, stats);
}

// The parts of a query's head, one work-group each: lanes along its quads, the rest of the threads along the parts.
__global__ __launch_bounds__(kThreads) void cached_join_kernel(CacheArgs a)
{
    __shared__ v4f sums[kThreads];
    __shared__ float scales[kMostParts], tops[kWaves], totals[kWaves];
    const int quads = (a.values + 3) / 4, row = (int)blockIdx.x % a.rows, head_at = (int)blockIdx.x / a.rows, b = head_at / a.kv_heads, kv = head_at % a.kv_heads;
    const int row0 = row / a.rows_each * a.rows_each;
    const Cut cut = cut_of(a, row0, min(a.rows_each, a.rows - row0), false, b);
    const auto at_part = [&](int p) { return ((long)kv * a.batch * a.parts + cut.first + p) * a.rows + row; };
    float2 mine[kMostParts / kThreads];
    float M = kNothing;
#pragma unroll
    for (int i = 0; i < kMostParts / kThreads; ++i) {
        const int p = (int)threadIdx.x + i * kThreads;
        mine[i] = p < cut.parts ? a.partial_stats[at_part(p)] : make_float2(0.0f, kNothing);
        M = fmaxf(M, mine[i].y);
    }
    for (int s = 1; s < 64; s *= 2) M = fmaxf(M, __shfl_xor(M, s, 64));
    if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, tops[w]);
    float part_sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kMostParts / kThreads; ++i) {
        const int p = (int)threadIdx.x + i * kThreads;
        const float f = mine[i].y == kNothing ? 0.0f : scale_between(mine[i].y, M);
        if (p < cut.parts) scales[p] = f;
        part_sum += mine[i].y == kNothing ? 0.0f : mine[i].x * f;
    }
    for (int s = 1; s < 64; s *= 2) part_sum += __shfl_xor(part_sum, s, 64);
    if (threadIdx.x % 64 == 0) totals[threadIdx.x / 64] = part_sum;
    __syncthreads();
    int columns = 1;                              // lanes along the quads: a power of two
    while (columns < quads) columns *= 2;
    const int column = threadIdx.x % columns, shares = kThreads / columns, share = threadIdx.x / columns;
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (column < quads)
#pragma unroll 4
        for (int p = share; p < cut.parts; p += shares) {
            const v4f x = *reinterpret_cast<const v4f*>(a.partial + at_part(p) * quads * 4 + column * 4);
            const float f = scales[p];
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += f != 0.0f ? x[c] * f : 0.0f;
        }
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (share != 0 || column >= quads) return;
    float total = 0.0f;
    for (int w = 0; w < kWaves; ++w) total += totals[w];
    for (int s = 1; s < shares; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] += sums[s * columns + column][c];
    const RowPlace at = place_of(a, kv, row);
    float* const to = a.y + (((long)b * a.tokens + at.token) * a.heads + at.head) * a.values + column * 4;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (column * 4 + c < a.values) to[c] = M == kNothing ? 0.0f : pad_div_off(sum[c], total, a.off, a.off != 1.0f);
}

// ---------------------------------------------------------------- host

// Rows of a work-group, how many work-groups the rows of a key head take, lanes of a group, parts of a sequence.
struct CachePlan { int rows_each, sets, lanes, parts; };
CachePlan cache_plan(long batch, long heads, long rows, long values, long capacity)
{
    CachePlan p;
    if (values % 4 != 0) p.rows_each = rows <= 1 ? 1 : 4;
    else {
        // (rows in as few sets as there can be, of one size)
        const long sets = (rows + kMostRows - 1) / kMostRows, each = (rows + sets - 1) / std::max(1L, sets);
        p.rows_each = each <= 1 ? 1 : each <= 2 ? 2 : (int)((each + 3) / 4 * 4);
    }
    p.sets = (int)((rows + p.rows_each - 1) / p.rows_each);
    p.lanes = values % 4 ? 4 : 8;
    while (p.lanes * 4 < values) p.lanes *= 2;
    // (the work-groups that 256 compute units have at once; a part of less than a span for each wavefront is not worth a second kernel)
    const long units = std::max(1L, heads * p.sets), wanted = 256 * groups_at_once(p.rows_each) / units, most = (capacity + kWaves * kSpan - 1) / (kWaves * kSpan);
    p.parts = (int)std::max(1L, std::min({wanted, most, (long)kMostParts / std::max(1L, std::min(batch, 64L))}));
    return p;
}
long padded(long values) { return (values + 3) / 4 * 4; }
size_t cache_bytes(const CachePlan& p, long heads, long rows, long values)
{
    if (p.parts == 1) return 0;
    const size_t n = (size_t)heads * rows * p.parts;
    return (n * sizeof(float2) + 255) / 256 * 256 + n * padded(values) * sizeof(float);
}

int check_cache(const char* what, const pam_hip_cache_shape* s)
{
    if (!s) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: null pointer", what);
    if (s->batch < 0 || s->tokens < 0 || s->heads < 0 || s->kv_heads < 0 || s->pages < 0 || s->per_sequence < 0 || s->window < 0)
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: negative size", what);
    if (s->dim < 1 || s->dim > 256) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: heads have up to 256 values, got %ld", what, s->dim);
    if (s->kv_heads == 0 ? s->heads != 0 : s->heads % s->kv_heads != 0)
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: %ld heads do not share %ld", what, s->heads, s->kv_heads);
    if (s->page < 1 || s->page > (1L << 20) || s->pages > (1L << 30) || s->per_sequence > (1L << 30) || s->batch > (1L << 20) || s->heads > (1L << 16)
        || s->tokens > (1L << 20) || s->batch * s->heads > (1L << 20) || s->batch * s->heads * s->tokens > (1L << 23))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: size out of range", what);
    if (s->per_sequence * s->page > (1L << 30)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the table of pages has up to 2^30 places", what);
    if (!(s->scale > 0x1p-40f && s->scale < 0x1p40f)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the scale lies between 2^-40 and 2^40", what);
    if (s->cap != 0.0f && !(s->cap > 0x1p-20f && s->cap < 0x1p20f)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the cap lies between 2^-20 and 2^20", what);
    if (!(s->offset > 0.75f && s->offset < 1.5f)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "%s: the offset lies between 0.75 and 1.5", what);
    return PAM_HIP_OK;
}

}  // namespace

extern "C" {

size_t pam_hip_cached_attention_workspace_bytes(const pam_hip_cache_shape* s)
{
    if (check_cache("cached_attention", s) != PAM_HIP_OK || s->batch * s->heads * s->tokens == 0) return 0;
    const long heads = s->batch * s->kv_heads, rows = s->heads / s->kv_heads * s->tokens;
    return cache_bytes(cache_plan(s->batch, heads, rows, s->dim, s->per_sequence * s->page), heads, rows, s->dim);
}

int pam_hip_cached_attention_fwd(const pam_hip_cache_shape* s, const pam_hip_tokens* q, const float* cache_k, const float* cache_v, long cache_sp, long cache_st,
                                 long cache_sh, const int* pages, const long long* lengths, const long long* counts, float* y, void* workspace, size_t workspace_bytes,
                                 void* stream)
{
    const int rc = check_cache("cached_attention", s);
    if (rc != PAM_HIP_OK || s->batch * s->heads * s->tokens == 0) return rc;
    // (without pages every key is one that is not there; it is not read, but an address is computed)
    if (!q || !q->p || !y || !lengths || (s->per_sequence && !pages) || (s->pages && (!cache_k || !cache_v)))
        return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "cached_attention: null pointer");
    CacheArgs a{};
    a.q = Tokens{q->p, q->sb, q->st, q->sh};
    a.k = s->pages ? cache_k : q->p; a.v = s->pages ? cache_v : q->p;
    a.c_sp = cache_sp; a.c_st = cache_st; a.c_sh = s->pages ? cache_sh : 0;
    a.table = pages; a.lengths = lengths; a.counts = counts; a.slopes = s->slopes; a.y = y;
    a.batch = (int)s->batch; a.tokens = (int)s->tokens; a.heads = (int)s->heads; a.kv_heads = (int)s->kv_heads; a.group = (int)(s->heads / s->kv_heads);
    a.values = (int)s->dim; a.rows = a.group * a.tokens;
    a.page = (int)s->page; a.pages = (int)s->pages; a.per_sequence = (int)s->per_sequence; a.capacity = (int)(s->per_sequence * s->page); a.window = (int)std::min(s->window, 1L << 30);
    a.scale = s->scale; a.cap = s->cap; a.off = s->offset;
    const long heads = s->batch * s->kv_heads;
    const CachePlan p = cache_plan(s->batch, heads, a.rows, a.values, s->per_sequence * s->page);
    a.lanes = p.lanes; a.parts = p.parts; a.sets = p.sets; a.rows_each = p.rows_each;
    const size_t need = cache_bytes(p, heads, a.rows, a.values);
    if (need && (!workspace || workspace_bytes < need)) return pamhost::fail(PAM_HIP_ERR_WORKSPACE, "cached_attention: workspace of %zu bytes needed", need);
    if (need) {
        a.partial_stats = (float2*)workspace;
        a.partial = (float*)((char*)workspace + ((size_t)heads * a.rows * p.parts * sizeof(float2) + 255) / 256 * 256);
    }
    const hipStream_t st = (hipStream_t)stream;
    const long units = heads * p.parts, groups = (units + 7) / 8 * 8 * p.sets;
    if (groups > (1L << 23)) return pamhost::fail(PAM_HIP_ERR_ARGUMENT, "cached_attention: size out of range");
    const dim3 grid((unsigned)groups);
    const bool whole = a.values % (4 * kSlice) == 0;
    Kernel kernel = nullptr;
    if (a.values % 4 != 0) kernel = p.rows_each == 1 ? cached_attention_kernel<1> : cached_attention_kernel<4>;
    else
        switch (p.rows_each) {
        case 1: kernel = whole ? cached_rows_kernel<1, true> : cached_rows_kernel<1, false>; break;
        case 2: kernel = whole ? cached_rows_kernel<2, true> : cached_rows_kernel<2, false>; break;
        case 4: kernel = whole ? cached_rows_kernel<4, true> : cached_rows_kernel<4, false>; break;
        case 8: kernel = whole ? cached_rows_kernel<8, true> : cached_rows_kernel<8, false>; break;
        default: kernel = whole ? cached_rows_kernel<kMostRows, true> : cached_rows_kernel<kMostRows, false>; break;
        }
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, a);
    int done = pamhost::check_launch("cached_attention");
    if (done != PAM_HIP_OK || !need) return done;
    hipLaunchKernelGGL(cached_join_kernel, dim3((unsigned)(heads * a.rows)), dim3(kThreads), 0, st, a);
    return pamhost::check_launch("cached_attention");
}

}  // extern "C"
