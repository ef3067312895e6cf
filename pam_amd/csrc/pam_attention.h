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
// A wavefront's lanes own 64 rows (queries; in the pass for dk and dv, keys), a slice of at most 64 of a row's values (32 in the gradients' passes, which hold
// three or four of them) in a lane's registers, and the other side streams by in scalar registers, that all lanes read: a product takes two
// instructions on 64 lanes, an integer addition and a float addition, and nothing else.  One piece of a streamed row (at most 20 values) is used
// while the next one is on its way, wherever that is: in this row, the next or the next phase's; pieces of 32 took scalar registers from
// everything else (forward 0.94, gradients 0.87 times as fast).  Longer rows are cut into slices with a wavefront each, which add up their parts of
// a score through LDS.  A work-group's wavefronts stream the same rows, so that the scalar cache has them.
// Rates of the inner loop alone, two wavefronts per SIMD: 28 T products/s; with the streamed values read from another lane inside the integer
// addition (a data-parallel primitive: everything around it issues half as fast) 18.6; copied out of one once for four rows 20.5; by lane reads 12.
// Whole passes: forward 18.7 T products/s where every row sees 4096 keys, 15.8 where the order is causal (the last turn of units is not full),
// gradients 13.8 and 10: a sixth to a third of the instructions are the weights', which slices make twice, and two or three wavefronts on a SIMD do not
// cover all waits for the scalar cache.
//
// The integer addition is the product while no exponent leaves the normal range.  Streamed values have to be in 2^[-40, 40), a lane's in 2^(-86, 80).  A
// lane's zero stands as 2^-86, and so does what lies behind a head's values: next to nothing in a score, and beside products that the sum has besides.  Where it may
// have none such: sums of approximate gradients that are that small make their unit begin again (below); exact slopes, which take the fraction of a score, have a lane with zeros
// in the loop that streamed rows with zeros take, which leaves those out by a factor.  Values in front of the places behind a head's are at least 2^28 times what stands there.
// With anything else in a streamed row, or in a lane's, a unit begins again with the full definition (`careful`), its lanes' rows read again as they are: kept apart
// from the usual loops, because side by side with them it took their registers.
// Every value of a block is looked at for that by one lane, with vector loads of its own.
#pragma once
#include "pam_activation.h"
#include "pam_common.h"
#include "../../include/pam_hip_attention.h"

namespace pamatt {
using namespace pamdev;

constexpr int kThreads = 256, kWaves = 4;         // (of the small kernels and of a cache's)
constexpr int kBlock = 8;                         // streamed rows at a time
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
    int windows;                                  // chunks begin where the window of a tile's first row does (in whole spans), else at row 0
    // forward
    float* y;                                     // [batch][tokens][heads][dim]
    float2* stats;                                // l and M, [batch][tokens][heads], or null
    float* partial; float2* partial_stats;        // [batch][kv_heads][chunks][rows][dim], [...][rows]; or null: chunks is 1
    // backward
    const float4* records;                        // [batch][kv_heads][rows]: M (+inf: the row sees nothing), dl, largest exponent of dn, slope
    const float* qs; const float* dn;             // [batch][kv_heads][rows][dim]
    float* out0; float* out1;                     // [batch][kv_heads][chunks][lanes' rows][dim]: dq, or dk and dv
    unsigned char* met;                           // [batch][kv_heads][chunks][tiles of 64 rows]: a tile saw something of a chunk
    int whole;                                    // ... or, of one chunk, the gradients themselves, [batch][tokens][heads][dim] and [batch][keys][kv_heads][dim]
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

constexpr uint32_t kStreamBase = (uint32_t)(127 - 40) << 24, kStreamSpan = 80u << 24;      // 2^[-40, 40) of bits << 1
constexpr uint32_t kLaneBase = (uint32_t)(127 - 86) << 24, kLaneSpan = 166u << 24;         // 2^[-86, 80)
constexpr uint32_t kStandIn = (uint32_t)(127 - 86) << 23;

// (comparisons with it are made where they are used, instead of kept from the beginning of a kernel to its end)
__device__ __forceinline__ int anew(int v) { asm volatile("" : "+v"(v)); return v; }
// (a lane's value, taken apart where it is used and not, for all rows, before the loop)
__device__ __forceinline__ uint32_t plain(uint32_t mine) { return (uint32_t)anew((int)mine); }

__device__ __forceinline__ uint32_t lane_pad(uint32_t shift) { return shift - kBias; }

template <int N, class T> __device__ __forceinline__ void turned(T (&v)[N])      // all one place down, the first to the end
{
    const T first = v[0];
#pragma unroll
    for (int i = 0; i + 1 < N; ++i) v[i] = v[i + 1];
    v[N - 1] = first;
}

// How a lane's values are held: they have to be in 2^(least, top); a zero and what lies behind the row's values have bits that no such value has.  ones: from that value of
// a quad on, what streams by behind the values is ones (keys and values of heads that are no whole quads); the products with those are zeros to the bit.
constexpr uint32_t bits_of_power(int e) { return (uint32_t)(127 + e) << 23; }
struct Form {
    int least, top; uint32_t zero, behind; int ones = 4;
    static __device__ __forceinline__ Form plain() { return Form{-86, 80, kStandIn, kStandIn}; }
};
// What a lane found in its part of a row: a value out of the window, a zero, anything but zeros.
struct Held { bool odd, zeros, numbers; };
// A lane's part of a row: bits(value) + scale + add, zeros and what lies behind the row's values stood in for (unscaled).  scale: of a factor in 2^[-41, 41];
// factor: a power of two of any size, multiplied (an addition to the bits would take what is far below it through the sign).
template <int W4>
__device__ __forceinline__ Held load_lane(const float* row, int first, int dim, int values, uint32_t scale, uint32_t add, uint32_t (&out)[4 * W4], const Form& form, float factor = 1.0f)
{
    uint32_t most = 0u;
    bool zeros = false, numbers = false;
    first = anew(first);
    const uint32_t base = ((uint32_t)(127 + form.least) << 24) + 2u;
#pragma unroll
    for (int n = 0; n < W4; ++n) {
        const v4f x = *reinterpret_cast<const v4f_any*>(row + min(first + 4 * n, dim - 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool behind = first + 4 * n + i >= values, zero = (f2u(x[i]) << 1) == 0u;
            const uint32_t b = f2u(x[i] * factor) + scale;
            most = max(most, zero || behind ? 0u : (b << 1) - base);
            zeros = zeros || (zero && !behind);
            numbers = numbers || !(zero || behind);
            out[4 * n + i] = behind && i >= form.ones ? lane_pad(0u) : (behind ? form.behind : zero ? form.zero : b) + add;
        }
    }
    return Held{most >= ((uint32_t)(form.top - form.least) << 24) - 2u, zeros, numbers};
}
// ... as the full definition takes it: the values themselves, zeros behind the row's
template <int W4, class Value>
__device__ __forceinline__ void load_plain(int first, int values, uint32_t (&out)[4 * W4], Value&& value)
{
#pragma unroll 1
    for (int d = 0; d < 4 * W4; ++d) {
        out[0] = first + d < values ? f2u(value(first + d)) : 0u;
        turned(out);
    }
}

// ---------------------------------------------------------------- streamed rows

typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f16_any __attribute__((ext_vector_type(16), aligned(4)));
typedef float f8_any __attribute__((ext_vector_type(8), aligned(4)));

// Rows of one head, of which a slice takes the quads first ... first + W4 - 1.  Where a row has fewer, the last one stands for the missing: lanes hold nothing there.
template <bool WHOLE> struct Stream {
    const float* p; long st, bytes; int last, first, quads;   // uniform; bytes: st as such; p: where the slice begins in row 0, or, not WHOLE, that row; quads: of a row
    __device__ __forceinline__ Stream(const float* base, long stride, int rows, int first_quad, int row_quads)
        : p(WHOLE ? base + 4 * first_quad : base), st(stride), bytes(stride * (long)sizeof(float)), last(rows - 1), first(first_quad), quads(row_quads) {}
    __device__ __forceinline__ const float* row(int j) const { return p + (long)min(j, last) * st; }
    __device__ __forceinline__ const float* after(const float* at, int j) const { return (const float*)((const char*)at + (j < last ? bytes : 0l)); }      // row j + 1, at being row j
    __device__ __forceinline__ int quad(int n) const { return WHOLE ? n : min(first + n, quads - 1); }
    // a lane of each sixteen has a quad
    template <int W4> __device__ __forceinline__ v4f across(int j) const
    { return *reinterpret_cast<const v4f_any*>(row(j) + 4 * quad(min((int)threadIdx.x % 16, W4 - 1))); }
};

// Q quads of a row in scalar registers.
struct Piece { f16v a; v4f b; };
template <int Q, bool WHOLE> __device__ __forceinline__ Piece piece_of(const Stream<WHOLE>& s, const float* row, int quad)
{
    typedef const __attribute__((address_space(4))) f16_any* P16;
    typedef const __attribute__((address_space(4))) f8_any* P8;
    typedef const __attribute__((address_space(4))) v4f_any* P4;
    Piece x;
    if constexpr (WHOLE) {
        const float* const p = row + 4 * quad;
        static_assert(Q >= 3 && Q <= 5);
        if constexpr (Q >= 4) x.a = *(P16)p;
        if constexpr (Q == 5) x.b = *(P4)(p + 16);
        if constexpr (Q == 3) {
            const f8_any y = *(P8)p; const v4f z = *(P4)(p + 8);
            const auto w = __builtin_shufflevector(z, z, 0, 1, 2, 3, 0, 1, 2, 3);
            x.a = __builtin_shufflevector(y, w, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 8, 9, 10, 11);
        }
    } else {
#pragma unroll
        for (int n = 0; n < Q; ++n) {
            const v4f z = *(P4)(row + 4 * s.quad(quad + n));
#pragma unroll
            for (int i = 0; i < 4; ++i) { if (n < 4) x.a[n * 4 + i] = z[i]; else x.b[i] = z[i]; }
        }
    }
    return x;
}
__device__ __forceinline__ float at(const Piece& x, int i) { return i < 16 ? x.a[i] : x.b[i - 16]; }

// Blocks of rows by pieces.  What asks for a phase's last piece asks for the next phase's first one.
template <int W4, bool WHOLE> struct Pipe {
    static constexpr int kPieces = W4 > 10 ? W4 / 4 : W4 > 5 ? 2 : 1, kQuads = W4 / kPieces;
    static_assert(kPieces * kQuads == W4);
    Piece now;
    const float* at;                              // the row that it is of
    __device__ __forceinline__ void request(const Stream<WHOLE>& s, int j) { at = s.row(j); now = piece_of<kQuads, WHOLE>(s, at, 0); }
    // f(row of the block, first value, piece) for the rows j1 ... j1 + 7 of s, whose first piece is asked for; then comes row j2 of `next`.
    // rolled: f gets row 0 every time and turns its arrays around
    template <class F> __device__ __forceinline__ void rolled(const Stream<WHOLE>& s, int j1, const Stream<WHOLE>& next, int j2, F&& f)
    {
#pragma unroll 1
        for (int j = 0; j < kBlock; ++j)
#pragma unroll
            for (int h = 0; h < kPieces; ++h) {
                const Piece x = piece_of<kQuads, WHOLE>(s, s.row(j1 + j), h * kQuads);
                f(h, h * kQuads * 4, x);
            }
        request(next, j2);
    }
    template <class F> __device__ __forceinline__ void block(const Stream<WHOLE>& s, int j1, const Stream<WHOLE>& next, int j2, F&& f)
    {
#pragma unroll
        for (int j = 0; j < kBlock; ++j) {
            const float* const after = j + 1 < kBlock ? s.after(at, j1 + j) : next.row(j2);
#pragma unroll
            for (int h = 0; h < kPieces; ++h) {
                if constexpr (kQuads > 4) asm volatile("" ::"s"(now.a), "s"(now.b));          // (the wait for it, before the next one is asked for: loads of this kind
                else asm volatile("" ::"s"(now.a));                                           // come back in any order, so that a wait is for all of them)
                __builtin_amdgcn_sched_barrier(0);
                const Piece later = h + 1 < kPieces ? piece_of<kQuads, WHOLE>(s, at, (h + 1) * kQuads) : piece_of<kQuads, WHOLE>(j + 1 < kBlock ? s : next, after, 0);
                __builtin_amdgcn_sched_barrier(0);
                f(j, h * kQuads * 4, now);
                __builtin_amdgcn_sched_barrier(0);
                now = later;
            }
            at = after;
        }
    }
};

// Eight values of a piece with eight of a lane's at a time, and what remains by four.  Written as instructions: the compiler gave each product the
// register of the one before, and the order below keeps dependent ones apart.
#define PAM_T8 [t0] "=&v"(t[0]), [t1] "=&v"(t[1]), [t2] "=&v"(t[2]), [t3] "=&v"(t[3]), [t4] "=&v"(t[4]), [t5] "=&v"(t[5]), [t6] "=&v"(t[6]), [t7] "=&v"(t[7])
#define PAM_T4 [t0] "=&v"(t[0]), [t1] "=&v"(t[1]), [t2] "=&v"(t[2]), [t3] "=&v"(t[3])
#define PAM_S4(n) [s0] "s"(at(x, n)), [s1] "s"(at(x, n + 1)), [s2] "s"(at(x, n + 2)), [s3] "s"(at(x, n + 3))
#define PAM_S8(n) PAM_S4(n), [s4] "s"(at(x, n + 4)), [s5] "s"(at(x, n + 5)), [s6] "s"(at(x, n + 6)), [s7] "s"(at(x, n + 7))
#define PAM_M4(n) [m0] "v"(m[n]), [m1] "v"(m[n + 1]), [m2] "v"(m[n + 2]), [m3] "v"(m[n + 3])
#define PAM_M8(n) PAM_M4(n), [m4] "v"(m[n + 4]), [m5] "v"(m[n + 5]), [m6] "v"(m[n + 6]), [m7] "v"(m[n + 7])
#define PAM_O4(n) [o0] "+v"(o[n]), [o1] "+v"(o[n + 1]), [o2] "+v"(o[n + 2]), [o3] "+v"(o[n + 3])
#define PAM_O8(n) PAM_O4(n), [o4] "+v"(o[n + 4]), [o5] "+v"(o[n + 5]), [o6] "+v"(o[n + 6]), [o7] "+v"(o[n + 7])
#define PAM_EACH4(op) op("0") op("1") op("2") op("3")
#define PAM_EACH8(op) PAM_EACH4(op) op("4") op("5") op("6") op("7")
// the product of a streamed value and a lane's, of a streamed one and the lane's weight, of the lane's weight and a lane's
#define PAM_OF_ROW(i) "v_add_u32 %[t" i "], %[s" i "], %[m" i "]\n"
#define PAM_OF_WEIGHT(i) "v_add_u32 %[t" i "], %[s" i "], %[w]\n"
#define PAM_OF_LANE(i) "v_add_u32 %[t" i "], %[w], %[m" i "]\n"
#define PAM_POWER(i) "v_and_b32 %[t" i "], %[mask], %[t" i "]\n"
#define PAM_SUM(i) "v_add_f32 %[sum], %[sum], %[t" i "]\n"
#define PAM_SUM_BY_LANE(i) "v_fmac_f32 %[sum], %[t" i "], %[m" i "]\n"
#define PAM_SUM_BY_ROW(i) "v_fmac_f32 %[sum], %[s" i "], %[t" i "]\n"
#define PAM_ADD(i) "v_fmac_f32 %[o" i "], %[f], %[t" i "]\n"
#define PAM_ADD_BY_ROW(i) "v_fmac_f32 %[o" i "], %[s" i "], %[t" i "]\n"

// sum over d of row (*) lane: `m` as load_lane left it with add = bits(offset) - 2 bias
template <int N> __device__ __forceinline__ void dot_piece(const Piece& x, const uint32_t* m, float& sum)
{
    float t[8];
#pragma unroll
    for (int n = 0; n + 8 <= N; n += 8) asm(PAM_EACH8(PAM_OF_ROW) PAM_EACH8(PAM_SUM) : [sum] "+v"(sum), PAM_T8 : PAM_S8(n), PAM_M8(n));
    if constexpr (N % 8 != 0) asm(PAM_EACH4(PAM_OF_ROW) PAM_EACH4(PAM_SUM) : [sum] "+v"(sum), PAM_T4 : PAM_S4(N - 4), PAM_M4(N - 4));
}
// out_d += f * (weight (*) row's d), the weight's bits with that added, f 0 or 1
template <int N> __device__ __forceinline__ void add_piece(const Piece& x, uint32_t w, float f, float* o)
{
    float t[8];
#pragma unroll
    for (int n = 0; n + 8 <= N; n += 8) asm(PAM_EACH8(PAM_OF_WEIGHT) PAM_EACH8(PAM_ADD) : PAM_O8(n), PAM_T8 : PAM_S8(n), [w] "v"(w), [f] "v"(f));
    if constexpr (N % 8 != 0) asm(PAM_EACH4(PAM_OF_WEIGHT) PAM_EACH4(PAM_ADD) : PAM_O4(N - 4), PAM_T4 : PAM_S4(N - 4), [w] "v"(w), [f] "v"(f));
}

// ... of a row with zeros, whose products count for nothing; so do a lane's, of which `lane` has what stands for them (with `add`)
struct Zeros { uint32_t zero, behind; };
// Lanes whose zeros stand as 2^ZERO and what lies behind as 2^BEHIND: whether there are zeros, and `add`.
template <int ZERO, int BEHIND> struct LaneZeros {
    static constexpr bool kLanes = true;
    int any; uint32_t add;
    __device__ __forceinline__ Zeros codes() const
    {
        uint32_t from = add;
        asm volatile("" : "+s"(from));            // (made where they are used: all the time they would take scalar registers from the usual loops)
        return Zeros{bits_of_power(ZERO) + from, bits_of_power(BEHIND) + from};
    }
};
struct NoLaneZeros {
    static constexpr bool kLanes = false;
    static constexpr int any = 0;
    __device__ __forceinline__ Zeros codes() const { return Zeros{}; }
};
template <int N, bool LANES> __device__ __forceinline__ void dot_piece_with_zeros(const Piece& x, const uint32_t* m, const Zeros& lane, float& sum)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t mine = LANES ? plain(m[i]) : m[i];
        const bool streamed = (f2u(at(x, i)) << 1) == 0u, none = streamed || (LANES && (mine == lane.zero || mine == lane.behind));
        sum = __builtin_fmaf(u2f((streamed ? kBias : f2u(at(x, i))) + mine), none ? 0.0f : 1.0f, sum);
    }
}
template <int N> __device__ __forceinline__ void add_piece_with_zeros(const Piece& x, uint32_t w, float f, float* o)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool none = (f2u(at(x, i)) << 1) == 0u;
        o[i] = __builtin_fmaf(u2f((none ? kBias : f2u(at(x, i))) + w) * f, none ? 0.0f : 1.0f, o[i]);
    }
}

// By the slopes of the pieces that the factors are in (a slope is a product's power of two over the own factor's, so that it takes the product without its
// mantissa; what it is to be over comes at the end).  mask: of the power, or zero where the product does not count.
// sum over d of power(weight (*) row's d) * lane's d
template <int N> __device__ __forceinline__ void dot_power_piece(const Piece& x, uint32_t w, uint32_t mask, const uint32_t* m, float& sum)
{
    float t[8];
#pragma unroll
    for (int n = 0; n + 8 <= N; n += 8)
        asm(PAM_EACH8(PAM_OF_WEIGHT) PAM_EACH8(PAM_POWER) PAM_EACH8(PAM_SUM_BY_LANE) : [sum] "+v"(sum), PAM_T8 : PAM_S8(n), PAM_M8(n), [w] "v"(w), [mask] "v"(mask));
    if constexpr (N % 8 != 0)
        asm(PAM_EACH4(PAM_OF_WEIGHT) PAM_EACH4(PAM_POWER) PAM_EACH4(PAM_SUM_BY_LANE) : [sum] "+v"(sum), PAM_T4 : PAM_S4(N - 4), PAM_M4(N - 4), [w] "v"(w), [mask] "v"(mask));
}
// sum over d of power(weight (*) lane's d) * row's d
template <int N> __device__ __forceinline__ void dot_lane_power_piece(const Piece& x, uint32_t w, uint32_t mask, const uint32_t* m, float& sum)
{
    float t[8];
#pragma unroll
    for (int n = 0; n + 8 <= N; n += 8)
        asm(PAM_EACH8(PAM_OF_LANE) PAM_EACH8(PAM_POWER) PAM_EACH8(PAM_SUM_BY_ROW) : [sum] "+v"(sum), PAM_T8 : PAM_S8(n), PAM_M8(n), [w] "v"(w), [mask] "v"(mask));
    if constexpr (N % 8 != 0)
        asm(PAM_EACH4(PAM_OF_LANE) PAM_EACH4(PAM_POWER) PAM_EACH4(PAM_SUM_BY_ROW) : [sum] "+v"(sum), PAM_T4 : PAM_S4(N - 4), PAM_M4(N - 4), [w] "v"(w), [mask] "v"(mask));
}
// ... with zeros in the lane
template <int N> __device__ __forceinline__ void dot_lane_power_piece_with_zeros(const Piece& x, uint32_t w, uint32_t mask, const uint32_t* m, const Zeros& lane, float& sum)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t mine = plain(m[i]);
        sum = __builtin_fmaf(at(x, i), u2f((w + mine) & (mine == lane.zero || mine == lane.behind ? 0u : mask)), sum);
    }
}
// out_d += f * power(row's d (*) lane's d)
template <int N> __device__ __forceinline__ void add_power_piece(const Piece& x, float f, uint32_t mask, const uint32_t* m, float* o)
{
    float t[8];
#pragma unroll
    for (int n = 0; n + 8 <= N; n += 8)
        asm(PAM_EACH8(PAM_OF_ROW) PAM_EACH8(PAM_POWER) PAM_EACH8(PAM_ADD) : PAM_O8(n), PAM_T8 : PAM_S8(n), PAM_M8(n), [f] "v"(f), [mask] "v"(mask));
    if constexpr (N % 8 != 0)
        asm(PAM_EACH4(PAM_OF_ROW) PAM_EACH4(PAM_POWER) PAM_EACH4(PAM_ADD) : PAM_O4(N - 4), PAM_T4 : PAM_S4(N - 4), PAM_M4(N - 4), [f] "v"(f), [mask] "v"(mask));
}
// ... of a row with zeros, whose slopes are none
template <int N> __device__ __forceinline__ void dot_power_piece_with_zeros(const Piece& x, uint32_t w, uint32_t mask, const uint32_t* m, float& sum)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool none = (f2u(at(x, i)) << 1) == 0u;
        sum = __builtin_fmaf(u2f(((none ? kBias : f2u(at(x, i))) + w) & (none ? 0u : mask)), u2f(m[i]), sum);
    }
}
template <int N> __device__ __forceinline__ void add_power_piece_with_zeros(const Piece& x, float f, uint32_t mask, const uint32_t* m, float* o)
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool none = (f2u(at(x, i)) << 1) == 0u;
        o[i] = __builtin_fmaf(u2f(((none ? kBias : f2u(at(x, i))) + m[i]) & (none ? 0u : mask)), f, o[i]);
    }
}
// out_d += row's d * power(weight (*) lane's d)
template <int N> __device__ __forceinline__ void add_lane_power_piece(const Piece& x, uint32_t w, uint32_t mask, const uint32_t* m, float* o)
{
    float t[8];
#pragma unroll
    for (int n = 0; n + 8 <= N; n += 8)
        asm(PAM_EACH8(PAM_OF_LANE) PAM_EACH8(PAM_POWER) PAM_EACH8(PAM_ADD_BY_ROW) : PAM_O8(n), PAM_T8 : PAM_S8(n), PAM_M8(n), [w] "v"(w), [mask] "v"(mask));
    if constexpr (N % 8 != 0)
        asm(PAM_EACH4(PAM_OF_LANE) PAM_EACH4(PAM_POWER) PAM_EACH4(PAM_ADD_BY_ROW) : PAM_O4(N - 4), PAM_T4 : PAM_S4(N - 4), PAM_M4(N - 4), [w] "v"(w), [mask] "v"(mask));
}

#undef PAM_ADD_BY_ROW
#undef PAM_ADD
#undef PAM_SUM_BY_ROW
#undef PAM_SUM_BY_LANE
#undef PAM_SUM
#undef PAM_POWER
#undef PAM_OF_LANE
#undef PAM_OF_WEIGHT
#undef PAM_OF_ROW
#undef PAM_EACH8
#undef PAM_EACH4
#undef PAM_O8
#undef PAM_O4
#undef PAM_M8
#undef PAM_M4
#undef PAM_S8
#undef PAM_S4
#undef PAM_T4
#undef PAM_T8

// A row's block as one lane in eight sees it: every value of the slice in one lane.
template <int W4, bool WHOLE> struct Look {
    static constexpr int kParts = (W4 + 7) / 8;
    v4f r[kParts];
    __device__ __forceinline__ static int mine(int i) { return min((int)threadIdx.x % 8 + 8 * i, W4 - 1); }
    __device__ __forceinline__ void load(const Stream<WHOLE>& s, int j1)
    {
        const float* const row = s.row(j1 + (int)threadIdx.x % 64 / 8);
#pragma unroll
        for (int i = 0; i < kParts; ++i) r[i] = *reinterpret_cast<const v4f_any*>(row + 4 * s.quad(mine(i)));
    }
    // (behind a head's values its last quad counts as the values in it)
    __device__ __forceinline__ void fill(const Stream<WHOLE>& s, int values)
    {
        if (values == 4 * s.quads) return;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const int d = 4 * min(s.first + mine(i), s.quads - 1);
#pragma unroll
            for (int c = 1; c < 4; ++c) r[i][c] = d + c < values ? r[i][c] : r[i][0];
        }
    }
};
// What is the matter with a block: zeros in it, or something else.
struct Verdict { bool zeros, wild; };
template <int W4, bool WHOLE> __device__ __forceinline__ Verdict judge(Look<W4, WHOLE>& look, const Stream<WHOLE>& s, int values, uint32_t shift)
{
    look.fill(s, values);
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < Look<W4, WHOLE>::kParts; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) most = max(most, ((f2u(look.r[i][c]) + shift) << 1) - kStreamBase);
    Verdict v{__ballot(most >= kStreamSpan) != 0ull, false};
    if (__builtin_expect(v.zeros, 0)) {
        bool wild = false;
#pragma unroll
        for (int i = 0; i < Look<W4, WHOLE>::kParts; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) wild = wild || ((f2u(look.r[i][c]) << 1) != 0u && ((f2u(look.r[i][c]) + shift) << 1) - kStreamBase >= kStreamSpan);
        v.wild = __ballot(wild) != 0ull;
    }
    return v;
}

// The power of two above a block's values.
template <int W4, bool WHOLE> __device__ __forceinline__ float above_all(const Look<W4, WHOLE>& look)
{
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < Look<W4, WHOLE>::kParts; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) most = max(most, f2u(look.r[i][c]) & ~kSign);
#pragma unroll
    for (int s = 1; s < 64; s *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, s, 64));
    return u2f((most & kExpo) + (1u << 23));
}

// ... where values are only factors of a float product: zeros and small ones are as good as any
template <int W4, bool WHOLE> __device__ __forceinline__ bool all_finite(Look<W4, WHOLE>& look, const Stream<WHOLE>& s, int values)
{
    look.fill(s, values);
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < Look<W4, WHOLE>::kParts; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) most = max(most, f2u(look.r[i][c]) << 1);
    return __ballot(most >= kExpo << 1) == 0ull;
}

// The same products by the full definition, for a row that lanes hold a quad each of and a lane's values as they are (load_plain).
struct Full { float off; bool has_off; };
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
            sum += full_product(f, plain(mine[4 * n.value + i]), from_lane<decltype(n)::value>(row[i]));
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

// A block's sums of products with the rows of s; then comes row j2 of `next`.  With LaneZeros a lane's zeros have products of zero to the bit, else of next to nothing,
// which is as good for a score alone.
template <int W4, bool WHOLE, class Lane>
__device__ __forceinline__ void block_dots(Pipe<W4, WHOLE>& pipe, const Stream<WHOLE>& s, int j1, const Stream<WHOLE>& next, int j2, bool zeros, const Lane& lane, const uint32_t (&mine)[4 * W4],
                                           float (&sum)[kBlock])
{
    constexpr int N = 4 * Pipe<W4, WHOLE>::kQuads;
#pragma unroll
    for (int j = 0; j < kBlock; ++j) sum[j] = 0.0f;
    if (__builtin_expect(zeros || lane.any != 0, 0)) {
        const Zeros codes = lane.codes();
        pipe.rolled(s, j1, next, j2, [&](int h, int d, const Piece& x) __attribute__((always_inline)) {
            dot_piece_with_zeros<N, Lane::kLanes>(x, mine + d, codes, sum[0]);
            if (h == Pipe<W4, WHOLE>::kPieces - 1) turned(sum);
        });
        return;
    }
    pipe.block(s, j1, next, j2, [&](int j, int d, const Piece& x) __attribute__((always_inline)) { dot_piece<N>(x, mine + d, sum[j]); });
}
// out += the block's weights times its rows; a weight that does not count is anything.  add: as in load_lane.  small, if there are some: weights below 2^-86, whose products with small
// values would leave the exponents' range: they come 2^kLift times as large, and the block takes the loop with factors, which scale their products back.
constexpr int kLift = 30;
template <int W4, bool WHOLE>
__device__ __forceinline__ void block_add(Pipe<W4, WHOLE>& pipe, const Stream<WHOLE>& s, int j1, const Stream<WHOLE>& next, int j2, bool zeros, float (&weight)[kBlock], uint32_t add, uint32_t counts,
                                          float (&out)[4 * W4], bool some_small = false, uint32_t small = 0u)
{
    constexpr int N = 4 * Pipe<W4, WHOLE>::kQuads;
    if (__builtin_expect(zeros || some_small, 0)) {
        pipe.rolled(s, j1, next, j2, [&](int h, int d, const Piece& x) __attribute__((always_inline)) {
            const bool in = counts & 1u;
            const float one = small & 1u ? 1.0f / (float)(1 << kLift) : 1.0f;
            add_piece_with_zeros<N>(x, in ? f2u(weight[0]) + add : 0u, in ? one : 0.0f, out + d);
            if (h == Pipe<W4, WHOLE>::kPieces - 1) { turned(weight); counts >>= 1; small >>= 1; }
        });
        return;
    }
    pipe.block(s, j1, next, j2, [&](int j, int d, const Piece& x) __attribute__((always_inline)) {
        const bool in = (counts >> j) & 1u;
        add_piece<N>(x, in ? f2u(weight[j]) + add : 0u, in ? 1.0f : 0.0f, out + d);
    });
}

// The same by slopes: out += the block's weights times the powers of its rows' products with `mine`.
template <int W4, bool WHOLE>
__device__ __forceinline__ void block_add_power(Pipe<W4, WHOLE>& pipe, const Stream<WHOLE>& s, int j1, const Stream<WHOLE>& next, int j2, bool zeros, uint32_t power,
                                                float (&weight)[kBlock], uint32_t counts, const uint32_t (&mine)[4 * W4], float (&out)[4 * W4])
{
    constexpr int N = 4 * Pipe<W4, WHOLE>::kQuads;
    if (__builtin_expect(zeros, 0)) {
        pipe.rolled(s, j1, next, j2, [&](int h, int d, const Piece& x) __attribute__((always_inline)) {
            const bool in = counts & 1u;
            add_power_piece_with_zeros<N>(x, in ? weight[0] : 0.0f, in ? power : 0u, mine + d, out + d);
            if (h == Pipe<W4, WHOLE>::kPieces - 1) { turned(weight); counts >>= 1; }
        });
        return;
    }
    pipe.block(s, j1, next, j2, [&](int j, int d, const Piece& x) __attribute__((always_inline)) {
        const bool in = counts >> j & 1u;
        add_power_piece<N>(x, in ? weight[j] : 0.0f, in ? power : 0u, mine + d, out + d);
    });
}

// A work-group is four wavefronts (eight, where a row has eight slices): NS of them for each of kTiles tiles of 64 rows, which stream the same rows by.  With
// slices all wavefronts have the same barriers: `Team` says what one of them found to all.
template <int NS> constexpr int kTiles = NS >= 4 ? 1 : 4 / NS;
template <int NS> constexpr int kWaveCount = NS * kTiles<NS>;
template <int NS> __device__ __forceinline__ bool in_team(bool x) { return NS == 1 ? __ballot(x) != 0ull : __syncthreads_or(x) != 0; }

// Slices' sums, in all of their wavefronts and in one order, and whether a wavefront of the team met something wild.  Two buffers in turn: who writes one
// again has passed the barrier before which the others read it.
template <int NS, int N> struct Slices {
    v4f part[2][kTiles<NS>][NS][N / 4][64];
    int wild[2][kWaveCount<NS>];
    __device__ __forceinline__ bool add_up(int turn, int wave, float (&v)[N], bool is_wild)
    {
        const int lane = (int)threadIdx.x % 64, tile = wave / NS, slice = wave % NS;
#pragma unroll
        for (int i = 0; i < N / 4; ++i) part[turn][tile][slice][i][lane] = v4f{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        if (lane == 0) wild[turn][wave] = is_wild;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            v4f x[NS];
#pragma unroll
            for (int s = 0; s < NS; ++s) x[s] = part[turn][tile][s][i][lane];
#pragma unroll
            for (int n = NS; n > 1; n /= 2)
#pragma unroll
                for (int s = 0; s < n / 2; ++s) x[s] = x[2 * s] + x[2 * s + 1];
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * i + c] = x[0][c];
        }
        int any = 0;
#pragma unroll
        for (int s = 0; s < kWaveCount<NS>; ++s) any |= wild[turn][s];
        return __builtin_amdgcn_readfirstlane(any) != 0;
    }
};
template <int N> struct Slices<1, N> { __device__ __forceinline__ bool add_up(int, int, float (&)[N], bool is_wild) { return is_wild; } };

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
    template <int NS> __device__ __forceinline__ void close_team()
    {
        if constexpr (NS > 1) {
            __shared__ int ends[kWaveCount<NS>][2];
            if (threadIdx.x % 64 == 0) { ends[threadIdx.x / 64][0] = first; ends[threadIdx.x / 64][1] = last; }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaveCount<NS>; ++w) { first = min(first, ends[w][0]); last = max(last, ends[w][1]); }
            first = __builtin_amdgcn_readfirstlane(first); last = __builtin_amdgcn_readfirstlane(last);
        }
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

// Whether a row of the team sees one of the rows begin ... end - 1: looked at before anything else is loaded, since half of the units of a causal pass
// see none.
template <int NS> __device__ __forceinline__ bool any_seen(const Sight& sight, int begin, int end)
{
    if (!sight.with_documents) return begin < end;
#pragma unroll 1
    for (int j0 = begin; j0 < end; j0 += kSpan)
        if (in_team<NS>(sight.span(j0) != 0ull)) return true;
    return false;
}

// ---------------------------------------------------------------- from a score to its exponent

// x (*) a positive constant below 2, whose bits less the bias (offset counted) are `add`, below zero for one below 1.  Underflow is zero; NaN, infinities and what is
// 2^127 or more are no number afterwards, whatever `add` is.
__device__ __forceinline__ float times(float x, uint32_t add)
{
    const uint32_t size = f2u(x) & ~kSign;
    const int m = max((int)(size + add), 0);
    return u2f(size >= 0x7f000000u ? kQNaN : (uint32_t)m | (f2u(x) & kSign));
}
// a (*) b of any finite numbers; an underflow (a zero's, too) is zero or next to nothing, an overflow an infinity
__device__ __forceinline__ float times_any(float a, float b, uint32_t off_add)
{
    const uint32_t m = __builtin_elementwise_sub_sat((f2u(a) & ~kSign) + (f2u(b) & ~kSign), kBias - off_add);
    return u2f(min(m, kExpo) | ((f2u(a) ^ f2u(b)) & kSign));
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

constexpr float kNothing = -0x1.fffffep127f;      // M of a row that has seen nothing yet: below every exponent of 2 that a score below 2^127 has

}  // namespace pamatt
