// Products of a few rows (single tokens, small batches while decoding): y[m][n] = sum over k of a[m][k] (*) w[n][k], with bias,
// activation, residual or the gated product behind the sums.
//
// Bound by reading w once.  33.5 MB of gated weights: one token 8.0 us (4.2 TB/s with the launch, copies reach 5.3), eight 10.7; the matrix
// kernel, whose tiles have 64 rows, 25.  8.4 MB: one token 3.9 us, eight 5.6.
// Up to eight tokens are one set of work-groups, up to 24 two or three, which read w from memory once between them (16 tokens through
// 33.5 MB 17.7 us, the matrix kernel 25; through 8.4 MB 6.9 and 16; 24 tokens 25 and 26.5, 10.6 and 16.6; 32 tokens 32 and 26, 11.5 and 16.5).
// A wavefront takes C rows of w and a part of k: its lanes lie along k with 128-bit loads, so that every load of a row is 1 KB in one
// piece, and keep C x ROWS sums, which are added up over the lanes through LDS.  How many rows a wavefront takes and over how many of a
// work-group's four wavefronts k is dealt out goes by the number of wavefronts (shape_for).  At these times a kernel's length counts:
// every compute unit fetches the instructions anew, and with the rare paths written out and the sums exchanged by shuffles eight tokens took 39 us.
// Order of a sum: per lane k ascending in quads 256 S apart (S wavefronts along k), then lanes, then
// wavefronts.  It depends on the sizes alone.
// Values: as in the matrix kernel, a step all of whose values are normal numbers in [2^-63, 2^64) takes one integer and one float addition per
// product; one with zeros besides selects their products away (they change no sum); anything else takes the full definition.
#include <algorithm>

#include "pam_activation.h"
#include "pam_common.h"
#include "pam_thin.h"

using namespace pamdev;

namespace {

constexpr int kThreads = 256, kWaves = 4, kStep = 256;       // kStep: k of a wavefront's step
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ uint32_t in_window(uint32_t u) { return (u << 1) - (64u << 24); }      // below kSpan: normal, in [2^-63, 2^64)
constexpr uint32_t kSpan = 127u << 24;

struct Quad { uint32_t v[4]; };
// (base in scalar registers, a 32-bit offset of the lane)
__device__ __forceinline__ Quad load_quad(const float* base, uint32_t bytes)
{
    const v4f_any q = *reinterpret_cast<const v4f_any*>(reinterpret_cast<const char*>(base) + bytes);
    return Quad{{f2u(q.x), f2u(q.y), f2u(q.z), f2u(q.w)}};
}

// The full definition, as a call: written out for every product of a step it made the kernels tens of kilobytes long.
__device__ __noinline__ float any_product(float a, float b) { return pam_mul(a, b); }

// Adds the products of ROWS quads of a with C quads of w.
template <int ROWS, int C>
__device__ __forceinline__ void add_products(const Quad (&x)[ROWS], const Quad (&w)[C], float (&acc)[ROWS][C])
{
    uint32_t seen = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) seen = max(seen, in_window(x[r].v[i]));
#pragma unroll
        for (int c = 0; c < C; ++c) seen = max(seen, in_window(w[c].v[i]));
    }
    if (__builtin_expect(__ballot(seen >= kSpan) == 0ull, 1)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int c = 0; c < C; ++c) acc[r][c] += u2f(x[r].v[i] + w[c].v[i] - kBias);
        return;
    }
    uint32_t odd = 0u;                            // ... without the zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) odd = max(odd, (x[r].v[i] << 1) != 0u ? in_window(x[r].v[i]) : 0u);
#pragma unroll
        for (int c = 0; c < C; ++c) odd = max(odd, (w[c].v[i] << 1) != 0u ? in_window(w[c].v[i]) : 0u);
    }
    if (__ballot(odd >= kSpan) == 0ull) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint32_t a = x[r].v[i], b = w[c].v[i];
                    acc[r][c] += min(a << 1, b << 1) != 0u ? u2f(a + b - kBias) : 0.0f;
                }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[r][c] += any_product(u2f(x[r].v[i]), u2f(w[c].v[i]));
}

// S wavefronts along k: 1, 2 or 4.  GATED: the C rows of a wavefront are C / 2 of the gate's and the same ones of the other half.
template <int ROWS, int C, bool GATED>
__global__ __launch_bounds__(kThreads) void thin_kernel(pamthin::Layer g, int S, int sets)
{
    constexpr int kSums = ROWS * C;
    constexpr int kColumns = GATED ? C / 2 : C;
    __shared__ float sums[kWaves][kSums], lanes[kWaves][kSums * 65];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);      // (so the rows' addresses are scalars)
    const int share = wave % S, set = wave / S;                            // which part of k, which rows of w
    // (work-groups go to the eight XCDs in turn: those that read the same rows of w for other tokens are eight apart, on one of them)
    const int of_set = (int)blockIdx.x / (8 * sets) * 8 + (int)blockIdx.x % 8, row0 = (int)blockIdx.x / 8 % sets * ROWS;
    const int column0 = (of_set * (kWaves / S) + set) * kColumns;
    const bool has_off = g.off != 1.0f;
    const float* wp[C];
    const float* ap[ROWS];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int column = min(column0 + c % kColumns, g.n - 1);           // (past the end the last one again)
        wp[c] = g.w + (long)(GATED && c >= kColumns ? column + g.n : column) * g.w_sr;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) ap[r] = g.a + (long)min(row0 + r, g.m - 1) * g.a_sr;
    float acc[ROWS][C];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[r][c] = 0.0f;
    auto scaled = [&](Quad q) {
        if (has_off)
#pragma unroll
            for (int i = 0; i < 4; ++i) q.v[i] = f2u(any_product(u2f(q.v[i]), g.off));
        return q;
    };
    const uint32_t whole = (uint32_t)g.k & ~3u;
    for (uint32_t k = (uint32_t)(share * kStep + lane * 4); k < whole; k += (uint32_t)(S * kStep)) {                                    // (lanes past the end idle)
        Quad x[ROWS], w[C];
#pragma unroll
        for (int c = 0; c < C; ++c) w[c] = load_quad(wp[c], k * 4u);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) x[r] = load_quad(ap[r], k * 4u);
#pragma unroll
        for (int c = 0; c < C; ++c) w[c] = scaled(w[c]);
        add_products(x, w, acc);
    }
    if (share == 0 && (uint32_t)lane < (uint32_t)g.k - whole) {                                // the last one to three k, one a lane
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float wv = wp[c][whole + lane], v = has_off ? any_product(wv, g.off) : wv;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) acc[r][c] += any_product(ap[r][whole + lane], v);
        }
    }
    // The lanes' sums through LDS: lane l adds kPart of value l / kLanes' sixty-four, the kLanes partial sums are exchanged.
    constexpr int kLanes = 64 / kSums, kPart = 64 / kLanes;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) lanes[wave][(r * C + c) * 65 + lane] = acc[r][c];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");            // (a wavefront's LDS accesses are in order)
    __builtin_amdgcn_wave_barrier();
    const float* part = lanes[wave] + lane / kLanes * 65 + lane % kLanes * kPart;
    float total = 0.0f;
#pragma unroll 4
    for (int i = 0; i < kPart; ++i) total += part[i];
#pragma unroll
    for (int s = kLanes / 2; s >= 1; s /= 2) total += __shfl_xor(total, s, 64);
    if (lane % kLanes == 0) sums[wave][lane / kLanes] = total;
    __syncthreads();
    if (share != 0 || lane >= ROWS * kColumns) return;
    auto sum_of = [&](int i) {
        float v = sums[wave][i];
        for (int s = 1; s < S; ++s) v += sums[wave + s][i];
        return v;
    };
    const int r = row0 + lane / kColumns, c = column0 + lane % kColumns, at = lane / kColumns * C + lane % kColumns;
    if (r >= g.m || c >= g.n) return;
    const Activation act{g.activation, g.off, has_off};
    float v = sum_of(at);
    if (g.bias) v += g.bias[c];
    if constexpr (GATED) {
        float u = sum_of(at + kColumns);
        if (g.bias) u += g.bias[c + g.n];
        if (g.z) { g.z[(long)r * 2 * g.n + c] = v; g.z[(long)r * 2 * g.n + g.n + c] = u; }
        g.y[(long)r * g.n + c] = pam_mul_off(act(v), u, g.off, has_off);
    } else {
        if (g.z) g.z[(long)r * g.n + c] = v;
        v = act(v);
        g.y[(long)r * g.n + c] = g.residual ? v + g.residual[(long)r * g.residual_sr + c] : v;
    }
}

constexpr long kMostRows = 24;

// Rows of w per wavefront and wavefronts along k: from four rows and one wavefront on, until there are enough wavefronts, first by dealing
// out k while a wavefront keeps two steps of it, then by taking fewer rows.  Enough keep the memory busy, sixteen on a compute
// unit for one or two tokens (1024 -> 8192: 8.8 us with eight, 7.4); each reads all the tokens' rows, so that for more tokens eight do better
// (33.5 MB, eight tokens: 10.7 us with eight, 13.5 with sixteen, 18.5 with thirty-two).
struct Shape { int C, S; };
Shape shape_for(long rows, long k, int tokens, int sets, bool gated)
{
    const long enough = tokens >= 4 ? 2048 : 4096;
    Shape s{4, 1};
    const long steps = (k + kStep - 1) / kStep, least = gated ? 2 : 1;
    while ((rows + s.C - 1) / s.C * s.S * sets < enough) {
        if (s.S < 4 && steps >= 2 * s.S) s.S *= 2;
        else if (s.C > least) s.C /= 2;
        else break;
    }
    return s;
}

}  // namespace

namespace pamthin {

// (a work-group takes sixteen rows of w where there are many, and a launch counts its work-items in 32 bits, 2^24 work-groups)
bool takes(long m, long rows, long k, long a_sc, long w_sc)
{
    return m <= kMostRows && k > 0 && k <= (1L << 28) && rows * ((m + 7) / 8) <= (1L << 27) && (a_sc == 1 || k == 1) && (w_sc == 1 || k == 1);
}

int launch(const char* what, const Layer& g, bool gated, hipStream_t st)
{
    const int rows = g.m <= 1 ? 1 : g.m <= 2 ? 2 : g.m <= 4 ? 4 : 8, sets = (g.m + rows - 1) / rows;
    const Shape s = shape_for((long)g.n * (gated ? 2 : 1), g.k, rows, sets, gated);
    const int columns = (gated ? s.C / 2 : s.C) * (kWaves / s.S);
    const unsigned each = (unsigned)((g.n + columns - 1) / columns);
    const dim3 grid(sets == 1 ? each : (each + 7) / 8 * 8 * (unsigned)sets);
#define PAM_THIN(ROWS, WIDE, GATED) \
    if (rows == ROWS && s.C == WIDE && gated == GATED) hipLaunchKernelGGL((thin_kernel<ROWS, WIDE, GATED>), grid, dim3(kThreads), 0, st, g, s.S, sets);
#define PAM_THIN_ROWS(ROWS) PAM_THIN(ROWS, 1, false) PAM_THIN(ROWS, 2, false) PAM_THIN(ROWS, 4, false) PAM_THIN(ROWS, 2, true) PAM_THIN(ROWS, 4, true)
    PAM_THIN_ROWS(1) PAM_THIN_ROWS(2) PAM_THIN_ROWS(4) PAM_THIN_ROWS(8)
#undef PAM_THIN_ROWS
#undef PAM_THIN
    return pamhost::check_launch(what);
}

}  // namespace pamthin
