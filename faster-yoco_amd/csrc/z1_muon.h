// The orthogonalised update of matrices: what its sources share (not part of the C ABI).
//   z1_muon.hip          the momentum and X's start, the host's part
//   z1_muon_steps.h      a step's products; compiled by z1_muon_fast.hip and z1_muon_precise.hip
//   z1_muon_small.hip    small matrices, whole
//
//   momentum   buf = mu buf + (1 - mu) g,  u = mu buf + (1 - mu) g (nesterov) or buf
//   start      X = u / max(|u|_F, eps), on its shorter side: r x c, r <= c (u's transpose where it has more rows)
//   step       A = X X^T,  B = b A + c A^2,  X <- a X + B X                  (r^2 c, r^3 and 2 r^2 c multiply-adds: A and
//                                                                            A^2 are symmetric, one half is computed)
//   end        the result, or p = keep p - lr X and its BF16 copy
//
// The products are matrix instructions on fp16 operands with fp32 sums.  Plain rounding of X, A and B to fp16 leaves 1e-3 to
// 1e-2 in the result (bf16: 1e-2 to 7e-2), since what is rounded off the few large directions grows as the many small ones do,
// 3.4 times a step, and since A and B are near multiples of 1 at the end, so that their diagonals lose most.  Hence
//   - the diagonals d of A and e of a + B stay in fp32, apart from the operands:  with A = D + A', B = E + B',
//     A^2 = D^2 + D A' + A' D + A'^2,  so B'[i][j] = c A'^2[i][j] + (b + c (d_i + d_j)) A'[i][j],
//     e_i = a + b d_i + c d_i^2 + c A'^2[i][i],  X <- e X + B' X;
//   - X is kept as a pair of fp16 (22 bits), of which e X takes both, and B' X too in the first steps (both_halves): what the
//     first half leaves out there goes into all directions, those of no size among them, and grows from step to step; what A and
//     B lose only turns the directions that are there.
// That leaves 4e-4 to 1e-3 of the result (2-norm) mostly and up to 2e-3 whatever the spectrum (many equal singular values), with
// more than 64 rows: about the rounding of a result in bf16, 1.7e-3, at the most.  Fewer rows, and PRECISE for results that hold
// more, take pairs for A and B as well and three products for one, hi hi + hi lo + lo hi: 1e-6 to 3e-5, and with few directions in
// the input 1e-4 (500 rows) to 4e-4 (3000), as plain fp32 products leave (1.8e-4 and 4.6e-4).
//
// Stored values are scaled by powers of two, so that fp16's range covers them: the host admits coefficients only if the
// iterates stay below 4 and B below 32, so |X| kX <= 2^14, |A| kA <= 2^15, |B| kB <= 2^15.
//
// Both products of X want their summed axis contiguous: c in A, r in B X.  X is written in both orders (t: [c][r], o: [r][c]).
// Rows are padded with zeros to whole blocks of 64; rows past an operand's end are zeros by the buffers' ranges.
#pragma once

#include "z1_tiles.h"

#pragma clang fp contract(off)

namespace z1muon __attribute__((visibility("hidden"))) {

using namespace z1blk;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float kX = 4096.0f, kA = 2048.0f, kB = 1024.0f;
constexpr int kHalves = 64;                            // columns of a staged block: 128 bytes
constexpr int kParts = 1024;                           // partial sums of a matrix's squares, at most
constexpr int kList = Z1_MAX_MATRICES;                 // matrices named one by one in a launch, and groups of them
constexpr int kMaxSteps = 64;
constexpr int kWholeSide = 128;                        // shorter side of the small matrices, at most

enum Mode { GRAM, SQUARE, UPDATE, LAST };

// What the last step writes: p and p16 of a list, or the result in a type.
struct Listed {};

// Where a launch's matrices lie: one by one, or `step` elements apart.
struct Inputs {
    const void* g[kList];
    int64_t stride[kList];                             // elements between rows
    float* buf[kList];
    float* p[kList];
    uint16_t* p16[kList];
};
struct Batch {
    const void* x;                                     // [count][m][n], rows `stride` and matrices `step` elements apart
    int64_t step, stride;
};

// A matrix's part of the workspace, with `planes` halves of X's second order, A and B (2: pairs): offsets of X in both orders (t
// twice: read and written), A, B and the diagonals, bytes from a pair's first halves to its second ones, and bytes in all.
// Every array starts at a multiple of 1024 bytes.
struct Layout {
    int64_t t[2], o, A, B, d, e, size;
    int64_t t_plane, o_plane, s_plane;
    int ldr, ldc;                                      // r and c rounded up to blocks
};
__host__ __device__ inline Layout layout_of(int r, int c, int planes) {
    Layout w;
    w.ldr = (r + kHalves - 1) / kHalves * kHalves;
    w.ldc = (c + kHalves - 1) / kHalves * kHalves;
    auto room = [](int64_t bytes) { return (bytes + 1023) / 1024 * 1024; };
    w.t_plane = room((int64_t)c * w.ldr * 2);
    w.o_plane = room((int64_t)r * w.ldc * 2);
    w.s_plane = room((int64_t)r * w.ldr * 2);
    w.t[0] = 0;
    w.t[1] = 2 * w.t_plane;
    w.o = 4 * w.t_plane;
    w.A = w.o + planes * w.o_plane;
    w.B = w.A + planes * w.s_plane;
    w.d = w.B + planes * w.s_plane;
    w.e = w.d + room((int64_t)w.ldr * 4);
    w.size = w.e + room((int64_t)w.ldr * 4);
    return w;
}

// Matrices of one shape, side by side in the workspace.
struct Group {
    int64_t base;                                      // of the first one's part
    int r, c;                                          // shorter and longer side
    int tall;                                          // the matrices have more rows than columns: their rows are c
    int first, count;                                  // matrices of the launch
    int tile0;                                         // the first one's first workgroup of the launch
    float lr, keep;
};
struct Plan {
    uint8_t* base;
    int groups;
    int cur;                                           // which t is read
    int both;                                          // B X on single operands takes both halves of X
    Group g[kList];
};
// The group of a workgroup, or of a matrix.
__device__ __forceinline__ const Group& group_of_tile(const Plan& w, int index) {
    int k = 0;
    while (k + 1 < w.groups && index >= w.g[k + 1].tile0) ++k;
    return w.g[k];
}
__device__ __forceinline__ const Group& group_of_matrix(const Plan& w, int z) {
    int k = 0;
    while (k + 1 < w.groups && z >= w.g[k + 1].first) ++k;
    return w.g[k];
}

struct Coefficients {
    float a, b, c;
};

struct Start {
    Inputs in;
    Batch batch;
    int list;
    const float* factor;                               // of g, or NULL
    float mu;
    int nesterov;
    double eps;
    double* partials;                                  // [matrices][kParts]
};

// Eight of a gradient and of its momentum; zeros past a row's end.
struct Eight {
    float g[8], buf[8];
};
template <typename T>
__device__ __forceinline__ void load_eight(const Start& a, int z, int64_t row, int n, int c, Eight& e) {
    const int left = n - c;
    const void* g = a.list ? a.in.g[z] : (const void*)((const typename T::elem*)a.batch.x + z * a.batch.step);
    load_row<T>(g, row * (a.list ? a.in.stride[z] : a.batch.stride) + c, left, e.g);
    if (a.list) load_row<F32>(a.in.buf[z], row * n + c, left, e.buf);
}
// u of them, and with MOVE the momentum's step before.
template <bool MOVE>
__device__ __forceinline__ void u_of(const Start& a, int z, int64_t row, int n, int c, float factor, Eight& e, float* u) {
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = e.g[j];
    if (!a.list) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float g = (u[j] * factor) * (1.0f - a.mu);
        if (MOVE) e.buf[j] = __builtin_fmaf(a.mu, e.buf[j], g);
        u[j] = a.nesterov ? __builtin_fmaf(a.mu, e.buf[j], g) : e.buf[j];
    }
    if (MOVE) store_row<F32>(a.in.buf[z], row * n + c, n - c, e.buf);
}
template <typename T, bool MOVE>
__device__ __forceinline__ void load_u(const Start& a, int z, int64_t row, int n, int c, float factor, float* u) {
    Eight e;
    load_eight<T>(a, z, row, n, c, e);
    u_of<MOVE>(a, z, row, n, c, factor, e, u);
}

// Eight values as fp16 at `at` (16-byte aligned), and what that leaves, `plane` bytes on.
template <bool PAIR>
__device__ __forceinline__ void put_halves(uint8_t* at, int64_t plane, const float* v) {
    const u4 hi = F16::close(v);
    *(Z1B_GLOBAL u4*)at = hi;
    if constexpr (PAIR) {
        float f[8], lo[8];
        F16::open(hi, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] = v[j] - f[j];
        *(Z1B_GLOBAL u4*)(at + plane) = F16::close(lo);
    }
}
constexpr int64_t kMaxSide = Z1_MAX_SIDE;
constexpr int64_t kMaxCount = 1 << 15;                 // of a call: a grid's second axis
constexpr int64_t kMaxTiles = 1ll << 22;               // of a launch: its threads count in 32 bits
constexpr int kCus = 256;

// All arguments of the steps' launches.
struct Steps {
    Plan plan;
    Coefficients co;
    void* out;
    Inputs in;
    hipStream_t st;
};
enum Kind { OUT_F32, OUT_BF16, OUT_F16, OUT_LIST };

// The steps' products over the plan's matrices, X's start in place; out by `kind`.
int iterate_fast(Steps& a, int steps, const float* coefficients, Kind kind);
int iterate_precise(Steps& a, int steps, const float* coefficients, Kind kind);
void ways_fast(Plan& w, int* way);
void ways_precise(Plan& w, int* way);

// Matrices of few rows take pairs in any case: the fewer rows, the less what A and B lose averages out (2 rows up to 5e-3, 3 x
// 2000 2e-3, 16 x 16 1.6e-3, 33 x 96 1.2e-3; 65 to 128 rows 1.0e-3 at most), and there it costs least (32 x 32: 12.7 -> 15.2
// us, 64 x 256 26.6 -> 35, 40 x 2000 91 -> 117).
constexpr int kPairSide = 64;
__host__ __device__ inline bool has_pairs(int m, int n, bool precise) { return precise || (m < n ? m : n) <= kPairSide; }

// In a kernel: a number that the compiler does not take apart into a truth value, as which it leaves the scalar unit, and every
// address that follows with it.
template <bool PRECISE>
__device__ __forceinline__ int planes_of(const Group& g) {
    return PRECISE ? 2 : __builtin_amdgcn_readfirstlane(has_pairs(g.r, g.c, false) ? 2 : 1);
}

// On single operands: the steps whose B X takes both halves of X, a bit each.  A direction of no size grows by `a` a step, and
// with it what the first half leaves out, 2^-12 of X in every element: both halves until no more than a factor of 4 is to come
// (the first three of five steps with the default coefficients.  Of 12,000 spectra of one to three levels, 65 to 352 rows, the
// worst, some 60 equal singular values of 96, come out 4.2e-3 off with two such steps, 1.9e-3 with three and with all five; ranks
// of one to four 4e-2 without.  Each such step is a tenth more work).
inline uint64_t both_halves(const float* coefficients, int steps) {
    uint64_t both = 0;
    double growth = 1.0;
    for (int k = steps - 1; k >= 0; --k) {
        if (growth > 4.0) both |= 1ull << k;
        growth *= coefficients[3 * k] < 0.0f ? -coefficients[3 * k] : coefficients[3 * k];
    }
    return both;
}

// The small matrices' kernel: fragments to a wave and bytes of LDS.  0: the matrix is too large for it.
struct WholeWay {
    int pieces, bytes;
};
WholeWay whole_way(int64_t m, int64_t n, bool precise);
inline bool is_whole(int64_t m, int64_t n, bool precise) { return whole_way(m, n, precise).pieces != 0; }

// By rows of fragments, which with `precise` decide on pairs: the largest of a launch's small matrices, or none.
struct WholeWays {
    WholeWay of[kWholeSide / 32];
    void add(int64_t m, int64_t n, bool precise) {
        const WholeWay w = whole_way(m, n, precise);
        WholeWay& own = of[((m < n ? m : n) - 1) / 32];
        if (w.pieces > own.pieces) own = w;
    }
};
// `count` matrices of the plan's groups, all of them small, in one launch for each number of rows of fragments.
int run_whole(const Start& start, const Plan& plan, const WholeWays& ways, int64_t count, int dtype, int steps,
              const float* coefficients, bool precise, void* out, int out_dtype, hipStream_t st);

}  // namespace z1muon
