// The orthogonalised update of matrices (declarations: include/yoco_z1.h).
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
//   - X is kept as a pair of fp16 (22 bits), of which products take the first and e X both.
// That leaves 1e-4 to 8e-4 for any spectrum, at the same number of products: enough for a result in bf16, whose own rounding is
// 1.7e-3.  For results that hold more, PRECISE takes pairs for A and B as well and three products for one, hi hi + hi lo +
// lo hi: 1e-6 to 3e-5, as plain fp32 products leave.
//
// Stored values are scaled by powers of two, so that fp16's range covers them: the host admits coefficients only if the
// iterates stay below 4 and B below 32, so |X| kX <= 2^14, |A| kA <= 2^15, |B| kB <= 2^15.
//
// Both products of X want their summed axis contiguous: c in A, r in B X.  X is written in both orders (t: [c][r], o: [r][c]).
// Rows are padded with zeros to whole blocks of 64; rows past an operand's end are zeros by the buffers' ranges.
#include "z1_tiles.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(off)

namespace {

using namespace z1blk;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float kX = 4096.0f, kA = 2048.0f, kB = 1024.0f;
constexpr int kHalves = 64;                            // columns of a staged block: 128 bytes
constexpr int kParts = 256;                            // partial sums of a matrix's squares
constexpr int kList = Z1_MAX_MATRICES;                 // matrices named one by one in a launch, and groups of them
constexpr int kMaxSteps = 64;

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

// A matrix's part of the workspace: offsets of X in both orders (t twice: read and written), A, B (pairs) and the diagonals, bytes
// from a pair's first halves to its second ones, and bytes in all.  Every array starts at a multiple of 1024 bytes.
struct Layout {
    int64_t t[2], o, A, B, d, e, size;
    int64_t t_plane, o_plane, s_plane;
    int ldr, ldc;                                      // r and c rounded up to blocks
};
__host__ __device__ inline Layout layout_of(int r, int c, bool precise) {
    Layout w;
    w.ldr = (r + kHalves - 1) / kHalves * kHalves;
    w.ldc = (c + kHalves - 1) / kHalves * kHalves;
    auto room = [](int64_t bytes) { return (bytes + 1023) / 1024 * 1024; };
    w.t_plane = room((int64_t)c * w.ldr * 2);
    w.o_plane = room((int64_t)r * w.ldc * 2);
    w.s_plane = room((int64_t)r * w.ldr * 2);
    const int planes = precise ? 2 : 1;
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

// ------------------------------------------------------------------------------------------------------ products
// A launch's i-th workgroup in an order that gives each XCD one run of neighbours.
__device__ __forceinline__ int in_runs() {
    const int total = gridDim.x, x = blockIdx.x & 7, share = total >> 3, more = total & 7;
    return x * share + (x < more ? x : more) + (int)(blockIdx.x >> 3);
}
struct Place {
    int down, across;
};
// The i-th tile of a lower triangle, in rows.
__device__ __forceinline__ Place in_triangle(int i) {
    int d = (int)((sqrtf(8.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
    while (d * (d + 1) / 2 > i) --d;
    while ((d + 1) * (d + 2) / 2 <= i) ++d;
    return {d, i - d * (d + 1) / 2};
}
// The i-th tile of `down` x `across`, in panels of 8 rows, each down its columns.
__device__ __forceinline__ Place in_panel(int i, int down, int across) {
    const int first = i / (8 * across) * 8, rest = i - first * across, rows = down - first < 8 ? down - first : 8;
    return {first + rest % rows, rest / rows};
}

// A wave's results change from the matrix instructions' layout to rows, and to columns, by way of its own LDS: up to 64 rows of
// 64 floats, whose groups of four lie at group ^ turn(row), so that no access of 16 neighbouring lanes meets in a bank: 16 rows'
// same group (out of the instructions' layout), two rows' groups of one parity (rows), and every eighth row's same columns
// (columns).
__device__ __forceinline__ int turn(int row) { return (row & 7) ^ (row & 8) ^ (row >> 3 & 6); }
__device__ __forceinline__ f4* group_at(float* own, int row, int group) {
    return (f4*)(own + row * 64 + ((group ^ turn(row)) << 2));
}
// A wave's own bytes: nobody to meet.
__device__ __forceinline__ void own_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

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
// Eight fp16 of a buffer, and eight floats; zeros past its end.
__device__ __forceinline__ u4 halves_of(__amdgpu_buffer_rsrc_t from, int at) {
    return __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0);
}
__device__ __forceinline__ void floats_of(__amdgpu_buffer_rsrc_t from, int at, float* v) {
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
        const u4 a = __builtin_amdgcn_raw_buffer_load_b128(from, at, k * 4, 0);
#pragma unroll
        for (int l = 0; l < 4; ++l) v[k + l] = as_f32(a[l]);
    }
}

// A launch's workgroups are the tiles from `first` on, or, with COARSE 2, the four quarters of tiles of twice the size.
//
// One launch of a step over `count` matrices: GRAM A = X X^T (operands o, o), SQUARE B from A A^T, UPDATE X from t and B, LAST
// the same into the result.  BT x BO results (t x o) of a workgroup, WT x WO of a wave, S blocks of 64 columns staged by direct
// loads; a block's two halves are read ahead by one half and the workgroup meets between them, as in the 8-bit products.
template <Mode MODE, bool PRECISE, typename Out, int COARSE, int BT, int BO, int WT, int WO, int S>
__global__ __launch_bounds__(BT / WT * (BO / WO) * 64) void step_kernel(Plan plan, Coefficients co, void* out, Inputs in, int first) {
    constexpr bool kSymmetric = MODE == GRAM || MODE == SQUARE;
    constexpr int kWaves = BT / WT * (BO / WO);
    constexpr int kPT = BT / 8 / kWaves, kPO = BO / 8 / kWaves;                // direct loads of a wave: 8 rows each
    constexpr int NT = WT / 32, NO = WO / 32;
    static_assert(!kSymmetric || BT == BO, "a triangle of square tiles");
    static_assert(S == 2 || S == 4, "a block's buffer is kb & (S - 1)");
    constexpr int kRow = kHalves * 2;
    __shared__ __align__(1024) uint8_t lds[S][(BT + BO) * kRow];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int run = in_runs(), index = first + run / (COARSE * COARSE);
    const Group& g = group_of_tile(plan, index);
    const Layout w = layout_of(g.r, g.c, PRECISE);
    const int64_t t_now = plan.cur ? w.t[1] : w.t[0], t_next = plan.cur ? w.t[0] : w.t[1];
    const int rows_t = kSymmetric ? g.r : g.c;
    const int down = (rows_t + COARSE * BT - 1) / (COARSE * BT), across = (g.r + COARSE * BO - 1) / (COARSE * BO);
    const int tiles = kSymmetric ? down * (down + 1) / 2 : down * across;
    const int nth = (index - g.tile0) / tiles, place = index - g.tile0 - nth * tiles, z = g.first + nth;
    const Place tile = kSymmetric ? in_triangle(place) : in_panel(place, down, across);
    const int part = run % (COARSE * COARSE);
    const int t0 = (tile.down * COARSE + part / COARSE) * BT, o0 = (tile.across * COARSE + part % COARSE) * BO;
    if (COARSE > 1 && (t0 >= rows_t || o0 >= g.r || (kSymmetric && o0 > t0))) return;          // past the end, or the upper half
    const int wt = wave / (BO / WO) * WT, wo = wave % (BO / WO) * WO;          // the wave's part of the tile
    uint8_t* const mine = plan.base + g.base + nth * w.size;

    const int ld = MODE == GRAM ? w.ldc : w.ldr, pitch = ld * 2, blocks = ld / kHalves;
    const uint8_t* const pt = mine + (MODE == GRAM ? w.o : MODE == SQUARE ? w.A : t_now) + (int64_t)t0 * pitch;
    const uint8_t* const po = mine + (MODE == GRAM ? w.o : MODE == SQUARE ? w.A : w.B) + (int64_t)o0 * pitch;
    const int64_t plane_t = MODE == GRAM ? w.o_plane : MODE == SQUARE ? w.s_plane : w.t_plane;
    const int64_t plane_o = MODE == GRAM ? w.o_plane : w.s_plane;
    const int64_t bytes_t = (int64_t)(rows_t - t0) * pitch, bytes_o = (int64_t)(g.r - o0) * pitch;
    // A row goes into a load's lane offset, which the buffer's range checks: rows past the end become zeros.  The block goes
    // into the scalar offset, which stays in the row: past the last block the last one is loaded again, not used.
    const __amdgpu_buffer_rsrc_t hi_t = buffer_of(pt, bytes_t), hi_o = buffer_of(po, bytes_o);
    const __amdgpu_buffer_rsrc_t lo_t = buffer_of(pt + (PRECISE ? plane_t : 0), bytes_t);
    const __amdgpu_buffer_rsrc_t lo_o = buffer_of(po + (PRECISE ? plane_o : 0), bytes_o);
    const int total = PRECISE ? 3 * blocks : blocks, last = total - 1;
    const int sub = lane >> 3, piece = lane & 7;
    const int from = sub * pitch + ((piece ^ (sub >> 1)) << 4);                // in 8 rows whose keys' third bit is 0
    auto stage = [&](int kb, int i) {                  // the i-th direct load of this wave's part of a block
        uint8_t* buf = lds[kb & (S - 1)];
        const int l = i < kPT ? wave * kPT + i : wave * kPO + i - kPT;
        int k = kb < last ? kb : last;
        bool t_lo = false, o_lo = false;
        if (PRECISE) {                                 // hi hi, hi lo, lo hi
            t_lo = k >= 2 * blocks;
            o_lo = k >= blocks && !t_lo;
            k -= t_lo ? 2 * blocks : o_lo ? blocks : 0;
        }
        const int row = l * 8 * pitch;
        if (i < kPT) load_lds(t_lo ? lo_t : hi_t, buf + l * 8 * kRow, row + (l & 1 ? from ^ 64 : from), k * kRow);
        else load_lds(o_lo ? lo_o : hi_o, buf + (BT + l * 8) * kRow, row + (l & 2 ? from ^ 64 : from), k * kRow);
    };
    const int r32 = lane & 31, half = lane >> 5, rs = spread(r32);

    f16 acc[NO][NT];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f16{};

    // what follows the meeting -- the next block's first reads, the direct loads into the buffer that has just been read --
    // runs beside the second half's products; past the last block the reads and loads are of no use, and in bounds
    constexpr int kReads = 2 * (NT + NO), kLoads = kPT + kPO, kProducts = 2 * NT * NO;
    i4 f[2][NT + NO][2];
    auto read = [&](int kb, int h, int q) {
        const int i = q >> 1, p = 4 * h + 2 * (q & 1) + half;
        const uint8_t* row = i < NT ? lds[kb & (S - 1)] + (wt + i * 32 + r32) * kRow
                                    : lds[kb & (S - 1)] + (BT + wo + (i - NT) * 32 + rs) * kRow;
        f[h][i][q & 1] = *(const i4*)(row + ((p ^ (i < NT ? key_plain(r32) : key_spread(rs))) << 4));
    };
    // products of half h; beside them, the reads of half 1 - h of block kb_read and the loads of block kb_load (< 0: none)
    auto products = [&](int h, int kb_read, int kb_load) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int m = 0; m < NO * NT; ++m) {
                const int i = m / NT, j = m % NT, at = s * NO * NT + m;
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, f[h][NT + i][s]),
                                                                   __builtin_bit_cast(h8, f[h][j][s]), acc[i][j], 0, 0, 0);
#pragma unroll
                for (int q = 0; q < kReads; ++q)
                    if (q * kProducts / kReads == at) read(kb_read, 1 - h, q);
#pragma unroll
                for (int l = 0; l < kLoads; ++l)
                    if (kb_load >= 0 && l * kProducts / kLoads == at) stage(kb_load, l);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int kb = 0; kb < S - 1; ++kb)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) stage(kb, i);
    meet<(S - 2) * kLoads>();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) stage(S - 1, i);
#pragma unroll
    for (int q = 0; q < kReads; ++q) read(0, 0, q);
#pragma unroll 1
    for (int kb = 0; kb < total; ++kb) {
        products(0, kb, -1);
        meet<(S - 2) * kLoads>();                      // block kb has been read, block kb + 1 has arrived
        products(1, kb + 1, kb + S);
    }
    meet();                                            // the staging buffers are free

    // The results, 64 columns (o) of the wave's rows (t) at a time: to LDS, back as rows of eight columns to a lane, which take
    // what they need of A or X (whole lines, all under way before the first is used) and go out, and back once more as columns
    // for the other order.  (Taken in the instructions' layout, 16 columns of a lane's row, the same loads are 64 requests to an
    // instruction and one latency after the other: an UPDATE's start and end of a 256 x 256 tile took 40 us.)
    constexpr int kRoom = (int)sizeof(lds) / kWaves, kCols = WO < 64 ? WO : 64;
    static_assert(WT <= 64 && WT * 64 * 4 <= kRoom, "room for a wave's rows");
    constexpr int kRowLanes = kCols / 8, kRows = 64 / kRowLanes, kRowTurns = WT / kRows;
    constexpr int kColumnLanes = WT / 8, kColumns = 64 / kColumnLanes, kColumnTurns = kCols / kColumns;
    constexpr bool kPlane = MODE == UPDATE || MODE == LAST || (MODE == SQUARE && PRECISE);      // the operand's second halves
    float* const own = (float*)(&lds[0][0] + wave * kRoom);
    float* const diagonal = (float*)(mine + (MODE == GRAM ? w.d : w.e));
    const uint8_t* const px = mine + (MODE == SQUARE ? w.A : t_now) + (int64_t)t0 * pitch;
    // a column past a row's end is the next row's: not stored
    const __amdgpu_buffer_rsrc_t buf_x = buffer_of(px, bytes_t);
    const __amdgpu_buffer_rsrc_t buf_y = buffer_of(px + (MODE == SQUARE ? w.s_plane : w.t_plane), bytes_t);
    const __amdgpu_buffer_rsrc_t buf_d = buffer_of(mine + (MODE == SQUARE ? w.d : w.e), (int64_t)w.ldr * 4);
    const int m = g.tall ? g.c : g.r, n = g.tall ? g.r : g.c;                  // of the result
    auto deliver = [&](int row, int c, const float* x) {
        const int left = n - c;
        if (row >= m || left <= 0) return;
        const int64_t at = (int64_t)row * n + c;
        if constexpr (std::is_same_v<Out, Listed>) {
            float p[8];
            load_row<F32>(in.p[z], at, left, p);
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = __builtin_fmaf(-g.lr, x[k], p[k] * g.keep);
            store_row<F32>(in.p[z], at, left, p);
            if (in.p16[z]) store_row<BF16>(in.p16[z], at, left, p);
        } else {
            store_row<Out>(out, z * ((int64_t)m * n) + at, left, x);
        }
    };
    const bool columns_too = kSymmetric ? t0 != o0 : MODE == UPDATE || !g.tall;
    const int row0 = lane / kRowLanes, c = lane % kRowLanes * 8;               // of a turn's rows
    const int col0 = lane / kColumnLanes, r = lane % kColumnLanes * 8;         // of a turn's columns
#pragma unroll
    for (int i0 = 0; i0 < NO; i0 += kCols / 32) {
        __builtin_amdgcn_sched_barrier(0);             // one pass's loads at a time: no registers for more
        const int o = o0 + wo + i0 * 32 + c;
        u4 x[kRowTurns], y[kPlane ? kRowTurns : 1];
        float near[8] = {}, dt[kRowTurns];
        if constexpr (MODE != GRAM) {
#pragma unroll
            for (int k = 0; k < kRowTurns; ++k) {
                const int row = wt + k * kRows + row0;
                x[k] = halves_of(buf_x, row * pitch + o * 2);
                if constexpr (kPlane) y[k] = halves_of(buf_y, row * pitch + o * 2);
                if constexpr (MODE == SQUARE) dt[k] = as_f32(__builtin_amdgcn_raw_buffer_load_b32(buf_d, (t0 + row) * 4, 0, 0));
            }
            floats_of(buf_d, o * 4, near);
        }
#pragma unroll
        for (int i = 0; i < kCols / 32; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f16& v = acc[i0 + i][j];
                    *group_at(own, j * 32 + r32, i * 8 + half * 4 + k) = f4{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
                }
        own_done();
#pragma unroll
        for (int k = 0; k < kRowTurns; ++k) {
            const int row = k * kRows + row0, t = t0 + wt + row;
            f4* const at[2] = {group_at(own, row, c / 4), group_at(own, row, c / 4 + 1)};
            float v[8], a[8] = {}, b[8] = {};
            F32::open({*at[0], *at[1]}, v);
            const bool on = kSymmetric && t0 == o0 && t >= o && t < o + 8;     // the diagonal's element is here
            float d = 0.0f;
            if (on) {
#pragma unroll
                for (int l = 0; l < 8; ++l) d = t == o + l ? v[l] : d;
            }
            if constexpr (MODE != GRAM) F16::open(x[k], a);
            if constexpr (kPlane) F16::open(y[k], b);
#pragma unroll
            for (int l = 0; l < 8; ++l) {
                if (MODE == GRAM) v[l] *= kA / (kX * kX);
                else if (MODE == SQUARE)
                    v[l] = __builtin_fmaf(v[l], co.c * (kB / (kA * kA)),
                                          __builtin_fmaf(co.c, dt[k] + near[l], co.b) * (kB / kA) * (a[l] + b[l]));
                else v[l] = __builtin_fmaf(near[l], a[l] + b[l], v[l] * (1.0f / kB)) * (MODE == LAST ? 1.0f / kX : 1.0f);
            }
            if (on) {
                d *= MODE == GRAM ? 1.0f / (kX * kX) : 1.0f / (kA * kA);
                if (t < w.ldr) diagonal[t] = MODE == GRAM ? d : co.a + co.b * dt[k] + co.c * (dt[k] * dt[k] + d);
#pragma unroll
                for (int l = 0; l < 8; ++l) v[l] = t == o + l ? 0.0f : v[l];
            }
            if (columns_too) {
                *at[0] = f4{v[0], v[1], v[2], v[3]};
                *at[1] = f4{v[4], v[5], v[6], v[7]};
            }
            if constexpr (kSymmetric) {
                if (t < g.r && o < w.ldr)
                    put_halves<PRECISE>(mine + (MODE == GRAM ? w.A : w.B) + ((int64_t)t * w.ldr + o) * 2, w.s_plane, v);
            } else if constexpr (MODE == UPDATE) {
                if (t < g.c && o < w.ldr) put_halves<true>(mine + t_next + ((int64_t)t * w.ldr + o) * 2, w.t_plane, v);
            } else if (g.tall) {
                deliver(t, o, v);
            }
        }
        own_done();
        if (columns_too) {
#pragma unroll
            for (int k = 0; k < kColumnTurns; ++k) {
                const int column = k * kColumns + col0, oc = o0 + wo + i0 * 32 + column, t = t0 + wt + r;
                float v[8];
#pragma unroll
                for (int l = 0; l < 8; ++l) v[l] = ((const float*)group_at(own, r + l, column >> 2))[column & 3];
                if constexpr (kSymmetric) {
                    if (oc < g.r && t < w.ldr)
                        put_halves<PRECISE>(mine + (MODE == GRAM ? w.A : w.B) + ((int64_t)oc * w.ldr + t) * 2, w.s_plane, v);
                } else if constexpr (MODE == UPDATE) {
                    if (oc < g.r && t < w.ldc) put_halves<PRECISE>(mine + w.o + ((int64_t)oc * w.ldc + t) * 2, w.o_plane, v);
                } else {
                    deliver(oc, t, v);
                }
            }
            own_done();
        }
    }
}

// ------------------------------------------------------------------------------------------------------ start
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

// Eight of u, and with MOVE the momentum's step before.
template <typename T, bool MOVE>
__device__ __forceinline__ void load_u(const Start& a, int z, int64_t row, int n, int c, float factor, float* u) {
    const int left = n - c;
    const void* g = a.list ? a.in.g[z] : (const void*)((const typename T::elem*)a.batch.x + z * a.batch.step);
    load_row<T>(g, row * (a.list ? a.in.stride[z] : a.batch.stride) + c, left, u);
    if (!a.list) return;
    const int64_t at = row * n + c;
    float buf[8];
    load_row<F32>(a.in.buf[z], at, left, buf);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float g = (u[j] * factor) * (1.0f - a.mu);
        if (MOVE) buf[j] = __builtin_fmaf(a.mu, buf[j], g);
        u[j] = a.nesterov ? __builtin_fmaf(a.mu, buf[j], g) : buf[j];
    }
    if (MOVE) store_row<F32>(a.in.buf[z], at, left, buf);
}

// The momentum's step, and u's squares summed in 64 bits (an fp32 u may be as large as its type goes): a workgroup's rows in
// turn, as many threads to a row as it has groups of eight columns.
constexpr int kStartThreads = 256;
template <typename T>
__global__ __launch_bounds__(kStartThreads) void momentum_kernel(Start a, Plan plan) {
    __shared__ double sums[kStartThreads];
    const int z = blockIdx.y;
    const Group& group = group_of_matrix(plan, z);
    const int m = group.tall ? group.c : group.r, n = group.tall ? group.r : group.c;
    int lanes = 1;
    while (lanes < kStartThreads && lanes * 8 < n) lanes *= 2;
    const int per = kStartThreads / lanes, first = threadIdx.x / lanes, lane = threadIdx.x % lanes;
    const float factor = a.factor ? *a.factor : 1.0f;
    double s = 0.0;
    for (int64_t row = (int64_t)blockIdx.x * per + first; row < m; row += (int64_t)gridDim.x * per) {
        for (int c = lane * 8; c < n; c += lanes * 8) {
            float u[8];
            load_u<T, true>(a, z, row, n, c, factor, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) s = __builtin_fma((double)u[j], (double)u[j], s);
        }
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    for (int k = kStartThreads / 2; k; k >>= 1) {
        if ((int)threadIdx.x < k) sums[threadIdx.x] += sums[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.partials[(int64_t)z * kParts + blockIdx.x] = sums[0];
}

// X in both orders from u: 64 x 64 of it to a workgroup.  parts: of each matrix's kParts sums, that are there.
template <typename T, bool PRECISE>
__global__ __launch_bounds__(kStartThreads) void start_kernel(Start a, Plan plan, int parts) {
    __shared__ double sums[kParts];
    __shared__ float turned[64][68];
    const Group& group = group_of_tile(plan, blockIdx.x);
    const int m = group.tall ? group.c : group.r, n = group.tall ? group.r : group.c;
    const Layout w = layout_of(group.r, group.c, PRECISE);
    const int across = (n + 63) / 64, down = (m + 63) / 64, nth = (blockIdx.x - group.tile0) / (across * down);
    const int index = blockIdx.x - group.tile0 - nth * across * down, i0 = index / across * 64, j0 = index % across * 64;
    const int z = group.first + nth;
    sums[threadIdx.x] = (int)threadIdx.x < parts ? a.partials[(int64_t)z * kParts + threadIdx.x] : 0.0;
    __syncthreads();
    for (int k = kParts / 2; k; k >>= 1) {
        if ((int)threadIdx.x < k) sums[threadIdx.x] += sums[threadIdx.x + k];
        __syncthreads();
    }
    const double norm = sqrt(sums[0]), scale = (double)kX / (norm < a.eps ? a.eps : norm);       // NaN stays
    const float factor = a.factor ? *a.factor : 1.0f;
    uint8_t* const mine = plan.base + group.base + nth * w.size;
    // u's own order is t's where it is tall, o's where it is wide
    const bool tall = group.tall;
    uint8_t* const plain = mine + (tall ? w.t[0] : w.o);
    uint8_t* const other = mine + (tall ? w.o : w.t[0]);
    const int64_t plane_plain = tall ? w.t_plane : w.o_plane, plane_other = tall ? w.o_plane : w.t_plane;
    const int ld_plain = tall ? w.ldr : w.ldc, ld_other = tall ? w.ldc : w.ldr;
    const int c = threadIdx.x % 8 * 8;
    auto put = [&](uint8_t* at, int64_t plane, bool pair, const float* v) {
        if (PRECISE || pair) put_halves<true>(at, plane, v);
        else put_halves<false>(at, plane, v);
    };
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int row = threadIdx.x / 8 + 32 * k;
        float u[8] = {};
        if (i0 + row < m && j0 + c < n) {
            load_u<T, false>(a, z, i0 + row, n, j0 + c, factor, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = j0 + c + j < n ? (float)((double)u[j] * scale) : 0.0f;
        }
        if (i0 + row < m) put(plain + ((int64_t)(i0 + row) * ld_plain + j0 + c) * 2, plane_plain, tall, u);
        *(f4*)&turned[row][c] = f4{u[0], u[1], u[2], u[3]};
        *(f4*)&turned[row][c + 4] = f4{u[4], u[5], u[6], u[7]};
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int row = threadIdx.x / 8 + 32 * k;
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = turned[c + j][row];
        if (j0 + row < n) put(other + ((int64_t)(j0 + row) * ld_other + i0 + c) * 2, plane_other, !tall, u);
    }
}

// ------------------------------------------------------------------------------------------------------ small matrices
// A matrix whose shorter side is at most 128 and that LDS holds: one workgroup does all of it in one launch (64 x 256: 17
// launches took 71 us).  X itself stays in registers, in fp32 and in the matrix instructions' layout (so e X is what their sums
// begin with), and its fp16 form in LDS is read by rows for A and turned, by transposing reads, for B X.
//
// The pieces: X's fragments of 32 x 32 are dealt to the eight waves, F at most to each; A's (all of them) too, and where they
// are fewer than the waves their summed axis is cut into parts that are added in order.  Rows in LDS are 16 bytes longer than a
// multiple of 64, so that 16 rows' pieces of 16 bytes lie in different banks.
struct Whole {
    Plan plan;                                         // the groups (base, tile0: not used)
    Start start;
    void* out;                                         // or p and p16 of the list
    int dtype, out_dtype;
    int steps;
    float co[3 * kMaxSteps];
};
constexpr int kWholeWaves = 8, kWholeSide = 128;
// Bytes of a matrix of R x C fragments, and where they are.
struct Places {
    int px, pa;                                        // bytes of a row of X, and of A and B
    int x_plane, a_plane, A, B, sums, d, e, size;
    int cuts;                                          // parts of A's summed axis
};
__host__ __device__ inline Places places_of(int R, int C, bool precise) {
    Places p;
    const int planes = precise ? 2 : 1;
    p.px = C * 64 + 16;
    p.pa = R * 64 + 16;
    p.x_plane = R * 32 * p.px;
    p.a_plane = R * 32 * p.pa;
    p.cuts = R == 1 ? 8 : R == 2 ? 2 : 1;
    p.A = planes * p.x_plane;
    p.B = p.A + planes * p.a_plane;
    p.d = p.B + planes * p.a_plane;
    p.e = p.d + R * 128;
    p.sums = p.e + R * 128;
    p.size = p.sums + (p.cuts > 1 ? p.cuts * R * R * 4096 : 0);
    return p;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
    return dtype == Z1_F32 ? F32::one(p, i) : dtype == Z1_BF16 ? BF16::one(p, i) : F16::one(p, i);
}

// 16 neighbours of a row as fp16, and what that leaves.
template <bool PAIR>
__device__ __forceinline__ void keep16(uint8_t* at, int plane, const float* v) {
#pragma unroll
    for (int k = 0; k < 16; k += 8) {
        const u4 hi = F16::close(v + k);
        *(u4*)(at + k * 2) = hi;
        if constexpr (PAIR) {
            float f[8], lo[8];
            F16::open(hi, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) lo[j] = v[k + j] - f[j];
            *(u4*)(at + plane + k * 2) = F16::close(lo);
        }
    }
}

template <bool PRECISE, int F, int BYTES>
__global__ __launch_bounds__(kWholeWaves * 64) void whole_kernel(Whole a) {
    __shared__ __align__(16) uint8_t lds[BYTES];
    __shared__ double norms[kWholeWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int z = blockIdx.x, l32 = lane & 31, half = lane >> 5, rs = spread(l32);
    const Group& g = group_of_matrix(a.plan, z);
    const int R = (g.r + 31) / 32, C = (g.c + 31) / 32, pieces = R * C;
    const Places at = places_of(R, C, PRECISE);
    const int m = g.tall ? g.c : g.r, n = g.tall ? g.r : g.c;
    // a lane's part of X's q-th fragment: row o, columns t .. t + 15
    auto o_of = [&](int q) { return (wave + q * kWholeWaves) % R * 32 + l32; };
    auto t_of = [&](int q) { return (wave + q * kWholeWaves) / R * 32 + half * 16; };
    auto on = [&](int q) { return wave + q * kWholeWaves < pieces; };          // the wave's

    f16 x[F];
    double s = 0.0;
    const float factor = a.start.factor ? *a.start.factor : 1.0f;
    const void* from = a.start.list ? a.start.in.g[z] : a.start.batch.x;
    const int64_t first = a.start.list ? 0 : z * a.start.batch.step, stride = a.start.list ? a.start.in.stride[z] : a.start.batch.stride;
#pragma unroll
    for (int q = 0; q < F; ++q) {
        x[q] = f16{};
        if (!on(q)) continue;
        const int o = o_of(q), t = t_of(q);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (o >= g.r || t + k >= g.c) continue;
            const int row = g.tall ? t + k : o, c = g.tall ? o : t + k;
            float u = load_any(from, first + row * stride + c, a.dtype);
            if (a.start.list) {
                float* const p = a.start.in.buf[z] + (int64_t)row * n + c;
                const float step = (u * factor) * (1.0f - a.start.mu), buf = __builtin_fmaf(a.start.mu, *p, step);
                *p = buf;
                u = a.start.nesterov ? __builtin_fmaf(a.start.mu, buf, step) : buf;
            }
            x[q][k] = u;
            s = __builtin_fma((double)u, (double)u, s);
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
    norms[wave] = s;                                   // every lane writes the same value
    __syncthreads();
    s = norms[0];
    for (int i = 1; i < kWholeWaves; ++i) s += norms[i];
    const double norm = sqrt(s), scale = 1.0 / (norm < a.start.eps ? a.start.eps : norm);        // NaN stays
    auto keep_x = [&](int q) {
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = x[q][k] * kX;
        keep16<PRECISE>(lds + o_of(q) * at.px + t_of(q) * 2, at.x_plane, v);
    };
#pragma unroll
    for (int q = 0; q < F; ++q) {
        if (!on(q)) continue;
#pragma unroll
        for (int k = 0; k < 16; ++k) x[q][k] = (float)((double)x[q][k] * scale);
        keep_x(q);
    }
    float* const d = (float*)(lds + at.d);
    float* const e = (float*)(lds + at.e);
    float* const sums = (float*)(lds + at.sums);
    // eight of a row's columns, the step-th 16 of them: a lane's operand
    auto by_row = [&](const uint8_t* rows, int pitch, int row, int step) {
        return __builtin_bit_cast(h8, *(const u4*)(rows + row * pitch + step * 32 + half * 16));
    };
    auto add = [&](f16 acc, h8 p, h8 q) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(p, q, acc, 0, 0, 0); };
    // rows i of one operand, in spread order, times rows j of the other, over steps of 16 of their columns
    auto square = [&](const uint8_t* rows, int pitch, int plane, int i, int j, int begin, int end) {
        f16 acc = f16{};
        for (int k = begin; k < end; ++k) {
            const h8 p = by_row(rows, pitch, i * 32 + rs, k), q = by_row(rows, pitch, j * 32 + l32, k);
            acc = add(acc, p, q);
            if constexpr (PRECISE) {
                acc = add(acc, p, by_row(rows + plane, pitch, j * 32 + l32, k));
                acc = add(acc, by_row(rows + plane, pitch, i * 32 + rs, k), q);
            }
        }
        return acc;
    };
    const int squares = R * R;

    for (int step = 0; step < a.steps; ++step) {
        const float ca = a.co[3 * step], cb = a.co[3 * step + 1], cc = a.co[3 * step + 2];
        __syncthreads();                               // X is there
        // A: row j, columns i .. i + 15 of a fragment to a lane
        auto finish_a = [&](int ij, f16 v) {
            const int i = ij / R * 32 + half * 16, j = ij % R * 32 + l32;
            float y[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                if (i + k == j) d[j] = v[k] * (1.0f / (kX * kX));
                y[k] = i + k == j ? 0.0f : v[k] * (kA / (kX * kX));
            }
            keep16<PRECISE>(lds + at.A + j * at.pa + i * 2, at.a_plane, y);
        };
        if (at.cuts == 1) {
            for (int ij = wave; ij < squares; ij += kWholeWaves)
                finish_a(ij, square(lds, at.px, at.x_plane, ij / R, ij % R, 0, 2 * C));
        } else {
            const int ij = wave / at.cuts, cut = wave % at.cuts;               // squares * cuts waves: all eight
            const f16 v = square(lds, at.px, at.x_plane, ij / R, ij % R, cut * 2 * C / at.cuts, (cut + 1) * 2 * C / at.cuts);
#pragma unroll
            for (int k = 0; k < 16; ++k) sums[(wave * 16 + k) * 64 + lane] = v[k];
            __syncthreads();
            if (wave < squares) {
                f16 t = f16{};
                for (int i = 0; i < at.cuts; ++i)
#pragma unroll
                    for (int k = 0; k < 16; ++k) t[k] += sums[((wave * at.cuts + i) * 16 + k) * 64 + lane];
                finish_a(wave, t);
            }
        }
        __syncthreads();
        for (int ij = wave; ij < squares; ij += kWholeWaves) {
            const f16 v = square(lds + at.A, at.pa, at.a_plane, ij / R, ij % R, 0, 2 * R);
            const int i = ij / R * 32 + half * 16, j = ij % R * 32 + l32;
            const uint8_t* own = lds + at.A + j * at.pa + i * 2;
            const float dj = d[j];
            float y[16], lo[16] = {};
            F16::open(*(const u4*)own, y);
            F16::open(*(const u4*)(own + 16), y + 8);
            if constexpr (PRECISE) {
                F16::open(*(const u4*)(own + at.a_plane), lo);
                F16::open(*(const u4*)(own + at.a_plane + 16), lo + 8);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                if (i + k == j) e[j] = ca + cb * dj + cc * (dj * dj + v[k] * (1.0f / (kA * kA)));
                const float w = __builtin_fmaf(v[k], cc * (kB / (kA * kA)), __builtin_fmaf(cc, dj + d[i + k], cb) * (kB / kA) * (y[k] + lo[k]));
                y[k] = i + k == j ? 0.0f : w;
            }
            keep16<PRECISE>(lds + at.B + j * at.pa + i * 2, at.a_plane, y);
        }
        __syncthreads();
        // a transposing read: the lane's row and four columns of it
        const int turned = (lane >> 5) * 8 + ((lane & 15) >> 2), column = spread((lane >> 4 & 1) * 16 + (lane & 3) * 4);
#pragma unroll
        for (int q = 0; q < F; ++q) {
            if (!on(q)) continue;
            const int o = (wave + q * kWholeWaves) % R * 32, t = (wave + q * kWholeWaves) / R * 32;
            const float scale_o = e[o + l32] * (kX * kB);
            f16 acc;
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[k] = x[q][k] * scale_o;
            for (int k = 0; k < 2 * R; ++k) {
                auto by_column = [&](const uint8_t* rows) {
                    const uint8_t* p = rows + (k * 16 + turned) * at.px + (t + column) * 2;
                    const s4 f0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)p);
                    const s4 f1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)(p + 4 * at.px));
                    return __builtin_bit_cast(h8, __builtin_shufflevector(f0, f1, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                const h8 p = by_column(lds), b = by_row(lds + at.B, at.pa, o + l32, k);
                acc = add(acc, p, b);
                if constexpr (PRECISE) {
                    acc = add(acc, p, by_row(lds + at.B + at.a_plane, at.pa, o + l32, k));
                    acc = add(acc, by_column(lds + at.x_plane), b);
                }
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) x[q][k] = acc[k] * (1.0f / (kX * kB));
        }
        if (step + 1 == a.steps) break;
        __syncthreads();                               // X has been read
#pragma unroll
        for (int q = 0; q < F; ++q)
            if (on(q)) keep_x(q);
    }
#pragma unroll
    for (int q = 0; q < F; ++q) {
        if (!on(q)) continue;
        const int o = o_of(q), t = t_of(q);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (o >= g.r || t + k >= g.c) continue;
            const int64_t to = g.tall ? (int64_t)(t + k) * n + o : (int64_t)o * n + t + k;
            const float v = x[q][k];
            if (a.start.list) {
                float* const p = a.start.in.p[z] + to;
                const float r = __builtin_fmaf(-g.lr, v, *p * g.keep);
                *p = r;
                if (a.start.in.p16[z]) BF16::put(a.start.in.p16[z], to, r);
            } else {
                const int64_t i = z * ((int64_t)m * n) + to;
                if (a.out_dtype == Z1_BF16) BF16::put(a.out, i, v);
                else if (a.out_dtype == Z1_F16) F16::put(a.out, i, v);
                else F32::put(a.out, i, v);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------ host
constexpr int64_t kMaxSide = 1 << 20;
constexpr int64_t kMaxCount = 1 << 15;                 // of a call: a grid's second axis
constexpr int64_t kMaxTiles = 1ll << 22;               // of a launch: its threads count in 32 bits
constexpr int kCus = 256;

// The small matrices' kernel: fragments to a wave and bytes of LDS.  0: the matrix is too large for it.
struct WholeWay {
    int pieces, bytes;
};
WholeWay whole_way(int64_t m, int64_t n, bool precise) {
    const int64_t r = m < n ? m : n, c = m < n ? n : m;
    if (r > kWholeSide || c > 64 * 32) return {0, 0};
    const int R = (int)(r + 31) / 32, C = (int)(c + 31) / 32, bytes = places_of(R, C, precise).size;
    for (const WholeWay way : {WholeWay{1, 64 << 10}, WholeWay{2, 64 << 10}, WholeWay{4, 159 << 10}, WholeWay{8, 159 << 10}})
        if (R * C <= way.pieces * kWholeWaves && bytes <= way.bytes && !(precise && way.pieces == 8)) return way;
    return {0, 0};
}
bool is_whole(int64_t m, int64_t n, bool precise) { return whole_way(m, n, precise).pieces != 0; }

template <bool PRECISE>
int launch_whole(const Whole& a, const WholeWay& way, int64_t count, hipStream_t st) {
    const dim3 grid((unsigned)count);
    switch (way.pieces) {
        case 1: whole_kernel<PRECISE, 1, 64 << 10><<<grid, kWholeWaves * 64, 0, st>>>(a); break;
        case 2: whole_kernel<PRECISE, 2, 64 << 10><<<grid, kWholeWaves * 64, 0, st>>>(a); break;
        case 4: whole_kernel<PRECISE, 4, 159 << 10><<<grid, kWholeWaves * 64, 0, st>>>(a); break;
        default:                                       // pairs of as many do not fit LDS
            if constexpr (!PRECISE) whole_kernel<false, 8, 159 << 10><<<grid, kWholeWaves * 64, 0, st>>>(a);
    }
    return (int)hipGetLastError();
}
// `count` matrices of the plan's groups, all of them small; way: the largest one's.
int run_whole(const Start& start, const Plan& plan, const WholeWay& way, int64_t count, int dtype, int steps,
              const float* coefficients, bool precise, void* out, int out_dtype, hipStream_t st) {
    Whole a{plan, start, out, dtype, out_dtype, steps, {}};
    for (int i = 0; i < 3 * steps; ++i) a.co[i] = coefficients[i];
    return precise ? launch_whole<true>(a, way, count, st) : launch_whole<false>(a, way, count, st);
}

// Whether the iterates stay in the stored ranges: |X| < 4 and |B| < 32 from singular values in [0, 1] on.
bool bounded(const float* coefficients, int steps) {
    double top = 1.0 + 1e-6;
    for (int k = 0; k < steps; ++k) {
        const double a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
        if (!(fabs(a) <= 64.0 && fabs(b) <= 1024.0 && fabs(c) <= 1024.0)) return false;         // NaN too
        auto f = [&](double s) { return s * (a + s * s * (b + c * s * s)); };
        auto p = [&](double l) { return l * (b + c * l); };
        double most = fabs(f(top)), large = fabs(p(top * top));
        auto try_x = [&](double q) {                   // a stationary point's s^2
            if (q > 0.0 && q < top * top) most = fmax(most, fabs(f(sqrt(q))));
        };
        if (c != 0.0) {
            const double disc = 9.0 * b * b - 20.0 * a * c;
            if (disc >= 0.0) {
                try_x((-3.0 * b + sqrt(disc)) / (10.0 * c));
                try_x((-3.0 * b - sqrt(disc)) / (10.0 * c));
            }
            const double l = -b / (2.0 * c);
            if (l > 0.0 && l < top * top) large = fmax(large, fabs(p(l)));
        } else if (b != 0.0) {
            try_x(-a / (3.0 * b));
        }
        top = most * (1.0 + 1e-3);                     // roundings on the way
        if (!(top < 4.0 && large < 32.0)) return false;
    }
    return true;
}

// Tiles of b x b in a launch, each group's first one noted in it.
template <Mode MODE>
int64_t tiles_of(Plan& w, int64_t b) {
    int64_t n = 0;
    for (int k = 0; k < w.groups; ++k) {
        Group& g = w.g[k];
        const int64_t across = (g.r + b - 1) / b, down = (g.c + b - 1) / b;
        g.tile0 = (int)n;
        n += g.count * (MODE == GRAM || MODE == SQUARE ? across * (across + 1) / 2 : down * across);
        if (n > kMaxTiles) return n;
    }
    return n;
}

// All arguments of the steps' launches.
struct Steps {
    Plan plan;
    Coefficients co;
    void* out;
    Inputs in;
    hipStream_t st;
};
template <Mode MODE, bool PRECISE, typename Out, int COARSE, int B, int WT, int WO, int S>
int launch(Steps& a, int64_t first, int64_t last) {
    const int64_t all = tiles_of<MODE>(a.plan, COARSE * B), tiles = ((last < 0 ? all : last) - first) * COARSE * COARSE;
    if (all > kMaxTiles || tiles > kMaxTiles) return Z1_E_SIZE;
    step_kernel<MODE, PRECISE, Out, COARSE, B, B, WT, WO, S>
        <<<dim3((unsigned)tiles), B / WT * (B / WO) * 64, 0, a.st>>>(a.plan, a.co, a.out, a.in, (int)first);
    return (int)hipGetLastError();
}
template <Mode MODE, bool PRECISE, typename Out = Listed>
int launch_step(Steps& a) {
    const int64_t large = tiles_of<MODE>(a.plan, 256), rounds = large / kCus, rest = large % kCus;
    if (rounds > 0) {
        const int64_t whole = rest * 2 > kCus ? large : large - rest;
        if (const int rc = launch<MODE, PRECISE, Out, 1, 256, 64, 128, 2>(a, 0, whole)) return rc;
        if (whole == large) return Z1_OK;
        if (4 * rest <= kCus) return launch<MODE, PRECISE, Out, 2, 128, 64, 64, 4>(a, whole, large);
        return launch<MODE, PRECISE, Out, 2, 128, 64, 64, 2>(a, whole, large);
    }
    const int64_t middle = tiles_of<MODE>(a.plan, 128);
    if (middle > kCus) return launch<MODE, PRECISE, Out, 1, 128, 64, 64, 2>(a, 0, -1);
    if (middle * 2 > kCus) return launch<MODE, PRECISE, Out, 1, 128, 64, 64, 4>(a, 0, -1);
    return launch<MODE, PRECISE, Out, 1, 64, 32, 32, 4>(a, 0, -1);
}

template <typename T>
int start_of(const Start& a, Plan& w, int64_t count, bool precise, hipStream_t st) {
    // enough workgroups for the largest matrix, 2048 elements or a row each
    int64_t parts = 1, tiles = 0;
    for (int k = 0; k < w.groups; ++k) {
        Group& g = w.g[k];
        const int64_t m = g.tall ? g.c : g.r, n = g.tall ? g.r : g.c, rows = 2048 / (n < 8 ? 8 : n) + 1, need = (m + rows - 1) / rows;
        parts = need > parts ? need : parts;
        g.tile0 = (int)tiles;
        tiles += g.count * ((n + 63) / 64) * ((m + 63) / 64);
        if (tiles > 2 * kMaxTiles) return Z1_E_SIZE;
    }
    if (parts > kParts) parts = kParts;
    momentum_kernel<T><<<dim3((unsigned)parts, (unsigned)count), kStartThreads, 0, st>>>(a, w);
    const dim3 grid((unsigned)tiles);
    if (precise) start_kernel<T, true><<<grid, kStartThreads, 0, st>>>(a, w, (int)parts);
    else start_kernel<T, false><<<grid, kStartThreads, 0, st>>>(a, w, (int)parts);
    return (int)hipGetLastError();
}

template <bool PRECISE, typename Out>
int iterate(Steps& a, int steps, const float* coefficients) {
    for (int k = 0; k < steps; ++k) {
        a.co = {coefficients[3 * k], coefficients[3 * k + 1], coefficients[3 * k + 2]};
        a.plan.cur = k & 1;
        if (const int rc = launch_step<GRAM, PRECISE>(a)) return rc;
        if (const int rc = launch_step<SQUARE, PRECISE>(a)) return rc;
        const int rc = k + 1 < steps ? launch_step<UPDATE, PRECISE>(a) : launch_step<LAST, PRECISE, Out>(a);
        if (rc) return rc;
    }
    return Z1_OK;
}

int64_t partials_of(int64_t count) { return (count * kParts * (int64_t)sizeof(double) + 1023) / 1024 * 1024; }
int64_t size_of(int64_t m, int64_t n, bool precise) {
    return layout_of((int)(m < n ? m : n), (int)(m < n ? n : m), precise).size;
}

bool bad_dtype(int d) { return d != Z1_F32 && d != Z1_BF16 && d != Z1_F16; }
bool bad_side(int64_t n) { return n < 1 || n > kMaxSide; }
int check(int dtype, int steps, const float* coefficients, float eps) {
    if (bad_dtype(dtype)) return Z1_E_DTYPE;
    if (steps < 1 || steps > kMaxSteps) return Z1_E_SIZE;
    if (!coefficients) return Z1_E_NULL;
    if (!(eps > 0.0f) || !bounded(coefficients, steps)) return Z1_E_MODE;
    return Z1_OK;
}

template <typename Out>
int run(Start a, Plan w, int64_t count, int dtype, int steps, const float* coefficients, bool precise, void* out, void* workspace,
        hipStream_t st) {
    a.partials = (double*)workspace;
    w.base = (uint8_t*)workspace + partials_of(count);
    int rc;
    switch (dtype) {
        case Z1_F32: rc = start_of<F32>(a, w, count, precise, st); break;
        case Z1_BF16: rc = start_of<BF16>(a, w, count, precise, st); break;
        default: rc = start_of<F16>(a, w, count, precise, st); break;
    }
    if (rc) return rc;
    Steps s{w, {}, out, a.in, st};
    return precise ? iterate<true, Out>(s, steps, coefficients) : iterate<false, Out>(s, steps, coefficients);
}

}  // namespace

extern "C" {

int64_t z1_orthogonalize_workspace(int64_t count, int64_t m, int64_t n, int precise) {
    if (count < 0 || count > kMaxCount || bad_side(m) || bad_side(n)) return Z1_E_SIZE;
    return is_whole(m, n, precise != 0) ? 0 : partials_of(count) + count * size_of(m, n, precise != 0);
}

int z1_orthogonalize(const void* x, int64_t step, int64_t stride, int64_t count, int64_t m, int64_t n, int dtype, void* out,
                     int out_dtype, int steps, const float* coefficients, float eps, int precise, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    const int64_t need = z1_orthogonalize_workspace(count, m, n, precise);
    if (need < 0) return (int)need;
    if (const int rc = check(dtype, steps, coefficients, eps)) return rc;
    if (step < 0 || stride < 0) return Z1_E_SIZE;
    if (bad_dtype(out_dtype)) return Z1_E_DTYPE;
    if (count == 0) return Z1_OK;
    if (!x || !out || (need && !workspace)) return Z1_E_NULL;
    if (workspace_bytes < need) return Z1_E_WORKSPACE;
    Start a{};
    a.batch = {x, step, stride};
    a.eps = eps;
    Plan w{};
    w.groups = 1;
    w.g[0] = {0, (int)(m < n ? m : n), (int)(m < n ? n : m), m > n, 0, (int)count, 0, 0.0f, 0.0f};
    const hipStream_t st = (hipStream_t)stream;
    if (!need)
        return run_whole(a, w, whole_way(m, n, precise != 0), count, dtype, steps, coefficients, precise != 0, out, out_dtype, st);
    switch (out_dtype) {
        case Z1_F32: return run<F32>(a, w, count, dtype, steps, coefficients, precise != 0, out, workspace, st);
        case Z1_BF16: return run<BF16>(a, w, count, dtype, steps, coefficients, precise != 0, out, workspace, st);
        default: return run<F16>(a, w, count, dtype, steps, coefficients, precise != 0, out, workspace, st);
    }
}

int64_t z1_muon_workspace(const z1_matrix* list, int count, int precise) {
    if (count < 0 || count > kList) return Z1_E_SIZE;
    if (count > 0 && !list) return Z1_E_NULL;
    int64_t bytes = 0, large = 0;
    for (int i = 0; i < count; ++i) {
        if (bad_side(list[i].m) || bad_side(list[i].n)) return Z1_E_SIZE;
        if (is_whole(list[i].m, list[i].n, precise != 0)) continue;
        bytes += size_of(list[i].m, list[i].n, precise != 0);
        ++large;
    }
    return bytes + partials_of(large);
}

int z1_muon_step(const z1_matrix* list, int count, int dtype, const z1_muon* how, void* workspace, int64_t workspace_bytes,
                 void* stream) {
    if (!how) return Z1_E_NULL;
    const int64_t need = z1_muon_workspace(list, count, how->precise);
    if (need < 0) return (int)need;
    if (const int rc = check(dtype, how->steps, how->coefficients, how->eps)) return rc;
    for (int i = 0; i < count; ++i) {
        if (!list[i].g || !list[i].momentum || !list[i].p) return Z1_E_NULL;
        if (list[i].g_stride < 0) return Z1_E_SIZE;
    }
    if (count == 0) return Z1_OK;
    if (need && !workspace) return Z1_E_NULL;
    if (workspace_bytes < need) return Z1_E_WORKSPACE;

    // the largest first, equal ones together: a launch then ends in its smallest work; the small ones by themselves
    const bool precise = how->precise != 0;
    int order[kList], small = 0;
    for (int i = 0; i < count; ++i) order[i] = i;
    std::stable_sort(order, order + count, [&](int i, int j) {
        const z1_matrix &a = list[i], &b = list[j];
        const bool wa = is_whole(a.m, a.n, precise), wb = is_whole(b.m, b.n, precise);
        if (wa != wb) return wa;
        if (a.m * a.n != b.m * b.n) return a.m * a.n > b.m * b.n;
        return a.m != b.m ? a.m < b.m : a.lr != b.lr ? a.lr < b.lr : a.keep < b.keep;
    });
    while (small < count && is_whole(list[order[small]].m, list[order[small]].n, precise)) ++small;
    auto run_some = [&](int first, int end) {
        Start a{};
        Plan w{};
        WholeWay way{0, 0};
        int64_t base = 0;
        for (int i = first; i < end; ++i) {
            const z1_matrix& x = list[order[i]];
            const int k = i - first;
            a.in.g[k] = x.g;
            a.in.stride[k] = x.g_stride;
            a.in.buf[k] = x.momentum;
            a.in.p[k] = x.p;
            a.in.p16[k] = x.p16;
            const z1_matrix* before = k ? &list[order[i - 1]] : nullptr;
            if (before && before->m == x.m && before->n == x.n && before->lr == x.lr && before->keep == x.keep) {
                ++w.g[w.groups - 1].count;
            } else {
                const int r = (int)(x.m < x.n ? x.m : x.n), c = (int)(x.m < x.n ? x.n : x.m);
                w.g[w.groups++] = {base, r, c, x.m > x.n, k, 1, 0, x.lr, x.keep};
            }
            base += size_of(x.m, x.n, precise);
            const WholeWay own = whole_way(x.m, x.n, precise);
            if (own.pieces > way.pieces) way = own;
        }
        a.list = 1;
        a.factor = how->factor;
        a.mu = how->momentum;
        a.nesterov = how->nesterov;
        a.eps = how->eps;
        const hipStream_t st = (hipStream_t)stream;
        if (end <= small)
            return run_whole(a, w, way, end - first, dtype, how->steps, how->coefficients, precise, nullptr, 0, st);
        return run<Listed>(a, w, end - first, dtype, how->steps, how->coefficients, precise, nullptr, workspace, st);
    };
    if (small > 0) {
        const int rc = run_some(0, small);
        if (rc) return rc;
    }
    return small < count ? run_some(small, count) : Z1_OK;
}

}  // extern "C"
