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

#include <type_traits>

#pragma clang fp contract(off)

namespace {

using namespace z1blk;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float kX = 4096.0f, kA = 2048.0f, kB = 1024.0f;
constexpr int kHalves = 64;                            // columns of a staged block: 128 bytes
constexpr int kParts = 256;                            // partial sums of a matrix's squares
constexpr int kList = 32;                              // matrices named one by one in a launch

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

// The workspace of a launch's matrices, `size` bytes each.
struct Work {
    uint8_t* base;
    int64_t size;
    int64_t t[2], o, A, B, d, e;                       // offsets in it: X in both orders, A, B (pairs), diagonals
    int64_t t_plane, o_plane, s_plane;                 // bytes from a pair's first halves to its second ones
    int r, c, ldr, ldc;                                // ldr, ldc: r and c rounded up to blocks
    int cur;                                           // which t is read
};

struct Coefficients {
    float a, b, c;
};

// What becomes of the last step's X.
struct Result {
    void* out;                                         // contiguous (else p and p16 of `in`)
    int tall;                                          // u has more rows than columns: its rows are c
    float lr, keep;
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
__global__ __launch_bounds__(BT / WT * (BO / WO) * 64) void step_kernel(Work w, Coefficients co, Result out, Inputs in, int first) {
    constexpr bool kSymmetric = MODE == GRAM || MODE == SQUARE;
    constexpr int kWaves = BT / WT * (BO / WO);
    constexpr int kPT = BT / 8 / kWaves, kPO = BO / 8 / kWaves;                // direct loads of a wave: 8 rows each
    constexpr int NT = WT / 32, NO = WO / 32;
    static_assert(!kSymmetric || BT == BO, "a triangle of square tiles");
    static_assert(S == 2 || S == 4, "a block's buffer is kb & (S - 1)");
    constexpr int kRow = kHalves * 2;
    __shared__ __align__(1024) uint8_t lds[S][(BT + BO) * kRow];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rows_t = kSymmetric ? w.r : w.c;
    const int down = (rows_t + COARSE * BT - 1) / (COARSE * BT), across = (w.r + COARSE * BO - 1) / (COARSE * BO);
    const int tiles = kSymmetric ? down * (down + 1) / 2 : down * across;
    const int run = in_runs(), index = first + run / (COARSE * COARSE), z = index / tiles;
    const Place tile = kSymmetric ? in_triangle(index - z * tiles) : in_panel(index - z * tiles, down, across);
    const int part = run % (COARSE * COARSE);
    const int t0 = (tile.down * COARSE + part / COARSE) * BT, o0 = (tile.across * COARSE + part % COARSE) * BO;
    if (COARSE > 1 && (t0 >= rows_t || o0 >= w.r || (kSymmetric && o0 > t0))) return;          // past the end, or the upper half
    const int wt = wave / (BO / WO) * WT, wo = wave % (BO / WO) * WO;          // the wave's part of the tile
    uint8_t* const mine = w.base + z * w.size;

    const int ld = MODE == GRAM ? w.ldc : w.ldr, pitch = ld * 2, blocks = ld / kHalves;
    const uint8_t* const pt = mine + (MODE == GRAM ? w.o : MODE == SQUARE ? w.A : w.t[w.cur]) + (int64_t)t0 * pitch;
    const uint8_t* const po = mine + (MODE == GRAM ? w.o : MODE == SQUARE ? w.A : w.B) + (int64_t)o0 * pitch;
    const int64_t plane_t = MODE == GRAM ? w.o_plane : MODE == SQUARE ? w.s_plane : w.t_plane;
    const int64_t plane_o = MODE == GRAM ? w.o_plane : w.s_plane;
    const int64_t bytes_t = (int64_t)(rows_t - t0) * pitch, bytes_o = (int64_t)(w.r - o0) * pitch;
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
        const int g = i < kPT ? wave * kPT + i : wave * kPO + i - kPT;
        int k = kb < last ? kb : last;
        bool t_lo = false, o_lo = false;
        if (PRECISE) {                                 // hi hi, hi lo, lo hi
            t_lo = k >= 2 * blocks;
            o_lo = k >= blocks && !t_lo;
            k -= t_lo ? 2 * blocks : o_lo ? blocks : 0;
        }
        const int row = g * 8 * pitch;
        if (i < kPT) load_lds(t_lo ? lo_t : hi_t, buf + g * 8 * kRow, row + (g & 1 ? from ^ 64 : from), k * kRow);
        else load_lds(o_lo ? lo_o : hi_o, buf + (BT + g * 8) * kRow, row + (g & 2 ? from ^ 64 : from), k * kRow);
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
    const uint8_t* const px = mine + (MODE == SQUARE ? w.A : w.t[w.cur]) + (int64_t)t0 * pitch;
    // a column past a row's end is the next row's: not stored
    const __amdgpu_buffer_rsrc_t buf_x = buffer_of(px, bytes_t);
    const __amdgpu_buffer_rsrc_t buf_y = buffer_of(px + (MODE == SQUARE ? w.s_plane : w.t_plane), bytes_t);
    const __amdgpu_buffer_rsrc_t buf_d = buffer_of(mine + (MODE == SQUARE ? w.d : w.e), (int64_t)w.ldr * 4);
    const int m = out.tall ? w.c : w.r, n = out.tall ? w.r : w.c;              // of the result
    auto deliver = [&](int row, int c, const float* x) {
        const int left = n - c;
        if (row >= m || left <= 0) return;
        const int64_t at = (int64_t)row * n + c;
        if constexpr (std::is_same_v<Out, Listed>) {
            float p[8];
            load_row<F32>(in.p[z], at, left, p);
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = __builtin_fmaf(-out.lr, x[k], p[k] * out.keep);
            store_row<F32>(in.p[z], at, left, p);
            if (in.p16[z]) store_row<BF16>(in.p16[z], at, left, p);
        } else {
            store_row<Out>(out.out, z * ((int64_t)m * n) + at, left, x);
        }
    };
    const bool columns_too = kSymmetric ? t0 != o0 : MODE == UPDATE || !out.tall;
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
                if (t < w.r && o < w.ldr)
                    put_halves<PRECISE>(mine + (MODE == GRAM ? w.A : w.B) + ((int64_t)t * w.ldr + o) * 2, w.s_plane, v);
            } else if constexpr (MODE == UPDATE) {
                if (t < w.c && o < w.ldr) put_halves<true>(mine + w.t[w.cur ^ 1] + ((int64_t)t * w.ldr + o) * 2, w.t_plane, v);
            } else if (out.tall) {
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
                    if (oc < w.r && t < w.ldr)
                        put_halves<PRECISE>(mine + (MODE == GRAM ? w.A : w.B) + ((int64_t)oc * w.ldr + t) * 2, w.s_plane, v);
                } else if constexpr (MODE == UPDATE) {
                    if (oc < w.r && t < w.ldc) put_halves<PRECISE>(mine + w.o + ((int64_t)oc * w.ldc + t) * 2, w.o_plane, v);
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
    int m, n;
    const float* factor;                               // of g, or NULL
    float mu;
    int nesterov;
    double eps;
    double* partials;                                  // [count][kParts]
    int parts;                                         // of kParts, that are used
};

// Eight of u, and with MOVE the momentum's step before.
template <typename T, bool MOVE>
__device__ __forceinline__ void load_u(const Start& a, int z, int64_t row, int c, float factor, float* u) {
    const int left = a.n - c;
    const void* g = a.list ? a.in.g[z] : (const void*)((const typename T::elem*)a.batch.x + z * a.batch.step);
    load_row<T>(g, row * (a.list ? a.in.stride[z] : a.batch.stride) + c, left, u);
    if (!a.list) return;
    const int64_t at = row * a.n + c;
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
// turn, `lanes` threads to a row.
constexpr int kStartThreads = 256;
template <typename T>
__global__ __launch_bounds__(kStartThreads) void momentum_kernel(Start a, int lanes) {
    __shared__ double sums[kStartThreads];
    const int z = blockIdx.y, per = kStartThreads / lanes, first = threadIdx.x / lanes, lane = threadIdx.x % lanes;
    const float factor = a.factor ? *a.factor : 1.0f;
    double s = 0.0;
    for (int64_t row = (int64_t)blockIdx.x * per + first; row < a.m; row += (int64_t)gridDim.x * per) {
        for (int c = lane * 8; c < a.n; c += lanes * 8) {
            float u[8];
            load_u<T, true>(a, z, row, c, factor, u);
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

// X in both orders from u: 64 x 64 of it to a workgroup.
template <typename T, bool PRECISE>
__global__ __launch_bounds__(kStartThreads) void start_kernel(Start a, Work w, int tall) {
    __shared__ double sums[kParts];
    __shared__ float turned[64][68];
    const int across = (a.n + 63) / 64, down = (a.m + 63) / 64, z = blockIdx.x / (across * down);
    const int index = blockIdx.x - z * across * down, i0 = index / across * 64, j0 = index % across * 64;
    sums[threadIdx.x] = (int)threadIdx.x < a.parts ? a.partials[(int64_t)z * kParts + threadIdx.x] : 0.0;
    __syncthreads();
    for (int k = kParts / 2; k; k >>= 1) {
        if ((int)threadIdx.x < k) sums[threadIdx.x] += sums[threadIdx.x + k];
        __syncthreads();
    }
    const double norm = sqrt(sums[0]), scale = (double)kX / (norm < a.eps ? a.eps : norm);       // NaN stays
    const float factor = a.factor ? *a.factor : 1.0f;
    uint8_t* const mine = w.base + z * w.size;
    // u's own order is t's where it is tall, o's where it is wide
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
        if (i0 + row < a.m && j0 + c < a.n) {
            load_u<T, false>(a, z, i0 + row, j0 + c, factor, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = j0 + c + j < a.n ? (float)((double)u[j] * scale) : 0.0f;
        }
        if (i0 + row < a.m) put(plain + ((int64_t)(i0 + row) * ld_plain + j0 + c) * 2, plane_plain, tall, u);
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
        if (j0 + row < a.n) put(other + ((int64_t)(j0 + row) * ld_other + i0 + c) * 2, plane_other, !tall, u);
    }
}

// ------------------------------------------------------------------------------------------------------ host
constexpr int64_t kMaxSide = 1 << 20;
constexpr int64_t kMaxCount = 1 << 15;                 // of a call: a grid's second axis
constexpr int64_t kMaxTiles = 1ll << 22;               // of a launch: its threads count in 32 bits
constexpr int kMaxSteps = 64;

int64_t blocks_of(int64_t n) { return (n + kHalves - 1) / kHalves * kHalves; }

// A matrix's part of the workspace; every array starts at a multiple of 1024 bytes.
Work work_of(int64_t m, int64_t n, bool precise) {
    Work w{};
    w.r = (int)(m < n ? m : n);
    w.c = (int)(m < n ? n : m);
    w.ldr = (int)blocks_of(w.r);
    w.ldc = (int)blocks_of(w.c);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t first = at;
        at += (bytes + 1023) / 1024 * 1024;
        return first;
    };
    auto pair = [&](int64_t bytes, bool both, int64_t* plane) {
        const int64_t first = take(bytes);
        *plane = at - first;
        if (both) take(bytes);
        return first;
    };
    for (int i = 0; i < 2; ++i) w.t[i] = pair((int64_t)w.c * w.ldr * 2, true, &w.t_plane);
    w.o = pair((int64_t)w.r * w.ldc * 2, precise, &w.o_plane);
    w.A = pair((int64_t)w.r * w.ldr * 2, precise, &w.s_plane);
    w.B = pair((int64_t)w.r * w.ldr * 2, precise, &w.s_plane);
    w.d = take((int64_t)w.ldr * 4);
    w.e = take((int64_t)w.ldr * 4);
    w.size = at;
    return w;
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

template <Mode MODE, bool PRECISE, typename Out, int COARSE, int B, int WT, int WO, int S>
int launch(const Work& w, int64_t first, int64_t tiles, const Coefficients& co, const Result& out, const Inputs& in,
           hipStream_t st) {
    if (tiles * COARSE * COARSE > kMaxTiles) return Z1_E_SIZE;
    const dim3 grid((unsigned)(tiles * COARSE * COARSE));
    step_kernel<MODE, PRECISE, Out, COARSE, B, B, WT, WO, S><<<grid, B / WT * (B / WO) * 64, 0, st>>>(w, co, out, in, (int)first);
    return (int)hipGetLastError();
}
constexpr int kCus = 256;
template <Mode MODE, bool PRECISE, typename Out = Listed>
int launch_step(const Work& w, int64_t count, const Coefficients& co, const Result& out, const Inputs& in, hipStream_t st) {
    auto tiles = [&](int64_t b) {
        const int64_t across = (w.r + b - 1) / b, down = (w.c + b - 1) / b;
        return count * (MODE == GRAM || MODE == SQUARE ? across * (across + 1) / 2 : down * across);
    };
    const int64_t large = tiles(256), rounds = large / kCus, rest = large % kCus;
    if (rounds > 0) {
        const int64_t whole = rest * 2 > kCus ? large : large - rest;
        if (const int rc = launch<MODE, PRECISE, Out, 1, 256, 64, 128, 2>(w, 0, whole, co, out, in, st)) return rc;
        if (whole == large) return Z1_OK;
        if (4 * rest <= kCus) return launch<MODE, PRECISE, Out, 2, 128, 64, 64, 4>(w, whole, rest, co, out, in, st);
        return launch<MODE, PRECISE, Out, 2, 128, 64, 64, 2>(w, whole, rest, co, out, in, st);
    }
    const int64_t middle = tiles(128);
    if (middle > kCus) return launch<MODE, PRECISE, Out, 1, 128, 64, 64, 2>(w, 0, middle, co, out, in, st);
    if (middle * 2 > kCus) return launch<MODE, PRECISE, Out, 1, 128, 64, 64, 4>(w, 0, middle, co, out, in, st);
    return launch<MODE, PRECISE, Out, 1, 64, 32, 32, 4>(w, 0, tiles(64), co, out, in, st);
}

template <typename T>
int start_of(const Start& a, const Work& w, int64_t count, bool precise, hipStream_t st) {
    int lanes = 1;
    while (lanes < kStartThreads && lanes * 8 < a.n) lanes *= 2;
    momentum_kernel<T><<<dim3((unsigned)a.parts, (unsigned)count), kStartThreads, 0, st>>>(a, lanes);
    const int64_t tiles = count * ((a.n + 63) / 64) * ((a.m + 63) / 64);
    if (tiles > kMaxTiles * 2) return Z1_E_SIZE;
    const int tall = a.m > a.n;
    if (precise) start_kernel<T, true><<<dim3((unsigned)tiles), kStartThreads, 0, st>>>(a, w, tall);
    else start_kernel<T, false><<<dim3((unsigned)tiles), kStartThreads, 0, st>>>(a, w, tall);
    return (int)hipGetLastError();
}

template <bool PRECISE, typename Out>
int iterate(Work w, int64_t count, int steps, const float* coefficients, const Result& out, const Inputs& in, hipStream_t st) {
    for (int k = 0; k < steps; ++k) {
        const Coefficients co{coefficients[3 * k], coefficients[3 * k + 1], coefficients[3 * k + 2]};
        w.cur = k & 1;
        if (const int rc = launch_step<GRAM, PRECISE>(w, count, co, out, in, st)) return rc;
        if (const int rc = launch_step<SQUARE, PRECISE>(w, count, co, out, in, st)) return rc;
        const int rc = k + 1 < steps ? launch_step<UPDATE, PRECISE>(w, count, co, out, in, st)
                                     : launch_step<LAST, PRECISE, Out>(w, count, co, out, in, st);
        if (rc) return rc;
    }
    return Z1_OK;
}

int64_t workspace_of(int64_t count, int64_t m, int64_t n, bool precise) {
    return (count * kParts * (int64_t)sizeof(double) + 1023) / 1024 * 1024 + count * work_of(m, n, precise).size;
}

int check(int64_t count, int64_t m, int64_t n, int dtype, int steps, const float* coefficients, float eps) {
    if (count < 0 || count > kMaxCount || m < 1 || n < 1 || m > kMaxSide || n > kMaxSide) return Z1_E_SIZE;
    if (dtype != Z1_F32 && dtype != Z1_BF16 && dtype != Z1_F16) return Z1_E_DTYPE;
    if (steps < 1 || steps > kMaxSteps) return Z1_E_SIZE;
    if (!coefficients) return Z1_E_NULL;
    if (!(eps > 0.0f) || !bounded(coefficients, steps)) return Z1_E_MODE;
    return Z1_OK;
}

template <typename Out>
int run(Start a, int64_t count, int dtype, int steps, const float* coefficients, bool precise, Result out, void* workspace,
        int64_t bytes, hipStream_t st) {
    if (count == 0) return Z1_OK;
    if (!workspace) return Z1_E_NULL;
    if (bytes < workspace_of(count, a.m, a.n, precise)) return Z1_E_WORKSPACE;
    Work w = work_of(a.m, a.n, precise);
    a.partials = (double*)workspace;
    w.base = (uint8_t*)workspace + (count * kParts * (int64_t)sizeof(double) + 1023) / 1024 * 1024;
    const int64_t rows = kStartThreads * 8 / (a.n < 8 ? 8 : a.n) + 1, need = (a.m + rows - 1) / rows;
    a.parts = (int)(need < kParts ? need : kParts);
    out.tall = a.m > a.n;
    int rc;
    switch (dtype) {
        case Z1_F32: rc = start_of<F32>(a, w, count, precise, st); break;
        case Z1_BF16: rc = start_of<BF16>(a, w, count, precise, st); break;
        default: rc = start_of<F16>(a, w, count, precise, st); break;
    }
    if (rc) return rc;
    return precise ? iterate<true, Out>(w, count, steps, coefficients, out, a.in, st)
                   : iterate<false, Out>(w, count, steps, coefficients, out, a.in, st);
}

}  // namespace

extern "C" {

int64_t z1_muon_workspace(int64_t count, int64_t m, int64_t n, int precise) {
    if (count < 0 || count > kMaxCount || m < 1 || n < 1 || m > kMaxSide || n > kMaxSide) return Z1_E_SIZE;
    return workspace_of(count, m, n, precise != 0);
}

int z1_orthogonalize(const void* x, int64_t step, int64_t stride, int64_t count, int64_t m, int64_t n, int dtype, void* out,
                     int out_dtype, int steps, const float* coefficients, float eps, int precise, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    if (const int rc = check(count, m, n, dtype, steps, coefficients, eps)) return rc;
    if (step < 0 || stride < 0) return Z1_E_SIZE;
    if (out_dtype != Z1_F32 && out_dtype != Z1_BF16 && out_dtype != Z1_F16) return Z1_E_DTYPE;
    if (count > 0 && (!x || !out)) return Z1_E_NULL;
    Start a{};
    a.batch = {x, step, stride};
    a.m = (int)m;
    a.n = (int)n;
    a.eps = eps;
    Result to{};
    to.out = out;
    const hipStream_t st = (hipStream_t)stream;
    switch (out_dtype) {
        case Z1_F32: return run<F32>(a, count, dtype, steps, coefficients, precise != 0, to, workspace, workspace_bytes, st);
        case Z1_BF16: return run<BF16>(a, count, dtype, steps, coefficients, precise != 0, to, workspace, workspace_bytes, st);
        default: return run<F16>(a, count, dtype, steps, coefficients, precise != 0, to, workspace, workspace_bytes, st);
    }
}

int z1_muon_step(const z1_matrix* list, int count, int64_t m, int64_t n, int dtype, const z1_muon* how, void* workspace,
                 int64_t workspace_bytes, void* stream) {
    if (!how) return Z1_E_NULL;
    if (const int rc = check(count, m, n, dtype, how->steps, how->coefficients, how->eps)) return rc;
    if (count > kList) return Z1_E_SIZE;
    if (count > 0 && !list) return Z1_E_NULL;
    Start a{};
    for (int i = 0; i < count; ++i) {
        if (!list[i].g || !list[i].momentum || !list[i].p) return Z1_E_NULL;
        if (list[i].g_stride < 0) return Z1_E_SIZE;
        a.in.g[i] = list[i].g;
        a.in.stride[i] = list[i].g_stride;
        a.in.buf[i] = list[i].momentum;
        a.in.p[i] = list[i].p;
        a.in.p16[i] = list[i].p16;
    }
    a.list = 1;
    a.m = (int)m;
    a.n = (int)n;
    a.factor = how->factor;
    a.mu = how->momentum;
    a.nesterov = how->nesterov;
    a.eps = how->eps;
    Result to{};
    to.lr = how->lr;
    to.keep = how->keep;
    return run<Listed>(a, count, dtype, how->steps, how->coefficients, how->precise != 0, to, workspace, workspace_bytes,
                       (hipStream_t)stream);
}

}  // extern "C"
