// A step's products over matrices of any size (the mathematics: z1_muon.h).  Included by one source for each PRECISE.
#pragma once

#include "z1_muon.h"

#include <type_traits>

namespace {

using namespace z1muon;

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
//
// Bound by the matrix instructions and the card's power: of 256 x 256 tiles a full round of 256 takes 98 us over 3072 columns in
// GRAM and LAST (1.05 PFLOP/s) and 119 in UPDATE, whose results are written in both orders and as pairs (192 with both halves of X
// as its operand); the quarters of 56 tiles 34.  On zeros, four 3072 x 3072 take 12 % less in all.  The largest library product of
// this card reaches 1.34 PFLOP/s, one of 3072^3 0.94.
//
// PART, JOINED: a long summed axis in parts, each a workgroup of its own, which leaves its sums as they are in its lanes (in the
// next t's place: free then), and a launch that adds them in order and goes on from there.
enum Phase { ALL, PART, JOINED };
template <Mode MODE, bool PRECISE, typename Out, int COARSE, int BT, int BO, int WT, int WO, int S, Phase PHASE>
__global__ __launch_bounds__(BT / WT * (BO / WO) * 64) void step_kernel(Plan plan, Coefficients co, void* out, Inputs in, int first,
                                                                            int parts) {
    constexpr bool kSymmetric = MODE == GRAM || MODE == SQUARE;
    constexpr int kWaves = BT / WT * (BO / WO);
    constexpr int kPT = BT / 8 / kWaves, kPO = BO / 8 / kWaves;                // direct loads of a wave: 8 rows each
    constexpr int NT = WT / 32, NO = WO / 32;
    static_assert(!kSymmetric || BT == BO, "a triangle of square tiles");
    static_assert(S == 2 || S == 4, "a block's buffer is kb & (S - 1)");
    // pairs: where LDS holds a block's both halves they are staged together and take three products, hi hi, hi lo and lo hi (A of
    // three of 777 x 401 12.0 -> 9.5 us, of 2048 x 2048 52 -> 43); larger tiles go through the axis three times
    constexpr bool kTogether = PRECISE && BT <= 128;
    constexpr int kPlanes = kTogether ? 2 : 1;
    constexpr int kRow = kHalves * 2, kSide = (BT + BO) * kRow;                // bytes of a block's first halves
    __shared__ __align__(1024) uint8_t lds[S][kPlanes * kSide];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // parts: one after another, so that an XCD's share is tiles of one part
    const int among = PHASE == PART ? gridDim.x / parts : 1, run_all = in_runs();
    const int axis = PHASE == PART ? run_all / among : 0, run = PHASE == PART ? run_all - axis * among : run_all;
    const int index = first + run / (COARSE * COARSE);
    const Group& g = group_of_tile(plan, index);
    const int planes = planes_of<PRECISE>(g);
    const bool pairs = planes == 2;
    const Layout w = layout_of(g.r, g.c, planes);
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
    // (a matrix without pairs has no second halves to read, but for t in UPDATE)
    const __amdgpu_buffer_rsrc_t lo_t = buffer_of(pt + plane_t, pairs || MODE == UPDATE ? bytes_t : 0);
    const __amdgpu_buffer_rsrc_t lo_o = buffer_of(po + plane_o, pairs ? bytes_o : 0);
    // times through the axis: pairs hi hi, hi lo and lo hi; single operands once, or X's second halves too
    const int times = kTogether ? 1 : pairs ? 3 : MODE == UPDATE && plan.both ? 2 : 1, all = times * blocks, last = all - 1;
    const int per = PHASE == PART ? (all + parts - 1) / parts : all, begin = axis * per;
    const int total = all - begin < per ? all - begin : per;                   // none where not positive: zeros are left
    const int sub = lane >> 3, piece = lane & 7;
    const int from = sub * pitch + ((piece ^ (sub >> 1)) << 4);                // in 8 rows whose keys' third bit is 0
    auto stage = [&](int kb, int i) {                  // the i-th direct load of this wave's part of a block
        const int plane = i / (kPT + kPO), ip = i % (kPT + kPO);
        uint8_t* buf = lds[kb & (S - 1)] + plane * kSide;
        const int l = ip < kPT ? wave * kPT + ip : wave * kPO + ip - kPT;
        int k = begin + kb < last ? begin + kb : last;
        bool t_lo = kTogether && plane, o_lo = t_lo;
        if (!kTogether) {
            const bool third = k >= 2 * blocks, second = k >= blocks && !third;
            t_lo = PRECISE ? third : second;
            o_lo = PRECISE ? second : third;
            k -= third ? 2 * blocks : second ? blocks : 0;
        }
        const int row = l * 8 * pitch;
        if (ip < kPT) load_lds(t_lo ? lo_t : hi_t, buf + l * 8 * kRow, row + (l & 1 ? from ^ 64 : from), k * kRow);
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
    constexpr int kEach = NT + NO, kReads = 2 * kEach * kPlanes, kLoads = kPlanes * (kPT + kPO);
    constexpr int kTimes = kTogether ? 3 : 1, kProducts = 2 * NT * NO * kTimes;
    i4 f[2][kEach * kPlanes][2];
    auto read = [&](int kb, int h, int q) {
        const int at = q >> 1, i = at % kEach, p = 4 * h + 2 * (q & 1) + half;
        const uint8_t* side = lds[kb & (S - 1)] + at / kEach * kSide;
        const uint8_t* row = i < NT ? side + (wt + i * 32 + r32) * kRow : side + (BT + wo + (i - NT) * 32 + rs) * kRow;
        f[h][at][q & 1] = *(const i4*)(row + ((p ^ (i < NT ? key_plain(r32) : key_spread(rs))) << 4));
    };
    // products of half h; beside them, the reads of half 1 - h of block kb_read and the loads of block kb_load (< 0: none)
    auto products = [&](int h, int kb_read, int kb_load) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int m = 0; m < NO * NT * kTimes; ++m) {
                const int i = m % (NO * NT) / NT, j = m % NT, time = m / (NO * NT), at = s * NO * NT * kTimes + m;
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    __builtin_bit_cast(h8, f[h][(time == 1 ? kEach : 0) + NT + i][s]),
                    __builtin_bit_cast(h8, f[h][(time == 2 ? kEach : 0) + j][s]), acc[i][j], 0, 0, 0);
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
    // a part's sums of a tile: the lanes' own, 16 bytes of neighbours beside each other
    auto left = [&](int part, int i, int j, int k) {
        const int64_t tile_of = ((int64_t)part * tiles + place) * kWaves + wave;
        return (Z1B_GLOBAL f4*)(mine + t_next) + ((tile_of * NO + i) * NT + j) * 256 + k * 64 + lane;
    };
    if constexpr (PHASE != JOINED) {
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
    }
    if constexpr (PHASE == PART) {
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *left(axis, i, j, k) = f4{acc[i][j][4 * k], acc[i][j][4 * k + 1], acc[i][j][4 * k + 2], acc[i][j][4 * k + 3]};
        return;
    }
    if constexpr (PHASE == JOINED) {
        for (int p = 0; p < parts; ++p) {
#pragma unroll
            for (int i = 0; i < NO; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const f4 v = *left(p, i, j, k);
#pragma unroll
                        for (int l = 0; l < 4; ++l) acc[i][j][4 * k + l] += v[l];
                    }
        }
    }

    // The results, 64 columns (o) of the wave's rows (t) at a time: to LDS, back as rows of eight columns to a lane, which take
    // what they need of A or X (whole lines, all under way before the first is used) and go out, and back once more as columns
    // for the other order.  (Taken in the instructions' layout, 16 columns of a lane's row, the same loads are 64 requests to an
    // instruction and one latency after the other: an UPDATE's start and end of a 256 x 256 tile took 40 us.)
    constexpr int kRoom = (int)sizeof(lds) / kWaves, kCols = WO < 64 ? WO : 64;
    static_assert(WT <= 64 && WT * 64 * 4 <= kRoom, "room for a wave's rows");
    constexpr int kRowLanes = kCols / 8, kRows = 64 / kRowLanes, kRowTurns = WT / kRows;
    constexpr int kColumnLanes = WT / 8, kColumns = 64 / kColumnLanes, kColumnTurns = kCols / kColumns;
    constexpr bool kPlane = MODE == UPDATE || MODE == LAST || (MODE == SQUARE && PRECISE);      // the operand's second halves
    auto put = [&](uint8_t* at, int64_t plane, const float* v) {
        if (pairs) put_halves<true>(at, plane, v);
        else put_halves<false>(at, plane, v);
    };
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
            // pairs among single operands are of few rows: loaded here, as registers for them would spill in every tile
            else if (MODE == SQUARE && pairs) F16::open(halves_of(buf_y, (wt + row) * pitch + o * 2), b);
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
                    put(mine + (MODE == GRAM ? w.A : w.B) + ((int64_t)t * w.ldr + o) * 2, w.s_plane, v);
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
                        put(mine + (MODE == GRAM ? w.A : w.B) + ((int64_t)oc * w.ldr + t) * 2, w.s_plane, v);
                } else if constexpr (MODE == UPDATE) {
                    if (oc < g.r && t < w.ldc) put(mine + w.o + ((int64_t)oc * w.ldc + t) * 2, w.o_plane, v);
                } else {
                    deliver(oc, t, v);
                }
            }
            own_done();
        }
    }
}

// ------------------------------------------------------------------------------------------------------ host
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

template <Mode MODE, bool PRECISE, typename Out, int COARSE, int B, int WT, int WO, int S, Phase PHASE = ALL>
int launch(Steps& a, int64_t first, int64_t last, int parts = 1) {
    const int64_t all = tiles_of<MODE>(a.plan, COARSE * B);
    const int64_t tiles = ((last < 0 ? all : last) - first) * COARSE * COARSE * (PHASE == PART ? parts : 1);
    if (all > kMaxTiles || tiles > kMaxTiles) return Z1_E_SIZE;
    step_kernel<MODE, PRECISE, Out, COARSE, B, B, WT, WO, S, PHASE>
        <<<dim3((unsigned)tiles), B / WT * (B / WO) * 64, 0, a.st>>>(a.plan, a.co, a.out, a.in, (int)first, parts);
    return (int)hipGetLastError();
}
// How a step's tiles run: all of one size, or whole rounds of 256 and what is left in quarters.
enum Kinds { ALL_256, WHOLE_256, ALL_128, ALL_64 };
struct Way {
    Kinds kind;
    int parts;                                         // of the summed axis
};

// The tiles of b x b, their mean number of blocks of the summed axis and the largest one.
struct Load {
    int64_t tiles;
    double blocks, most;
};
template <Mode MODE, bool PRECISE>
Load load_of(Plan& w, int64_t b) {
    Load l{tiles_of<MODE>(w, b), 0.0, 0.0};
    for (int k = 0; k < w.groups; ++k) {
        const Group& g = w.g[k];
        const double n = (double)((k + 1 < w.groups ? w.g[k + 1].tile0 : l.tiles) - g.tile0);
        const bool apart = !PRECISE || b == 256;       // a time after the other
        const double times = !apart ? 1.0 : has_pairs(g.r, g.c, PRECISE) ? 3.0 : MODE == UPDATE && w.both ? 2.0 : 1.0;
        const double blocks = times * (((MODE == GRAM ? g.c : g.r) + kHalves - 1) / kHalves);
        l.blocks += n * blocks;
        l.most = blocks > l.most ? blocks : l.most;
    }
    l.blocks /= (double)(l.tiles > 0 ? l.tiles : 1);
    return l;
}
// Estimates in us, as measured on launches of 10 to 9216 tiles over 16 to 128 blocks.  256: one to a CU, a start and an end of 15
// us and 1.0 us a block, which the card's power makes 1.8 when all CUs are at it (78 tiles over 48 and 128 blocks 67 and 149 us,
// 256 tiles over 48 105); X's update moves more (117).  128: 7 us and 0.42 alone on a CU (136 over 32 and 128 blocks 20 and 61),
// two to a CU 9 us and 1.1 (512 over 48 57 to 66).  64: 3.3 us and 0.19 alone (136 over 64 15), two to a CU 2 us and 0.56.
// Pairs: 256 has three times the blocks.  128: a CU holds one, 8 us and 0.82 (36 over 16 and 64 blocks 22 and 64), with all CUs
// at it 12 us and 1.27 (256 over 16 and 32 33 and 53; longer axes take more: 1200 over 48 to 128 895, where this says 604).  64:
// 4.7 us and 0.36 alone (136 over 16 and 64 11 and 28), two to a CU 4.1 us and 0.88 (1024 over 16 and 32 36 and 65).
template <bool PRECISE>
double time_256(double tiles, double blocks, bool update) {
    constexpr double kCool = PRECISE ? 0.45 : 0.3;     // of the CUs
    const double fill = tiles < kCus ? tiles / kCus : 1.0, hot = fill > kCool ? (fill - kCool) / (1.0 - kCool) : 0.0;
    return 15.0 + blocks * (1.0 + 0.8 * hot) + (update ? 12.0 * fill : 0.0);
}
constexpr int kMostParts = 16;
// Rounds of which the last is not full: it takes more than its part of one.
double rounds_of(double tiles, double round) {
    const double n = tiles / round;
    return n + 0.6 * (ceil(n) - n);
}
// Tiles of which a CU holds two: up to one to each, `alone`; beyond, those that share a CU take about half as long again at once.
template <bool PRECISE>
double shared(double tiles, double alone, double two) {
    if (tiles <= kCus) return alone;
    if (tiles > 2 * kCus) return (PRECISE ? rounds_of(tiles, 2 * kCus) : tiles / (2 * kCus) + 0.3) * two;
    return two > alone ? alone + (two - alone) * (0.45 + 0.55 * (tiles - kCus) / kCus) : alone;
}
template <bool PRECISE>
double time_128(double tiles, double blocks, double most, bool update) {
    if (!PRECISE) return shared<PRECISE>(tiles, 7.0 + 0.42 * most, 9.0 + 1.1 * blocks + (update ? 8.0 : 0.0));
    const double fill = tiles < kCus ? tiles / kCus : 1.0;
    const double one = 8.0 + (update ? 7.0 : 4.0) * fill + (0.82 + 0.45 * fill) * (tiles > kCus ? blocks : most);
    return tiles > kCus ? rounds_of(tiles, kCus) * one : one;
}
template <bool PRECISE>
double time_64(double tiles, double blocks, double most) {
    const double alone = PRECISE ? 4.7 + 0.36 * most : 3.3 + 0.19 * most;
    const double all = shared<PRECISE>(tiles, alone, PRECISE ? 4.1 + 0.88 * blocks : 2.0 + 0.56 * blocks);
    return all > alone ? all : alone;
}
// A last round of 256 tiles in quarters: triangles of pairs leave 256 to 128 tiles before it comes to that.
template <Mode MODE, bool PRECISE>
constexpr bool quarters = !PRECISE || MODE == UPDATE || MODE == LAST;
template <Mode MODE, bool PRECISE>
Way way_of(Plan& w) {
    const bool update = MODE == UPDATE || (PRECISE && MODE == LAST);
    const Load a = load_of<MODE, PRECISE>(w, 256), b = load_of<MODE, PRECISE>(w, 128), c = load_of<MODE, PRECISE>(w, 64);
    const int64_t rounds = a.tiles / kCus, rest = a.tiles % kCus;
    const double full = (double)rounds * time_256<PRECISE>(kCus, a.blocks, update);
    double best = full + (rest ? time_256<PRECISE>((double)rest, rounds ? a.blocks : a.most, update) : 0.0);
    Way way{ALL_256, 1};
    auto take = [&](Kinds kind, double time, int parts = 1) {
        if (time < best) best = time, way = {kind, parts};
    };
    const double axis = PRECISE ? a.blocks / 3.0 : a.blocks;
    if (rounds && rest && quarters<MODE, PRECISE>)
        take(WHOLE_256, full + time_128<PRECISE>(4.0 * (double)rest, axis, axis, update));
    take(ALL_128, time_128<PRECISE>((double)b.tiles, b.blocks, b.most, update));
    take(ALL_64, time_64<PRECISE>((double)c.tiles, c.blocks, c.most));
    if (MODE != GRAM) return way;
    // The long axis of A in parts, where few tiles leave CUs idle: 6.5 us for a second launch, less what the first does not do at
    // its end (pairs: 3), and its reads of what the parts leave at 80 bytes/ns a CU (400 x 8000: 23.3 us, 14.9 of 4 to 8 parts;
    // 200 x 4000: 13.8, 11.5; 1536 x 6144: 40.8, 31.4 of 3; 2048 x 8192: 61, 54 of 3; but 1024 x 4096 15.3, 17.5 of 3, and 300 x
    // 1000 6.5, 9.7.  Pairs: 400 x 8000 43.0, 19.0 of 4; 1024 x 4096 28.4, 25.3 of 3; but three of 777 x 401 9.5, 11.9 of 2).
    auto fits = [&](int64_t side) {                    // parts that the next t's place holds
        int64_t n = kMostParts;
        for (int k = 0; k < w.groups; ++k) {
            const Group& g = w.g[k];
            const int64_t d = (g.r + side - 1) / side, room = 2 * layout_of(g.r, g.c, 1).t_plane / (d * (d + 1) / 2 * side * side * 4);
            n = room < n ? room : n;
        }
        return n;
    };
    auto join = [](double parts, double side) { return (PRECISE ? 3.0 : 6.5) + (parts + 1.0) * side * side * 4.0 / 80000.0; };
    const int64_t most_b = fits(128), most_c = fits(64);
    for (int p = 2; p <= most_b && b.tiles * p <= 4 * kCus; ++p)
        take(ALL_128, time_128<PRECISE>((double)(b.tiles * p), b.blocks / p, b.most / p, false) + join(p, 128), p);
    for (int p = 2; p <= most_c && c.tiles * p <= 4 * kCus; ++p)
        take(ALL_64, time_64<PRECISE>((double)(c.tiles * p), c.blocks / p, c.most / p) + join(p, 64), p);
    return way;
}

// Tiles of 64 or 128: as many blocks staged as LDS holds where a CU has one tile, and as leave room for a second one where not.
template <Mode MODE, bool PRECISE, typename Out, Phase PHASE>
int launch_small(Steps& a, Kinds way, int parts) {
    if (way == ALL_64) {
        if constexpr (PRECISE)
            if (tiles_of<MODE>(a.plan, 64) * parts > kCus) return launch<MODE, PRECISE, Out, 1, 64, 32, 32, 2, PHASE>(a, 0, -1, parts);
        return launch<MODE, PRECISE, Out, 1, 64, 32, 32, 4, PHASE>(a, 0, -1, parts);
    }
    if constexpr (!PRECISE)
        if (tiles_of<MODE>(a.plan, 128) * parts <= kCus) return launch<MODE, PRECISE, Out, 1, 128, 64, 64, 4, PHASE>(a, 0, -1, parts);
    return launch<MODE, PRECISE, Out, 1, 128, 64, 64, 2, PHASE>(a, 0, -1, parts);
}
template <Mode MODE, bool PRECISE, typename Out = Listed>
int launch_step(Steps& a) {
    const auto [way, parts] = way_of<MODE, PRECISE>(a.plan);
    if constexpr (MODE == GRAM) {
        if (parts > 1) {
            if (const int rc = launch_small<MODE, PRECISE, Out, PART>(a, way, parts)) return rc;
            return way == ALL_64 ? launch<MODE, PRECISE, Out, 1, 64, 32, 32, PRECISE ? 2 : 4, JOINED>(a, 0, -1, parts)
                                 : launch<MODE, PRECISE, Out, 1, 128, 64, 64, 2, JOINED>(a, 0, -1, parts);
        }
    }
    if (way == ALL_256) return launch<MODE, PRECISE, Out, 1, 256, 64, 128, 2>(a, 0, -1);
    if constexpr (quarters<MODE, PRECISE>) {
        if (way == WHOLE_256) {
            const int64_t large = tiles_of<MODE>(a.plan, 256), rest = large % kCus;
            if (const int rc = launch<MODE, PRECISE, Out, 1, 256, 64, 128, 2>(a, 0, large - rest)) return rc;
            if constexpr (!PRECISE)
                if (4 * rest <= kCus) return launch<MODE, PRECISE, Out, 2, 128, 64, 64, 4>(a, large - rest, large);
            return launch<MODE, PRECISE, Out, 2, 128, 64, 64, 2>(a, large - rest, large);
        }
    }
    return launch_small<MODE, PRECISE, Out, ALL>(a, way, 1);
}

template <bool PRECISE, typename Out>
int iterate(Steps& a, int steps, const float* coefficients) {
    const uint64_t both = both_halves(coefficients, steps);
    for (int k = 0; k < steps; ++k) {
        a.co = {coefficients[3 * k], coefficients[3 * k + 1], coefficients[3 * k + 2]};
        a.plan.cur = k & 1;
        a.plan.both = both >> k & 1;
        if (const int rc = launch_step<GRAM, PRECISE>(a)) return rc;
        if (const int rc = launch_step<SQUARE, PRECISE>(a)) return rc;
        const int rc = k + 1 < steps ? launch_step<UPDATE, PRECISE>(a) : launch_step<LAST, PRECISE, Out>(a);
        if (rc) return rc;
    }
    return Z1_OK;
}

// How the three products run (z1_orthogonalize_way).
template <bool PRECISE, Mode MODE>
void way_into(Plan& w, int* way) {
    const auto [kind, parts] = way_of<MODE, PRECISE>(w);
    const int64_t rest = tiles_of<MODE>(w, 256) % kCus, middle = tiles_of<MODE>(w, 128) * parts, small = tiles_of<MODE>(w, 64) * parts;
    way[0] = kind == ALL_64 ? 64 : kind == ALL_128 ? 128 : 256;
    way[1] = kind == WHOLE_256 ? (int)rest : 0;
    way[2] = parts;
    if (kind == ALL_64) way[3] = PRECISE && small > kCus ? 2 : 4;
    else way[3] = !PRECISE && (kind == ALL_128 ? middle <= kCus : kind == WHOLE_256 && 4 * rest <= kCus) ? 4 : 2;
}
template <bool PRECISE>
void ways_of(Plan& w, int* way) {
    w.both = 1;
    way_into<PRECISE, GRAM>(w, way);
    way_into<PRECISE, SQUARE>(w, way + 4);
    way_into<PRECISE, UPDATE>(w, way + 8);
}

template <bool PRECISE>
int iterate_of(Steps& a, int steps, const float* coefficients, Kind kind) {
    switch (kind) {
        case OUT_F32: return iterate<PRECISE, F32>(a, steps, coefficients);
        case OUT_BF16: return iterate<PRECISE, BF16>(a, steps, coefficients);
        case OUT_F16: return iterate<PRECISE, F16>(a, steps, coefficients);
        default: return iterate<PRECISE, Listed>(a, steps, coefficients);
    }
}

}  // namespace
