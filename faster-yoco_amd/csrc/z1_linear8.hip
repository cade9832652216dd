// Products of 8-bit rows with 8-bit weights, and the weight's gradient from 8-bit rows (format: z1_block.h; declarations:
// include/yoco_z1.h).
//
//   product    y[t, o] = sum over blocks j of 2^(e[t, j] + f[o / 128, j]) * sum over k in j of a[t, k] w[o, k]
//   gradient   dw[o, k] = sum over t of dy[t, o] * a[t, k] 2^e[t, k / 128]
//
// Both open their 8-bit operands to bf16, which holds values and scales exactly, and multiply by the bf16 instructions, whose
// products and sums are fp32: a product on the way from LDS into the instructions, so that 8 bits are moved and staged; the
// gradient, whose sum runs over tokens, on the way into LDS.
#include "z1_block.h"

#pragma clang fp contract(off)

namespace {

using namespace z1blk;

typedef int i8 __attribute__((ext_vector_type(8)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

#define Z1B_LDS __attribute__((address_space(3)))

// The 32 x 32 result of a matrix instruction gives lane l column l % 32 and rows 8 (i/4) + 4 (l/32) + i%4, i = 0..15.
// Reading its first operand's rows in this order makes those 16 consecutive: 16 (l/32) + i.
__device__ __forceinline__ int spread(int row) { return 16 * ((row >> 2) & 1) + 4 * (row >> 3) + (row & 3); }

// Eight bytes of a row and its scale, opened to bf16 (exact: 4 significant bits, and bf16 has fp32's exponents; what is below
// its least value, 2^-133, rounds to a multiple of that, and 256 * 2^120, to which the largest fp32 values round, is infinite).
__device__ __forceinline__ u4 open_bf16(u2 q, float f) {
    u4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[0], f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[0], f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[1], f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[1], f, true));
    return r;
}

// Adds the products of NO by NT fragments of 32 rows, the s-th 16 of their 64 columns (8 bytes of a lane): both operands are
// opened to bf16 with their scales (exact) for the bf16 instructions, whose products and sums are fp32.  The 8-bit
// instructions have twice the rate but sum 8 products at a time on a common exponent and cut what lies more than 13 bits
// below the largest (probed: 256 + 2^-5 arrives, 256 + 2^-6 does not): up to 7 * 2^-13 of it is lost, a sum in fewer bits
// than 32.  after(m): what is issued beside the m-th product.
template <int NO, int NT, int NB, typename After>
__device__ __forceinline__ void multiply(f16 (&acc)[NO][NT], int s, const i8 (&fo)[NO], const i8 (&ft)[NT],
                                         const uint32_t (&so)[NB], const uint32_t (&st)[NT], After after) {
    auto open = [&](const i8& f, uint32_t scale) {
        return __builtin_bit_cast(b8, open_bf16(u2{(uint32_t)f[2 * s], (uint32_t)f[2 * s + 1]}, scale_value(scale & 0xffu)));
    };
    b8 bo[NO], bt[NT];
#pragma unroll
    for (int i = 0; i < NO; ++i) bo[i] = open(fo[i], so[NB == 1 ? 0 : i]);
#pragma unroll
    for (int j = 0; j < NT; ++j) bt[j] = open(ft[j], st[j]);
#pragma unroll
    for (int m = 0; m < NO * NT; ++m) {
        const int i = m / NT, j = m % NT;
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bo[i], bt[j], acc[i][j], 0, 0, 0);
        after(m);
    }
}

// A wave's 32 rows of C columns of a result, out of the matrix instructions' layout by way of its own ROOM bytes of LDS: a
// lane holds 16 columns of one row, whose pieces of 16 bytes would go out as requests of their own (64 to an instruction),
// while the rows read back go out as whole lines.  row0, col0: the first of them in out[rows][cols].
template <typename T, int C, int ROOM>
struct Flush {
    static constexpr int kElem = (int)sizeof(typename T::elem);
    static constexpr int pitch(int c) { return c * kElem + 16; }               // 16 neighbouring rows in different banks
    static constexpr int kC = C & (C - 1) ? 32 : 32 * pitch(C) <= ROOM ? C : 32 * pitch(C / 2) <= ROOM ? C / 2 : 32;
    static constexpr int kPitch = pitch(kC);
    static_assert(32 * kPitch <= ROOM, "room for a wave's rows");
    static __device__ __forceinline__ void run(uint8_t* own, int lane, const f16 (&acc)[C / 32], void* out, int64_t row0,
                                               int64_t rows, int col0, int cols) {
        const int r32 = lane & 31, half = lane >> 5;
        constexpr int kGroups = kC / kLane, kRows = 64 / kGroups;              // rows of one access
        const int c = lane % kGroups * kLane, r = lane / kGroups;
#pragma unroll
        for (int c0 = 0; c0 < C; c0 += kC) {
#pragma unroll
            for (int i = 0; i < kC / 32; ++i) {
                float x[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) x[k] = acc[c0 / 32 + i][k];
                uint8_t* to = own + r32 * kPitch;
                T::store_local(to, i * 32 + half * 16, x);
                T::store_local(to, i * 32 + half * 16 + 8, x + 8);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // a wave's own bytes: nobody to meet
            const int n = cols - col0 - c0 - c;
#pragma unroll
            for (int k = 0; k < 32 / kRows; ++k) {
                const int row = k * kRows + r;
                if (row0 + row >= rows || n <= 0) continue;
                const uint8_t* from = own + row * kPitch;
                const int64_t at = (row0 + row) * cols + col0 + c0 + c;
                if (n >= kLane) {
                    T::copy_local(out, at, from, c);
                } else {
#pragma unroll
                    for (int j = 0; j < kLane; ++j)
                        if (j < n) ((Z1B_GLOBAL typename T::elem*)out)[at + j] = ((const typename T::elem*)from)[c + j];
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // before the next rows overwrite them
        }
    }
};

// All waves of the workgroup are here, their reads from LDS are done, and of their loads all but the LATER last ones have
// arrived, direct loads into LDS among them.
template <int LATER = 0>
__device__ __forceinline__ void meet() {
    static_assert(LATER < 64, "the counter's range");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LATER) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A raw buffer of `bytes` (none where negative) from p: loads whose lane offset lies past it give zeros (word 3: the raw
// 32-bit data format).  The scalar offset of a load need not count in that check: it only moves within a row's own bytes.
// Without a branch: a loop around it keeps its loads on their way.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int64_t bytes) {
    const uint32_t low = (uint32_t)bytes, high = (uint32_t)(bytes >> 32);
    const uint32_t n = (low | (uint32_t)-(int)(high != 0)) & ~(uint32_t)((int)high >> 31);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)n, 0x00020000);
}
// 16 bytes a lane, straight into LDS at `to` + 16 * lane.
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t from, void* to, int lane_at, int at) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Z1B_LDS void*)to, 16, lane_at, at, 0, 0);
}

// A workgroup's tile, of gridDim.x in rows of `across`.  Workgroups go to the eight XCDs in turn.  In order, an XCD has every
// eighth tile; in panels, it has one run of them, which goes down `panel` rows of tiles, then to the next column, so that
// those it has at a time share both operands in its L2.
struct At {
    int down, across;
};
__device__ __forceinline__ At in_order(int across) { return {(int)blockIdx.x / across, (int)blockIdx.x % across}; }
__device__ __forceinline__ At in_panels(int across, int panel) {
    const int total = gridDim.x;
    if (total & 7) return in_order(across);
    const int i = (int)(blockIdx.x & 7) * (total >> 3) + (int)(blockIdx.x >> 3), first = i / (panel * across) * panel;
    const int rest = i - first * across, rows = total / across - first < panel ? total / across - first : panel;
    return {first + rest % rows, rest / rows};
}

struct Product {
    const uint8_t* a;                                  // [M, wide]
    const uint8_t* as;                                 // [M, pitch]
    const uint8_t* w;                                  // [N, wide]
    const uint8_t* ws;                                 // [ceil(N / 128), pitch]
    void* y;                                           // [M, N], or [parts, M, N] fp32
    int per;                                           // blocks of K to a part: all, or a multiple of four
    int64_t M;
    int N, blocks, pitch;                              // blocks of 128 along K
    int64_t wide;
};

// Staging keeps rows of 128 bytes (one block of K).  A lane of a direct load writes 16 bytes at its own place in a run of
// 1024, so the order of a row's eight 16-byte pieces is changed at the source: piece p of a row lies at p ^ key(row).  LDS
// has 64 banks of 4 bytes, two rows: the 16 rows that neighbouring lanes read together are eight of either parity, with
// eight different keys.
__device__ __forceinline__ int key_plain(int row) { return row >> 1 & 7; }
__device__ __forceinline__ int key_spread(int row) { return (row >> 1 & 3) | (row >> 4 & 1) << 2; }

// BT x BO outputs (tokens x outputs) of a workgroup, WT x WO of a wave, S blocks of K staged: two leave room for a second
// workgroup on a CU (of 128 x 128), four cover the loads' way where there is no second one.
//
// Large products are bound by the card's power: 8192 x 8192 x 8192 takes 739 us (1.49 PFLOP/s) with random operands and 582
// with zeros; what counts there is products to an opened value, hence eight waves of 64 x 128 (128 x 128 tiles: 869 to 892).
// Smaller ones are bound by the opening, which a wave does for itself (32 x 32 of a wave: 8 conversions to a product, 64 x 64:
// 4), and by CUs without a tile (below, where the tile is chosen).
template <typename T, int BT, int BO, int WT, int WO, int S>
__global__ __launch_bounds__(BT / WT * (BO / WO) * 64) void product_kernel(Product a) {
    constexpr int kWaves = BT / WT * (BO / WO);
    constexpr int kPT = BT / 8 / kWaves, kPO = BO / 8 / kWaves;                // direct loads of a wave: 8 rows each
    constexpr int NT = WT / 32, NO = WO / 32;
    static_assert(S == 2 || S == 4, "a block's buffer is kb & (S - 1)");
    __shared__ __align__(1024) uint8_t lds[S][(BT + BO) * kBlock];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_o = (a.N + BO - 1) / BO;
    // 16384 rows, in order against panels of 8 (panels of 4): 8192 -> 3072 566 us, 551 (556); 4096 -> 4096 384, 380 (381);
    // 2048 -> 5120 255, 251 (250); 1536 -> 6144 242, 239 (236); 3072 -> 8192 577, 578 (576).
    const At tile = in_panels(tiles_o, 8);
    const int64_t t0 = (int64_t)tile.down * BT;
    const int o0 = tile.across * BO;
    const int wt = wave / (BO / WO) * WT, wo = wave % (BO / WO) * WO;          // the wave's part of the tile

    const int kb0 = blockIdx.y * a.per;                // this part's blocks of K
    const int blocks = a.blocks - kb0 < a.per ? a.blocks - kb0 : a.per;
    a.a += (int64_t)kb0 * kBlock;
    a.w += (int64_t)kb0 * kBlock;
    a.as += kb0;
    a.ws += kb0;
    const int64_t before = (int64_t)kb0 * kBlock;
    // A row goes into a load's lane offset, which the buffer's range checks: rows past the end become zeros.  The block of K
    // goes into the scalar offset, which stays in the row: past the last block the last one is loaded again, not used.
    const __amdgpu_buffer_rsrc_t buf_t = buffer_of(a.a + t0 * a.wide, (a.M - t0) * a.wide - before);
    const __amdgpu_buffer_rsrc_t buf_o = buffer_of(a.w + o0 * a.wide, (a.N - o0) * a.wide - before);
    const int wide = (int)a.wide, last = blocks - 1;
    const int sub = lane >> 3, piece = lane & 7;
    const int from = sub * wide + ((piece ^ (sub >> 1)) << 4);                 // in 8 rows whose keys' third bit is 0
    auto stage = [&](int kb, int i) {                  // the i-th direct load of this wave's part of a block
        uint8_t* buf = lds[kb & (S - 1)];
        const int g = i < kPT ? wave * kPT + i : wave * kPO + i - kPT;
        const int at = (kb < last ? kb : last) * kBlock, row = g * 8 * wide;
        if (i < kPT) load_lds(buf_t, buf + g * 8 * kBlock, row + (g & 1 ? from ^ 64 : from), at);
        else load_lds(buf_o, buf + (BT + g * 8) * kBlock, row + (g & 2 ? from ^ 64 : from), at);
    };
    // scales: four blocks' bytes at a time, the next four loaded ahead
    const __amdgpu_buffer_rsrc_t buf_s = buffer_of(a.as + t0 * a.pitch, (a.M - t0) * a.pitch - kb0);
    const int r32 = lane & 31, half = lane >> 5, rs = spread(r32);
    // a wave of 64 or 128 outputs lies in one block of the weight, one of 96 in two
    constexpr int NB = WO == 96 ? NO : 1;
    __amdgpu_buffer_rsrc_t sw[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int ob = (o0 + wo + i * 32) / kBlock, end = (a.N - 1) / kBlock;
        sw[i] = buffer_of(a.ws + (int64_t)(ob < end ? ob : end) * a.pitch, a.pitch - kb0);
    }
    uint32_t now[NT] = {}, next[NT], now_w[NB] = {}, next_w[NB];
    auto scales = [&](int kb) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
            next[j] = __builtin_amdgcn_raw_buffer_load_b32(buf_s, (wt + j * 32 + r32) * a.pitch, kb, 0);
#pragma unroll
        for (int i = 0; i < NB; ++i) next_w[i] = __builtin_amdgcn_raw_buffer_load_b32(sw[i], 0, kb, 0);
    };
    scales(0);

    f16 acc[NO][NT];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f16{};

    // A block's two halves of 64 columns are read ahead by one half, and the workgroup meets between them: what follows
    // the meeting -- the next block's first reads, the direct loads into the buffer that has just been read -- runs beside
    // the second half's products, spread over them, and what it waits for was issued S - 1 blocks before.  Past the last
    // block the reads and loads are of no use, and in bounds.  (2048 rows of 8192 -> 3072: 88 us, with all reads and loads
    // before the products 92.)
    constexpr int kReads = 2 * (NT + NO), kLoads = kPT + kPO, kProducts = 4 * NT * NO;
    i4 f[2][NT + NO][2];
    auto read = [&](int kb, int h, int q) {
        const int i = q >> 1, p = 4 * h + 2 * half + (q & 1);
        const uint8_t* row = i < NT ? lds[kb & (S - 1)] + (wt + i * 32 + r32) * kBlock
                                    : lds[kb & (S - 1)] + (BT + wo + (i - NT) * 32 + rs) * kBlock;
        f[h][i][q & 1] = *(const i4*)(row + ((p ^ (i < NT ? key_plain(r32) : key_spread(rs))) << 4));
    };
    // products of half h; beside them, the reads of half 1 - h of block kb_read and the loads of block kb_load (< 0: none)
    auto products = [&](int h, int kb_read, int kb_load) {
        auto beside = [&](int m) {
#pragma unroll
            for (int q = 0; q < kReads; ++q)
                if (q * kProducts / kReads == m) read(kb_read, 1 - h, q);
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (kb_load >= 0 && i * kProducts / kLoads == m) stage(kb_load, i);
        };
        auto pair = [&](int i) { return __builtin_shufflevector(f[h][i][0], f[h][i][1], 0, 1, 2, 3, 4, 5, 6, 7); };
        i8 ft[NT], fo[NO];
#pragma unroll
        for (int j = 0; j < NT; ++j) ft[j] = pair(j);
#pragma unroll
        for (int i = 0; i < NO; ++i) fo[i] = pair(NT + i);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            multiply(acc, s, fo, ft, now_w, now, [&](int m) { beside(s * NO * NT + m); });
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
    for (int kb4 = 0; kb4 < blocks; kb4 += 4) {
#pragma unroll
        for (int j = 0; j < NT; ++j) now[j] = next[j];
#pragma unroll
        for (int i = 0; i < NB; ++i) now_w[i] = next_w[i];
        scales(kb4 + 4 < blocks ? kb4 + 4 : 0);
        const int end = kb4 + 4 < blocks ? kb4 + 4 : blocks;
#pragma unroll 1
        for (int kb = kb4; kb < end; ++kb) {
            products(0, kb, -1);
            meet<(S - 2) * kLoads>();                  // block kb has been read, block kb + 1 has arrived
            products(1, kb + 1, kb + S);
#pragma unroll
            for (int j = 0; j < NT; ++j) now[j] >>= 8;
#pragma unroll
            for (int i = 0; i < NB; ++i) now_w[i] >>= 8;
        }
    }
    meet();                                            // the staging buffers are free
    constexpr int kRoom = (int)sizeof(lds) / kWaves;
    void* y = (typename T::elem*)a.y + blockIdx.y * a.M * a.N;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        f16 part[NO];
#pragma unroll
        for (int i = 0; i < NO; ++i) part[i] = acc[i][j];
        Flush<T, WO, kRoom>::run(&lds[0][0] + wave * kRoom, lane, part, y, t0 + wt + j * 32, a.M, o0 + wo, a.N);
    }
}

// Few rows: the weight is read once by workgroups of OB outputs whose waves share K and whose sums meet in LDS; R * OB rows
// at most.  With OB 8 or 16 the instruction's 32 rows and columns are 32 / OB groups, each of the same outputs and rows with
// a block of K of its own: the results on its diagonal are that many partial sums, so that a narrow output has workgroups for
// all CUs.  A wave stages its own steps by direct loads, two under way: a lane's 16 bytes lie beside its neighbours', where
// fragments loaded into registers would be pieces of 32 rows to an instruction, and the address unit the bound (32 rows of
// 8192 -> 3072: 18 us, 9.8 this way).  Bound by the weight's bytes where they are many (one row of 3072 -> 100288: 56 us, 5.5
// TB/s), else by the launch and the loads' latency (3072 -> 8192: 6.6 us, 3.8 TB/s, from the last cache).  Three or four steps
// under way, or eight waves, leave room for fewer workgroups and lost.
constexpr int kFewWaves = 4;
template <typename T, int OB, int R>
__global__ __launch_bounds__(kFewWaves * 64) void product_few_kernel(Product a) {
    static_assert(R == 1 || OB == 32, "more row fragments than one are whole ones");
    constexpr int G = 32 / OB, U = 2, W = kFewWaves;   // blocks of K to an instruction; steps under way
    constexpr int kRows = 32 * kBlock;                 // bytes: 32 rows of the weight, R times 32 of a, and their scales
    constexpr int kScales = (1 + R) * kRows, kStep = kScales + (1 + R) * 256, kStepLoads = (1 + R) * 5;
    __shared__ __align__(1024) uint8_t lds[W][U][kStep];
    static_assert(U * kStep >= R * 32 * 33 * (int)sizeof(float), "a wave's sums take its staging's place");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o0 = blockIdx.x * OB, r32 = lane & 31, half = lane >> 5, g = r32 / OB;
    const int sub = lane >> 3, piece = lane & 7, last_row = (int)a.M - 1;
    const int64_t wide = a.wide;
    const uint8_t* from[1 + R][4];                     // a lane's 16 bytes of 8 rows, in the first block
    const uint8_t* scale[1 + R];
#pragma unroll
    for (int j = 0; j <= R; ++j) {                     // rows past the end repeat the last one and are not used
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 8 * i + sub, o = o0 + row % OB, t = (j - 1) * 32 + row % OB;
            const uint8_t* p = j == 0 ? a.w + (o < a.N ? o : a.N - 1) * wide : a.a + (t < last_row ? t : last_row) * wide;
            from[j][i] = p + ((piece ^ key_plain(row)) << 4);
        }
        const int t = (j - 1) * 32 + r32 % OB;
        scale[j] = j == 0 ? a.ws + (int64_t)(o0 / kBlock) * a.pitch : a.as + (t < last_row ? t : last_row) * a.pitch;
    }
    const int steps = (a.blocks + G - 1) / G, last = a.blocks - 1;
    auto stage = [&](int step, uint8_t* to) {          // past K's end: the last block, not used
        int kb = step * G + g;
        kb = (kb < last ? kb : last) & ~3;             // the dword that holds the lane's scale
#pragma unroll
        for (int j = 0; j <= R; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = step * G + i * 8 / OB;
                __builtin_amdgcn_global_load_lds((const Z1B_GLOBAL void*)(from[j][i] + (int64_t)(k < last ? k : last) * kBlock),
                                                 (Z1B_LDS void*)(to + j * kRows + i * 1024), 16, 0, 0);
            }
            __builtin_amdgcn_global_load_lds((const Z1B_GLOBAL void*)(scale[j] + kb),
                                             (Z1B_LDS void*)(to + kScales + j * 256), 4, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);             // a step's loads stay together: the waits count them
    };
    f16 acc[1][R] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) stage(wave + u * W, lds[wave][u]);
    for (int first = wave; first < steps; first += W * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int step = first + u * W, kb = step * G + g;         // the lane's block
            uint8_t* own = lds[wave][u];
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((U - 1) * kStepLoads) : "memory");
            i4 f[1 + R][4];
            uint32_t e[1 + R];
#pragma unroll
            for (int j = 0; j <= R; ++j) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    f[j][q] = *(const i4*)(own + j * kRows + r32 * kBlock +
                                           (((q >> 1) * 4 + half * 2 + (q & 1)) ^ key_plain(r32)) * 16);
                e[j] = ((const uint32_t*)(own + kScales + j * 256))[lane] >> (8 * (kb & 3));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // read, before it is overwritten
            __builtin_amdgcn_sched_barrier(0);
            stage(step + W * U, own);
            const uint32_t so[1] = {e[0]};
            uint32_t st[R];
#pragma unroll
            for (int j = 0; j < R; ++j) st[j] = e[1 + j];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                auto pair = [&](int j) {
                    const i8 v = __builtin_shufflevector(f[j][2 * h], f[j][2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                    return j == 0 || kb <= last ? v : i8{};                    // past K's end: times nothing
                };
                const i8 fw[1] = {pair(0)};
                i8 fx[R];
#pragma unroll
                for (int j = 0; j < R; ++j) fx[j] = pair(1 + j);
#pragma unroll
                for (int s = 0; s < 4; ++s) multiply(acc, s, fw, fx, so, st, [](int) {});
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing more arrives where the sums go
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            ((float*)lds[wave])[(j * 32 + r32) * 33 + 8 * (i >> 2) + 4 * half + (i & 3)] = acc[0][j][i];
    __syncthreads();
    for (int n = threadIdx.x; n < R * OB * OB; n += W * 64) {
        const int row = n / OB, c = n % OB;
        if (row > last_row || o0 + c >= a.N) continue;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < G; ++k)
#pragma unroll
            for (int i = 0; i < W; ++i) v += ((const float*)lds[i])[(k * OB + row) * 33 + k * OB + c];
        T::put(a.y, (int64_t)row * a.N + o0 + c, v);
    }
}

// ------------------------------------------------------------------------------------------------ weight gradient
struct Gradient {
    const uint16_t* dy;                                // bf16 [T, N], rows `stride` apart
    int64_t stride;
    const uint8_t* q;                                  // [T, wide]
    const uint8_t* s;                                  // [T, pitch]
    void* dw;                                          // [N, K], or [parts, N, K] fp32
    int64_t per;                                       // tokens to a part: all, or a multiple of the step
    int64_t T;
    int N, K, wide, pitch;
};

// The workgroup's part of the tokens.
__device__ __forceinline__ void take_part(Gradient& a) {
    const int64_t first = blockIdx.y * a.per;
    a.dy += first * a.stride;
    a.q += first * a.wide;
    a.s += first * a.pitch;
    a.T = a.T - first < a.per ? a.T - first : a.per;
}

// Four rows (tokens) of 16 columns by 16 lanes, transposed on the way out of LDS: each lane a column's four.
__device__ __forceinline__ s8 column_pair(const uint16_t* lo, const uint16_t* hi) {
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)lo);
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)hi);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Eight 16-bit values moved down by n (0..7) places.
__device__ __forceinline__ u4 shift_pieces(u4 v, int n) {
    v = n & 4 ? u4{v[2], v[3], 0, 0} : v;
    v = n & 2 ? u4{v[1], v[2], v[3], 0} : v;
    const u4 w = {v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    return n & 1 ? w : v;
}

// Where dy's rows do not start at whole dwords, as with an odd N, both operands are staged through registers (8191 x 3072 over
// 2048 tokens: 143 us, where 8192 x 3072 takes 95 by the direct loads below; 7 x 3072 over 16384 tokens 47, in parts).
// BN x BK of dw to a workgroup, WN x WK to a wave, TS tokens staged at a time, twice buffered.  While a step's products
// run, the next step's pieces go from registers into the other buffer, and the pieces of the step after that are loaded
// into those registers: a load has a whole step to arrive, and neither staging nor opening stands between two steps.  The
// loop has no branch (a branch around a load makes the waits for all of them complete): the first step has the rows that
// do not fill one, every other is full, and past the last one the same rows are loaded again and not used.
enum Edge { kCut, kFew };                              // N is at least 8, or less
template <typename T, Edge EDGE, int BN, int BK, int WN, int WK, int TS>
__global__ __launch_bounds__(BN / WN * (BK / WK) * 64) void weight_grad_kernel(Gradient a) {
    constexpr int kThreads = BN / WN * (BK / WK) * 64;
    constexpr int kPitchN = BN + 32, kPitchK = BK + 32;                        // elements: rows 64 bytes apart in the banks
    constexpr int kDy = TS * BN / 8 / kThreads, kX = TS * BK / 8 / kThreads;   // 8-element pieces of a thread
    constexpr int kDyRows = kThreads / (BN / 8), kXRows = kThreads / (BK / 8); // rows between a thread's pieces
    constexpr int NN = WN / 32, NK = WK / 32, KK = TS / 16;
    static_assert(kThreads % (BN / 8) == 0 && kThreads % (BK / 8) == 0, "a thread keeps its columns");
    __shared__ __align__(16) uint16_t lds[2 * TS * (kPitchN + kPitchK)];
    auto lds_n = [&](int buf) { return lds + buf * TS * kPitchN; };
    auto lds_k = [&](int buf) { return lds + (2 * kPitchN + buf * kPitchK) * TS; };
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_k = (a.K + BK - 1) / BK;
    const At tile = in_panels(tiles_k, 4);             // 7 x 3072 over 16384 tokens: 53 us in order, 47
    const int n0 = tile.down * BN, k0 = tile.across * BK;
    const int wn = wave / (BK / WK) * WN, wk = wave % (BK / WK) * WK;
    take_part(a);

    // Loads ask nothing: rows past the end repeat the last one (zeroed when kept), columns past it repeat columns whose
    // results are dropped.  A piece that the row's end cuts starts 8 columns before the end and is shifted when kept.
    const int last_n = a.N - 8, cut = a.N & 7;
    const int row_n = threadIdx.x / (BN / 8), row_k = threadIdx.x / (BK / 8);
    const int my_n = threadIdx.x % (BN / 8) * 8, my_k = threadIdx.x % (BK / 8) * 8;
    const int from_n = n0 + my_n < last_n ? n0 + my_n : last_n;
    const int from_k = k0 + my_k < a.wide ? k0 + my_k : a.wide - 8;
    const bool shifted = EDGE == kCut && n0 + my_n > last_n;
    u4 dy[kDy];
    u2 x[kX];
    uint32_t xs[kX];
    uint32_t at_n[kDy], at_k[kX], at_s[kX];            // offsets of the pieces from a step's first row
    auto place = [&](int rows) {                       // of a step with that many rows
#pragma unroll
        for (int i = 0; i < kDy; ++i) {
            const int t = row_n + i * kDyRows < rows ? row_n + i * kDyRows : rows - 1;
            at_n[i] = (uint32_t)t * (uint32_t)a.stride + (EDGE == kFew ? 0u : (uint32_t)from_n);
        }
#pragma unroll
        for (int i = 0; i < kX; ++i) {
            const int t = row_k + i * kXRows < rows ? row_k + i * kXRows : rows - 1;
            at_k[i] = (uint32_t)t * (uint32_t)a.wide + (uint32_t)from_k;
            at_s[i] = (uint32_t)t * (uint32_t)a.pitch + (uint32_t)from_k / kBlock;
        }
    };
    auto fetch = [&](int64_t t0, int part, int parts) {
        const uint16_t* dy0 = a.dy + t0 * a.stride;
        const uint8_t* q0 = a.q + t0 * a.wide;
        const uint8_t* s0 = a.s + t0 * a.pitch;
#pragma unroll
        for (int i = 0; i < kDy; ++i) {
            if (i * parts / kDy != part) continue;
            if (EDGE == kFew) {
                dy[i] = u4{};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < a.N) dy[i][j / 2] |= (uint32_t)((const Z1B_GLOBAL uint16_t*)dy0)[at_n[i] + j] << (16 * (j % 2));
            } else {
                dy[i] = *(const Z1B_GLOBAL u4_any2*)(dy0 + at_n[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kX; ++i) {
            if (i * parts / kX != part) continue;
            x[i] = *(const Z1B_GLOBAL u2*)(q0 + at_k[i]);
            xs[i] = s0[at_s[i]];
        }
    };
    auto keep = [&](int rows, int buf, int part, int parts) {
#pragma unroll
        for (int i = 0; i < kDy; ++i) {
            if (i * parts / kDy != part) continue;
            const int t = row_n + i * kDyRows;
            u4 v = dy[i];
            if (EDGE == kCut) v = shift_pieces(v, shifted ? 8 - cut : 0);
            if (rows < TS && t >= rows) v = u4{};
            *(u4*)(lds_n(buf) + t * kPitchN + my_n) = v;
        }
#pragma unroll
        for (int i = 0; i < kX; ++i) {
            if (i * parts / kX != part) continue;
            const int t = row_k + i * kXRows;
            u4 v = open_bf16(x[i], scale_value(xs[i]));
            if (rows < TS && t >= rows) v = u4{};
            *(u4*)(lds_k(buf) + t * kPitchK + my_k) = v;
        }
    };

    f16 acc[NK][NN];
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int j = 0; j < NN; ++j) acc[i][j] = f16{};

    // lane -> the row and the four columns whose address it gives to a transposing read
    const int group = lane >> 4, p = lane & 15;
    const int row = (group >> 1) * 8 + (p >> 2);
    const int col_n = (group & 1) * 16 + (p & 3) * 4;
    const int col_k = spread((group & 1) * 16 + (p & 3) * 4);                  // rows of the result in spread order
    const int64_t steps = (a.T + TS - 1) / TS;
    const int first = (int)(a.T - (steps - 1) * TS);   // rows of the first step
    if (steps > 0) {
        place(first);
        fetch(0, 0, 1);
        keep(first, 0, 0, 1);
        if (steps > 1) {
            place(TS);
            fetch(first, 0, 1);
        }
    }
    const int64_t end = steps > 1 ? a.T - TS : 0;      // first row of the last step
    int64_t next = end < first + TS ? end : first + TS;
    for (int64_t step = 0; step < steps; ++step) {
        const int buf = (int)(step & 1);
        __syncthreads();
        const uint16_t* bn = lds_n(buf) + row * kPitchN + wn + col_n;
        const uint16_t* bk = lds_k(buf) + row * kPitchK + wk + col_k;
        s8 fn[2][NN], fk[2][NK];
        auto read = [&](int kk) {
#pragma unroll
            for (int j = 0; j < NN; ++j)
                fn[kk & 1][j] = column_pair(bn + kk * 16 * kPitchN + j * 32, bn + (kk * 16 + 4) * kPitchN + j * 32);
#pragma unroll
            for (int i = 0; i < NK; ++i)
                fk[kk & 1][i] = column_pair(bk + kk * 16 * kPitchK + i * 32, bk + (kk * 16 + 4) * kPitchK + i * 32);
        };
        read(0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            if (kk + 1 < KK) read(kk + 1);
            keep(TS, buf ^ 1, kk, KK);
            fetch(next, kk, KK);
            __builtin_amdgcn_sched_barrier(0);         // the compiler would gather the loads at the step's end
#pragma unroll
            for (int i = 0; i < NK; ++i)
#pragma unroll
                for (int j = 0; j < NN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, fk[kk & 1][i]),
                                                                        __builtin_bit_cast(b8, fn[kk & 1][j]), acc[i][j],
                                                                        0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        next = next + TS < end ? next + TS : end;
    }
    __syncthreads();                                   // the staging buffers are free
    constexpr int kRoom = (int)sizeof(lds) / (kThreads / 64) & ~15;
    void* dw = (typename T::elem*)a.dw + (int64_t)blockIdx.y * a.N * a.K;
#pragma unroll
    for (int j = 0; j < NN; ++j) {
        f16 part[NK];
#pragma unroll
        for (int i = 0; i < NK; ++i) part[i] = acc[i][j];
        Flush<T, WK, kRoom>::run((uint8_t*)lds + wave * kRoom, lane, part, dw, n0 + wn + j * 32, a.N, k0 + wk, a.K);
    }
}

// A token's 64-byte run in LDS rows of R runs: rows of whole 256 bytes start in the same banks, ones of 384 bytes in two
// places in turn.
template <int R>
__device__ __forceinline__ int placed(int run, int token) {
    static_assert(R % 2 == 0, "rows of 128 bytes or more");
    return run ^ (R % 4 == 0 ? token & 3 : token >> 1 & 1);
}

// The same where dy's rows start at whole dwords: dy goes straight into LDS, and both operands are staged the way the
// product's are.  8192 x 8192 over 8192 tokens: 880 us, 1.25 PFLOP/s (715 with zeros: power again; without opening a's values
// 746), 8192 x 3072 over 2048: 95 us, over 16384: 736.  a's values opened once more beside the products instead of on the way
// into LDS: 1058 us; four waves of 128 x 128 924, 128 x 128 tiles 1117.  Rows of both lie whole in LDS; a transposing read
// takes 64 bytes of four tokens at a time, so a row's 64-byte runs are placed (`placed`) so that the four lie in different
// banks.  What lies past the last token or past a tensor's end is zero (the buffers' ranges).
//
// A step of TS tokens is TS / 16 parts.  Each part's operands are read a part ahead, and the workgroup meets before the
// last part: all of the step has been read by then.  From one meeting to the next (`between`) everything is read from one
// buffer, the next step's, while the direct loads of dy and the opened rows of a two steps on (loaded into registers a
// step before) go into the other.  It is one function of four restricted pointers because the compiler else takes every
// transposing read for one of the bytes on their way and waits for them.
template <typename T, int BN, int BK, int WN, int WK, int TS>
__global__ __launch_bounds__(BN / WN * (BK / WK) * 64) void weight_grad_direct_kernel(Gradient a) {
    constexpr int kThreads = BN / WN * (BK / WK) * 64, kWaves = kThreads / 64;
    constexpr int NN = WN / 32, NK = WK / 32, KK = TS / 16;
    constexpr int kRowN = BN * 2, kRowK = BK * 2;                              // bytes of a row in LDS
    constexpr int kLoadRows = 1024 / kRowN;                                    // rows of a wave's direct load
    constexpr int kLoads = TS / kLoadRows / kWaves;
    constexpr int P = BK == 192 ? 8 : 16;              // columns of a thread's piece of a's rows
    constexpr int kX = TS * BK / P / kThreads;
    static_assert(kX * kThreads * P == TS * BK, "every thread has as many");
    static_assert(kLoadRows == 2 || kLoadRows == 4 || kLoadRows == 8, "rows of 128, 256 or 512 bytes");
    __shared__ __align__(1024) uint8_t lds[2 * TS * (kRowN + kRowK)];
    auto lds_n = [&](int64_t step) { return lds + (step & 1) * TS * kRowN; };
    auto lds_k = [&](int64_t step) { return lds + (2 * kRowN + (step & 1) * kRowK) * TS; };
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_k = (a.K + BK - 1) / BK;
    // in order against panels of 4 (of 8), 2048 tokens: 8192 x 3072 99 us, 96 (97); 4096 x 4096 63, 63 (63); 6144 x 1536 47, 44
    // (44); 16384 tokens: 4096 x 4096 454, 441 (445); 6144 x 1536 345, 332 (334); 5120 x 2048 360, 360 (360)
    const At tile = in_panels(tiles_k, 4);
    const int n0 = tile.down * BN, k0 = tile.across * BK;
    const int wn = wave / (BK / WK) * WN, wk = wave % (BK / WK) * WK;
    take_part(a);
    const int64_t steps = (a.T + TS - 1) / TS;

    // direct loads: a lane's row and piece of 16 bytes within a load's rows
    const int sub = lane / (64 / kLoadRows), piece = lane % (64 / kLoadRows);
    const int row_bytes = (int)a.stride * 2;
    int from[kLoadRows == 2 ? 2 : 1];                  // by the parity of the load: two rows are half of four
#pragma unroll
    for (int i = 0; i < (int)(sizeof(from) / sizeof(int)); ++i)
        from[i] = sub * row_bytes + (placed<BN / 32>(piece >> 2, i * kLoadRows + sub) << 2 | (piece & 3)) * 16;
    // from the tile's first column to dy's end, in whole dwords (an odd N's last one holds nothing that is used); a load's
    // token goes into its lane offset, which this range checks
    const int64_t bytes_n = a.T > 0 ? (a.T - 1) * row_bytes + ((a.N - n0 + 1) & ~1) * 2 : 0;
    auto stage = [&](int64_t step, int i, uint8_t* to) {
        const int64_t t0 = step * TS;
        const int g = wave * kLoads + i;
        const __amdgpu_buffer_rsrc_t rows = buffer_of(a.dy + t0 * a.stride + n0, bytes_n - t0 * row_bytes);
        load_lds(rows, to + g * 1024, from[kLoadRows == 2 ? g & 1 : 0] + g * kLoadRows * row_bytes, 0);
    };
    uint32_t x[kX][P / 4], xs[kX];
    int at_q[kX], at_s[kX], at_k[kX];                  // of the pieces: offsets in a step's rows, and in LDS
#pragma unroll
    for (int i = 0; i < kX; ++i) {
        const int e = i * kThreads + threadIdx.x, t = e / (BK / P), c = e % (BK / P) * P;
        at_q[i] = t * a.wide + k0 + c;
        at_s[i] = t * a.pitch + (k0 + c) / kBlock;
        at_k[i] = t * kRowK + (placed<BK / 32>(c >> 5, t) << 6) + (c & 31) * 2;
    }
    auto fetch = [&](int64_t step, int i) {
        const int64_t t0 = step * TS, left = a.T - t0;
        const __amdgpu_buffer_rsrc_t rows = buffer_of(a.q + t0 * a.wide, left * a.wide);
        if constexpr (P == 16) {
            const u4 v = __builtin_amdgcn_raw_buffer_load_b128(rows, at_q[i], 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i][j] = v[j];
        } else {
            const u2 v = __builtin_amdgcn_raw_buffer_load_b64(rows, at_q[i], 0, 0);
#pragma unroll
            for (int j = 0; j < 2; ++j) x[i][j] = v[j];
        }
        xs[i] = __builtin_amdgcn_raw_buffer_load_b8(buffer_of(a.s + t0 * a.pitch, left * a.pitch), at_s[i], 0, 0);
    };
    auto keep = [&](int i, uint8_t* rows) {
        const float f = scale_value(xs[i]);
        u4* to = (u4*)(rows + at_k[i]);
        if constexpr (P == 16) {
            // half of the lanes write their second half first: neighbours' pieces, 32 bytes apart, then differ in banks
            const bool flip = (threadIdx.x >> 2 ^ threadIdx.x >> 3) & 1;
            to[flip ? 1 : 0] = open_bf16(flip ? u2{x[i][2], x[i][3]} : u2{x[i][0], x[i][1]}, f);
            to[flip ? 0 : 1] = open_bf16(flip ? u2{x[i][0], x[i][1]} : u2{x[i][2], x[i][3]}, f);
        } else {
            to[0] = open_bf16(u2{x[i][0], x[i][1]}, f);
        }
    };

    // lane -> the token and the four columns whose address it gives to a transposing read
    const int group = lane >> 4, p = lane & 15;
    const int token = (group >> 1) * 8 + (p >> 2);
    const int col_n = (group & 1) * 16 + (p & 3) * 4;
    const int col_k = spread((group & 1) * 16 + (p & 3) * 4);                  // rows of the result in spread order
    s4 f[2][NK + NN][2] = {};                          // in the order in which the products want them
    constexpr int kReads = 2 * (NN + NK), kProducts = NN * NK;
    f16 acc[NN][NK];
#pragma unroll
    for (int i = 0; i < NN; ++i)
#pragma unroll
        for (int j = 0; j < NK; ++j) acc[i][j] = f16{};
    auto product = [&](int h, int m) {
        const int i = m / NK, j = m % NK;
        auto pair = [&](int k) {
            return __builtin_bit_cast(b8, __builtin_shufflevector(f[h][k][0], f[h][k][1], 0, 1, 2, 3, 4, 5, 6, 7));
        };
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pair(j), pair(NK + i), acc[i][j], 0, 0, 0);
    };
    // the last part of step - 1, and all parts but the last of `step`, which lies in from_n and from_k
    auto between = [&](int64_t step, const uint8_t* __restrict__ from_n, const uint8_t* __restrict__ from_k,
                       uint8_t* __restrict__ to_n, uint8_t* __restrict__ to_k) {
#pragma unroll
        for (int kk = -1; kk < KK - 1; ++kk) {
#pragma unroll
            for (int m = 0; m < kProducts; ++m) {
                product((kk + KK) & 1, m);
#pragma unroll
                for (int q = 0; q < kReads; ++q) {
                    if (q * kProducts / kReads != m) continue;
                    const int i = q >> 1, t = token + (kk + 1) * 16 + (q & 1) * 4;
                    const int run = i < NK ? wk / 32 + i : wn / 32 + i - NK;
                    const uint8_t* at = i < NK ? from_k + t * kRowK + (placed<BK / 32>(run, p >> 2) << 6) + col_k * 2
                                               : from_n + t * kRowN + (placed<BN / 32>(run, p >> 2) << 6) + col_n * 2;
                    f[(kk + 1) & 1][i][q & 1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)at);
                }
                if (kk < 0) {
#pragma unroll
                    for (int l = 0; l < kLoads; ++l)
                        if (l * kProducts / kLoads == m) stage(step + 1, l, to_n);
                }
                if (kk == 0) {
#pragma unroll
                    for (int l = 0; l < kX; ++l)
                        if (l * kProducts / kX == m) {
                            keep(l, to_k);
                            fetch(step + 2, l);
                        }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    static_assert(KK % 2 == 0, "the parts' registers alternate");

#pragma unroll
    for (int i = 0; i < kLoads; ++i) stage(0, i, lds_n(0));
#pragma unroll
    for (int i = 0; i < kX; ++i) fetch(0, i);
#pragma unroll
    for (int i = 0; i < kX; ++i) keep(i, lds_k(0));
#pragma unroll
    for (int i = 0; i < kX; ++i) fetch(1, i);
    for (int64_t step = 0; step < steps; ++step) {
        meet();                                        // step - 1 has been read, `step` has arrived
        between(step, lds_n(step), lds_k(step), lds_n(step + 1), lds_k(step + 1));
    }
#pragma unroll
    for (int m = 0; m < kProducts; ++m) product(1, m);
    meet();                                            // the staging buffers are free
    constexpr int kRoom = (int)sizeof(lds) / kWaves & ~15;
    void* dw = (typename T::elem*)a.dw + (int64_t)blockIdx.y * a.N * a.K;
#pragma unroll
    for (int i = 0; i < NN; ++i)
        Flush<T, WK, kRoom>::run(lds + wave * kRoom, lane, acc[i], dw, n0 + wn + i * 32, a.N, k0 + wk, a.K);
}

constexpr int64_t kMaxRows = 1ll << 40;
constexpr int64_t kMaxDim = 1 << 24;                   // outputs, and elements between rows of dy
constexpr int64_t kMaxInner = 1 << 22;                 // columns: 256 rows of them lie within 31 bits
constexpr int kMaxParts = 64;
constexpr int64_t kMaxTiles = 1ll << 22;               // of a launch: its threads count in 32 bits

bool bad_dtype(int d) { return d != Z1_F32 && d != Z1_BF16 && d != Z1_F16; }

constexpr int kCus = 256;

// The sum of `parts` partial results, in order: bound by their way through the last cache (four of 128 x 3072: 2.5 us and
// their bytes at 5 TB/s).
constexpr int kJoinThreads = 256;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const float* part, int parts, int64_t count, void* out) {
    const int64_t i = ((int64_t)blockIdx.x * kJoinThreads + threadIdx.x) * kLane;
    if (i >= count) return;
    const int n = count - i < kLane ? (int)(count - i) : kLane;
    float s[kLane] = {};
#pragma unroll 8
    for (int p = 0; p < parts; ++p) {
        float v[kLane];
        load_row<F32>(part, p * count + i, n, v);
#pragma unroll
        for (int j = 0; j < kLane; ++j) s[j] += v[j];
    }
    store_row<T>(out, i, n, s);
}
template <typename T>
int join(const float* part, int parts, int64_t count, void* out, hipStream_t st) {
    const int64_t per = kJoinThreads * kLane;
    join_kernel<T><<<dim3((unsigned)((count + per - 1) / per)), kJoinThreads, 0, st>>>(part, parts, count, out);
    return (int)hipGetLastError();
}

// The number of parts into which the long axis of a product in small tiles is cut, `steps` of it in multiples of `unit`:
// the one with the least estimate of the time, which *ns is.  A step takes `alone` where a CU has one tile, `shared` where
// it has two (0: it has no room for two); joining takes 3.3 us and 0.05 a part, and the partial results' way out and back, at
// `rate` bytes/ns.
constexpr int kProductRate = 16000, kGradientRate = 5000;          // as the shapes that these rules decide measured
int parts_of(int64_t tiles, int64_t steps, int unit, int64_t results, int rate, int alone, int shared, int64_t* ns) {
    int best = 1;
    *ns = 0;
    for (int p = 1; p <= kMaxParts; ++p) {
        const int64_t per = (steps + p * unit - 1) / (p * unit) * unit;
        if (p > 1 && (per * (p - 1) >= steps || tiles * p > (shared ? 2 * kCus : kCus))) continue;     // no steps; no room
        const int64_t time = per * (tiles * p <= kCus ? alone : shared) + (p > 1 ? 3300 + p * (50 + results * 8 / rate) : 0);
        if (p == 1 || time < *ns) best = p, *ns = time;
    }
    return best;
}

// How a product runs.
//
// Many tiles: large ones (256 x 256) open fewer values per product, smaller ones leave fewer CUs without work.  A round of
// large ones, one to a CU, takes 100; of 128 x 128, two to a CU, 59; of 128 x 192, one to a CU, 51 (us: 3072 -> 8192 with 2048
// rows 76 in 256 x 256, 86 in 128 x 128, 98 in 128 x 192; 8192 -> 3072 142, 94, 87, and with 4096 rows 157, 169, 179; 1536 ->
// 6144 with 2048 rows 36, 36, 41).
//
// Up to one of 128 x 128 to a CU: smaller tiles on more CUs win while there are CUs (kSmall: a start and a block of K, in ns,
// as measured), and where even they leave CUs idle, a long K is cut into parts, joined by a second launch.  1000 -> 1501, 333
// rows: 6.4 us in 64 x 64, 11.6 in 128 x 128; 4100 -> 3000, 600 rows: 24.1 in 64 x 128, 27.0 without it; 4096 -> 4096, 1024
// rows: 34.9 in 128 x 128, 45.3 in 64 x 64; 8192 -> 3072, 512 rows: 34.6 in 128 x 128 of four parts, 39.6 in 64 x 64; 128 rows:
// 31.3 in 64 x 64, 17.9 of four parts.
//
// Up to 64 rows the few rows' kernel runs where it is faster, a workgroup to a CU, at 3.3 us and 0.12 to 0.25 us a block of K,
// more with more of them and more rows (33 rows, 3072 -> 3072: 6.9 us against 13.4, 3072 -> 8192: 8.3 against 13.5; 64 rows,
// 8192 -> 3072: 14.4 against 14.3 in 64 x 64 of eight parts).
struct Way {
    int rows, outputs;                                 // of a tile
    int stages;                                        // blocks of K staged; 0: the few rows' kernel
    int parts, per;                                    // of K's blocks
};
struct Small {
    int rows, outputs, start, alone, shared;
};
constexpr Small kSmall[] = {{128, 128, 5400, 940, 1590}, {64, 128, 4000, 600, 0}, {64, 64, 3100, 450, 630}};
// The best of them for M x N results (M x N 128 x 128 tiles at most one to a CU, or the first is taken).
struct Cut {
    const Small* tile;
    int parts;
    int64_t ns;
};
template <int COUNT>
Cut best_of(const Small (&small)[COUNT], int64_t M, int64_t N, int64_t steps, int unit, int rate) {
    Cut best{nullptr, 1, 0};
    for (const Small& t : small) {
        const int64_t n = (M + t.rows - 1) / t.rows * ((N + t.outputs - 1) / t.outputs);
        if (best.tile && n > (t.shared ? 2 * kCus : kCus)) continue;
        int64_t ns;
        const int parts = parts_of(n, steps, unit, M * N, rate, t.alone, t.shared, &ns);
        if (!best.tile || t.start + ns < best.ns) best = {&t, parts, t.start + ns};
    }
    return best;
}
Way few_way(int64_t M, int64_t N, int blocks) {
    if (M > 32) return {64, 32, 0, 1, blocks};
    // the fewest outputs that hold the rows, or more while there are 192 workgroups: one row of 3072 -> 8192 takes 9.8 us with
    // 8 outputs, 8.1 with 16, 6.6 with 32; 8192 -> 3072 8.2, 7.3, 9.2; 4096 -> 4096 6.1, 6.1, 6.2; 5120 -> 1280 4.1, 4.9, 6.0
    int outputs = M <= 8 ? 8 : M <= 16 ? 16 : 32;
    while (outputs < 32 && N >= 2 * outputs * 192) outputs *= 2;
    return {outputs, outputs, 0, 1, blocks};
}
Way product_way(int64_t M, int64_t N, int blocks) {
    if (M <= 32) return few_way(M, N, blocks);
    auto tiles = [&](int rows, int outputs) { return (M + rows - 1) / rows * ((N + outputs - 1) / outputs); };
    auto rounds = [&](int rows, int outputs, int at_once) { return (tiles(rows, outputs) + at_once - 1) / at_once; };
    if (tiles(128, 128) > kCus) {
        const int64_t large_time = 100 * rounds(256, 256, kCus), middle_time = 51 * rounds(128, 192, kCus);
        if (59 * rounds(128, 128, 2 * kCus) <= (large_time < middle_time ? large_time : middle_time))
            return {128, 128, 2, 1, blocks};
        if (large_time <= middle_time) return {256, 256, 2, 1, blocks};
        return {128, 192, 4, 1, blocks};
    }
    const Cut cut = best_of(kSmall, M, N, blocks, 4, kProductRate);
    const int64_t groups = (N + 31) / 32;              // workgroups of few rows; with less than 64, the parts read K sooner
    const int64_t few_rounds = (groups + kCus - 1) / kCus, at_once = groups < kCus ? groups : kCus;
    if (M <= 64 && groups >= 64 && 3300 + few_rounds * blocks * (120 + at_once * M / 128) <= cut.ns)
        return few_way(M, N, blocks);
    const int stages = cut.tile->rows == 128 && tiles(128, 128) * cut.parts > kCus ? 2 : 4;
    return {cut.tile->rows, cut.tile->outputs, stages, cut.parts,
            cut.parts == 1 ? blocks : (blocks + 4 * cut.parts - 1) / (4 * cut.parts) * 4};
}

template <typename T, int BT, int BO, int WT, int WO, int S>
int launch_tiles(const Product& a, int parts, hipStream_t st) {
    const int64_t tiles = (a.M + BT - 1) / BT * ((a.N + BO - 1) / BO);
    if (tiles > kMaxTiles) return Z1_E_SIZE;
    product_kernel<T, BT, BO, WT, WO, S><<<dim3((unsigned)tiles, parts), BT / WT * (BO / WO) * 64, 0, st>>>(a);
    return (int)hipGetLastError();
}

template <typename T, int OB, int R>
int launch_few(const Product& a, hipStream_t st) {
    product_few_kernel<T, OB, R><<<dim3((unsigned)((a.N + OB - 1) / OB)), kFewWaves * 64, 0, st>>>(a);
    return (int)hipGetLastError();
}

template <typename T>
int launch_small(const Product& a, const Way& way, hipStream_t st) {
    if (way.outputs == 64) return launch_tiles<T, 64, 64, 32, 32, 4>(a, way.parts, st);
    if (way.rows == 64) return launch_tiles<T, 64, 128, 32, 64, 4>(a, way.parts, st);
    if (way.stages == 4) return launch_tiles<T, 128, 128, 64, 64, 4>(a, way.parts, st);
    return launch_tiles<T, 128, 128, 64, 64, 2>(a, way.parts, st);
}

template <typename T>
int launch_product(Product a, const Way& way, float* workspace, hipStream_t st) {
    if (way.stages == 0) {
        if (way.rows == 64) return launch_few<T, 32, 2>(a, st);
        if (way.outputs == 8) return launch_few<T, 8, 1>(a, st);
        if (way.outputs == 16) return launch_few<T, 16, 1>(a, st);
        return launch_few<T, 32, 1>(a, st);
    }
    a.per = way.per;
    if (way.outputs == 256) return launch_tiles<T, 256, 256, 64, 128, 2>(a, 1, st);
    if (way.outputs == 192) return launch_tiles<T, 128, 192, 64, 96, 4>(a, 1, st);
    if (way.parts == 1) return launch_small<T>(a, way, st);
    void* y = a.y;
    a.y = workspace;
    if (const int rc = launch_small<F32>(a, way, st)) return rc;
    return join<T>(workspace, way.parts, a.M * a.N, y, st);
}

template <typename T, Edge EDGE, int BN, int BK, int WN, int WK, int TS>
int launch_gradient(const Gradient& a, int parts, hipStream_t st) {
    const int64_t tiles = (int64_t)((a.N + BN - 1) / BN) * ((a.K + BK - 1) / BK);
    if (tiles > kMaxTiles) return Z1_E_SIZE;
    weight_grad_kernel<T, EDGE, BN, BK, WN, WK, TS><<<dim3((unsigned)tiles, parts), BN / WN * (BK / WK) * 64, 0, st>>>(a);
    return (int)hipGetLastError();
}
// How a weight gradient runs: by direct loads where dy's rows are whole dwords, in large tiles of 256 x 256 or 256 x 192 (a
// round of which takes 0.87 of the time: 3072 columns in 12 or 16 tiles, 2048 tokens: 112 or 98 us), or in small ones (their
// start and 64 tokens in ns, as for the products) with the tokens cut into parts where those leave CUs idle (512 x 512 over
// 16384 tokens: 106 us in 128 x 128, 17 of 16 parts; 128 x 128 over 65536: 409 us, 15 of 64 parts; 2048 x 1024 over 2048: 16.0
// in 128 x 128, 13.3 in 64 x 64; odd rows, 2047 x 1024 over 2048: 19.2 in 128 x 128 of four parts, 16.1 in 64 x 64).
struct GradientWay {
    bool direct;
    int rows, columns;                                 // of a tile
    int parts;
    int64_t per;
};
constexpr int kStep = 64;
constexpr Small kSmallDirect[] = {{128, 128, 2900, 420, 800}, {64, 64, 2700, 280, 420}};
constexpr Small kSmallStaged[] = {{128, 128, 2900, 1300, 1480}, {64, 64, 2700, 550, 630}};
constexpr Small kSmallFew[] = {kSmallStaged[1]};
GradientWay gradient_way(int64_t T, int64_t N, int64_t K, bool direct) {
    const int64_t small = (N + 127) / 128 * ((K + 127) / 128);
    if (direct) {
        const int64_t large_rounds = ((N + 255) / 256 * ((K + 255) / 256) + kCus - 1) / kCus;
        const int64_t middle_rounds = ((N + 255) / 256 * ((K + 191) / 192) + kCus - 1) / kCus;
        const int64_t small_rounds = (small + 2 * kCus - 1) / (2 * kCus);
        const bool middle = 87 * middle_rounds < 100 * large_rounds;
        if ((middle ? 87 * middle_rounds : 100 * large_rounds) <= 62 * small_rounds)
            return {true, 256, middle ? 192 : 256, 1, T};
    }
    const bool few = !direct && N < 8;
    if (small > kCus && !few) return {direct, 128, 128, 1, T};
    const int64_t steps = (T + kStep - 1) / kStep;
    const Cut cut = direct ? best_of(kSmallDirect, N, K, steps, 1, kGradientRate)
                    : few  ? best_of(kSmallFew, N, K, steps, 1, kGradientRate)
                           : best_of(kSmallStaged, N, K, steps, 1, kGradientRate);
    return {direct, cut.tile->rows, cut.tile->outputs, cut.parts,
            cut.parts == 1 ? T : (steps + cut.parts - 1) / cut.parts * kStep};
}
// Rows of whole dwords that do not overlap: a row past the last then lies past the buffer's range.
bool is_direct(const void* dy, int64_t stride, int64_t N) {
    return stride % 2 == 0 && stride >= N && reinterpret_cast<uintptr_t>(dy) % 4 == 0;
}

template <typename T, int BN, int BK, int WN, int WK>
int launch_direct(const Gradient& a, int parts, hipStream_t st) {
    const int64_t tiles = (int64_t)((a.N + BN - 1) / BN) * ((a.K + BK - 1) / BK);
    if (tiles > kMaxTiles) return Z1_E_SIZE;
    weight_grad_direct_kernel<T, BN, BK, WN, WK, kStep><<<dim3((unsigned)tiles, parts), BN / WN * (BK / WK) * 64, 0, st>>>(a);
    return (int)hipGetLastError();
}
template <typename T>
int small_gradient(const Gradient& a, const GradientWay& way, hipStream_t st) {
    const bool tiny = way.rows == 64;
    if (way.direct)
        return tiny ? launch_direct<T, 64, 64, 32, 32>(a, way.parts, st) : launch_direct<T, 128, 128, 64, 64>(a, way.parts, st);
    if (a.N < 8) return launch_gradient<T, kFew, 64, 64, 32, 32, 64>(a, way.parts, st);
    return tiny ? launch_gradient<T, kCut, 64, 64, 32, 32, 64>(a, way.parts, st)
                : launch_gradient<T, kCut, 128, 128, 64, 64, 32>(a, way.parts, st);
}
template <typename T>
int gradient(Gradient a, const GradientWay& way, float* workspace, hipStream_t st) {
    a.per = way.per;
    if (way.columns == 256) return launch_direct<T, 256, 256, 128, 64>(a, 1, st);
    if (way.columns == 192) return launch_direct<T, 256, 192, 64, 96>(a, 1, st);
    if (way.parts == 1) return small_gradient<T>(a, way, st);
    void* dw = a.dw;
    a.dw = workspace;
    if (const int rc = small_gradient<F32>(a, way, st)) return rc;
    return join<T>(workspace, way.parts, (int64_t)a.N * a.K, dw, st);
}

}  // namespace

extern "C" {

int z1_product8_way(int64_t M, int64_t N, int64_t K, int* way) {
    if (M < 1 || M > kMaxRows || N < 1 || N > kMaxDim || K < 1 || K > kMaxInner) return Z1_E_SIZE;
    if (!way) return Z1_E_NULL;
    const Way w = product_way(M, N, wide_of(K) / kBlock);
    way[0] = w.rows, way[1] = w.outputs, way[2] = w.stages, way[3] = w.parts;
    return Z1_OK;
}

int z1_weight_grad8_way(int64_t T, int64_t N, int64_t K, int whole_dwords, int* way) {
    if (T < 0 || T > kMaxRows || N < 1 || N > kMaxDim || K < 1 || K > kMaxInner) return Z1_E_SIZE;
    if (!way) return Z1_E_NULL;
    const GradientWay w = gradient_way(T, N, K, whole_dwords != 0);
    way[0] = w.rows, way[1] = w.columns, way[2] = w.direct, way[3] = w.parts;
    return Z1_OK;
}

int64_t z1_product8_workspace(int64_t M, int64_t N, int64_t K, int dtype) {
    if (M < 0 || M > kMaxRows || N < 0 || N > kMaxDim || K < 1 || K > kMaxInner) return Z1_E_SIZE;
    if (bad_dtype(dtype)) return Z1_E_DTYPE;
    if (M == 0 || N == 0) return 0;
    const int blocks = wide_of(K) / kBlock;
    const Way way = product_way(M, N, blocks);
    return way.parts > 1 ? way.parts * M * N : 0;
}

int z1_product8(const void* a, const void* as, int64_t M, const void* w, const void* ws, int64_t N, int64_t K, void* y,
                int dtype, float* workspace, int64_t workspace_floats, void* stream) {
    const int64_t need = z1_product8_workspace(M, N, K, dtype);
    if (need < 0) return (int)need;
    if (M == 0 || N == 0) return Z1_OK;
    if (!a || !as || !w || !ws || !y || (need && !workspace)) return Z1_E_NULL;
    if (workspace_floats < need) return Z1_E_WORKSPACE;
    const int blocks = wide_of(K) / kBlock;
    const Product p{(const uint8_t*)a, (const uint8_t*)as, (const uint8_t*)w, (const uint8_t*)ws, y, blocks, M, (int)N,
                    blocks, pitch_of(K), wide_of(K)};
    const Way way = product_way(M, N, blocks);
    const hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case Z1_F32: return launch_product<F32>(p, way, workspace, st);
        case Z1_BF16: return launch_product<BF16>(p, way, workspace, st);
        default: return launch_product<F16>(p, way, workspace, st);
    }
}

int64_t z1_weight_grad8_workspace(int64_t T, int64_t N, int64_t K) {
    if (T < 0 || T > kMaxRows || N < 0 || N > kMaxDim || K < 1 || K > kMaxInner) return Z1_E_SIZE;
    if (N == 0) return 0;
    const int direct = gradient_way(T, N, K, true).parts, staged = gradient_way(T, N, K, false).parts;
    const int64_t parts = direct > staged ? direct : staged;                   // dy's rows may be either
    return parts > 1 ? parts * N * K : 0;
}

int z1_weight_grad8(const uint16_t* dy, int64_t stride, const void* q, const void* s, int64_t T, int64_t N, int64_t K,
                    void* dw, int dtype, float* workspace, int64_t workspace_floats, void* stream) {
    // a step's rows lie within 32 bits of its first
    if (T < 0 || T > kMaxRows || N < 0 || N > kMaxDim || K < 1 || K > kMaxInner || stride < 0 || stride > kMaxDim) return Z1_E_SIZE;
    if (bad_dtype(dtype)) return Z1_E_DTYPE;
    if (N == 0) return Z1_OK;
    if (!dw || (T > 0 && (!dy || !q || !s))) return Z1_E_NULL;
    const int64_t need = z1_weight_grad8_workspace(T, N, K);
    if (need && !workspace) return Z1_E_NULL;
    if (workspace_floats < need) return Z1_E_WORKSPACE;
    const GradientWay way = gradient_way(T, N, K, is_direct(dy, stride, N));
    const Gradient g{dy, stride, (const uint8_t*)q, (const uint8_t*)s, dw, T, T, (int)N, (int)K, wide_of(K), pitch_of(K)};
    const hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case Z1_F32: return gradient<F32>(g, way, workspace, st);
        case Z1_BF16: return gradient<BF16>(g, way, workspace, st);
        default: return gradient<F16>(g, way, workspace, st);
    }
}

}  // extern "C"
