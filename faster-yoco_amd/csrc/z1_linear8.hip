// Products of 8-bit rows with 8-bit weights, and the weight's gradient from 8-bit rows (format: z1_block.h; declarations:
// include/yoco_z1.h).
//
//   product    y[t, o] = sum over blocks j of 2^(e[t, j] + f[o / 128, j]) * sum over k in j of a[t, k] w[o, k]
//   gradient   dw[o, k] = sum over t of dy[t, o] * a[t, k] 2^e[t, k / 128]
//
// The matrix instructions apply the powers of two themselves (v_mfma_scale_f32_32x32x64_f8f6f4 takes one E8M0 byte for
// each lane's 32 values), so a product accumulates over all of K in its fp32 accumulators without a pass of its own for
// the scales.  The gradient's sum runs over tokens, each with a scale of its own: its rows are opened to bf16, which
// holds them exactly, while they are staged, and multiplied by the bf16 instructions.
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

constexpr int kE4M3 = 0;                               // the matrix instructions' code of the format

// The 32 x 32 result of a matrix instruction gives lane l column l % 32 and rows 8 (i/4) + 4 (l/32) + i%4, i = 0..15.
// Reading its first operand's rows in this order makes those 16 consecutive: 16 (l/32) + i.
__device__ __forceinline__ int spread(int row) { return 16 * ((row >> 2) & 1) + 4 * (row >> 3) + (row & 3); }

// Eight bytes of a row and its scale, opened to bf16 (exact: 4 significant bits, and bf16 has fp32's exponents).
__device__ __forceinline__ u4 open_bf16(u2 q, float f) {
    u4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[0], f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[0], f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[1], f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[1], f, true));
    return r;
}

// Adds the products of two 32-row fragments of 64 columns.  The 8-bit instructions sum 8 products at a time on a common
// exponent and cut what is more than 13 bits below the largest (probed: 256 + 2^-5 arrives, 256 + 2^-6 does not, while
// sums across groups keep 24 bits), an error of 1.5e-5 of the result on activations: far below a 16-bit result's own
// rounding, not below an fp32 one's.  PRECISE opens both operands to bf16 (exact) for the bf16 instructions, whose sums
// are fp32 throughout, at half the rate.
template <bool PRECISE, int NO, int NT>
__device__ __forceinline__ void multiply(f16 (&acc)[NO][NT], const i8 (&fo)[NO], const i8 (&ft)[NT], uint32_t so,
                                         const uint32_t (&st)[NT]) {
    if (!PRECISE) {
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fo[i], ft[j], acc[i][j], kE4M3, kE4M3, 0, (int)so,
                                                                            0, (int)st[j]);
        return;
    }
    const float go = scale_value(so & 0xffu);
#pragma unroll
    for (int s = 0; s < 4; ++s) {                      // 8 bytes of a lane: 16 columns of the wave
        u4 bo[NO], bt[NT];
#pragma unroll
        for (int i = 0; i < NO; ++i) bo[i] = open_bf16(u2{(uint32_t)fo[i][2 * s], (uint32_t)fo[i][2 * s + 1]}, go);
#pragma unroll
        for (int j = 0; j < NT; ++j)
            bt[j] = open_bf16(u2{(uint32_t)ft[j][2 * s], (uint32_t)ft[j][2 * s + 1]}, scale_value(st[j] & 0xffu));
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, bo[i]),
                                                                    __builtin_bit_cast(b8, bt[j]), acc[i][j], 0, 0, 0);
    }
}

// A lane's 16 consecutive outputs of one row; n of them are in the row.
template <typename T>
__device__ __forceinline__ void put16(void* out, int64_t at, int64_t n, const f16& v) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = v[i];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (n > 8 * h) store_row<T>(out, at + 8 * h, n - 8 * h < kLane ? (int)(n - 8 * h) : kLane, x + 8 * h);
}

struct Product {
    const uint8_t* a;                                  // [M, wide]
    const uint8_t* as;                                 // [M, pitch]
    const uint8_t* w;                                  // [N, wide]
    const uint8_t* ws;                                 // [ceil(N / 128), pitch]
    void* y;                                           // [M, N]
    int64_t M;
    int N, blocks, pitch;                              // blocks of 128 along K
    int64_t wide;
};

// Staging keeps rows of 128 bytes (one block of K).  A lane of a direct load writes 16 bytes at its own place in a run of
// 1024, so the order of a row's eight 16-byte pieces is changed at the source: piece p of a row lies at p ^ key(row), and
// the eight rows that neighbouring lanes read together have eight different keys.
__device__ __forceinline__ int key_plain(int row) { return row & 7; }
__device__ __forceinline__ int key_spread(int row) { return (row & 3) | ((row >> 4 & 1) << 2); }

__device__ __forceinline__ i8 piece_pair(const uint8_t* row, int p, int key) {
    const i4 lo = *(const i4*)(row + ((p ^ key) << 4)), hi = *(const i4*)(row + (((p + 1) ^ key) << 4));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// BT x BO outputs (tokens x outputs) of a workgroup, WT x WO of a wave.
template <typename T, bool PRECISE, int BT, int BO, int WT, int WO>
__global__ __launch_bounds__(BT / WT * (BO / WO) * 64) void product_kernel(Product a) {
    constexpr int kWaves = BT / WT * (BO / WO);
    constexpr int kPT = BT / 8 / kWaves, kPO = BO / 8 / kWaves;                // direct loads of a wave: 8 rows each
    constexpr int NT = WT / 32, NO = WO / 32;
    __shared__ __align__(1024) uint8_t lds[2][(BT + BO) * kBlock];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_o = (a.N + BO - 1) / BO;
    const int64_t t0 = (int64_t)(blockIdx.x / tiles_o) * BT;
    const int o0 = (int)(blockIdx.x % tiles_o) * BO;
    const int wt = wave / (BO / WO) * WT, wo = wave % (BO / WO) * WO;          // the wave's part of the tile

    const uint8_t* src_t[kPT];
    const uint8_t* src_o[kPO];
    const int sub = lane >> 3, piece = lane & 7;
#pragma unroll
    for (int i = 0; i < kPT; ++i) {
        const int row = (wave * kPT + i) * 8 + sub;
        int64_t t = t0 + row;
        t = t < a.M ? t : a.M - 1;                     // rows past the end repeat the last; their results are dropped
        src_t[i] = a.a + t * a.wide + ((piece ^ key_plain(row)) << 4);
    }
#pragma unroll
    for (int i = 0; i < kPO; ++i) {
        const int row = (wave * kPO + i) * 8 + sub;
        int o = o0 + row;
        o = o < a.N ? o : a.N - 1;
        src_o[i] = a.w + o * a.wide + ((piece ^ key_spread(row)) << 4);
    }
    auto stage = [&](int kb, uint8_t* buf) {
#pragma unroll
        for (int i = 0; i < kPT; ++i)
            __builtin_amdgcn_global_load_lds((const Z1B_GLOBAL void*)(src_t[i] + (int64_t)kb * kBlock),
                                             (Z1B_LDS void*)(buf + (wave * kPT + i) * 8 * kBlock), 16, 0, 0);
#pragma unroll
        for (int i = 0; i < kPO; ++i)
            __builtin_amdgcn_global_load_lds((const Z1B_GLOBAL void*)(src_o[i] + (int64_t)kb * kBlock),
                                             (Z1B_LDS void*)(buf + (BT + (wave * kPO + i) * 8) * kBlock), 16, 0, 0);
    };
    // scales: four blocks' bytes at a time, the next four loaded ahead
    const uint8_t* sa[NT];
    uint32_t now[NT], next[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        int64_t t = t0 + wt + j * 32 + (lane & 31);
        t = t < a.M ? t : a.M - 1;
        sa[j] = a.as + t * a.pitch;
        next[j] = *(const Z1B_GLOBAL uint32_t*)sa[j];
    }
    const int ob = (o0 + wo) / kBlock, ob_last = (a.N - 1) / kBlock;
    const uint8_t* sw = a.ws + (int64_t)(ob < ob_last ? ob : ob_last) * a.pitch;
    uint32_t now_w = 0, next_w = *(const Z1B_GLOBAL uint32_t*)sw;

    f16 acc[NO][NT];
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f16{};

    const int r32 = lane & 31, half = lane >> 5, rs = spread(r32);
    stage(0, lds[0]);
    for (int kb = 0; kb < a.blocks; ++kb) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                       // this wave's direct loads of block kb
        __syncthreads();                               // every wave's, and block kb - 1 has been read
        if (kb + 1 < a.blocks) stage(kb + 1, lds[(kb + 1) & 1]);
        if ((kb & 3) == 0) {
#pragma unroll
            for (int j = 0; j < NT; ++j) now[j] = next[j];
            now_w = next_w;
            if (kb + 4 < a.blocks) {
#pragma unroll
                for (int j = 0; j < NT; ++j) next[j] = *(const Z1B_GLOBAL uint32_t*)(sa[j] + kb + 4);
                next_w = *(const Z1B_GLOBAL uint32_t*)(sw + kb + 4);
            }
        }
        const uint8_t* bt = lds[kb & 1] + (wt + r32) * kBlock;
        const uint8_t* bo = lds[kb & 1] + (BT + wo + rs) * kBlock;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i8 ft[NT], fo[NO];
#pragma unroll
            for (int j = 0; j < NT; ++j) ft[j] = piece_pair(bt + j * 32 * kBlock, 4 * h + 2 * half, key_plain(r32));
#pragma unroll
            for (int i = 0; i < NO; ++i) fo[i] = piece_pair(bo + i * 32 * kBlock, 4 * h + 2 * half, key_spread(rs));
            multiply<PRECISE>(acc, fo, ft, now_w, now);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) now[j] >>= 8;
        now_w >>= 8;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t t = t0 + wt + j * 32 + r32;
        if (t >= a.M) continue;
#pragma unroll
        for (int i = 0; i < NO; ++i) {
            const int o = o0 + wo + i * 32 + half * 16;
            put16<T>(a.y, t * a.N + o, a.N - o, acc[i][j]);
        }
    }
}

// Up to 32 rows: the weight is read once, straight into the matrix instructions' registers, 32 outputs to a workgroup and
// K shared by its waves, whose sums meet in LDS.
constexpr int kFewWaves = 8;
template <typename T, bool PRECISE>
__global__ __launch_bounds__(kFewWaves * 64) void product_few_kernel(Product a) {
    __shared__ float sums[kFewWaves][32 * 33];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o0 = blockIdx.x * 32, r32 = lane & 31, half = lane >> 5;
    int o = o0 + spread(r32);
    o = o < a.N ? o : a.N - 1;
    const int64_t t = r32 < a.M ? r32 : a.M - 1;
    const uint8_t* pa = a.a + t * a.wide + half * 32;
    const uint8_t* pw = a.w + o * a.wide + half * 32;
    const uint8_t* sa = a.as + t * a.pitch;
    const uint8_t* sw = a.ws + (int64_t)(o0 / kBlock) * a.pitch;
    f16 acc[1][1] = {};
    for (int kb = wave; kb < a.blocks; kb += kFewWaves) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const Z1B_GLOBAL i4* x = (const Z1B_GLOBAL i4*)(pa + (int64_t)kb * kBlock + h * 64);
            const Z1B_GLOBAL i4* w = (const Z1B_GLOBAL i4*)(pw + (int64_t)kb * kBlock + h * 64);
            const i8 fx[1] = {__builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7)};
            const i8 fw[1] = {__builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7)};
            const uint32_t sx[1] = {sa[kb]};
            multiply<PRECISE>(acc, fw, fx, sw[kb], sx);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sums[wave][r32 * 33 + half * 16 + i] = acc[0][0][i];
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * 32; e += kFewWaves * 64) {
        const int row = e >> 5, col = e & 31;
        if (row >= a.M || o0 + col >= a.N) continue;
        float v = sums[0][row * 33 + col];
#pragma unroll
        for (int i = 1; i < kFewWaves; ++i) v += sums[i][row * 33 + col];
        T::put(a.y, (int64_t)row * a.N + o0 + col, v);
    }
}

// ------------------------------------------------------------------------------------------------ weight gradient
struct Gradient {
    const uint16_t* dy;                                // bf16 [T, N], rows `stride` apart
    int64_t stride;
    const uint8_t* q;                                  // [T, wide]
    const uint8_t* s;                                  // [T, pitch]
    void* dw;                                          // [N, K]
    int64_t T;
    int N, K, wide, pitch;
};

// Four rows (tokens) of 16 columns by 16 lanes, transposed on the way out of LDS: each lane a column's four.
__device__ __forceinline__ s8 column_pair(const uint16_t* lo, const uint16_t* hi) {
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)lo);
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)hi);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

// BN x BK of dw to a workgroup, WN x WK to a wave, TS tokens staged at a time.
template <typename T, int BN, int BK, int WN, int WK, int TS>
__global__ __launch_bounds__(BN / WN * (BK / WK) * 64) void weight_grad_kernel(Gradient a) {
    constexpr int kThreads = BN / WN * (BK / WK) * 64;
    constexpr int kPitchN = BN + 32, kPitchK = BK + 32;                        // elements: rows 64 bytes apart in the banks
    constexpr int kDy = TS * BN / 8 / kThreads, kX = TS * BK / 8 / kThreads;   // 8-element pieces of a thread
    constexpr int NN = WN / 32, NK = WK / 32;
    __shared__ __align__(16) uint16_t lds_n[2][TS * kPitchN];
    __shared__ __align__(16) uint16_t lds_k[2][TS * kPitchK];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_k = (a.K + BK - 1) / BK;
    const int n0 = (int)(blockIdx.x / tiles_k) * BN, k0 = (int)(blockIdx.x % tiles_k) * BK;
    const int wn = wave / (BK / WK) * WN, wk = wave % (BK / WK) * WK;

    u4 dy[kDy];
    u2 x[kX];
    uint32_t xs[kX];
    auto fetch = [&](int64_t t0) {
#pragma unroll
        for (int i = 0; i < kDy; ++i) {
            const int e = i * kThreads + threadIdx.x, c = e % (BN / 8) * 8;
            const int64_t t = t0 + e / (BN / 8);
            const int n = t < a.T ? a.N - n0 - c : 0;
            if (n >= 8) {
                dy[i] = *(const Z1B_GLOBAL u4_any2*)(a.dy + t * a.stride + n0 + c);
            } else {
                dy[i] = u4{};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) dy[i][j / 2] |= (uint32_t)((const Z1B_GLOBAL uint16_t*)a.dy)[t * a.stride + n0 + c + j] << (16 * (j % 2));
            }
        }
#pragma unroll
        for (int i = 0; i < kX; ++i) {
            const int e = i * kThreads + threadIdx.x, c = e % (BK / 8) * 8;
            const int64_t t = t0 + e / (BK / 8);
            const bool in = t < a.T && k0 + c < a.wide;
            x[i] = in ? *(const Z1B_GLOBAL u2*)(a.q + t * a.wide + k0 + c) : u2{0, 0};
            xs[i] = in ? a.s[t * a.pitch + (k0 + c) / kBlock] : 127u;
        }
    };
    auto keep = [&](int buf) {
#pragma unroll
        for (int i = 0; i < kDy; ++i) {
            const int e = i * kThreads + threadIdx.x;
            *(u4*)(lds_n[buf] + e / (BN / 8) * kPitchN + e % (BN / 8) * 8) = dy[i];
        }
#pragma unroll
        for (int i = 0; i < kX; ++i) {
            const int e = i * kThreads + threadIdx.x;
            *(u4*)(lds_k[buf] + e / (BK / 8) * kPitchK + e % (BK / 8) * 8) = open_bf16(x[i], scale_value(xs[i]));
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
    fetch(0);
    keep(0);
    int buf = 0;
    for (int64_t t0 = 0; t0 < a.T; t0 += TS) {
        __syncthreads();
        if (t0 + TS < a.T) fetch(t0 + TS);
        const uint16_t* bn = lds_n[buf] + row * kPitchN + wn + col_n;
        const uint16_t* bk = lds_k[buf] + row * kPitchK + wk + col_k;
#pragma unroll
        for (int kk = 0; kk < TS / 16; ++kk) {
            s8 fn[NN], fk[NK];
#pragma unroll
            for (int j = 0; j < NN; ++j)
                fn[j] = column_pair(bn + kk * 16 * kPitchN + j * 32, bn + (kk * 16 + 4) * kPitchN + j * 32);
#pragma unroll
            for (int i = 0; i < NK; ++i)
                fk[i] = column_pair(bk + kk * 16 * kPitchK + i * 32, bk + (kk * 16 + 4) * kPitchK + i * 32);
#pragma unroll
            for (int i = 0; i < NK; ++i)
#pragma unroll
                for (int j = 0; j < NN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, fk[i]),
                                                                        __builtin_bit_cast(b8, fn[j]), acc[i][j], 0, 0, 0);
        }
        if (t0 + TS < a.T) keep(buf ^ 1);
        buf ^= 1;
    }
    const int half = lane >> 5;
#pragma unroll
    for (int j = 0; j < NN; ++j) {
        const int n = n0 + wn + j * 32 + (lane & 31);
        if (n >= a.N) continue;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int k = k0 + wk + i * 32 + half * 16;
            put16<T>(a.dw, (int64_t)n * a.K + k, a.K - k, acc[i][j]);
        }
    }
}

constexpr int64_t kMaxRows = 1ll << 40;
constexpr int64_t kMaxDim = 1 << 24;
constexpr int64_t kMaxTiles = 1ll << 22;               // of a launch: its threads count in 32 bits

bool bad_dtype(int d) { return d != Z1_F32 && d != Z1_BF16 && d != Z1_F16; }

template <typename T, bool PRECISE>
int launch_product(const Product& a, hipStream_t st) {
    if (a.M <= 32) {
        product_few_kernel<T, PRECISE><<<dim3((unsigned)((a.N + 31) / 32)), kFewWaves * 64, 0, st>>>(a);
        return (int)hipGetLastError();
    }
    constexpr int B = 128;
    const int64_t tiles = (a.M + B - 1) / B * ((a.N + B - 1) / B);
    if (tiles > kMaxTiles) return Z1_E_SIZE;
    product_kernel<T, PRECISE, B, B, 64, 64><<<dim3((unsigned)tiles), 256, 0, st>>>(a);
    return (int)hipGetLastError();
}

// fp32 results are always precise; 16-bit ones where K is short, since a short sum has few groups over which the cuts
// average out, and its time goes into the result's writes anyway.
constexpr int kPreciseBlocks = 3;
template <typename T>
int product(const Product& a, hipStream_t st) {
    return a.blocks <= kPreciseBlocks ? launch_product<T, true>(a, st) : launch_product<T, false>(a, st);
}
template <>
int product<F32>(const Product& a, hipStream_t st) {
    return launch_product<F32, true>(a, st);
}

template <typename T>
int gradient(const Gradient& a, hipStream_t st) {
    constexpr int B = 128;
    const int64_t tiles = (int64_t)((a.N + B - 1) / B) * ((a.K + B - 1) / B);
    if (tiles > kMaxTiles) return Z1_E_SIZE;
    weight_grad_kernel<T, B, B, 64, 64, 32><<<dim3((unsigned)tiles), 256, 0, st>>>(a);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

int z1_product8(const void* a, const void* as, int64_t M, const void* w, const void* ws, int64_t N, int64_t K, void* y,
                int dtype, void* stream) {
    if (M < 0 || M > kMaxRows || N < 0 || N > kMaxDim || K < 1 || K > kMaxDim) return Z1_E_SIZE;
    if (bad_dtype(dtype)) return Z1_E_DTYPE;
    if (M == 0 || N == 0) return Z1_OK;
    if (!a || !as || !w || !ws || !y) return Z1_E_NULL;
    const Product p{(const uint8_t*)a, (const uint8_t*)as, (const uint8_t*)w, (const uint8_t*)ws, y, M, (int)N,
                    wide_of(K) / kBlock, pitch_of(K), wide_of(K)};
    const hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case Z1_F32: return product<F32>(p, st);
        case Z1_BF16: return product<BF16>(p, st);
        default: return product<F16>(p, st);
    }
}

int z1_weight_grad8(const uint16_t* dy, int64_t stride, const void* q, const void* s, int64_t T, int64_t N, int64_t K,
                    void* dw, int dtype, void* stream) {
    if (T < 0 || T > kMaxRows || N < 0 || N > kMaxDim || K < 1 || K > kMaxDim || stride < 0) return Z1_E_SIZE;
    if (bad_dtype(dtype)) return Z1_E_DTYPE;
    if (N == 0) return Z1_OK;
    if (!dw || (T > 0 && (!dy || !q || !s))) return Z1_E_NULL;
    const Gradient g{dy, stride, (const uint8_t*)q, (const uint8_t*)s, dw, T, (int)N, (int)K, wide_of(K), pitch_of(K)};
    const hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case Z1_F32: return gradient<F32>(g, st);
        case Z1_BF16: return gradient<BF16>(g, st);
        default: return gradient<F16>(g, st);
    }
}

}  // extern "C"
