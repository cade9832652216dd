// 8-bit activations and weights: rows in blocks of 128 columns with a power-of-two scale each, and 128 x 128 blocks of a
// weight in both orders (format: z1_block.h; declarations: include/yoco_z1.h).
#include "z1_block.h"

#pragma clang fp contract(off)

namespace {

using namespace z1blk;

constexpr int kThreads = 256;
constexpr int kPer = 4;                                // most groups of 8 columns to a thread
constexpr int64_t kMaxRows = 1ll << 40;
constexpr int64_t kMaxDim = 1 << 24;
constexpr int64_t kFewBlocks = 1024;                   // of kPer groups a thread
constexpr int64_t kMaxBlocks = (1ll << 24) - 1;        // of a launch: its threads count in 32 bits

// The rows are one run of groups of 8 columns, wide / 8 to a row: a workgroup takes kThreads of them, or kThreads *
// PER in turn, and 16 neighbouring lanes always hold one block, since a row is whole blocks.  Packing takes one a thread
// at every size (16384 x 8192 BF16: 75 us, 5.4 TB/s, the same with four; 4099 x 1001: 4.8 us against 6.7), unpacking four
// for large ones (72 us against 82, and 69, 5.8 TB/s, with stores past the caches; the norms' stores gain nothing by it).
struct Place {
    int64_t row;
    int c;
};
__device__ __forceinline__ Place place(int64_t row0, uint32_t rest, uint32_t i, uint32_t per_row) {
    const uint32_t u = rest + i;                       // < per_row + kThreads * kPer
    const uint32_t down = u / per_row;
    return {row0 + down, (int)((u - down * per_row) * kLane)};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void act8_pack_kernel(const void* x, int64_t stride, uint8_t* q, uint8_t* s,
                                                             int64_t rows, int dim, int wide, int pitch) {
    const uint32_t per_row = wide / kLane;
    const int64_t first = (int64_t)blockIdx.x * kThreads;
    const int64_t row0 = first / per_row;
    const Place p = place(row0, (uint32_t)(first - row0 * per_row), threadIdx.x, per_row);
    float v[kLane];
    load_row<T>(x, p.row * stride + p.c, p.row < rows ? dim - p.c : 0, v);
    uint32_t byte;
    const u2 w = quantize8(v, byte);                   // every lane
    if (p.row >= rows) return;
    *(Z1B_GLOBAL u2*)(q + p.row * wide + p.c) = w;
    uint8_t* sr = s + p.row * pitch + p.c / kBlock;
    if ((p.c & (kBlock - 1)) == 0) *sr = (uint8_t)byte;
    if (p.c + kLane == wide)
        for (int j = wide / kBlock; j < pitch; ++j) sr[j - wide / kBlock + 1] = 127;
}

template <typename T, int PER>
__global__ __launch_bounds__(kThreads) void act8_unpack_kernel(const uint8_t* q, const uint8_t* s, void* out,
                                                               int64_t rows, int dim, int wide, int pitch) {
    const uint32_t per_row = wide / kLane;
    const int64_t first = (int64_t)blockIdx.x * (kThreads * PER);
    const int64_t row0 = first / per_row;
    const uint32_t rest = (uint32_t)(first - row0 * per_row);
    u2 w[PER];
    uint32_t byte[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const Place p = place(row0, rest, k * kThreads + threadIdx.x, per_row);
        if (p.row < rows) {
            w[k] = *(const Z1B_GLOBAL u2*)(q + p.row * wide + p.c);
            byte[k] = s[p.row * pitch + p.c / kBlock];
        }
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const Place p = place(row0, rest, k * kThreads + threadIdx.x, per_row);
        if (p.row >= rows || p.c >= dim) continue;
        float v[kLane];
        open8(w[k], v);
        const float f = scale_value(byte[k]);
        // a value that rounded up to a power of two past the type's largest stays finite; NaN stays NaN
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            const float x = v[j] * f;
            v[j] = x != x ? x : fminf(fmaxf(x, -T::kMax), T::kMax);
        }
        if (dim - p.c >= kLane) T::stream(out, p.row * dim + p.c, v);
        else store_row<T>(out, p.row * dim + p.c, dim - p.c, v);
    }
}

// One 128 x 128 block of a weight.  A thread holds 8 rows of 8 columns, so a wave's load covers 256 bytes of four rows,
// and the transposed order is whole 8-byte groups of rows, gathered in LDS into the other order's 128-byte rows.  Bound by
// memory: 8192 x 3072 BF16 in both orders 18.9 us, 5.3 TB/s.
constexpr int kTilePitch = kBlock + 8;

template <typename T>
__global__ __launch_bounds__(kThreads) void weight8_pack_kernel(const void* w, int64_t stride, uint8_t* q, uint8_t* s,
                                                                uint8_t* qt, uint8_t* st, int N, int K, int kb_count,
                                                                int nb_count, int pitch, int pitch_t) {
    __shared__ __align__(16) uint8_t tile[kBlock * kTilePitch];
    __shared__ float red[2][kThreads / 64];
    const int nb = blockIdx.x / kb_count, kb = blockIdx.x - nb * kb_count;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = (threadIdx.x & 15) * kLane, r = (threadIdx.x >> 4) * 8;      // column and first row in the block
    const int k0 = kb * kBlock, n0 = nb * kBlock;
    const int64_t wide = (int64_t)kb_count * kBlock, tall = (int64_t)nb_count * kBlock;
    float v[8][kLane], a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = n0 + r + i;
        load_row<T>(w, (int64_t)row * stride + k0 + c, row < N ? K - k0 - c : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int j = 0; j < kLane; ++j) {              // an infinity becomes NaN, and neither counts for the scale
            v[i][j] = nan_of_infinite(v[i][j]);
            a = fmaxf(a, fabsf(v[i][j]));
        }
    }
    a = max16(a);
    a = fmaxf(a, __shfl_xor(a, 16));
    a = fmaxf(a, __shfl_xor(a, 32));
    if (lane == 0) red[0][wave] = a;
    __syncthreads();
    a = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const uint32_t byte = scale_byte(a);
    u2 b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        b[i] = close8(v[i], byte);
        if (n0 + r + i < N) *(Z1B_GLOBAL u2*)(q + (int64_t)(n0 + r + i) * wide + k0 + c) = b[i];
    }
    if (threadIdx.x == 0) {
        s[(int64_t)nb * pitch + kb] = (uint8_t)byte;
        if (kb == kb_count - 1)
            for (int j = kb_count; j < pitch; ++j) s[(int64_t)nb * pitch + j] = 127;
        if (st) {
            st[(int64_t)kb * pitch_t + nb] = (uint8_t)byte;
            if (nb == nb_count - 1)
                for (int j = nb_count; j < pitch_t; ++j) st[(int64_t)kb * pitch_t + j] = 127;
        }
    }
    if (!qt) return;
#pragma unroll
    for (int j = 0; j < kLane; ++j) {                  // column c + j: its bytes of rows r .. r + 7
        u2 t = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i / 4] |= ((b[i][j / 4] >> (8 * (j % 4))) & 0xffu) << (8 * (i % 4));
        *(u2*)(tile + (c + j) * kTilePitch + r) = t;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBlock * 8; i += kThreads) {                 // 16 bytes each
        const int row = i >> 3, at = (i & 7) * 16;
        if (k0 + row >= K) continue;
        const u2 lo = *(const u2*)(tile + row * kTilePitch + at), hi = *(const u2*)(tile + row * kTilePitch + at + 8);
        *(Z1B_GLOBAL u4*)(qt + (int64_t)(k0 + row) * tall + n0 + at) = u4{lo[0], lo[1], hi[0], hi[1]};
    }
}

bool bad_dtype(int d) { return d != Z1_F32 && d != Z1_BF16 && d != Z1_F16; }

int shape(int64_t rows, int64_t dim, int64_t stride, int64_t* groups) {
    if (rows < 0 || rows > kMaxRows || dim < 1 || dim > kMaxDim || stride < 0) return Z1_E_SIZE;
    *groups = rows * (wide_of(dim) / kLane);
    return *groups > kMaxBlocks * kThreads ? Z1_E_SIZE : Z1_OK;
}

template <typename T>
int pack(const void* x, int64_t rows, int64_t dim, int64_t stride, uint8_t* q, uint8_t* s, int64_t groups, hipStream_t st) {
    const dim3 grid((unsigned)((groups + kThreads - 1) / kThreads));
    act8_pack_kernel<T><<<grid, kThreads, 0, st>>>(x, stride, q, s, rows, (int)dim, wide_of(dim), pitch_of(dim));
    return (int)hipGetLastError();
}
template <typename T>
int unpack(const uint8_t* q, const uint8_t* s, int64_t rows, int64_t dim, void* out, int64_t groups, hipStream_t st) {
    const int d = (int)dim, wide = wide_of(dim), pitch = pitch_of(dim);
    const int64_t per = groups <= kFewBlocks * kThreads * kPer ? kThreads : kThreads * kPer;
    const dim3 blocks((unsigned)((groups + per - 1) / per));
    if (per == kThreads) act8_unpack_kernel<T, 1><<<blocks, kThreads, 0, st>>>(q, s, out, rows, d, wide, pitch);
    else act8_unpack_kernel<T, kPer><<<blocks, kThreads, 0, st>>>(q, s, out, rows, d, wide, pitch);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

int64_t z1_act8_columns(int64_t dim) { return dim < 1 || dim > kMaxDim ? Z1_E_SIZE : wide_of(dim); }
int64_t z1_act8_scales(int64_t dim) { return dim < 1 || dim > kMaxDim ? Z1_E_SIZE : pitch_of(dim); }

int z1_act8_pack(const void* x, int64_t rows, int64_t dim, int64_t stride, int dtype, void* q, void* s, void* stream) {
    int64_t groups;
    if (const int rc = shape(rows, dim, stride, &groups)) return rc;
    if (bad_dtype(dtype)) return Z1_E_DTYPE;
    if (rows == 0) return Z1_OK;
    if (!x || !q || !s) return Z1_E_NULL;
    const hipStream_t st = (hipStream_t)stream;
    uint8_t *qb = (uint8_t*)q, *sb = (uint8_t*)s;
    switch (dtype) {
        case Z1_F32: return pack<F32>(x, rows, dim, stride, qb, sb, groups, st);
        case Z1_BF16: return pack<BF16>(x, rows, dim, stride, qb, sb, groups, st);
        default: return pack<F16>(x, rows, dim, stride, qb, sb, groups, st);
    }
}

int z1_act8_unpack(const void* q, const void* s, int64_t rows, int64_t dim, void* out, int dtype, void* stream) {
    int64_t groups;
    if (const int rc = shape(rows, dim, 0, &groups)) return rc;
    if (bad_dtype(dtype)) return Z1_E_DTYPE;
    if (rows == 0) return Z1_OK;
    if (!q || !s || !out) return Z1_E_NULL;
    const hipStream_t st = (hipStream_t)stream;
    const uint8_t *qb = (const uint8_t*)q, *sb = (const uint8_t*)s;
    switch (dtype) {
        case Z1_F32: return unpack<F32>(qb, sb, rows, dim, out, groups, st);
        case Z1_BF16: return unpack<BF16>(qb, sb, rows, dim, out, groups, st);
        default: return unpack<F16>(qb, sb, rows, dim, out, groups, st);
    }
}

int z1_weight8_pack(const void* w, int64_t N, int64_t K, int64_t stride, int dtype, void* q, void* s, void* qt, void* st,
                    void* stream) {
    if (N < 0 || N > kMaxDim || K < 1 || K > kMaxDim || stride < 0) return Z1_E_SIZE;
    const int64_t nb = (N + kBlock - 1) / kBlock, kb = (K + kBlock - 1) / kBlock;
    if (nb * kb > kMaxBlocks) return Z1_E_SIZE;
    if (bad_dtype(dtype)) return Z1_E_DTYPE;
    if (N == 0) return Z1_OK;
    if (!w || !q || !s || !qt != !st) return Z1_E_NULL;
    const hipStream_t str = (hipStream_t)stream;
    const dim3 grid((unsigned)(nb * kb));
#define Z1_PACK(T)                                                                                                       \
    weight8_pack_kernel<T><<<grid, kThreads, 0, str>>>(w, stride, (uint8_t*)q, (uint8_t*)s, (uint8_t*)qt, (uint8_t*)st,  \
                                                       (int)N, (int)K, (int)kb, (int)nb, pitch_of(K), pitch_of(N))
    switch (dtype) {
        case Z1_F32: Z1_PACK(F32); break;
        case Z1_BF16: Z1_PACK(BF16); break;
        default: Z1_PACK(F16); break;
    }
#undef Z1_PACK
    return (int)hipGetLastError();
}

}  // extern "C"
