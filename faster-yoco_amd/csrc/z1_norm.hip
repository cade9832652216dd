// Layer norm and RMS norm over rows, forward and backward (declarations: include/yoco_z1.h).
//
//   forward   mu = mean(x) (0 for RMS), r = 1/sqrt(mean((x-mu)^2) + eps), y = (x-mu) r w + b
//   backward  xh = (x-mu) r, g = dy w:  dx = r (g - mean(g) - xh mean(g xh)) (no mean(g) for RMS),
//             dw = sum over rows of dy xh, db = sum over rows of dy
//
// All of it is bound by memory: a row is read once, held in registers (kLane = 8 columns of a lane at a time), and the
// variance is taken about the mean in a second pass over the registers, so that a large common offset costs no digits.
// Statistics and sums are fp32.
#include "z1_block.h"

#include <type_traits>

#pragma clang fp contract(off)

namespace {

using namespace z1blk;

constexpr int kFwdThreads = 256;
constexpr int kRowThreads = 512;
constexpr int kUnit = 64 * kLane;                      // columns of one wave's access
constexpr int kLongThreads = 1024;                     // of those that read them again

struct Forward {
    const void* x;
    int64_t stride;                                    // elements between rows
    const void* w;
    const void* b;
    void* y;                                           // y in x's type, or
    uint8_t* yq;                                       // its 8-bit form
    uint8_t* ys;
    uint8_t* cq;                                       // the 8-bit form of x
    uint8_t* cs;
    float* mean;
    float* rstd;
    int64_t row0, rows;                                // a launch's first row (long rows only), and the end of all rows
    int dim, wide, pitch;
    int wpr;                                           // waves of a row: 1, 2 or 4
    int w32;                                           // w and b are fp32 (else x's type)
    float eps;
};

template <typename T>
__device__ __forceinline__ void load_weight(const void* p, int w32, int64_t c, int n, float* v) {
    if (w32) load_row<F32>(p, c, n, v);
    else load_row<T>(p, c, n, v);
}

// Sum over a row's wpr waves (red: one slot per wave of the workgroup).  Every wave of the workgroup is here.
__device__ __forceinline__ float row_sum(float s, float* red, int wave, int wpr) {
    s = wave_sum(s);
    if (wpr == 1) return s;
    red[wave] = s;                                     // every lane writes the same value
    __syncthreads();
    const int first = wave & ~(wpr - 1);
    s = red[first];
    for (int i = 1; i < wpr; ++i) s += red[first + i];
    return s;
}

// The 8-bit form of eight columns from c on, of which n are in the row (the rest are zeros): bytes, scale, padding.
__device__ __forceinline__ void put8(uint8_t* q, uint8_t* s, int64_t row, int c, const Forward& a, const float* v) {
    uint32_t byte;
    const u2 w = quantize8(v, byte);
    if (c < a.wide) {
        *(Z1B_GLOBAL u2*)(q + row * a.wide + c) = w;
        if ((c & (kBlock - 1)) == 0) s[row * a.pitch + c / kBlock] = (uint8_t)byte;
    }
}
__device__ __forceinline__ void pad_scales(uint8_t* s, int64_t row, int lane, int wide, int pitch) {
    if (lane < pitch - wide / kBlock) s[row * pitch + wide / kBlock + lane] = 127;
}

template <typename T, bool CENTER>
__device__ __forceinline__ void finish8(const Forward& a, int64_t row, int c, int n, float mu, float r, const float* v) {
    float y[kLane];
#pragma unroll
    for (int j = 0; j < kLane; ++j) y[j] = (CENTER ? v[j] - mu : v[j]) * r;
    if (a.w) {
        float w[kLane];
        load_weight<T>(a.w, a.w32, c, n, w);
        if (CENTER && a.b) {
            float b[kLane];
            load_weight<T>(a.b, a.w32, c, n, b);
#pragma unroll
            for (int j = 0; j < kLane; ++j) y[j] = __builtin_fmaf(y[j], w[j], b[j]);
        } else {
#pragma unroll
            for (int j = 0; j < kLane; ++j) y[j] *= w[j];
        }
    } else if (CENTER && a.b) {
        float b[kLane];
        load_weight<T>(a.b, a.w32, c, n, b);
#pragma unroll
        for (int j = 0; j < kLane; ++j) y[j] += b[j];
    }
    if (a.y) {
        store_row<T>(a.y, row * a.dim + c, n, y);
    } else {
        if (n < kLane) {
#pragma unroll
            for (int j = 0; j < kLane; ++j) y[j] = j < n ? y[j] : 0.0f;
        }
        put8(a.yq, a.ys, row, c, a, y);
    }
    if (a.cq) put8(a.cq, a.cs, row, c, a, v);
}

// Rows of 8 to 4 * NV * 512 columns: a row's wpr waves hold it in registers.  One row to them: a grid of rows, which the
// hardware hands out, is faster here than one that takes rows in turn and loads ahead (layer norm of 16384 x 3072 BF16 37.6
// us, 5.4 TB/s, against 48-65; RMS norm of 8192 x 3072 with 8-bit result and checkpoint 18.9 us, 5.3 TB/s).
// All loads are under way before the first sum, and none stands behind a branch (settle).
template <typename T, typename W, int NV, bool CENTER>
__global__ __launch_bounds__(kFwdThreads) void norm_forward_kernel(Forward a) {
    __shared__ float red[2][kFwdThreads / 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wpr = a.wpr, group = wave / wpr, wi = wave - group * wpr;
    int64_t row = a.row0 + (int64_t)blockIdx.x * (kFwdThreads / 64 / wpr) + group;
    const bool live = row < a.rows;                    // every wave stays for the barriers
    if (!live) row = a.rows - 1;
    const int c0 = (wi * 64 + lane) * kLane, step = wpr * kUnit, last = a.dim - kLane;
    typename T::raw x[NV];
    typename W::raw w[NV], b[NV];
    const void* p = (const typename T::elem*)a.x + row * a.stride;
    const void* pw = a.w ? a.w : a.b ? a.b : a.x;      // something to load, where there is no weight
    const void* pb = a.b ? a.b : pw;
#pragma unroll
    for (int k = 0; k < NV; ++k) x[k] = T::load(p, c0 + k * step < last ? c0 + k * step : last);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = c0 + k * step < last ? c0 + k * step : last;
        w[k] = W::load(pw, c);
        if (CENTER) b[k] = W::load(pb, c);
    }
    float v[NV][kLane], s = 0.0f, mu = 0.0f;
    const float inv = 1.0f / (float)a.dim;
    // whether the row ends in this wave's k-th part, or before it; what then is the lane's
    auto edge = [&](int k) { return (wi + 1) * kUnit + k * step > a.dim; };
    auto by = [&](int k) { return c0 + k * step < last ? 0 : c0 + k * step - last; };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        T::open(x[k], v[k]);
        if (edge(k)) settle<T>(v[k], by(k));
    }
    if (CENTER) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < kLane; ++j) s += v[k][j];
        mu = row_sum(s, red[0], wave, wpr) * inv;
    }
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const bool cut = CENTER && edge(k);
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            float d = v[k][j] - mu;
            if (cut) d = j + by(k) < kLane ? d : 0.0f;
            s = __builtin_fmaf(d, d, s);
        }
    }
    s = row_sum(s, red[1], wave, wpr);
    const float r = 1.0f / sqrtf(s * inv + a.eps);
    if (!live) return;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = c0 + k * step;
        if (c - lane * kLane >= a.wide) continue;      // no lane of the wave has a column here
        float y[kLane], f[kLane], g[kLane];
        W::open(w[k], f);
        if (CENTER) W::open(b[k], g);
        if (edge(k)) {
            settle<W>(f, by(k));
            if (CENTER) settle<W>(g, by(k));
        }
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            y[j] = (CENTER ? v[k][j] - mu : v[k][j]) * r;
            if (!CENTER) y[j] = a.w ? y[j] * f[j] : y[j];
            else y[j] = __builtin_fmaf(y[j], a.w ? f[j] : 1.0f, a.b ? g[j] : 0.0f);
        }
        if (edge(k)) {                                 // y's padding
#pragma unroll
            for (int j = 0; j < kLane; ++j) y[j] = j + by(k) < kLane ? y[j] : 0.0f;
        }
        if (a.y) {
            void* out = (typename T::elem*)a.y + row * a.dim;
            if (edge(k)) store_row<T>(out, c, a.dim - c, y);
            else T::store(out, c, y);
        } else {
            put8(a.yq, a.ys, row, c, a, y);
        }
        if (a.cq) put8(a.cq, a.cs, row, c, a, v[k]);
    }
    if (wi == 0) {
        if (lane == 0) {
            if (CENTER) a.mean[row] = mu;
            a.rstd[row] = r;
        }
        if (a.yq) pad_scales(a.ys, row, lane, a.wide, a.pitch);
        if (a.cq) pad_scales(a.cs, row, lane, a.wide, a.pitch);
    }
}

__device__ __forceinline__ float block_sum(float s, float* red, int wave, int waves) {
    s = wave_sum(s);
    __syncthreads();
    red[wave] = s;
    __syncthreads();
    s = red[0];
    for (int i = 1; i < waves; ++i) s += red[i];
    return s;
}

// Longer rows: one workgroup reads its row again for each pass, from a cache (2048 x 20000 BF16: 44 us, 3.7 TB/s).
template <typename T, bool CENTER>
__global__ __launch_bounds__(kLongThreads) void norm_forward_long_kernel(Forward a) {
    __shared__ float red[kLongThreads / 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = a.row0 + blockIdx.x, at = row * a.stride;
    const int step = kLongThreads * kLane;
    float mu = 0.0f, s = 0.0f, v[kLane];
    if (CENTER) {
        for (int c = threadIdx.x * kLane; c < a.dim; c += step) {
            load_row<T>(a.x, at + c, a.dim - c, v);
#pragma unroll
            for (int j = 0; j < kLane; ++j) s += v[j];
        }
        mu = block_sum(s, red, wave, kLongThreads / 64) / (float)a.dim;
    }
    s = 0.0f;
    for (int c = threadIdx.x * kLane; c < a.dim; c += step) {
        load_row<T>(a.x, at + c, a.dim - c, v);
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            const float d = j < a.dim - c ? v[j] - mu : 0.0f;
            s = __builtin_fmaf(d, d, s);
        }
    }
    s = block_sum(s, red, wave, kLongThreads / 64);
    const float r = 1.0f / sqrtf(s / (float)a.dim + a.eps);
    for (int base = wave * kUnit; base < a.wide; base += step) {        // whole waves: the 8-bit forms need 16 lanes
        const int c = base + lane * kLane;
        load_row<T>(a.x, at + c, a.dim - c, v);
        finish8<T, CENTER>(a, row, c, a.dim - c, mu, r, v);
    }
    if (wave == 0) {
        if (lane == 0) {
            if (CENTER) a.mean[row] = mu;
            a.rstd[row] = r;
        }
        if (a.yq) pad_scales(a.ys, row, lane, a.wide, a.pitch);
        if (a.cq) pad_scales(a.cs, row, lane, a.wide, a.pitch);
    }
}

// ------------------------------------------------------------------------------------------------------ backward
struct Backward {
    const void* dy;
    int64_t dy_stride;
    const void* x;                                     // x in dy's type, or
    int64_t x_stride;
    const uint8_t* q;                                  // its 8-bit form
    const uint8_t* s;
    const float* mean;
    const float* rstd;
    const void* w;
    void* dx;
    float* part;                                       // [blocks][2][dim]: sums of dy xh and of dy; NULL: none
    int64_t row0, rows;                                // a launch's first row (long rows only), and the end of all rows
    int dim, wide, pitch;
    int wpr;                                           // waves of a row: 1, 2, 4 or 8
    int w32;
};

// xh of eight columns (zeros past the row's end).
template <typename T, bool Q, bool CENTER>
__device__ __forceinline__ void load_xh(const Backward& a, int64_t row, int c, int n, float mu, float r, float* xh) {
    if (Q) {
        if (n > 0) {
            const float f = scale_value(a.s[row * a.pitch + c / kBlock]);
            open8(*(const Z1B_GLOBAL u2*)(a.q + row * a.wide + c), xh);
#pragma unroll
            for (int j = 0; j < kLane; ++j) xh[j] *= f;
        } else {
#pragma unroll
            for (int j = 0; j < kLane; ++j) xh[j] = 0.0f;
        }
    } else {
        load_row<T>(a.x, row * a.x_stride + c, n, xh);
    }
#pragma unroll
    for (int j = 0; j < kLane; ++j) xh[j] = (CENTER ? (j < n ? xh[j] - mu : 0.0f) : xh[j]) * r;
}

// Both sums of a row over its wpr waves.
__device__ __forceinline__ void row_sums(float& s1, float& s2, float (*red)[2], int wave, int wpr) {
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if (wpr == 1) return;
    red[wave][0] = s1;
    red[wave][1] = s2;
    __syncthreads();
    const int first = wave & ~(wpr - 1);
    s1 = red[first][0];
    s2 = red[first][1];
    for (int i = 1; i < wpr; ++i) s1 += red[first + i][0], s2 += red[first + i][1];
}

// Eight columns of a row as they are loaded: x in T, or its 8-bit rows' bytes and scale.  open: their values, and `fill` past
// the row's end.
template <typename T, bool Q>
struct Input {
    typename T::raw r;
    static __device__ __forceinline__ Input load(const Backward& a, int64_t row, int c, int from) {
        return {T::load((const typename T::elem*)a.x + row * a.x_stride, from)};
    }
    __device__ __forceinline__ void open(float* v, bool edge, int by, float fill) const {
        T::open(r, v);
        if (edge) settle<T>(v, by, fill);
    }
};
template <typename T>
struct Input<T, true> {
    u2 q;
    uint32_t s;
    static __device__ __forceinline__ Input load(const Backward& a, int64_t row, int c, int from) {
        c = c < a.wide ? c : a.wide - kLane;           // past the row's end: zeros, or not used
        const uint8_t* q = a.q + row * a.wide;
        const uint8_t* s = a.s + row * a.pitch;
        return {*(const Z1B_GLOBAL u2*)(q + (uint32_t)c), ((const Z1B_GLOBAL uint8_t*)s)[(uint32_t)c / kBlock]};
    }
    __device__ __forceinline__ void open(float* v, bool edge, int by, float fill) const {
        const float f = scale_value(s);
        open8(q, v);
#pragma unroll
        for (int j = 0; j < kLane; ++j) v[j] = edge && j + by >= kLane ? fill : v[j] * f;
    }
};

// Rows of 8 to 8 * NV * 512 columns.  A workgroup's groups of wpr waves take rows in turn; a lane keeps its columns' dw and
// db sums in registers over all of them, the groups' sums meet in LDS at the end, and the workgroup writes one partial row
// of each, which norm_reduce_kernel adds in order.  The next rows are loaded while the present ones are computed, and no
// load stands behind a branch.  Bound by memory (layer norm of 16384 x 3072 BF16 57 us, 5.3 TB/s; RMS norm from the checkpoint
// 46 us, 5.5); one workgroup to a CU, as 128 of them (73 us) have too few loads under way and 512 (65) twice the partial rows.
template <typename T, int NV, bool Q, bool CENTER>
__global__ __launch_bounds__(kRowThreads) void norm_backward_kernel(Backward a) {
    __shared__ float red[2][kRowThreads / 64][2];
    __shared__ float sums[kRowThreads * NV * kLane];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wpr = a.wpr, groups = kRowThreads / 64 / wpr, group = wave / wpr, wi = wave - group * wpr;
    const int c0 = (wi * 64 + lane) * kLane, step = wpr * kUnit;
    int from[NV], by[NV];
    bool edge[NV];                                     // the row ends in this wave's k-th part, or before it
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = c0 + k * step, last = a.dim - kLane;
        from[k] = c < last ? c : last;
        by[k] = c - from[k];
        edge[k] = (wi + 1) * kUnit + k * step > a.dim;
    }
    float w[NV][kLane];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < kLane; ++j) w[k][j] = 1.0f;
        if (a.w) {
            if (a.w32) F32::open(F32::load(a.w, from[k]), w[k]);
            else T::open(T::load(a.w, from[k]), w[k]);
            settle<T>(w[k], by[k]);
        }
    }
    float dw[NV][kLane] = {}, db[NV][kLane] = {};
    const float inv = 1.0f / (float)a.dim;
    typename T::raw dy[NV];
    Input<T, Q> x[NV];
    float r_next = 0.0f, mu_next = 0.0f;
    auto fetch = [&](int64_t row) {                    // past the last row: the last, not used
        row = row < a.rows ? row : a.rows - 1;
        r_next = a.rstd[row];
        mu_next = CENTER ? a.mean[row] : 0.0f;
        const void* d = (const typename T::elem*)a.dy + row * a.dy_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            dy[k] = T::load(d, from[k]);
            x[k] = Input<T, Q>::load(a, row, c0 + k * step, from[k]);
        }
    };
    const int64_t stride = (int64_t)gridDim.x * groups;
    int64_t row = (int64_t)blockIdx.x * groups + group;
    const int64_t end = a.rows + group;                // every wave stays for the barriers: the group's last turn
    int turn = 0;
    fetch(row);
    for (; row < end; row += stride) {
        const bool live = row < a.rows;
        const float r = r_next, mu = mu_next;
        float xh[NV][kLane], g[NV][kLane], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            T::open(dy[k], g[k]);
            if (edge[k]) settle<T>(g[k], by[k]);
            x[k].open(xh[k], edge[k], by[k], mu);
        }
        fetch(row + stride);
        if (!live) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < kLane; ++j) g[k][j] = 0.0f, xh[k][j] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < kLane; ++j) {
                // past the row's end dy and w are zeros, x is mu (mu r may be infinite), and so is all that xh enters
                xh[k][j] = (CENTER ? xh[k][j] - mu : xh[k][j]) * r;
                dw[k][j] = __builtin_fmaf(g[k][j], xh[k][j], dw[k][j]);
                if (CENTER) db[k][j] += g[k][j];
                g[k][j] *= w[k][j];
                if (CENTER) s1 += g[k][j];
                s2 = __builtin_fmaf(g[k][j], xh[k][j], s2);
            }
        }
        row_sums(s1, s2, red[turn], wave, wpr);
        turn ^= 1;                                     // the next row's sums need no barrier before they are written
        if (!live) continue;
        const float m1 = s1 * inv, m2 = s2 * inv;
        void* out = (typename T::elem*)a.dx + row * a.dim;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float dx[kLane];
#pragma unroll
            for (int j = 0; j < kLane; ++j)
                dx[j] = __builtin_fmaf(-xh[k][j], m2, CENTER ? g[k][j] - m1 : g[k][j]) * r;
            if (edge[k]) store_row<T>(out, c0 + k * step, a.dim - c0 - k * step, dx);
            else T::store(out, c0 + k * step, dx);
        }
    }
    if (!a.part) return;
    float* out = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    const int columns = step * NV;                     // of a group, in column order below
#pragma unroll
    for (int which = 0; which < (CENTER ? 2 : 1); ++which) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < kLane; ++j) sums[group * columns + c0 + k * step + j] = which ? db[k][j] : dw[k][j];
        __syncthreads();
        for (int c = threadIdx.x; c < a.dim; c += kRowThreads) {
            float t = sums[c];
            for (int i = 1; i < groups; ++i) t += sums[i * columns + c];
            out[which * a.dim + c] = t;
        }
    }
}

// The same in one launch, for few rows: the first workgroups sum dw and db over all rows, kStrip columns each, straight from
// dy and x, and the others give a row's dx to each group of wpr waves.  The rows are read twice, the second time from a
// cache, instead of partial sums written, read and added by a second launch.  What bounds it is the 50 GB/s that one CU gets
// from beyond its XCD's L2: hence narrow strips, and eight neighbours, which share lines of 128 bytes, on one XCD (layer
// norm of 2048 x 3072 BF16: 13.3 us; in two launches 17.5; strips of 32 columns 14.7, of 8 15.0, in launch order 17.1).
constexpr int kStrip = 16, kStripLanes = kStrip / kLane, kStripRows = kRowThreads / kStripLanes;
template <typename T, bool Q, bool CENTER>
__device__ __forceinline__ void strip_sums(const Backward& a, int strip, float (*sums)[2][kStrip]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = strip * kStrip + lane % kStripLanes * kLane, last = a.dim - kLane;
    const int from = c < last ? c : last, by = c - from;
    const int first = threadIdx.x / kStripLanes;
    constexpr int kTurns = 4;                          // of kStripRows rows under way
    float dw[kLane] = {}, db[kLane] = {};
    // kTurns turns from row0 on; `left` rows where those are fewer: past them the last, times nothing
    auto turns = [&](int64_t row0, int left, auto whole) {
        typename T::raw dy[kTurns];
        Input<T, Q> x[kTurns];
        float r[kTurns], mu[kTurns];
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            int t = first + i * kStripRows;
            if (!whole) t = t < left ? t : left - 1;
            const int64_t row = row0 + t;
            dy[i] = T::load((const typename T::elem*)a.dy + row * a.dy_stride, from);
            x[i] = Input<T, Q>::load(a, row, c, from);
            r[i] = a.rstd[row];
            mu[i] = CENTER ? a.mean[row] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            float g[kLane], xh[kLane];
            T::open(dy[i], g);
            x[i].open(xh, !whole && by > 0, by, mu[i]);
            if (!whole) {
                if (by > 0) settle<T>(g, by);
            }
            const bool in = whole || first + i * kStripRows < left;
#pragma unroll
            for (int j = 0; j < kLane; ++j) {
                float h = (CENTER ? xh[j] - mu[i] : xh[j]) * r[i];
                if (!whole) {
                    g[j] = in ? g[j] : 0.0f;
                    h = in ? h : 0.0f;
                }
                dw[j] = __builtin_fmaf(g[j], h, dw[j]);
                if (CENTER) db[j] += g[j];
            }
        }
    };
    constexpr int kAll = kStripRows * kTurns;
    int64_t row0 = 0;
    if (by == 0)
        for (; row0 + kAll <= a.rows; row0 += kAll) turns(row0, kAll, std::true_type{});
    for (; row0 < a.rows; row0 += kAll) turns(row0, (int)(a.rows - row0 < kAll ? a.rows - row0 : kAll), std::false_type{});
    // the wave's rows of one column lie kStripLanes lanes apart
#pragma unroll
    for (int d = kStripLanes; d < 64; d *= 2) {
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            dw[j] += __shfl_xor(dw[j], d);
            if (CENTER) db[j] += __shfl_xor(db[j], d);
        }
    }
    if (lane < kStripLanes) {
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            sums[wave][0][lane * kLane + j] = dw[j];
            if (CENTER) sums[wave][1][lane * kLane + j] = db[j];
        }
    }
    __syncthreads();
}

template <typename T, int NV, bool Q, bool CENTER>
__global__ __launch_bounds__(kRowThreads) void norm_backward_once_kernel(Backward a, int strips, void* out_w, void* out_b,
                                                                         int grad) {
    __shared__ float red[kRowThreads / 64][2];
    __shared__ float sums[kRowThreads / 64][2][kStrip];
    if ((int)blockIdx.x < strips) {
        const int strip = (int)(blockIdx.x & 7) * (strips >> 3) + (int)(blockIdx.x >> 3);
        if (strip * kStrip >= a.dim) return;
        strip_sums<T, Q, CENTER>(a, strip, sums);
        const int which = threadIdx.x / kStrip, c = threadIdx.x % kStrip, at = strip * kStrip + c;
        void* out = which ? out_b : out_w;
        if (which >= (CENTER ? 2 : 1) || at >= a.dim || !out) return;
        float t = sums[0][which][c];
#pragma unroll
        for (int i = 1; i < kRowThreads / 64; ++i) t += sums[i][which][c];
        if (grad == Z1_F32) F32::put(out, at, t);
        else if (grad == Z1_BF16) BF16::put(out, at, t);
        else F16::put(out, at, t);
        return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wpr = a.wpr, groups = kRowThreads / 64 / wpr, group = wave / wpr, wi = wave - group * wpr;
    int64_t row = (int64_t)(blockIdx.x - strips) * groups + group;
    const bool live = row < a.rows;                    // every wave stays for the barrier
    if (!live) row = a.rows - 1;
    const int c0 = (wi * 64 + lane) * kLane, step = wpr * kUnit, last = a.dim - kLane;
    auto edge = [&](int k) { return (wi + 1) * kUnit + k * step > a.dim; };
    auto from = [&](int k) { return c0 + k * step < last ? c0 + k * step : last; };
    typename T::raw dy[NV];
    Input<T, Q> x[NV];
    const void* d = (const typename T::elem*)a.dy + row * a.dy_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        dy[k] = T::load(d, from(k));
        x[k] = Input<T, Q>::load(a, row, c0 + k * step, from(k));
    }
    const float r = a.rstd[row], mu = CENTER ? a.mean[row] : 0.0f;
    float xh[NV][kLane], g[NV][kLane], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int by = c0 + k * step - from(k);
        T::open(dy[k], g[k]);
        if (edge(k)) settle<T>(g[k], by);
        x[k].open(xh[k], edge(k), by, mu);
        if (a.w) {
            float w[kLane];
            if (a.w32) F32::open(F32::load(a.w, from(k)), w);
            else T::open(T::load(a.w, from(k)), w);
            if (edge(k)) settle<T>(w, by);
#pragma unroll
            for (int j = 0; j < kLane; ++j) g[k][j] *= w[j];
        }
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            xh[k][j] = (CENTER ? xh[k][j] - mu : xh[k][j]) * r;
            if (CENTER) s1 += g[k][j];
            s2 = __builtin_fmaf(g[k][j], xh[k][j], s2);
        }
    }
    row_sums(s1, s2, red, wave, wpr);
    if (!live) return;
    const float inv = 1.0f / (float)a.dim, m1 = s1 * inv, m2 = s2 * inv;
    void* out = (typename T::elem*)a.dx + row * a.dim;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float dx[kLane];
#pragma unroll
        for (int j = 0; j < kLane; ++j) dx[j] = __builtin_fmaf(-xh[k][j], m2, CENTER ? g[k][j] - m1 : g[k][j]) * r;
        if (edge(k)) store_row<T>(out, c0 + k * step, a.dim - c0 - k * step, dx);
        else T::store(out, c0 + k * step, dx);
    }
}

// Longer rows: dx by one workgroup a row, which reads it twice; the columns' sums apart (norm_columns_kernel).  2048 x 20000
// BF16: 104 us in all, 2.4 TB/s of what the gradient has to move.
template <typename T, bool Q, bool CENTER>
__global__ __launch_bounds__(kLongThreads) void norm_backward_long_kernel(Backward a) {
    __shared__ float red[kLongThreads / 64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = a.row0 + blockIdx.x;
    const int step = kLongThreads * kLane;
    const float r = a.rstd[row], mu = CENTER ? a.mean[row] : 0.0f;
    float s1 = 0.0f, s2 = 0.0f, xh[kLane], g[kLane];
    for (int pass = 0; pass < 2; ++pass) {
        const float m1 = s1 / (float)a.dim, m2 = s2 / (float)a.dim;
        for (int c = threadIdx.x * kLane; c < a.dim; c += step) {
            const int n = a.dim - c;
            load_xh<T, Q, CENTER>(a, row, c, n, mu, r, xh);
            load_row<T>(a.dy, row * a.dy_stride + c, n, g);
            if (a.w) {
                float w[kLane];
                load_weight<T>(a.w, a.w32, c, n, w);
#pragma unroll
                for (int j = 0; j < kLane; ++j) g[j] *= w[j];
            }
            if (pass == 0) {
#pragma unroll
                for (int j = 0; j < kLane; ++j) s1 += g[j], s2 = __builtin_fmaf(g[j], xh[j], s2);
            } else {
#pragma unroll
                for (int j = 0; j < kLane; ++j)
                    g[j] = __builtin_fmaf(-xh[j], m2, CENTER ? g[j] - m1 : g[j]) * r;
                store_row<T>(a.dx, row * a.dim + c, n, g);
            }
        }
        if (pass == 0) {
            s1 = block_sum(s1, red, wave, kLongThreads / 64);
            s2 = block_sum(s2, red, wave, kLongThreads / 64);
        }
    }
}

constexpr int kColumnThreads = 256;
// dw and db partials of kColumnThreads * 8 columns (blockIdx.x) over the blockIdx.y-th of gridDim.y shares of the rows.
template <typename T, bool Q, bool CENTER>
__global__ __launch_bounds__(kColumnThreads) void norm_columns_kernel(Backward a) {
    const int c = (blockIdx.x * kColumnThreads + threadIdx.x) * kLane, n = a.dim - c;
    if (n <= 0) return;
    float dw[kLane] = {}, db[kLane] = {}, xh[kLane], g[kLane];
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        load_xh<T, Q, CENTER>(a, row, c, n, CENTER ? a.mean[row] : 0.0f, a.rstd[row], xh);
        load_row<T>(a.dy, row * a.dy_stride + c, n, g);
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            dw[j] = __builtin_fmaf(g[j], xh[j], dw[j]);
            if (CENTER) db[j] += g[j];
        }
    }
    float* out = a.part + (int64_t)blockIdx.y * 2 * a.dim;
    store_row<F32>(out, c, n, dw);
    if (CENTER) store_row<F32>(out, (int64_t)a.dim + c, n, db);
}

// dw and db from `parts` partial rows of `columns` sums (dw's, then db's): a few columns to a workgroup, four to a lane, and
// the partial rows in shares, each added in order and the shares in order after that (256 rows of 6144 sums: 4.7 us; 16 or
// 64 shares no better).
constexpr int kReduceShares = 32, kReduceColumns = 1024 / kReduceShares;
template <typename T>
__global__ __launch_bounds__(256) void norm_reduce_kernel(const float* part, int parts, int dim, int columns, void* dw,
                                                          void* db) {
    __shared__ float sums[kReduceShares][kReduceColumns];
    const int lane = threadIdx.x % (kReduceColumns / 4), share = threadIdx.x / (kReduceColumns / 4);
    const int c = blockIdx.x * kReduceColumns + lane * 4;
    const int64_t row = 2 * (int64_t)dim;
    f4 t = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c + 4 <= columns) {
        const float* p = part + c;
        int i = share;
        for (; i + 7 * kReduceShares < parts; i += 8 * kReduceShares) {
            f4 v[8];                                   // loads side by side
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = *(const Z1B_GLOBAL f4_any4*)(p + (i + k * kReduceShares) * row);
#pragma unroll
            for (int k = 0; k < 8; ++k) t += v[k];
        }
        for (; i < parts; i += kReduceShares) t += *(const Z1B_GLOBAL f4_any4*)(p + i * row);
    } else {
        for (int i = share; i < parts; i += kReduceShares)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < columns) t[j] += part[i * row + c + j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[share][lane * 4 + j] = t[j];
    __syncthreads();
    const int at = blockIdx.x * kReduceColumns + threadIdx.x;
    if (threadIdx.x >= kReduceColumns || at >= columns) return;
    float s = sums[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < kReduceShares; ++i) s += sums[i][threadIdx.x];
    if (at < dim) {
        if (dw) T::put(dw, at, s);
    } else if (db) {
        T::put(db, at - dim, s);
    }
}

// ------------------------------------------------------------------------------------------------------ host
constexpr int kMaxVectors = 4;
constexpr int kMaxBlocks = 256;                        // workgroups of the backward pass: one partial row each

// A launch counts its threads in 32 bits: at most this many rows (a multiple of every workgroup's rows) to one.
constexpr int64_t kLaunchRows = 1 << 21;
unsigned launch_rows(int64_t left) { return (unsigned)(left < kLaunchRows ? left : kLaunchRows); }

// Waves of a row of `units` * 512 columns: up to three 8-column groups to a lane while that is enough.
int waves_of(int units) { return units <= 3 ? 1 : units <= 6 ? 2 : units <= 12 ? 4 : 8; }

template <typename T, typename W, bool CENTER>
int forward_rows(Forward& a, int nv, hipStream_t st) {
    const int per = kFwdThreads / 64 / a.wpr;
    for (; a.row0 < a.rows; a.row0 += kLaunchRows) {
        const dim3 grid((launch_rows(a.rows - a.row0) + per - 1) / per);
        switch (nv) {
            case 1: norm_forward_kernel<T, W, 1, CENTER><<<grid, kFwdThreads, 0, st>>>(a); break;
            case 2: norm_forward_kernel<T, W, 2, CENTER><<<grid, kFwdThreads, 0, st>>>(a); break;
            case 3: norm_forward_kernel<T, W, 3, CENTER><<<grid, kFwdThreads, 0, st>>>(a); break;
            case 4: norm_forward_kernel<T, W, 4, CENTER><<<grid, kFwdThreads, 0, st>>>(a); break;
            default: norm_forward_kernel<T, W, 6, CENTER><<<grid, kFwdThreads, 0, st>>>(a); break;
        }
    }
    return (int)hipGetLastError();
}

template <typename T, bool CENTER>
int forward(Forward& a, hipStream_t st) {
    const int units = (a.dim + kUnit - 1) / kUnit;
    if (units > 4 * 6 || a.dim < kLane) {
        for (; a.row0 < a.rows; a.row0 += kLaunchRows)
            norm_forward_long_kernel<T, CENTER><<<launch_rows(a.rows - a.row0), kLongThreads, 0, st>>>(a);
        return (int)hipGetLastError();
    }
    a.wpr = units <= 3 ? 1 : units <= 6 ? 2 : 4;       // two to a lane: 43.4 us, four the same as three, six 47.3
    const int nv = (units + a.wpr - 1) / a.wpr;
    if constexpr (sizeof(typename T::elem) == 2) {
        if (a.w32 && (a.w || a.b)) return forward_rows<T, F32, CENTER>(a, nv, st);
    }
    return forward_rows<T, T, CENTER>(a, nv, st);
}

struct Shape { int wpr, nv, blocks; };                 // wpr 0: the long rows' kernels, `blocks` shares of the rows

Shape backward_shape(int64_t rows, int dim) {
    const int units = (dim + kUnit - 1) / kUnit;
    if (units > 8 * kMaxVectors || dim < kLane) return {0, 0, (int)(rows < 64 ? rows : 64)};
    const int wpr = waves_of(units);
    const int groups = kRowThreads / 64 / wpr;
    const int64_t need = (rows + groups - 1) / groups;
    return {wpr, (units + wpr - 1) / wpr, (int)(need < kMaxBlocks ? need : kMaxBlocks)};
}

template <typename T, bool Q, bool CENTER>
int backward(Backward& a, const Shape& s, hipStream_t st) {
    if (s.wpr == 0) {
        for (; a.row0 < a.rows; a.row0 += kLaunchRows)
            norm_backward_long_kernel<T, Q, CENTER><<<launch_rows(a.rows - a.row0), kLongThreads, 0, st>>>(a);
        if (a.part) {
            const dim3 grid((unsigned)((a.dim + kColumnThreads * kLane - 1) / (kColumnThreads * kLane)), s.blocks);
            norm_columns_kernel<T, Q, CENTER><<<grid, kColumnThreads, 0, st>>>(a);
        }
        return (int)hipGetLastError();
    }
    a.wpr = s.wpr;
    switch (s.nv) {
        case 1: norm_backward_kernel<T, 1, Q, CENTER><<<s.blocks, kRowThreads, 0, st>>>(a); break;
        case 2: norm_backward_kernel<T, 2, Q, CENTER><<<s.blocks, kRowThreads, 0, st>>>(a); break;
        case 3: norm_backward_kernel<T, 3, Q, CENTER><<<s.blocks, kRowThreads, 0, st>>>(a); break;
        default: norm_backward_kernel<T, 4, Q, CENTER><<<s.blocks, kRowThreads, 0, st>>>(a); break;
    }
    return (int)hipGetLastError();
}

// Whether one launch takes it: few rows, since a strip has them all, and few enough in all for the second reading to come
// from a cache.  Layer norm, one launch against two, BF16: 777 x 1537 7.7 us, 12.4; 1024 x 8192 17.2, 19.6; 2560 x 3072
// 15.4, 18.3; but 1536 x 8192 23.3, 22.0; 4096 x 3072 22.3, 21.5; 4096 x 256 14.3, 11.5.
constexpr int64_t kOnceRows = 2560, kOnceElements = 1 << 23;
bool is_once(int64_t rows, int64_t dim) {
    return rows <= kOnceRows && rows * dim <= kOnceElements && dim >= kLane && (dim + kUnit - 1) / kUnit <= 8 * kMaxVectors;
}

template <typename T, bool Q, bool CENTER>
int backward_once(Backward& a, const Shape& s, void* dw, void* db, int grad, hipStream_t st) {
    a.wpr = s.wpr;
    const int strips = dw || db ? (a.dim + 8 * kStrip - 1) / (8 * kStrip) * 8 : 0;       // as many to each XCD
    const int groups = kRowThreads / 64 / s.wpr;
    const dim3 grid((unsigned)(strips + (a.rows + groups - 1) / groups));
    switch (s.nv) {
        case 1: norm_backward_once_kernel<T, 1, Q, CENTER><<<grid, kRowThreads, 0, st>>>(a, strips, dw, db, grad); break;
        case 2: norm_backward_once_kernel<T, 2, Q, CENTER><<<grid, kRowThreads, 0, st>>>(a, strips, dw, db, grad); break;
        case 3: norm_backward_once_kernel<T, 3, Q, CENTER><<<grid, kRowThreads, 0, st>>>(a, strips, dw, db, grad); break;
        default: norm_backward_once_kernel<T, 4, Q, CENTER><<<grid, kRowThreads, 0, st>>>(a, strips, dw, db, grad); break;
    }
    return (int)hipGetLastError();
}
template <typename T>
int once_of(Backward& a, bool center, const Shape& s, void* dw, void* db, int grad, hipStream_t st) {
    if (a.q)
        return center ? backward_once<T, true, true>(a, s, dw, db, grad, st)
                      : backward_once<T, true, false>(a, s, dw, db, grad, st);
    return center ? backward_once<T, false, true>(a, s, dw, db, grad, st)
                  : backward_once<T, false, false>(a, s, dw, db, grad, st);
}

template <typename T>
int backward_of(Backward& a, bool center, const Shape& s, hipStream_t st) {
    if (a.q) return center ? backward<T, true, true>(a, s, st) : backward<T, true, false>(a, s, st);
    return center ? backward<T, false, true>(a, s, st) : backward<T, false, false>(a, s, st);
}

bool bad_dtype(int d) { return d != Z1_F32 && d != Z1_BF16 && d != Z1_F16; }

constexpr int64_t kMaxRows = 1ll << 38;                // rows times columns fit 63 bits
constexpr int64_t kMaxDim = 1 << 24;                   // a whole number in fp32, and columns fit an int

int bad_shape(int64_t rows, int64_t dim, int64_t stride) {
    if (rows < 0 || rows > kMaxRows || dim < 1 || dim > kMaxDim || stride < 0) return Z1_E_SIZE;
    return Z1_OK;
}

}  // namespace

extern "C" {

int z1_norm_forward(const void* x, int64_t rows, int64_t dim, int64_t stride, int dtype, const void* w, const void* b,
                    int w_dtype, float eps, int center, void* y, void* yq, void* ys, void* cq, void* cs, float* mean,
                    float* rstd, void* stream) {
    if (const int rc = bad_shape(rows, dim, stride)) return rc;
    if (bad_dtype(dtype) || (w_dtype != dtype && w_dtype != Z1_F32)) return Z1_E_DTYPE;
    if (center != 0 && center != 1) return Z1_E_MODE;
    if (rows == 0) return Z1_OK;
    if (!x || !rstd || (center && !mean) || !y == !yq || !yq != !ys || !cq != !cs || (b && !center)) return Z1_E_NULL;
    Forward a{x, stride, w, b, y, (uint8_t*)yq, (uint8_t*)ys, (uint8_t*)cq, (uint8_t*)cs, mean, rstd, 0, rows, (int)dim,
              wide_of(dim), pitch_of(dim), 1, w_dtype == Z1_F32, eps};
    const hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case Z1_F32: return center ? forward<F32, true>(a, st) : forward<F32, false>(a, st);
        case Z1_BF16: return center ? forward<BF16, true>(a, st) : forward<BF16, false>(a, st);
        default: return center ? forward<F16, true>(a, st) : forward<F16, false>(a, st);
    }
}

int64_t z1_norm_backward_workspace(int64_t rows, int64_t dim) {
    if (bad_shape(rows, dim, 0)) return Z1_E_SIZE;
    if (is_once(rows, dim)) return 0;
    return (int64_t)backward_shape(rows, (int)dim).blocks * 2 * dim;
}

int z1_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const void* q, const void* s,
                     int64_t rows, int64_t dim, int dtype, const float* mean, const float* rstd, const void* w,
                     int w_dtype, int center, void* dx, void* dw, void* db, int grad_dtype, float* workspace,
                     int64_t workspace_floats, void* stream) {
    if (const int rc = bad_shape(rows, dim, dy_stride)) return rc;
    if (x && x_stride < 0) return Z1_E_SIZE;
    if (bad_dtype(dtype) || (w_dtype != dtype && w_dtype != Z1_F32) || bad_dtype(grad_dtype)) return Z1_E_DTYPE;
    if (center != 0 && center != 1) return Z1_E_MODE;
    if (db && !center) return Z1_E_NULL;
    const hipStream_t st = (hipStream_t)stream;
    const Shape sh = backward_shape(rows, (int)dim);
    if (rows > 0) {
        if (!dy || !x == !q || !q != !s || !rstd || (center && !mean) || !dx) return Z1_E_NULL;
        const bool once = is_once(rows, dim);
        if (!once && (dw || db)) {
            if (!workspace) return Z1_E_NULL;
            if (workspace_floats < (int64_t)sh.blocks * 2 * dim) return Z1_E_WORKSPACE;
        }
        Backward a{dy, dy_stride, x, x_stride, (const uint8_t*)q, (const uint8_t*)s, mean, rstd, w, dx,
                   dw || db ? workspace : nullptr, 0, rows, (int)dim, wide_of(dim), pitch_of(dim), 1, w_dtype == Z1_F32};
        if (once) {
            switch (dtype) {
                case Z1_F32: return once_of<F32>(a, center, sh, dw, db, grad_dtype, st);
                case Z1_BF16: return once_of<BF16>(a, center, sh, dw, db, grad_dtype, st);
                default: return once_of<F16>(a, center, sh, dw, db, grad_dtype, st);
            }
        }
        int rc;
        switch (dtype) {
            case Z1_F32: rc = backward_of<F32>(a, center, sh, st); break;
            case Z1_BF16: rc = backward_of<BF16>(a, center, sh, st); break;
            default: rc = backward_of<F16>(a, center, sh, st); break;
        }
        if (rc) return rc;
    }
    if (!dw && !db) return Z1_OK;
    const int columns = (int)dim * (center ? 2 : 1);
    const dim3 grid((unsigned)((columns + kReduceColumns - 1) / kReduceColumns));
    const int parts = rows > 0 ? sh.blocks : 0;
    switch (grad_dtype) {
        case Z1_F32: norm_reduce_kernel<F32><<<grid, 256, 0, st>>>(workspace, parts, (int)dim, columns, dw, db); break;
        case Z1_BF16: norm_reduce_kernel<BF16><<<grid, 256, 0, st>>>(workspace, parts, (int)dim, columns, dw, db); break;
        default: norm_reduce_kernel<F16><<<grid, 256, 0, st>>>(workspace, parts, (int)dim, columns, dw, db); break;
    }
    return (int)hipGetLastError();
}

}  // extern "C"
