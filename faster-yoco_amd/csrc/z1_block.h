// Device helpers shared by the block-side kernels (norms, 8-bit activations, 8-bit products); not part of the C ABI.
//
// 8-bit values: a row in blocks of kBlock = 128 columns; a block's scale is 2^e, held as the byte e + 127, with e the
// least integer >= -127 such that max |x| <= 448 * 2^e over the block's finite elements; an element is e4m3(x * 2^-e),
// nearest, ties to even.  Powers of two make the scaling exact, so an element has one rounding, and what it stands for
// (4 significant bits) is exact in bf16 too.  448 = 1.75 * 2^8: with max |x| = m * 2^E, 1 <= m < 2, e is E - 8 where
// m <= 1.75 and E - 7 where not, which is a carry out of the mantissa of its fp32 bits plus 0x1fffff.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "yoco_z1.h"

namespace z1blk {

constexpr int kBlock = 128;                  // columns of one scale
constexpr int kLane = 8;                     // columns of one lane in a pass over rows: 16 lanes hold one block

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

#define Z1B_GLOBAL __attribute__((address_space(1)))

// Rows may start at any element: 16-byte accesses need no more than the elements' own alignment.
typedef u4 u4_any2 __attribute__((aligned(2)));
typedef f4 f4_any4 __attribute__((aligned(4)));

__device__ __forceinline__ float as_f32(uint32_t u) { return __uint_as_float(u); }

// Eight elements of a row as they lie in memory (`raw`), and as fp32.
struct F32 {
    typedef float elem;
    struct raw { f4 a, b; };
    static __device__ __forceinline__ raw load(const void* p, int64_t i) {
        const Z1B_GLOBAL f4_any4* q = (const Z1B_GLOBAL f4_any4*)((const float*)p + i);
        return {q[0], q[1]};
    }
    static __device__ __forceinline__ void open(const raw& r, float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = r.a[j], v[4 + j] = r.b[j];
    }
    static __device__ __forceinline__ float one(const void* p, int64_t i) { return ((const Z1B_GLOBAL float*)p)[i]; }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float* v) {
        Z1B_GLOBAL f4_any4* q = (Z1B_GLOBAL f4_any4*)((float*)p + i);
        f4 a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = v[j], b[j] = v[4 + j];
        q[0] = a;
        q[1] = b;
    }
    // past the caches
    static __device__ __forceinline__ void stream(void* p, int64_t i, const float* v) {
        Z1B_GLOBAL f4_any4* q = (Z1B_GLOBAL f4_any4*)((float*)p + i);
        __builtin_nontemporal_store((f4_any4)f4{v[0], v[1], v[2], v[3]}, q);
        __builtin_nontemporal_store((f4_any4)f4{v[4], v[5], v[6], v[7]}, q + 1);
    }
    static __device__ __forceinline__ void put(void* p, int64_t i, float v) { ((Z1B_GLOBAL float*)p)[i] = v; }
    // eight elements to a row in LDS from element i (a multiple of 8) on, and from there to memory
    static __device__ __forceinline__ void store_local(uint8_t* row, int i, const float* v) {
        f4* q = (f4*)(row + i * 4);
        q[0] = f4{v[0], v[1], v[2], v[3]};
        q[1] = f4{v[4], v[5], v[6], v[7]};
    }
    static __device__ __forceinline__ void copy_local(void* p, int64_t at, const uint8_t* row, int i) {
        const f4* q = (const f4*)(row + i * 4);
        Z1B_GLOBAL f4_any4* to = (Z1B_GLOBAL f4_any4*)((float*)p + at);
        to[0] = q[0];
        to[1] = q[1];
    }
    static constexpr float kMax = 3.402823466e38f;
};

struct BF16 {
    typedef __bf16 elem;
    typedef u4 raw;
    static __device__ __forceinline__ raw load(const void* p, int64_t i) {
        return *(const Z1B_GLOBAL u4_any2*)((const uint16_t*)p + i);
    }
    static __device__ __forceinline__ void open(const raw& r, float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = as_f32(r[j] << 16), v[2 * j + 1] = as_f32(r[j] & 0xffff0000u);
    }
    static __device__ __forceinline__ float one(const void* p, int64_t i) {
        return as_f32((uint32_t)((const Z1B_GLOBAL uint16_t*)p)[i] << 16);
    }
    static __device__ __forceinline__ u4 close(const float* v) {
        u4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f2 x = {v[2 * j], v[2 * j + 1]};
            w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, b2));
        }
        return w;
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float* v) {
        *(Z1B_GLOBAL u4_any2*)((uint16_t*)p + i) = close(v);
    }
    static __device__ __forceinline__ void stream(void* p, int64_t i, const float* v) {
        __builtin_nontemporal_store((u4_any2)close(v), (Z1B_GLOBAL u4_any2*)((uint16_t*)p + i));
    }
    static __device__ __forceinline__ void store_local(uint8_t* row, int i, const float* v) { *(u4*)(row + i * 2) = close(v); }
    static __device__ __forceinline__ void copy_local(void* p, int64_t at, const uint8_t* row, int i) {
        *(Z1B_GLOBAL u4_any2*)((uint16_t*)p + at) = *(const u4*)(row + i * 2);
    }
    static __device__ __forceinline__ void put(void* p, int64_t i, float v) { ((Z1B_GLOBAL __bf16*)p)[i] = (__bf16)v; }
    static constexpr float kMax = 3.3895313893e38f;
};

struct F16 {
    typedef _Float16 elem;
    typedef u4 raw;
    static __device__ __forceinline__ raw load(const void* p, int64_t i) { return BF16::load(p, i); }
    static __device__ __forceinline__ void open(const raw& r, float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w = r[j];                   // a bit cast of r[j] itself would take the vector's first word
            const h2 x = __builtin_bit_cast(h2, w);
            v[2 * j] = (float)x[0], v[2 * j + 1] = (float)x[1];
        }
    }
    static __device__ __forceinline__ float one(const void* p, int64_t i) {
        return (float)((const Z1B_GLOBAL _Float16*)p)[i];
    }
    static __device__ __forceinline__ u4 close(const float* v) {
        u4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f2 x = {v[2 * j], v[2 * j + 1]};
            w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, h2));
        }
        return w;
    }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float* v) {
        *(Z1B_GLOBAL u4_any2*)((uint16_t*)p + i) = close(v);
    }
    static __device__ __forceinline__ void stream(void* p, int64_t i, const float* v) {
        __builtin_nontemporal_store((u4_any2)close(v), (Z1B_GLOBAL u4_any2*)((uint16_t*)p + i));
    }
    static __device__ __forceinline__ void store_local(uint8_t* row, int i, const float* v) { *(u4*)(row + i * 2) = close(v); }
    static __device__ __forceinline__ void copy_local(void* p, int64_t at, const uint8_t* row, int i) {
        BF16::copy_local(p, at, row, i);
    }
    static __device__ __forceinline__ void put(void* p, int64_t i, float v) {
        ((Z1B_GLOBAL _Float16*)p)[i] = (_Float16)v;
    }
    static constexpr float kMax = 65504.0f;
};

// The same eight elements where only the first n (0..8) are there: the others are zeros, and are not touched.
template <typename T>
__device__ __forceinline__ void load_some(const void* p, int64_t i, int n, float* v) {
#pragma unroll
    for (int j = 0; j < kLane; ++j) v[j] = j < n ? T::one(p, i + j) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void load_row(const void* p, int64_t i, int n, float* v) {
    if (n >= kLane) {
        T::open(T::load(p, i), v);
    } else {
        load_some<T>(p, i, n, v);
    }
}
template <typename T>
__device__ __forceinline__ void store_row(void* p, int64_t i, int n, const float* v) {
    if (n >= kLane) {
        T::store(p, i, v);
    } else {
#pragma unroll
        for (int j = 0; j < kLane; ++j)
            if (j < n) T::put(p, i + j, v[j]);
    }
}

// A lane's eight elements of a row of `dim` >= 8 from column c on without a branch: it loads eight that are there, from
// column min(c, dim - 8) on, and what the row's end cuts off is moved down and filled up (`settle`) afterwards.
// `by`: c - (dim - 8) where positive; 8 and more: no element is the lane's.
template <typename T>
__device__ __forceinline__ void settle(float* v, int by, float fill = 0.0f) {
#pragma unroll
    for (int s = 4; s; s >>= 1) {
#pragma unroll
        for (int j = 0; j < kLane; ++j) v[j] = by & s ? (j + s < kLane ? v[j + s] : fill) : v[j];
    }
#pragma unroll
    for (int j = 0; j < kLane; ++j) v[j] = by >= kLane ? fill : v[j];
}

// The largest of 16 neighbouring lanes (one DPP row), in every lane of them.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float max16(float x) {
    x = fmaxf(x, dpp<0x128>(x));             // row_ror 8, 4, 2, 1
    x = fmaxf(x, dpp<0x124>(x));
    x = fmaxf(x, dpp<0x122>(x));
    return fmaxf(x, dpp<0x121>(x));
}

__device__ __forceinline__ uint32_t scale_byte(float amax) {                   // amax finite, >= 0
    const uint32_t b = (__float_as_uint(amax) + 0x1fffffu) >> 23;
    return b > 8 ? b - 8 : 0;                                                   // (E + 127) - 8, or one more
}
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return as_f32((254u - byte) << 23); }
// 2^(byte - 127), subnormal for byte 0
__device__ __forceinline__ float scale_value(uint32_t byte) { return as_f32(byte ? byte << 23 : 0x400000u); }

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ float only_finite(float x) {                         // |x| where finite, else 0
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}
__device__ __forceinline__ float nan_of_infinite(float x) {
    return fabsf(x) <= 3.402823466e38f ? x : __builtin_nanf("");
}
__device__ __forceinline__ float amax8(const float* v) {
    float a = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < kLane; ++j) a = fmaxf(a, fabsf(v[j]));
    return a;
}
__device__ __forceinline__ bool not_finite(float amax) { return !(amax <= 3.402823466e38f); }
__device__ __forceinline__ u2 close8(const float* v, uint32_t byte) {
    const float f = scale_inverse(byte);
    u2 q;
    q[0] = e4m3x4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
    q[1] = e4m3x4(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
    return q;
}
// Eight of a block's 128 elements in each of 16 neighbouring lanes, all of them active (with zeros past the row's end):
// the lane's eight bytes, and the block's scale byte in every lane.  fmaxf passes NaN over, so only an infinity (or a
// block of NaN alone) shows in the maximum; e4m3 has no infinity: both become its NaN and do not count for the scale.
__device__ __forceinline__ u2 quantize8(const float* v, uint32_t& byte) {
    float a = max16(amax8(v));
    if (__builtin_expect(not_finite(a), 0)) {
        float w[kLane], m = 0.0f;
#pragma unroll
        for (int j = 0; j < kLane; ++j) w[j] = nan_of_infinite(v[j]), m = fmaxf(m, only_finite(v[j]));
        byte = scale_byte(max16(m));                    // the 16 lanes agree on `a`: all of them are here
        return close8(w, byte);
    }
    byte = scale_byte(a);
    return close8(v, byte);
}

// The eight values that eight bytes stand for, before their scale.
__device__ __forceinline__ void open8(u2 q, float* v) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[j], false);
        const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[j], true);
        v[4 * j] = lo[0], v[4 * j + 1] = lo[1], v[4 * j + 2] = hi[0], v[4 * j + 3] = hi[1];
    }
}

// Sum over the 64 lanes of a wave, in every lane; the same tree for every call.  All lanes are active.
__device__ __forceinline__ float wave_sum(float x) {
    x += dpp<0x128>(x);
    x += dpp<0x124>(x);
    x += dpp<0x122>(x);
    x += dpp<0x121>(x);
    const int i = __builtin_bit_cast(int, x);
    const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 0));
    const float b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 16));
    const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 32));
    const float d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, 48));
    return (a + b) + (c + d);
}

inline int wide_of(int64_t dim) { return (int)((dim + kBlock - 1) / kBlock * kBlock); }
inline int pitch_of(int64_t dim) { return (int)((dim + 4 * kBlock - 1) / (4 * kBlock) * 4); }

}  // namespace z1blk
