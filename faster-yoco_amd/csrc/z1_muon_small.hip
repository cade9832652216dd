// A matrix whose shorter side is at most 128 and that LDS holds: one workgroup does all of it in one launch (64 x 256: 34 us,
// where 17 launches took 71 without pairs; 16 x 16 15).  Bound by latency: fifteen products in a row, each a few fragments to a
// wave.  X itself stays in registers, in fp32 and in the matrix instructions' layout (so e X is what their sums begin with),
// and its fp16 form in LDS is read by rows for A and turned, by transposing reads, for B X.
//
// The pieces: X's fragments of 32 x 32 are dealt to the eight waves, F at most to each; A's (all of them) too, and where they
// are fewer than the waves their summed axis is cut into parts that are added in order.  Rows in LDS are 16 bytes longer than a
// multiple of 64, so that 16 rows' pieces of 16 bytes lie in different banks.
#include "z1_muon.h"

namespace {

using namespace z1muon;

struct Whole {
    Plan plan;                                         // the groups (base, tile0: not used)
    Start start;
    void* out;                                         // or p and p16 of the list
    int dtype, out_dtype;
    int steps;
    uint64_t both;                                     // both_halves
    float co[3 * kMaxSteps];
};
constexpr int kWholeWaves = 8;
// Bytes of a matrix of R x C fragments, and where they are.  X is a pair in any case.
struct Places {
    int px, pa;                                        // bytes of a row of X, and of A and B
    int x_plane, a_plane, A, B, sums, d, e, size;
    int cuts;                                          // parts of A's summed axis
};
__host__ __device__ constexpr Places places_of(int R, int C, bool precise) {
    Places p{};
    const int planes = precise ? 2 : 1;
    p.px = C * 64 + 16;
    p.pa = R * 64 + 16;
    p.x_plane = R * 32 * p.px;
    p.a_plane = R * 32 * p.pa;
    const int most = R > 2 ? 1 : 8 / (R * R), half = C / 2;                    // four steps of 16 columns to a part at least
    p.cuts = 1;
    while (p.cuts < most && p.cuts < half) p.cuts *= 2;
    p.A = 2 * p.x_plane;
    p.B = p.A + planes * p.a_plane;
    p.d = p.B + planes * p.a_plane;
    p.e = p.d + R * 128;
    p.sums = p.e + R * 128;
    p.size = p.sums + (p.cuts > 1 ? p.cuts * R * R * 4096 : 0);
    if (p.size < R * C * 4096) p.size = R * C * 4096;  // u and the result pass through as fp32
    return p;
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

template <int R, bool PRECISE, int F, int BYTES>
__global__ __launch_bounds__(kWholeWaves * 64) void whole_kernel(Whole a) {
    __shared__ __align__(16) uint8_t lds[BYTES];
    __shared__ double norms[kWholeWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int z = blockIdx.x, l32 = lane & 31, half = lane >> 5, rs = spread(l32);
    const Group& g = group_of_matrix(a.plan, z);
    if ((g.r + 31) / 32 != R) return;                  // another launch's
    const int C = (g.c + 31) / 32, pieces = R * C;
    const Places at = places_of(R, C, PRECISE);
    const int m = g.tall ? g.c : g.r, n = g.tall ? g.r : g.c;
    // a lane's part of X's q-th fragment: row o, columns t .. t + 15
    auto o_of = [&](int q) { return (wave + q * kWholeWaves) % R * 32 + l32; };
    auto t_of = [&](int q) { return (wave + q * kWholeWaves) / R * 32 + half * 16; };
    auto on = [&](int q) { return wave + q * kWholeWaves < pieces; };          // the wave's

    // u and the result pass through LDS as rows of fp32, whose groups of four lie at group ^ (row & 7)
    float* const all = (float*)lds;
    auto four = [&](int o, int t) { return (f4*)(all + o * (C * 32) + (((t >> 2) ^ (o & 7)) << 2)); };
    auto one = [&](int o, int t) -> float& { return ((float*)four(o, t))[t & 3]; };
    // eight neighbours of a row of the matrix at a time, put(row, column), over whole fragments
    const int groups = (g.tall ? R : C) * 4, total = pieces * 128;
    auto each = [&](auto put) {
        for (int i = threadIdx.x; i < total; i += kWholeWaves * 64) put(i / groups, i % groups * 8);
    };
    double s = 0.0;
    const float factor = a.start.factor ? *a.start.factor : 1.0f;
    auto load = [&](auto type) {
        each([&](int row, int c) {
            float u[8] = {};
            if (row < m && c < n) load_u<decltype(type), true>(a.start, z, row, n, c, factor, u);
#pragma unroll
            for (int k = 0; k < 8; ++k) s = __builtin_fma((double)u[k], (double)u[k], s);
            if (g.tall) {
#pragma unroll
                for (int k = 0; k < 8; ++k) one(c + k, row) = u[k];
            } else {
                *four(row, c) = f4{u[0], u[1], u[2], u[3]};
                *four(row, c + 4) = f4{u[4], u[5], u[6], u[7]};
            }
        });
    };
    if (a.dtype == Z1_F32) load(F32{});
    else if (a.dtype == Z1_BF16) load(BF16{});
    else load(F16{});
#pragma unroll
    for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
    norms[wave] = s;                                   // every lane writes the same value
    __syncthreads();
    s = norms[0];
    for (int i = 1; i < kWholeWaves; ++i) s += norms[i];
    f16 x[F];
#pragma unroll
    for (int q = 0; q < F; ++q) {
        x[q] = f16{};
        if (!on(q)) continue;
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            const f4 v = *four(o_of(q), t_of(q) + k);
#pragma unroll
            for (int l = 0; l < 4; ++l) x[q][k + l] = v[l];
        }
    }
    __syncthreads();                                   // u has been read
    const double norm = sqrt(s), scale = 1.0 / (norm < a.start.eps ? a.start.eps : norm);        // NaN stays
    auto keep_x = [&](int q) {
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = x[q][k] * kX;
        keep16<true>(lds + o_of(q) * at.px + t_of(q) * 2, at.x_plane, v);
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
        auto one = [&](int k) {
            const h8 p = by_row(rows, pitch, i * 32 + rs, k), q = by_row(rows, pitch, j * 32 + l32, k);
            acc = add(acc, p, q);
            if constexpr (PRECISE) {
                acc = add(acc, p, by_row(rows + plane, pitch, j * 32 + l32, k));
                acc = add(acc, by_row(rows + plane, pitch, i * 32 + rs, k), q);
            }
        };
        int k = begin;
        for (; k + 4 <= end; k += 4) one(k), one(k + 1), one(k + 2), one(k + 3);
        for (; k < end; ++k) one(k);
        return acc;
    };
    constexpr int squares = R * R;

    for (int step = 0; step < a.steps; ++step) {
        const float ca = a.co[3 * step], cb = a.co[3 * step + 1], cc = a.co[3 * step + 2];
        const bool both = PRECISE || (a.both >> step & 1);
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
            const int ij = wave / at.cuts, cut = wave % at.cuts;
            if (ij < squares) {
                const f16 v = square(lds, at.px, at.x_plane, ij / R, ij % R, cut * 2 * C / at.cuts, (cut + 1) * 2 * C / at.cuts);
#pragma unroll
                for (int k = 0; k < 16; ++k) sums[(wave * 16 + k) * 64 + lane] = v[k];
            }
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
#pragma unroll
            for (int k = 0; k < 2 * R; ++k) {
                auto by_column = [&](const uint8_t* rows) {
                    const uint8_t* p = rows + (k * 16 + turned) * at.px + (t + column) * 2;
                    const s4 f0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)p);
                    const s4 f1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Z1B_LDS s4*)(p + 4 * at.px));
                    return __builtin_bit_cast(h8, __builtin_shufflevector(f0, f1, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                const h8 p = by_column(lds), b = by_row(lds + at.B, at.pa, o + l32, k);
                acc = add(acc, p, b);
                if constexpr (PRECISE) acc = add(acc, p, by_row(lds + at.B + at.a_plane, at.pa, o + l32, k));
                if (both) acc = add(acc, by_column(lds + at.x_plane), b);
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
    __syncthreads();                                   // the last step has been read
#pragma unroll
    for (int q = 0; q < F; ++q) {
        if (!on(q)) continue;
#pragma unroll
        for (int k = 0; k < 16; k += 4) *four(o_of(q), t_of(q) + k) = f4{x[q][k], x[q][k + 1], x[q][k + 2], x[q][k + 3]};
    }
    __syncthreads();
    const int64_t own = z * ((int64_t)m * n);
    auto store = [&](auto put) {
        each([&](int row, int c) {
            const int left = n - c;
            if (row >= m || left <= 0) return;
            float v[8];
            if (g.tall) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = one(c + k, row);
            } else {
                F32::open({*four(row, c), *four(row, c + 4)}, v);
            }
            put((int64_t)row * n + c, left, v);
        });
    };
    if (a.start.list) {
        float* const p = a.start.in.p[z];
        uint16_t* const p16 = a.start.in.p16[z];
        store([&](int64_t i, int left, const float* v) {
            float r[8];
            load_row<F32>(p, i, left, r);
#pragma unroll
            for (int k = 0; k < 8; ++k) r[k] = __builtin_fmaf(-g.lr, v[k], r[k] * g.keep);
            store_row<F32>(p, i, left, r);
            if (p16) store_row<BF16>(p16, i, left, r);
        });
    } else if (a.out_dtype == Z1_BF16) {
        store([&](int64_t i, int left, const float* v) { store_row<BF16>(a.out, own + i, left, v); });
    } else if (a.out_dtype == Z1_F16) {
        store([&](int64_t i, int left, const float* v) { store_row<F16>(a.out, own + i, left, v); });
    } else {
        store([&](int64_t i, int left, const float* v) { store_row<F32>(a.out, own + i, left, v); });
    }
}

template <int R, bool PRECISE>
int launch_whole(const Whole& a, const WholeWay& way, int64_t count, hipStream_t st) {
    // what a matrix of R rows of fragments takes at least (it has as many columns of them)
    constexpr int kLeast = places_of(R, R, PRECISE).size;
    const dim3 grid((unsigned)count);
    if constexpr (kLeast <= 64 << 10) {
        if (way.pieces == 2) {
            whole_kernel<R, PRECISE, 2, 64 << 10><<<grid, kWholeWaves * 64, 0, st>>>(a);
            return (int)hipGetLastError();
        }
    }
    if constexpr (kLeast <= 159 << 10) whole_kernel<R, PRECISE, 4, 159 << 10><<<grid, kWholeWaves * 64, 0, st>>>(a);
    return (int)hipGetLastError();
}
template <int R>
int run_rows(const Whole& a, const WholeWays& ways, int64_t count, bool precise, hipStream_t st) {
    const WholeWay& way = ways.of[R - 1];
    if (!way.pieces) return Z1_OK;
    if constexpr (R * 32 > kPairSide)
        if (!precise) return launch_whole<R, false>(a, way, count, st);
    return launch_whole<R, true>(a, way, count, st);
}
static_assert(kPairSide % 32 == 0, "rows of fragments decide on pairs");
}  // namespace

namespace z1muon {

WholeWay whole_way(int64_t m, int64_t n, bool precise) {
    const int64_t r = m < n ? m : n, c = m < n ? n : m;
    if (r > kWholeSide || c > 32 * 32) return {0, 0};
    const int R = (int)(r + 31) / 32, C = (int)(c + 31) / 32, bytes = places_of(R, C, has_pairs((int)r, (int)c, precise)).size;
    for (const WholeWay way : {WholeWay{2, 64 << 10}, WholeWay{4, 159 << 10}})
        if (R * C <= way.pieces * kWholeWaves && bytes <= way.bytes) return way;
    return {0, 0};
}

int run_whole(const Start& start, const Plan& plan, const WholeWays& ways, int64_t count, int dtype, int steps,
              const float* coefficients, bool precise, void* out, int out_dtype, hipStream_t st) {
    Whole a{plan, start, out, dtype, out_dtype, steps, both_halves(coefficients, steps), {}};
    for (int i = 0; i < 3 * steps; ++i) a.co[i] = coefficients[i];
    if (const int rc = run_rows<1>(a, ways, count, precise, st)) return rc;
    if (const int rc = run_rows<2>(a, ways, count, precise, st)) return rc;
    if (const int rc = run_rows<3>(a, ways, count, precise, st)) return rc;
    return run_rows<4>(a, ways, count, precise, st);
}

}  // namespace z1muon
