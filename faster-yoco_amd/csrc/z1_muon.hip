// The orthogonalised update of matrices: momentum, X's start, and the host's part (declarations: include/yoco_z1.h; the
// mathematics and the other parts: z1_muon.h).
#include "z1_muon.h"

#include <math.h>

#include <algorithm>

namespace {

using namespace z1muon;

// ------------------------------------------------------------------------------------------------------ start
// The momentum's step, and u's squares summed in 64 bits (an fp32 u may be as large as its type goes).  Bound by memory: the
// workgroups of a matrix pass over its groups of eight columns side by side, kAhead of them on the way to a thread (8192 x 3072
// in BF16: 16 us, 37 by 256 workgroups, 44 with one on the way as well; the matrices of two blocks, 690 MB, 130 us, 5.3 TB/s, and
// 148).
constexpr int kStartThreads = 256, kAhead = 4;
template <typename T>
__global__ __launch_bounds__(kStartThreads) void momentum_kernel(Start a, Plan plan) {
    __shared__ double sums[kStartThreads];
    const int z = blockIdx.y;
    const Group& group = group_of_matrix(plan, z);
    const int m = group.tall ? group.c : group.r, n = group.tall ? group.r : group.c;
    const int groups = (n + 7) / 8, step = gridDim.x * kStartThreads, begin = blockIdx.x * kStartThreads + threadIdx.x;
    const int rows = step / groups, more = step % groups;
    int row = begin / groups, i = begin % groups;      // rows below 2^20 and some 2^20 more
    const float factor = a.factor ? *a.factor : 1.0f;
    double s = 0.0;
    while (row < m) {
        Eight e[kAhead];
        int at[kAhead], c[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            at[k] = row;
            c[k] = i * 8;
            if (row < m) load_eight<T>(a, z, row, n, c[k], e[k]);
            row += rows;
            i += more;
            if (i >= groups) i -= groups, ++row;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (at[k] >= m) break;
            float u[8];
            u_of<true>(a, z, at[k], n, c[k], factor, e[k], u);
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

// X in both orders from u: 64 x 64 of it to a workgroup, turned by way of LDS.  Bound by memory (the matrices of two blocks,
// 830 MB, 164 us, 5.1 TB/s; four of 3072 x 3072 59; u again from the gradient and the momentum is as much as a stored u).
// parts: of each matrix's kParts sums, that are there.
template <typename T, bool PRECISE>
__global__ __launch_bounds__(kStartThreads) void start_kernel(Start a, Plan plan, int parts) {
    __shared__ double sums[kStartThreads];
    __shared__ float turned[64][68];
    const Group& group = group_of_tile(plan, blockIdx.x);
    const int m = group.tall ? group.c : group.r, n = group.tall ? group.r : group.c;
    const int planes = planes_of<PRECISE>(group);
    const bool pairs = planes == 2;
    const Layout w = layout_of(group.r, group.c, planes);
    const int across = (n + 63) / 64, down = (m + 63) / 64, nth = (blockIdx.x - group.tile0) / (across * down);
    const int index = blockIdx.x - group.tile0 - nth * across * down, i0 = index / across * 64, j0 = index % across * 64;
    const int z = group.first + nth;
    double s = 0.0;
    for (int k = threadIdx.x; k < parts; k += kStartThreads) s += a.partials[(int64_t)z * kParts + k];
    sums[threadIdx.x] = s;
    __syncthreads();
    for (int k = kStartThreads / 2; k; k >>= 1) {
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
        if (pairs || pair) put_halves<true>(at, plane, v);
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

// ------------------------------------------------------------------------------------------------------ host
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

template <typename T>
int start_of(const Start& a, Plan& w, int64_t count, bool precise, hipStream_t st) {
    // enough workgroups for the largest matrix, a group of eight columns to a thread, and for the card: four of them to a CU
    int64_t parts = 1, tiles = 0;
    for (int k = 0; k < w.groups; ++k) {
        Group& g = w.g[k];
        const int64_t m = g.tall ? g.c : g.r, n = g.tall ? g.r : g.c;
        const int64_t need = (m * ((n + 7) / 8) + kStartThreads - 1) / kStartThreads;
        parts = need > parts ? need : parts;
        g.tile0 = (int)tiles;
        tiles += g.count * ((n + 63) / 64) * ((m + 63) / 64);
        if (tiles > 2 * kMaxTiles) return Z1_E_SIZE;
    }
    const int64_t most = count < 4 ? kParts / count : 256;
    if (parts > most) parts = most;
    momentum_kernel<T><<<dim3((unsigned)parts, (unsigned)count), kStartThreads, 0, st>>>(a, w);
    const dim3 grid((unsigned)tiles);
    if (precise) start_kernel<T, true><<<grid, kStartThreads, 0, st>>>(a, w, (int)parts);
    else start_kernel<T, false><<<grid, kStartThreads, 0, st>>>(a, w, (int)parts);
    return (int)hipGetLastError();
}

int64_t partials_of(int64_t count) { return (count * kParts * (int64_t)sizeof(double) + 1023) / 1024 * 1024; }
int64_t size_of(int64_t m, int64_t n, bool precise) {
    return layout_of((int)(m < n ? m : n), (int)(m < n ? n : m), has_pairs((int)m, (int)n, precise) ? 2 : 1).size;
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

int run(Start a, Plan w, int64_t count, int dtype, int steps, const float* coefficients, bool precise, void* out, Kind kind,
        void* workspace, hipStream_t st) {
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
    return precise ? iterate_precise(s, steps, coefficients, kind) : iterate_fast(s, steps, coefficients, kind);
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
    if (!need) {
        WholeWays ways{};
        ways.add(m, n, precise != 0);
        return run_whole(a, w, ways, count, dtype, steps, coefficients, precise != 0, out, out_dtype, st);
    }
    const Kind kind = out_dtype == Z1_F32 ? OUT_F32 : out_dtype == Z1_BF16 ? OUT_BF16 : OUT_F16;
    return run(a, w, count, dtype, steps, coefficients, precise != 0, out, kind, workspace, st);
}

int z1_orthogonalize_way(int64_t count, int64_t m, int64_t n, int precise, int* way) {
    if (!way) return Z1_E_NULL;
    if (count < 1 || count > kMaxCount || bad_side(m) || bad_side(n)) return Z1_E_SIZE;
    for (int i = 0; i < 12; ++i) way[i] = 0;
    const WholeWay small = whole_way(m, n, precise != 0);
    if (small.pieces) {
        way[1] = small.pieces;
        way[2] = has_pairs((int)m, (int)n, precise != 0);
        return Z1_OK;
    }
    Plan w{};
    w.groups = 1;
    w.g[0] = {0, (int)(m < n ? m : n), (int)(m < n ? n : m), m > n, 0, (int)count, 0, 0.0f, 0.0f};
    if (precise) ways_precise(w, way);
    else ways_fast(w, way);
    return Z1_OK;
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
        WholeWays ways{};
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
            if (end <= small) ways.add(x.m, x.n, precise);
        }
        a.list = 1;
        a.factor = how->factor;
        a.mu = how->momentum;
        a.nesterov = how->nesterov;
        a.eps = how->eps;
        const hipStream_t st = (hipStream_t)stream;
        if (end <= small)
            return run_whole(a, w, ways, end - first, dtype, how->steps, how->coefficients, precise, nullptr, 0, st);
        return run(a, w, end - first, dtype, how->steps, how->coefficients, precise, nullptr, OUT_LIST, workspace, st);
    };
    if (small > 0) {
        const int rc = run_some(0, small);
        if (rc) return rc;
    }
    return small < count ? run_some(small, count) : Z1_OK;
}

}  // extern "C"
