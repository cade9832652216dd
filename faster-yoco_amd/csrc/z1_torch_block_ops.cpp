/*
 * The block-side kernels (norms, 8-bit activations and weights, 8-bit products) as PyTorch operators of the namespace
 * yoco_z1: schemas, CUDA (HIP) kernels -- argument checks and one call of the C ABI on torch's current stream -- and CPU
 * kernels that only raise.  Host code only.  Results and workspaces come from torch's allocator, on the call's stream,
 * so the operators may be captured in a graph and used on any stream.  z1t_init_block(path) resolves the C ABI, as
 * z1t_init does for the update's operators.
 */
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <dlfcn.h>

#include <cstdint>
#include <optional>
#include <tuple>
#include <vector>

#include "yoco_z1.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Api {
    decltype(&::z1_norm_forward) norm_forward;
    decltype(&::z1_norm_backward) norm_backward;
    decltype(&::z1_norm_backward_workspace) norm_backward_workspace;
    decltype(&::z1_act8_columns) act8_columns;
    decltype(&::z1_act8_scales) act8_scales;
    decltype(&::z1_act8_pack) act8_pack;
    decltype(&::z1_act8_unpack) act8_unpack;
    decltype(&::z1_weight8_pack) weight8_pack;
    decltype(&::z1_product8) product8;
    decltype(&::z1_product8_workspace) product8_workspace;
    decltype(&::z1_weight_grad8) weight_grad8;
    decltype(&::z1_weight_grad8_workspace) weight_grad8_workspace;
    decltype(&::z1_strerror) strerror;
};

Api g_api{};
bool g_api_ok = false;

const Api& api() {
    TORCH_CHECK(g_api_ok, "yoco_z1: the block-side operators are not bound: faster_yoco_amd.library is not imported, or the "
                         "selected build of libyoco_z1.so lacks them");
    return g_api;
}

void check_rc(int64_t rc, const char* what) {
    if (rc != 0) {
        const char* s = g_api.strerror ? g_api.strerror(static_cast<int>(rc)) : nullptr;
        TORCH_CHECK(false, "yoco_z1: ", what, " failed: ", s ? s : "?", " (code ", rc, ")");
    }
}

// ------------------------------------------------------------------------------------------ argument checks
int dtype_code(at::ScalarType t, const char* what) {
    switch (t) {
        case at::kFloat: return Z1_F32;
        case at::kBFloat16: return Z1_BF16;
        case at::kHalf: return Z1_F16;
        default: TORCH_CHECK(false, what, ": expected fp32, bf16 or fp16, got ", c10::toString(t));
    }
}

void require_gpu(const Tensor& t, const char* what, const char* name) {
    TORCH_CHECK(t.defined() && t.is_cuda(), what, ": ", name, ": expected a GPU tensor (there is no CPU path)");
}

void require_on(const Tensor& t, const Tensor& other, const char* what, const char* name) {
    require_gpu(t, what, name);
    TORCH_CHECK(t.device() == other.device(), what, ": ", name, " is on ", t.device(), ", the launch runs on ",
                other.device());
}

// Rows [rows, dim] whose elements are neighbours; any stride between rows.
struct Rows {
    const void* p;
    int64_t rows, dim, stride;
    int dtype;
};
Rows rows_of(const Tensor& t, const char* what, const char* name) {
    TORCH_CHECK(t.dim() == 2, what, ": ", name, ": expected rows [n, dim], got ", t.dim(), " dimensions");
    const int64_t n = t.size(0), d = t.size(1);
    TORCH_CHECK(d >= 1, what, ": ", name, ": expected at least one column");
    TORCH_CHECK((d == 1 || t.stride(1) == 1) && (n <= 1 || t.stride(0) >= 0), what, ": ", name,
                ": expected rows of neighbouring elements");
    return {t.const_data_ptr(), n, d, t.stride(0), dtype_code(t.scalar_type(), what)};
}

// A column vector [dim] in `like`'s type or fp32, or none.
const void* weight_of(const OptTensor& t, const Tensor& x, int64_t dim, const char* what, const char* name) {
    if (!t.has_value() || !t->defined()) return nullptr;
    require_on(*t, x, what, name);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == dim && t->is_contiguous(), what, ": ", name, ": expected a contiguous [",
                dim, "]");
    TORCH_CHECK(t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type(), what, ": ", name,
                ": expected fp32 or the rows' type");
    return t->const_data_ptr();
}

const float* stat_of(const Tensor& t, const Tensor& x, int64_t rows, const char* what, const char* name) {
    require_on(t, x, what, name);
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == rows && t.is_contiguous(), what, ": ", name,
                ": expected contiguous fp32 [", rows, "]");
    return static_cast<const float*>(t.const_data_ptr());
}

int64_t wide_of(int64_t dim, const char* what) {
    const int64_t w = api().act8_columns(dim);
    if (w < 0) check_rc(w, what);
    return w;
}

// 8-bit rows: q [rows, wide(dim)] and s [scale_rows, pitch(dim)].
void check8(const Tensor& q, const Tensor& s, int64_t rows, int64_t dim, int64_t scale_rows, const char* what,
            const char* name) {
    require_gpu(q, what, name);
    require_on(s, q, what, name);
    TORCH_CHECK(q.scalar_type() == at::kFloat8_e4m3fn && s.scalar_type() == at::kFloat8_e8m0fnu, what, ": ", name,
                ": expected float8_e4m3fn values and float8_e8m0fnu scales");
    const int64_t wide = wide_of(dim, what), pitch = api().act8_scales(dim);
    TORCH_CHECK(q.dim() == 2 && q.size(0) == rows && q.size(1) == wide && q.is_contiguous(), what, ": ", name,
                ": expected contiguous values [", rows, ", ", wide, "]");
    TORCH_CHECK(s.dim() == 2 && s.size(0) == scale_rows && s.size(1) == pitch && s.is_contiguous(), what, ": ", name,
                ": expected contiguous scales [", scale_rows, ", ", pitch, "]");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(q.const_data_ptr()) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(s.const_data_ptr()) % 4 == 0,
                what, ": ", name, ": values must be 16-byte aligned and scales 4-byte aligned");
}

// A new tensor on the current device, from torch's allocator.  (at::empty goes through the dispatcher again: a norm's four
// to six results then cost 2 us more.)
Tensor fresh(at::IntArrayRef size, at::ScalarType dtype) {
    return Tensor(at::detail::empty_cuda(size, dtype, c10::Device(c10::DeviceType::CUDA), std::nullopt));
}

// Scratch floats of one call.  Freed when the call returns, which torch's allocator orders behind the call's launches.
struct Workspace {
    Tensor t;
    float* p = nullptr;
    int64_t floats;
    Workspace(int64_t n, const char* what) : floats(n) {
        if (n < 0) check_rc(n, what);
        if (n > 0) {
            t = fresh({n}, at::kFloat);
            p = static_cast<float*>(t.data_ptr());
        }
    }
};

struct Pair {
    Tensor q, s;
};
Pair empty8(int64_t rows, int64_t dim, int64_t scale_rows, const char* what) {
    const int64_t wide = wide_of(dim, what);
    return {fresh({rows, wide}, at::kFloat8_e4m3fn), fresh({scale_rows, api().act8_scales(dim)}, at::kFloat8_e8m0fnu)};
}

struct OnDevice {
    c10::DeviceGuard guard;
    void* stream;
    explicit OnDevice(const Tensor& t)
        : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

// ------------------------------------------------------------------------------------------ norms
// [y or (yq, ys), mean (center), rstd, (cq, cs) (checkpoint)]
std::vector<Tensor> norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, bool center,
                                 bool y8, bool checkpoint) {
    const char* what = "norm";
    require_gpu(x, what, "x");
    const Rows r = rows_of(x, what, "x");
    const void* w = weight_of(weight, x, r.dim, what, "weight");
    const void* b = weight_of(bias, x, r.dim, what, "bias");
    TORCH_CHECK(!b || center, what, ": the uncentred norm takes no bias");
    TORCH_CHECK(!w || !b || weight->scalar_type() == bias->scalar_type(), what, ": weight and bias must have one type");
    TORCH_CHECK(eps >= 0, what, ": eps must not be negative");
    const int w_dtype = w || b ? dtype_code((w ? *weight : *bias).scalar_type(), what) : Z1_F32;
    OnDevice on(x);
    std::vector<Tensor> out;
    void *y = nullptr, *yq = nullptr, *ys = nullptr, *cq = nullptr, *cs = nullptr;
    float* mean = nullptr;
    out.reserve(6);
    if (y8) {
        Pair p = empty8(r.rows, r.dim, r.rows, what);
        yq = p.q.data_ptr();
        ys = p.s.data_ptr();
        out.push_back(std::move(p.q));
        out.push_back(std::move(p.s));
    } else {
        out.push_back(fresh({r.rows, r.dim}, x.scalar_type()));
        y = out.back().data_ptr();
    }
    if (center) {
        out.push_back(fresh({r.rows}, at::kFloat));
        mean = static_cast<float*>(out.back().data_ptr());
    }
    out.push_back(fresh({r.rows}, at::kFloat));
    float* rstd = static_cast<float*>(out.back().data_ptr());
    if (checkpoint) {
        Pair p = empty8(r.rows, r.dim, r.rows, what);
        cq = p.q.data_ptr();
        cs = p.s.data_ptr();
        out.push_back(std::move(p.q));
        out.push_back(std::move(p.s));
    }
    check_rc(api().norm_forward(r.p, r.rows, r.dim, r.stride, r.dtype, w, b, w_dtype, static_cast<float>(eps), center, y,
                                yq, ys, cq, cs, mean, rstd, on.stream), "z1_norm_forward");
    return out;
}

// [dx, dw (need_dw), db (need_db)]; x, or its 8-bit rows q, s; dw and db in grad_dtype, else the weight's, else dy's
std::vector<Tensor> norm_backward(const Tensor& dy, const OptTensor& x, const OptTensor& q, const OptTensor& s,
                                  const OptTensor& mean, const Tensor& rstd, const OptTensor& weight, bool center,
                                  bool need_dw, bool need_db, std::optional<at::ScalarType> grad_dtype) {
    const char* what = "norm_backward";
    require_gpu(dy, what, "dy");
    const Rows r = rows_of(dy, what, "dy");
    const bool packed = q.has_value() && q->defined();
    const bool plain = x.has_value() && x->defined();
    TORCH_CHECK(packed != plain, what, ": expected x or its 8-bit rows");
    Rows xr{nullptr, r.rows, r.dim, r.dim, r.dtype};
    if (packed) {
        TORCH_CHECK(s.has_value() && s->defined(), what, ": expected the scales of the 8-bit rows");
        require_on(*q, dy, what, "x");
        check8(*q, *s, r.rows, r.dim, r.rows, what, "x");
    } else {
        require_on(*x, dy, what, "x");
        xr = rows_of(*x, what, "x");
        TORCH_CHECK(xr.rows == r.rows && xr.dim == r.dim && xr.dtype == r.dtype, what, ": dy and x must have one shape "
                    "and type");
    }
    TORCH_CHECK(center || !need_db, what, ": the uncentred norm has no bias");
    const float* mp = nullptr;
    if (center) {
        TORCH_CHECK(mean.has_value() && mean->defined(), what, ": expected the rows' means");
        mp = stat_of(*mean, dy, r.rows, what, "mean");
    }
    const float* rp = stat_of(rstd, dy, r.rows, what, "rstd");
    const void* w = weight_of(weight, dy, r.dim, what, "weight");
    const at::ScalarType gt = grad_dtype.value_or((w ? *weight : dy).scalar_type());
    const int grad_code = dtype_code(gt, what);
    OnDevice on(dy);
    std::vector<Tensor> out;
    out.reserve(3);
    out.push_back(fresh({r.rows, r.dim}, dy.scalar_type()));
    if (need_dw) out.push_back(fresh({r.dim}, gt));
    if (need_db) out.push_back(fresh({r.dim}, gt));
    const Workspace parts(need_dw || need_db ? api().norm_backward_workspace(r.rows, r.dim) : 0,
                          "z1_norm_backward_workspace");
    check_rc(api().norm_backward(r.p, r.stride, plain ? xr.p : nullptr, xr.stride, packed ? q->const_data_ptr() : nullptr,
                                 packed ? s->const_data_ptr() : nullptr, r.rows, r.dim, r.dtype, mp, rp, w,
                                 w ? dtype_code(weight->scalar_type(), what) : Z1_F32, center, out[0].data_ptr(),
                                 need_dw ? out[1].data_ptr() : nullptr, need_db ? out.back().data_ptr() : nullptr,
                                 grad_code, parts.p, parts.floats, on.stream), "z1_norm_backward");
    return out;
}

// ------------------------------------------------------------------------------------------ 8-bit rows and weights
std::tuple<Tensor, Tensor> act8_pack(const Tensor& x) {
    const char* what = "act8.pack";
    require_gpu(x, what, "x");
    const Rows r = rows_of(x, what, "x");
    OnDevice on(x);
    Pair p = empty8(r.rows, r.dim, r.rows, what);
    check_rc(api().act8_pack(r.p, r.rows, r.dim, r.stride, r.dtype, p.q.data_ptr(), p.s.data_ptr(), on.stream),
             "z1_act8_pack");
    return {std::move(p.q), std::move(p.s)};
}

Tensor act8_unpack(const Tensor& q, const Tensor& s, int64_t dim, at::ScalarType dtype) {
    const char* what = "act8.unpack";
    require_gpu(q, what, "q");
    TORCH_CHECK(q.dim() == 2, what, ": expected 8-bit rows");
    check8(q, s, q.size(0), dim, q.size(0), what, "a");
    const int code = dtype_code(dtype, what);
    OnDevice on(q);
    Tensor out = fresh({q.size(0), dim}, dtype);
    check_rc(api().act8_unpack(q.const_data_ptr(), s.const_data_ptr(), q.size(0), dim, out.data_ptr(), code, on.stream),
             "z1_act8_unpack");
    return out;
}

// [q, s] or [q, s, qt, st]
std::vector<Tensor> weight8_pack(const Tensor& w, bool transposed) {
    const char* what = "linear8.pack_weight";
    require_gpu(w, what, "w");
    const Rows r = rows_of(w, what, "w");
    TORCH_CHECK(r.rows >= 1, what, ": expected at least one row");
    OnDevice on(w);
    Pair p = empty8(r.rows, r.dim, blocks_of(r.rows), what), t;
    if (transposed) t = empty8(r.dim, r.rows, blocks_of(r.dim), what);
    check_rc(api().weight8_pack(r.p, r.rows, r.dim, r.stride, r.dtype, p.q.data_ptr(), p.s.data_ptr(),
                                transposed ? t.q.data_ptr() : nullptr, transposed ? t.s.data_ptr() : nullptr, on.stream),
             "z1_weight8_pack");
    std::vector<Tensor> out{std::move(p.q), std::move(p.s)};
    if (transposed) {
        out.push_back(std::move(t.q));
        out.push_back(std::move(t.s));
    }
    return out;
}

// ------------------------------------------------------------------------------------------ products
Tensor product8(const Tensor& q, const Tensor& s, const Tensor& wq, const Tensor& ws, int64_t inner, at::ScalarType dtype) {
    const char* what = "linear8.matmul";
    require_gpu(q, what, "a");
    TORCH_CHECK(q.dim() == 2 && wq.dim() == 2, what, ": expected 8-bit rows and an 8-bit weight");
    const int64_t M = q.size(0), N = wq.size(0);
    check8(q, s, M, inner, M, what, "a");
    require_on(wq, q, what, "w");
    check8(wq, ws, N, inner, blocks_of(N), what, "w");
    const int code = dtype_code(dtype, what);
    OnDevice on(q);
    Tensor y = fresh({M, N}, dtype);
    const Workspace parts(api().product8_workspace(M, N, inner, code), "z1_product8_workspace");
    check_rc(api().product8(q.const_data_ptr(), s.const_data_ptr(), M, wq.const_data_ptr(), ws.const_data_ptr(), N, inner,
                            y.data_ptr(), code, parts.p, parts.floats, on.stream), "z1_product8");
    return y;
}

Tensor weight_grad8(const Tensor& dy_given, const Tensor& q, const Tensor& s, int64_t inner, at::ScalarType dtype) {
    const char* what = "linear8.weight_grad";
    require_gpu(dy_given, what, "dy");
    // a step's rows lie within 32 bits of its first
    const Tensor dy = dy_given.dim() == 2 && dy_given.stride(0) > (1 << 24) ? dy_given.contiguous() : dy_given;
    const Rows r = rows_of(dy, what, "dy");
    TORCH_CHECK(r.dtype == Z1_BF16, what, ": expected bf16 gradient rows");
    require_on(q, dy, what, "a");
    check8(q, s, r.rows, inner, r.rows, what, "a");
    const int code = dtype_code(dtype, what);
    OnDevice on(dy);
    Tensor dw = fresh({r.dim, inner}, dtype);
    const Workspace parts(api().weight_grad8_workspace(r.rows, r.dim, inner), "z1_weight_grad8_workspace");
    check_rc(api().weight_grad8(static_cast<const uint16_t*>(r.p), r.rows > 1 ? r.stride : r.dim, q.const_data_ptr(),
                                s.const_data_ptr(), r.rows, r.dim, inner, dw.data_ptr(), code, parts.p, parts.floats,
                                on.stream), "z1_weight_grad8");
    return dw;
}

// ------------------------------------------------------------------------------------------ CPU: refuse
void refuse_cpu(const c10::OperatorHandle& op, torch::jit::Stack*) {
    TORCH_CHECK(false, op.schema().name(), ": expected GPU tensors (there is no CPU path)");
}

const char* const kOps[] = {"norm_forward", "norm_backward", "act8_pack", "act8_unpack", "weight8_pack", "product8",
                            "weight_grad8"};

}  // namespace

TORCH_LIBRARY_FRAGMENT(yoco_z1, m) {
    m.def("norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps, bool center, bool y8, bool checkpoint) "
          "-> Tensor[]");
    m.def("norm_backward(Tensor dy, Tensor? x, Tensor? q, Tensor? s, Tensor? mean, Tensor rstd, Tensor? weight, "
          "bool center, bool need_dw, bool need_db, ScalarType? grad_dtype=None) -> Tensor[]");
    m.def("act8_pack(Tensor x) -> (Tensor, Tensor)");
    m.def("act8_unpack(Tensor q, Tensor s, int dim, ScalarType dtype) -> Tensor");
    m.def("weight8_pack(Tensor w, bool transposed) -> Tensor[]");
    m.def("product8(Tensor q, Tensor s, Tensor wq, Tensor ws, int inner, ScalarType dtype) -> Tensor");
    m.def("weight_grad8(Tensor dy, Tensor q, Tensor s, int inner, ScalarType dtype) -> Tensor");
}

TORCH_LIBRARY_IMPL(yoco_z1, CUDA, m) {
    m.impl("norm_forward", &norm_forward);
    m.impl("norm_backward", &norm_backward);
    m.impl("act8_pack", &act8_pack);
    m.impl("act8_unpack", &act8_unpack);
    m.impl("weight8_pack", &weight8_pack);
    m.impl("product8", &product8);
    m.impl("weight_grad8", &weight_grad8);
}

TORCH_LIBRARY_IMPL(yoco_z1, CPU, m) {
    for (const char* name : kOps) m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse_cpu>());
}

extern "C" {

/* Resolves the C ABI from the already loaded library at `path`: 0, or -1 when it is not loaded, -2 when a function is
 * missing (an older build of the ABI: the update's operators work without these). */
int z1t_init_block(const char* path) {
    void* h = dlopen(path, RTLD_NOW | RTLD_NOLOAD);
    if (!h) return -1;
    Api a{};
#define Z1T_RESOLVE(field)                                                        \
    a.field = reinterpret_cast<decltype(a.field)>(dlsym(h, "z1_" #field));        \
    if (!a.field) return -2;
    Z1T_RESOLVE(norm_forward)
    Z1T_RESOLVE(norm_backward)
    Z1T_RESOLVE(norm_backward_workspace)
    Z1T_RESOLVE(act8_columns)
    Z1T_RESOLVE(act8_scales)
    Z1T_RESOLVE(act8_pack)
    Z1T_RESOLVE(act8_unpack)
    Z1T_RESOLVE(weight8_pack)
    Z1T_RESOLVE(product8)
    Z1T_RESOLVE(product8_workspace)
    Z1T_RESOLVE(weight_grad8)
    Z1T_RESOLVE(weight_grad8_workspace)
    Z1T_RESOLVE(strerror)
#undef Z1T_RESOLVE
    g_api = a;
    g_api_ok = true;
    return 0;
}

}  // extern "C"
