/*
 * The matrices' update (momentum, orthogonalisation, decay) as PyTorch operators of the namespace yoco_z1: schemas, CUDA (HIP)
 * kernels -- argument checks and calls of the C ABI on torch's current stream -- and CPU kernels that only raise.  Host code
 * only.  Results and workspaces come from torch's allocator, on the call's stream, so the operators may be captured in a graph
 * and used on any stream.  z1t_init_matrix(path) resolves the C ABI, as z1t_init does for the update's operators.
 */
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <dlfcn.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <utility>
#include <vector>

#include "yoco_z1.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Api {
    decltype(&::z1_orthogonalize) orthogonalize;
    decltype(&::z1_orthogonalize_workspace) orthogonalize_workspace;
    decltype(&::z1_muon_step) muon_step;
    decltype(&::z1_muon_workspace) muon_workspace;
    decltype(&::z1_strerror) strerror;
};

Api g_api{};
bool g_api_ok = false;

const Api& api() {
    TORCH_CHECK(g_api_ok, "yoco_z1: the matrices' operators are not bound: faster_yoco_amd.library is not imported, or the "
                         "selected build of libyoco_z1.so lacks them");
    return g_api;
}

void check_rc(int64_t rc, const char* what) {
    if (rc != 0) {
        const char* s = g_api.strerror ? g_api.strerror(static_cast<int>(rc)) : nullptr;
        TORCH_CHECK(false, "yoco_z1: ", what, " failed: ", s ? s : "?", " (code ", rc, ")");
    }
}

int dtype_code(at::ScalarType t, const char* what, const char* name) {
    switch (t) {
        case at::kFloat: return Z1_F32;
        case at::kBFloat16: return Z1_BF16;
        case at::kHalf: return Z1_F16;
        default: TORCH_CHECK(false, what, ": ", name, ": expected fp32, bf16 or fp16, got ", c10::toString(t));
    }
}

void require_gpu(const Tensor& t, const char* what, const char* name) {
    TORCH_CHECK(t.defined() && t.is_cuda(), what, ": ", name, ": expected a GPU tensor (there is no CPU path)");
}

std::vector<float> coefficients_of(at::ArrayRef<double> c, int64_t steps, const char* what) {
    TORCH_CHECK(steps >= 1 && steps <= 64, what, ": expected 1 to 64 steps, got ", steps);
    TORCH_CHECK(static_cast<int64_t>(c.size()) == 3 * steps, what, ": expected three coefficients a step, got ", c.size(),
                " for ", steps);
    std::vector<float> f(c.begin(), c.end());
    return f;
}

void check_sides(int64_t m, int64_t n, const char* what) {
    TORCH_CHECK(m <= Z1_MAX_SIDE && n <= Z1_MAX_SIDE, what, ": expected matrices with sides of 1 to ", Z1_MAX_SIDE, ", got ", m,
                " x ", n);
}

// A call's matrices run in launches whose workspace stays near 2 GiB.
constexpr int64_t kRoom = int64_t{1} << 31;
Tensor workspace_of(int64_t bytes) {
    if (bytes < 0) check_rc(bytes, "the matrices' workspace");
    return Tensor(at::detail::empty_cuda({bytes}, at::kByte, c10::Device(c10::DeviceType::CUDA), std::nullopt));
}

struct OnDevice {
    c10::DeviceGuard guard;
    void* stream;
    explicit OnDevice(const Tensor& t)
        : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

const char* const kMode = "the coefficients let the iterates leave their range (singular values of at most 1 must stay below 4), "
                          "or eps is not positive";

// x [count, m, n], rows of neighbouring elements
Tensor orthogonalize(const Tensor& x, int64_t steps, at::ArrayRef<double> coefficients, double eps, at::ScalarType dtype,
                     bool precise) {
    const char* what = "muon.orthogonalize";
    require_gpu(x, what, "x");
    TORCH_CHECK(x.dim() == 3, what, ": expected matrices [count, m, n], got ", x.dim(), " dimensions");
    const int64_t count = x.size(0), m = x.size(1), n = x.size(2);
    TORCH_CHECK((n <= 1 || x.stride(2) == 1) && (m <= 1 || x.stride(1) >= 0) && (count <= 1 || x.stride(0) >= 0), what,
                ": expected rows of neighbouring elements");
    const int code = dtype_code(x.scalar_type(), what, "x"), out_code = dtype_code(dtype, what, "dtype");
    const std::vector<float> c = coefficients_of(coefficients, steps, what);
    OnDevice on(x);
    Tensor out(at::detail::empty_cuda({count, m, n}, dtype, c10::Device(c10::DeviceType::CUDA), std::nullopt));
    if (out.numel() == 0) return out;
    check_sides(m, n, what);
    const int64_t one = api().orthogonalize_workspace(1, m, n, precise);
    if (one < 0) check_rc(one, "z1_orthogonalize_workspace");
    const int64_t most = std::max<int64_t>(1, std::min({count, int64_t{1} << 15, kRoom / std::max<int64_t>(1, one)}));
    const Tensor room = workspace_of(api().orthogonalize_workspace(most, m, n, precise));
    const auto* from = static_cast<const char*>(x.const_data_ptr());
    auto* to = static_cast<char*>(out.data_ptr());
    for (int64_t i = 0; i < count; i += most) {
        const int rc = api().orthogonalize(from + i * x.stride(0) * x.element_size(), x.stride(0), x.stride(1),
                                           std::min(most, count - i), m, n, code, to + i * m * n * out.element_size(),
                                           out_code, static_cast<int>(steps), c.data(), static_cast<float>(eps), precise,
                                           room.data_ptr(), room.numel(), on.stream);
        TORCH_CHECK(rc != Z1_E_MODE, what, ": ", kMode);
        check_rc(rc, "z1_orthogonalize");
    }
    return out;
}

void check_matrix(const Tensor& t, const Tensor& like, at::ScalarType dtype, const char* what, const char* name, size_t i) {
    require_gpu(t, what, name);
    TORCH_CHECK(t.device() == like.device(), what, ": ", name, "[", i, "] is on ", t.device(), ", the launch runs on ",
                like.device());
    TORCH_CHECK(t.scalar_type() == dtype && t.is_contiguous() && t.sizes() == like.sizes(), what, ": ", name, "[", i,
                "]: expected a contiguous ", c10::toString(dtype), " matrix of p's shape");
}

// A matrix's bytes, from its first one to its last one's end.
using Span = std::pair<const char*, const char*>;
Span span_of(const Tensor& t) {
    const auto* at = static_cast<const char*>(t.const_data_ptr());
    const int64_t rows = t.size(0) > 1 ? (t.size(0) - 1) * t.stride(0) : 0;
    return {at, at + (rows + t.size(1)) * t.element_size()};
}

// p = keep p - lr X, each matrix with its own
void muon_step_(at::TensorList p, at::TensorList g, at::TensorList momentum, at::TensorList p16, const OptTensor& factor,
                at::ArrayRef<double> lr, at::ArrayRef<double> keep, double mu, bool nesterov,
                int64_t steps, at::ArrayRef<double> coefficients, double eps, bool precise) {
    const char* what = "muon.step_";
    const size_t count = p.size();
    TORCH_CHECK(g.size() == count && momentum.size() == count && (p16.empty() || p16.size() == count) && lr.size() == count &&
                    keep.size() == count,
                what, ": expected as many gradients, momenta, copies and rates as matrices");
    const std::vector<float> c = coefficients_of(coefficients, steps, what);
    TORCH_CHECK(mu >= 0 && mu < 1, what, ": momentum must be in [0, 1)");
    if (count == 0) return;
    require_gpu(p[0], what, "p");
    std::vector<Span> written, read;
    for (size_t i = 0; i < count; ++i) {
        TORCH_CHECK(p[i].dim() == 2, what, ": p[", i, "]: expected a matrix, got ", p[i].dim(), " dimensions");
        require_gpu(p[i], what, "p");
        TORCH_CHECK(p[i].device() == p[0].device(), what, ": the matrices are on different devices");
        check_matrix(p[i], p[i], at::kFloat, what, "p", i);
        check_matrix(momentum[i], p[i], at::kFloat, what, "momentum", i);
        if (!p16.empty()) check_matrix(p16[i], p[i], at::kBFloat16, what, "p16", i);
        require_gpu(g[i], what, "g");
        TORCH_CHECK(g[i].device() == p[0].device() && g[i].sizes() == p[i].sizes() &&
                        (g[i].size(1) <= 1 || g[i].stride(1) == 1) && (g[i].size(0) <= 1 || g[i].stride(0) >= 0),
                    what, ": g[", i, "]: expected rows of neighbouring elements of p's shape, on its device");
        dtype_code(g[i].scalar_type(), what, "g");
        if (p[i].numel() == 0) continue;
        check_sides(p[i].size(0), p[i].size(1), what);
        written.push_back(span_of(p[i]));
        written.push_back(span_of(momentum[i]));
        if (!p16.empty()) written.push_back(span_of(p16[i]));
        read.push_back(span_of(g[i]));
    }
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
        TORCH_CHECK(written[i - 1].second <= written[i].first, what, ": tensors that are written overlap, or one is named twice");
    auto apart = [&](const Span& s) {                  // of all that is written
        auto next = std::lower_bound(written.begin(), written.end(), s);
        return (next == written.end() || s.second <= next->first) && (next == written.begin() || (--next)->second <= s.first);
    };
    for (const Span& s : read) TORCH_CHECK(apart(s), what, ": a gradient overlaps what is written");
    const float* f = nullptr;
    if (factor.has_value() && factor->defined()) {
        require_gpu(*factor, what, "factor");
        TORCH_CHECK(factor->scalar_type() == at::kFloat && factor->numel() == 1 && factor->device() == p[0].device(), what,
                    ": factor: expected one fp32 value on the matrices' device");
        f = static_cast<const float*>(factor->const_data_ptr());
        const auto* at = reinterpret_cast<const char*>(f);
        TORCH_CHECK(apart({at, at + sizeof(float)}), what, ": factor overlaps what is written");
    }
    OnDevice on(p[0]);

    // launches of one gradient type, as many matrices as may be named and as the workspace holds
    std::vector<std::vector<z1_matrix>> launches;
    std::vector<int> codes;
    int64_t bytes = 0;
    auto room_of = [&](const std::vector<z1_matrix>& list) {
        const int64_t n = api().muon_workspace(list.data(), static_cast<int>(list.size()), precise);
        if (n < 0) check_rc(n, "z1_muon_workspace");
        return n;
    };
    for (const at::ScalarType type : {at::kFloat, at::kBFloat16, at::kHalf}) {
        const size_t first = launches.size();
        for (size_t i = 0; i < count; ++i) {
            if (p[i].numel() == 0 || g[i].scalar_type() != type) continue;
            const z1_matrix x{g[i].const_data_ptr(), g[i].stride(0), static_cast<float*>(momentum[i].data_ptr()),
                              static_cast<float*>(p[i].data_ptr()),
                              p16.empty() ? nullptr : static_cast<uint16_t*>(p16[i].data_ptr()), p[i].size(0), p[i].size(1),
                              static_cast<float>(lr[i]), static_cast<float>(keep[i])};
            if (launches.size() == first || launches.back().size() == Z1_MAX_MATRICES) {
                launches.push_back({x});
                codes.push_back(dtype_code(type, what, "g"));
            } else {
                launches.back().push_back(x);
                if (room_of(launches.back()) > kRoom) {
                    launches.back().pop_back();
                    launches.push_back({x});
                    codes.push_back(codes.back());
                }
            }
            bytes = std::max(bytes, room_of(launches.back()));
        }
    }
    if (launches.empty()) return;
    const Tensor room = workspace_of(bytes);
    const z1_muon how{f, static_cast<float>(mu), nesterov, static_cast<int>(steps), c.data(), static_cast<float>(eps), precise};
    for (size_t i = 0; i < launches.size(); ++i) {
        const int rc = api().muon_step(launches[i].data(), static_cast<int>(launches[i].size()), codes[i], &how, room.data_ptr(),
                                       room.numel(), on.stream);
        TORCH_CHECK(rc != Z1_E_MODE, what, ": ", kMode);
        check_rc(rc, "z1_muon_step");
    }
}

// The step below autograd; then what it wrote counts as written there, as after torch's own in-place operators: a backward pass
// over values saved before it is refused.  (Tensors made in inference mode have no version.)
void muon_step_versions_(at::TensorList p, at::TensorList g, at::TensorList momentum, at::TensorList p16, const OptTensor& factor,
                         at::ArrayRef<double> lr, at::ArrayRef<double> keep, double mu, bool nesterov, int64_t steps,
                         at::ArrayRef<double> coefficients, double eps, bool precise) {
    static const auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("yoco_z1::muon_step_", "").typed<decltype(muon_step_)>();
    {
        at::AutoDispatchBelowADInplaceOrView below;
        op.call(p, g, momentum, p16, factor, lr, keep, mu, nesterov, steps, coefficients, eps, precise);
    }
    for (const at::TensorList& list : {p, momentum, p16})
        for (const Tensor& t : list)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void refuse_cpu(const c10::OperatorHandle& op, torch::jit::Stack*) {
    TORCH_CHECK(false, op.schema().name(), ": expected GPU tensors (there is no CPU path)");
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(yoco_z1, m) {
    m.def("orthogonalize(Tensor x, int steps, float[] coefficients, float eps, ScalarType dtype, bool precise) -> Tensor");
    m.def("muon_step_(Tensor(a!)[] p, Tensor[] g, Tensor(b!)[] momentum, Tensor(c!)[] p16, Tensor? factor, float[] lr, "
          "float[] keep, float mu, bool nesterov, int steps, float[] coefficients, float eps, "
          "bool precise) -> ()");
}

TORCH_LIBRARY_IMPL(yoco_z1, CUDA, m) {
    m.impl("orthogonalize", &orthogonalize);
    m.impl("muon_step_", &muon_step_);
}

TORCH_LIBRARY_IMPL(yoco_z1, ADInplaceOrView, m) { m.impl("muon_step_", &muon_step_versions_); }

TORCH_LIBRARY_IMPL(yoco_z1, CPU, m) {
    for (const char* name : {"orthogonalize", "muon_step_"})
        m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse_cpu>());
}

extern "C" {

/* Resolves the C ABI from the already loaded library at `path`: 0, or -1 when it is not loaded, -2 when a function is
 * missing (an older build of the ABI: the other operators work without these). */
int z1t_init_matrix(const char* path) {
    void* h = dlopen(path, RTLD_NOW | RTLD_NOLOAD);
    if (!h) return -1;
    Api a{};
#define Z1T_RESOLVE(field)                                                        \
    a.field = reinterpret_cast<decltype(a.field)>(dlsym(h, "z1_" #field));        \
    if (!a.field) return -2;
    Z1T_RESOLVE(orthogonalize)
    Z1T_RESOLVE(orthogonalize_workspace)
    Z1T_RESOLVE(muon_step)
    Z1T_RESOLVE(muon_workspace)
    Z1T_RESOLVE(strerror)
#undef Z1T_RESOLVE
    g_api = a;
    g_api_ok = true;
    return 0;
}

}  // extern "C"
