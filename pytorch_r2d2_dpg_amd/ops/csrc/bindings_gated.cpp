// Bindings of the layer norm, gated recurrence and gated linear kernels
// (K9-K11): checks, outputs and workspaces; the kernels sit behind extern "C"
// launchers as in bindings.cpp.
//
// Every entry runs on its first argument's device and that device's current
// stream. Workspaces are allocated per call on that stream, so calls on several
// streams and captured graphs share none.

#include <torch/extension.h>
#include <torch/csrc/autograd/variable.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <hip/hip_runtime.h>

#include <limits>
#include <tuple>
#include <vector>

extern "C" int launch_norm_fwd(int, const void*, const void*, const void*, const void*, void*,
                               void*, int64_t, int, float, hipStream_t);
extern "C" int norm_bwd_parts(int, int64_t, int);
extern "C" int64_t norm_bwd_stats(int, int64_t, int);
extern "C" int launch_norm_bwd(int, const void*, const void*, const void*, const void*,
                               const void*, void*, float*, float*, void*, int64_t, int, int, float, hipStream_t);
extern "C" int recurrence_chunk();
extern "C" int64_t recurrence_maps(int, int, int);
extern "C" int launch_recurrence_fwd(int, const void*, const float*, const int*, void*, float*,
                                     float*, float*, int, int, int, hipStream_t);
extern "C" int launch_recurrence_bwd(int, const void*, const float*, const int*, const void*,
                                     const float*, void*, float*, float*, int, int, int,
                                     hipStream_t);
extern "C" int launch_gated_linear_fwd(int, const void*, const void*, const void*, void*, int,
                                       int, int, hipStream_t);
extern "C" int gated_linear_bias_parts(int, int, int, int);
extern "C" int64_t gated_linear_split_sums(int, int, int, int, int, int);
extern "C" int launch_gated_linear_bwd(int, const void*, const void*, const void*, const void*,
                                       void*, void*, void*, void*, float*, float*, int, int, int,
                                       hipStream_t);

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

constexpr int64_t MOST = std::numeric_limits<int>::max() / 2;

hipStream_t stream() { return at::hip::getCurrentHIPStream().stream(); }

// On the first argument's device, contiguous, of its type.
void check_first(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat32, name,
                " must be bf16 or fp32 (got ", t.scalar_type(), ")");
}

void check(const Tensor& t, const char* name, const Tensor& first, torch::ScalarType dt,
           at::IntArrayRef shape) {
    TORCH_CHECK(t.device() == first.device(), name, " must be on ", first.device());
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == dt, name, " must be ", dt, " (got ", t.scalar_type(), ")");
    TORCH_CHECK(t.sizes() == shape, name, " must have shape ", shape, " (got ", t.sizes(), ")");
}

const void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }
int is_bf16(const Tensor& t) { return t.scalar_type() == torch::kBFloat16 ? 1 : 0; }

// ---- K9: layer norm --------------------------------------------------------
std::tuple<Tensor, Tensor> layer_norm_fwd(Tensor x, Tensor weight, OptTensor bias,
                                          OptTensor residual, double eps) {
    check_first(x, "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "x must have a last axis to normalise");
    const c10::DeviceGuard guard(x.device());
    const int64_t dim = x.size(-1), rows = x.numel() / dim;
    TORCH_CHECK(dim <= MOST && rows <= MOST, "x is too large");
    check(weight, "weight", x, x.scalar_type(), {dim});
    if (bias) check(*bias, "bias", x, x.scalar_type(), {dim});
    if (residual) check(*residual, "residual", x, x.scalar_type(), x.sizes());
    auto y = torch::empty_like(x);
    Tensor s;
    if (residual) s = torch::empty_like(x);
    const int rc = launch_norm_fwd(is_bf16(x), x.data_ptr(), ptr(residual), weight.data_ptr(),
                                   ptr(bias), y.data_ptr(), residual ? s.data_ptr() : nullptr,
                                   rows, (int)dim, (float)eps, stream());
    TORCH_CHECK(rc == 0, "layer norm launch failed");
    return {y, s};
}

std::tuple<Tensor, Tensor> layer_norm_bwd(Tensor x, OptTensor residual, Tensor weight, Tensor dy,
                                          OptTensor ds, double eps) {
    check_first(x, "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, "x must have a last axis to normalise");
    const c10::DeviceGuard guard(x.device());
    const int64_t dim = x.size(-1), rows = x.numel() / dim;
    TORCH_CHECK(dim <= MOST && rows <= MOST, "x is too large");
    check(weight, "weight", x, x.scalar_type(), {dim});
    check(dy, "dy", x, x.scalar_type(), x.sizes());
    if (residual) check(*residual, "residual", x, x.scalar_type(), x.sizes());
    if (ds) check(*ds, "ds", x, x.scalar_type(), x.sizes());
    const int parts = norm_bwd_parts(is_bf16(x), rows, (int)dim);
    const auto f32 = x.options().dtype(torch::kFloat32);
    auto dx = torch::empty_like(x);
    auto dwb = torch::empty({2, dim}, x.options());
    auto part = torch::empty({parts, 2 * dim}, f32);
    auto stats = torch::empty({norm_bwd_stats(is_bf16(x), rows, (int)dim)}, f32);
    const int rc = launch_norm_bwd(is_bf16(x), x.data_ptr(), ptr(residual), weight.data_ptr(),
                                   dy.data_ptr(), ptr(ds), dx.data_ptr(), part.data_ptr<float>(),
                                   stats.data_ptr<float>(), dwb.data_ptr(), rows, (int)dim, parts,
                                   (float)eps, stream());
    TORCH_CHECK(rc == 0, "layer norm backward launch failed");
    return {dx, dwb};
}

// ---- K10: gated linear recurrence ------------------------------------------
std::tuple<Tensor, Tensor, Tensor> gated_recurrence_fwd(Tensor gates, OptTensor h0,
                                                        OptTensor lengths, bool keep) {
    check_first(gates, "gates");
    TORCH_CHECK(gates.dim() == 3 && gates.size(2) % 3 == 0, "gates must be [T, B, 3H]");
    const c10::DeviceGuard guard(gates.device());
    const int64_t T = gates.size(0), B = gates.size(1), H = gates.size(2) / 3;
    // places in a step are counted in 32 bits, of the whole in 64
    TORCH_CHECK(T <= MOST && B <= MOST && H <= MOST && 3 * B * (H + 1) <= MOST,
                "gates is too large");
    if (h0) check(*h0, "h0", gates, torch::kFloat32, {B, H});
    if (lengths) check(*lengths, "lengths", gates, torch::kInt32, {B});
    const auto f32 = gates.options().dtype(torch::kFloat32);
    auto y = torch::empty({T, B, H}, gates.options());
    auto hT = torch::empty({B, H}, f32);
    const int64_t chunk = recurrence_chunk();
    Tensor kept;
    if (keep) kept = torch::empty({(T + chunk - 1) / chunk, B, H}, f32);
    auto maps = torch::empty({recurrence_maps((int)T, (int)B, (int)H)}, f32);
    const int rc = launch_recurrence_fwd(
        is_bf16(gates), gates.data_ptr(), (const float*)ptr(h0), (const int*)ptr(lengths),
        y.data_ptr(), hT.data_ptr<float>(), keep ? kept.data_ptr<float>() : nullptr,
        maps.data_ptr<float>(), (int)T, (int)B, (int)H, stream());
    TORCH_CHECK(rc == 0, "gated recurrence launch failed");
    return {y, hT, kept};
}

std::tuple<Tensor, Tensor> gated_recurrence_bwd(Tensor gates, Tensor kept, OptTensor lengths,
                                                Tensor dy, OptTensor dhT) {
    check_first(gates, "gates");
    TORCH_CHECK(gates.dim() == 3 && gates.size(2) % 3 == 0, "gates must be [T, B, 3H]");
    const c10::DeviceGuard guard(gates.device());
    const int64_t T = gates.size(0), B = gates.size(1), H = gates.size(2) / 3;
    const int64_t chunk = recurrence_chunk();
    check(kept, "kept", gates, torch::kFloat32, {(T + chunk - 1) / chunk, B, H});
    check(dy, "dy", gates, gates.scalar_type(), {T, B, H});
    if (dhT) check(*dhT, "dhT", gates, torch::kFloat32, {B, H});
    if (lengths) check(*lengths, "lengths", gates, torch::kInt32, {B});
    auto dgates = torch::empty_like(gates);
    auto dh0 = torch::empty({B, H}, kept.options());
    auto maps = torch::empty({recurrence_maps((int)T, (int)B, (int)H)}, kept.options());
    const int rc = launch_recurrence_bwd(
        is_bf16(gates), gates.data_ptr(), kept.data_ptr<float>(), (const int*)ptr(lengths),
        dy.data_ptr(), (const float*)ptr(dhT), dgates.data_ptr(), dh0.data_ptr<float>(),
        maps.data_ptr<float>(), (int)T, (int)B, (int)H, stream());
    TORCH_CHECK(rc == 0, "gated recurrence backward launch failed");
    return {dgates, dh0};
}

// ---- K11: gated linear unit ------------------------------------------------
struct LinearSizes {
    int64_t M, K, F;
};

LinearSizes check_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias) {
    check_first(x, "x");
    TORCH_CHECK(x.dim() >= 1, "x must have a last axis");
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) % 2 == 0, "weight must be [2F, K]");
    const int64_t K = x.size(-1), F = weight.size(0) / 2;
    check(weight, "weight", x, x.scalar_type(), {2 * F, K});
    if (bias) check(*bias, "bias", x, x.scalar_type(), {2 * F});
    int64_t M = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) M *= x.size(i);
    // tiles of 64 by 64 at the least lie on one grid axis
    const int64_t m = M / 64 + 1, k = K / 64 + 1, f = 2 * F / 64 + 1;
    TORCH_CHECK(M <= MOST && K <= MOST && F <= MOST / 2 && m * f <= MOST && m * k <= MOST &&
                    k * f <= MOST, "x or weight is too large");
    return {M, K, F};
}

Tensor gated_linear_fwd(Tensor x, Tensor weight, OptTensor bias) {
    const auto n = check_linear(x, weight, bias);
    const c10::DeviceGuard guard(x.device());
    auto shape = x.sizes().vec();
    shape.back() = n.F;
    auto y = torch::empty(shape, x.options());
    const int rc = launch_gated_linear_fwd(is_bf16(x), x.data_ptr(), weight.data_ptr(), ptr(bias),
                                           y.data_ptr(), (int)n.M, (int)n.K, (int)n.F, stream());
    TORCH_CHECK(rc == 0, "gated linear launch failed");
    return y;
}

std::tuple<Tensor, Tensor, Tensor> gated_linear_bwd(Tensor x, Tensor weight, OptTensor bias,
                                                    Tensor dy, bool need_x, bool need_w,
                                                    bool need_b) {
    const auto n = check_linear(x, weight, bias);
    const c10::DeviceGuard guard(x.device());
    auto shape = x.sizes().vec();
    shape.back() = n.F;
    check(dy, "dy", x, x.scalar_type(), shape);
    const auto f32 = x.options().dtype(torch::kFloat32);
    auto dp = torch::empty({n.M, 2 * n.F}, x.options());
    Tensor dx, dw, db, part_db;
    const int M = (int)n.M, K = (int)n.K, F = (int)n.F, half = is_bf16(x);
    if (need_x) dx = torch::empty_like(x);
    if (need_w) dw = torch::empty_like(weight);
    if (need_b) {
        db = torch::empty({2 * n.F}, x.options());
        part_db = torch::empty({gated_linear_bias_parts(half, M, K, F), 2 * n.F}, f32);
    }
    auto part = torch::empty({gated_linear_split_sums(half, M, K, F, need_x, need_w)}, f32);
    const int rc = launch_gated_linear_bwd(
        half, x.data_ptr(), weight.data_ptr(), ptr(bias), dy.data_ptr(), dp.data_ptr(),
        need_x ? dx.data_ptr() : nullptr, need_w ? dw.data_ptr() : nullptr,
        need_b ? db.data_ptr() : nullptr, need_b ? part_db.data_ptr<float>() : nullptr,
        part.data_ptr<float>(), M, K, F, stream());
    TORCH_CHECK(rc == 0, "gated linear backward launch failed");
    return {dx, dw, db};
}

// A leaf whose gradient accumulator was made by a graph that still lives keeps
// that graph's stream. Where that is not the stream being captured, a captured
// backward pass would wait on a stream outside of the capture, which ends the
// process. Refused here, while the forward pass is being captured.
void check_capture(const std::vector<OptTensor>& inputs) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    (void)hipStreamIsCapturing(stream(), &status);
    if (status == hipStreamCaptureStatusNone) return;
    for (const auto& t : inputs) {
        if (!t.has_value() || !t->defined() || !t->is_leaf() || !t->requires_grad()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node) continue;
        const auto made_on = node->stream();
        TORCH_CHECK(!made_on || made_on->id() == at::hip::getCurrentHIPStream().id(),
                    "an eager graph of a leaf that this capture differentiates is alive: delete "
                    "its outputs (or detach them) before the capture");
    }
}

}  // namespace

void bind_gated(py::module_& m) {
    m.def("layer_norm_fwd", &layer_norm_fwd, "layer norm forward (K9)", py::arg("x"),
          py::arg("weight"), py::arg("bias"), py::arg("residual"), py::arg("eps"));
    m.def("layer_norm_bwd", &layer_norm_bwd, "layer norm backward (K9)");
    m.def("gated_recurrence_fwd", &gated_recurrence_fwd, "gated linear recurrence forward (K10)",
          py::arg("gates"), py::arg("h0"), py::arg("lengths"), py::arg("keep"));
    m.def("gated_recurrence_bwd", &gated_recurrence_bwd,
          "gated linear recurrence backward (K10)");
    m.def("gated_linear_fwd", &gated_linear_fwd, "gated linear unit forward (K11)");
    m.def("gated_linear_bwd", &gated_linear_bwd, "gated linear unit backward (K11)");
    m.def("check_capture", &check_capture,
          "refuse to capture a graph over leaves of a live eager graph");
}
