// Bindings of the layer norm, gated recurrence and gated linear kernels
// (K9-K11): checks, outputs and workspaces; the kernels sit behind extern "C"
// launchers as in bindings.cpp.
//
// Each operator is one call: checks, launches and its autograd node, in C++ and
// of plain members: a small batch's training step is bound by the host, 62 us
// with torch's custom functions and their maps of saved values, 56 with these
// nodes, 44 for a bare product by two. It runs on its first argument's device and
// that device's current stream. Workspaces are allocated per call on that stream,
// so calls on several streams and captured graphs share none.

#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

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
extern "C" void gated_linear_cut(int, int, int, int, int, int*, int*, int*);
extern "C" int gated_linear_bias_parts(int, int, int, int);
extern "C" int64_t gated_linear_split_sums(int, int, int, int, int, int);
extern "C" int launch_gated_linear_bwd(int, const void*, const void*, const void*, const void*,
                                       void*, void*, void*, void*, float*, float*, int, int, int,
                                       hipStream_t);

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

constexpr int64_t MOST = std::numeric_limits<int>::max() / 2;
// Blocks of 256 threads, or columns of 64: a launch has less than 2^32 of them.
constexpr int64_t MOST_BLOCKS = (1 << 24) - 1;

hipStream_t stream() { return at::hip::getCurrentHIPStream().stream(); }

void check_first(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
    TORCH_CHECK_TYPE(t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat32,
                     name, " must be bf16 or fp32 (got ", t.scalar_type(), ")");
}

// An argument after the first one, on whose device it has to be.
void check(const Tensor& t, const char* name, const Tensor& first, torch::ScalarType dt,
           at::IntArrayRef shape) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == dt, name, " must be ", dt, ", got ", t.scalar_type());
    TORCH_CHECK(t.device() == first.device(), name, " must be on ", first.device());
}

// The values as they lie in the kernels' order, with a sign that is only noted applied.
Tensor contiguous(const Tensor& t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }
OptTensor contiguous(const OptTensor& t) { return t ? OptTensor(contiguous(*t)) : t; }

// An input that an eager graph computed, or a leaf whose gradient accumulator was
// made by an eager graph that still lives, hands its gradient to a node that keeps
// that graph's stream. Another stream joins a capture when it waits for one of its
// events, as a captured backward pass has it do, and is waited for at the pass's end;
// the default stream cannot, which ends the process. Refused here, while the forward
// pass is being captured.
void check_capture(std::initializer_list<OptTensor> inputs) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    (void)hipStreamIsCapturing(stream(), &status);
    if (status == hipStreamCaptureStatusNone) return;
    for (const auto& t : inputs) {
        if (!t || !t->requires_grad()) continue;
        const auto node = t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t)
                                       : t->grad_fn();
        if (!node) continue;
        const auto made_on = node->stream();
        TORCH_CHECK(!made_on || made_on->id() != 0,
                    "an eager graph of an input that this capture differentiates is alive on the "
                    "default stream: delete its outputs (or detach them) before the capture, and "
                    "compute inputs that are no leaves within it");
    }
}

// Whether torch's operations are being recorded or only simulated: by jit.trace,
// make_fx (before or after dispatch), fake or functional tensors. The allocation of
// an output would be recorded, and not the launch that fills it. Modes that only
// watch are none of these.
bool recorded() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Mode = c10::impl::TorchDispatchModeKey;
    if (torch::jit::tracer::isTracing()) return true;
    if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)) return true;
    if (!Modes::any_modes_set()) return false;
    return Modes::get_mode(Mode::PROXY) || Modes::get_mode(Mode::FAKE) ||
           Modes::get_mode(Mode::FUNCTIONAL);
}

// What a launch that torch's dispatcher does not see cannot serve: a recording, tensors
// without memory (a fake one that outlived its mode has a null pointer and is on GPU by
// its own account), and tangents, which the kernels would drop. Forward mode has a
// switch of its own: inference mode turns it off, no_grad does not. Both passes look: a
// recording or a tangent may begin with the outputs' gradients.
template <typename... T>
void check_modes(const T&... t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!recorded(), "the kernels' launches cannot be recorded (traced, "
                                             "exported or run on fake tensors): use the "
                                             "reference on CPU");
    const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const auto& v : std::initializer_list<OptTensor>{t...}) {
        if (!v || !v->defined()) continue;
        TORCH_CHECK_NOT_IMPLEMENTED(
            v->has_storage() && (v->numel() == 0 || v->storage().data() != nullptr),
            "a tensor without memory (fake, wrapped by a transform, or a zero that is only said "
            "to be one) has nothing for a kernel to read");
        TORCH_CHECK_NOT_IMPLEMENTED(!forward || !v->_fw_grad(0).defined(),
                                    "no forward-mode derivatives: use the reference on CPU");
    }
}

// Whether a gradient may be asked for: then a capture's inputs are looked at too.
template <typename... T>
bool tracked(const T&... t) {
    if (!torch::GradMode::is_enabled()) return false;
    const std::initializer_list<OptTensor> all{t...};
    bool any = false;
    for (const auto& v : all) any = any || (v && v->requires_grad());
    if (any) check_capture(all);
    return any;
}

// What the nodes below share: the lock that a node holds while it runs, saved
// tensors, and the edges to the inputs.
template <typename N, typename... T>
std::shared_ptr<N> node_of(const T&... inputs) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return node;
}

SavedVariable save(const OptTensor& t) { return SavedVariable(t ? *t : Tensor(), false); }
OptTensor optional(const SavedVariable& s) {
    Tensor t = s.unpack();
    return t.defined() ? OptTensor(t) : OptTensor();
}

// The kernels' gradients are not differentiable themselves: asked for with
// create_graph, they raise when someone differentiates them, and are no constants.
variable_list once(variable_list grads, const char* name) {
    if (!torch::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(name) + " is differentiable once", (int)grads.size());
    return (*error)(std::move(grads));
}

const void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }
int is_bf16(const Tensor& t) { return t.scalar_type() == torch::kBFloat16 ? 1 : 0; }

// ---- K9: layer norm --------------------------------------------------------
std::tuple<Tensor, Tensor> layer_norm_fwd(const Tensor& x, const Tensor& weight,
                                          const OptTensor& bias, const OptTensor& residual,
                                          double eps) {
    const int64_t dim = x.size(-1), rows = x.numel() / dim;
    auto y = torch::empty_like(x);
    Tensor s;
    if (residual) s = torch::empty_like(x);
    const int rc = launch_norm_fwd(is_bf16(x), x.data_ptr(), ptr(residual), weight.data_ptr(),
                                   ptr(bias), y.data_ptr(), residual ? s.data_ptr() : nullptr,
                                   rows, (int)dim, (float)eps, stream());
    TORCH_CHECK(rc == 0, "layer norm launch failed");
    return {y, s};
}

std::tuple<Tensor, Tensor> layer_norm_bwd(const Tensor& x, const OptTensor& residual,
                                          const Tensor& weight, const Tensor& dy,
                                          const OptTensor& ds, double eps) {
    const c10::DeviceGuard guard(x.device());
    const int64_t dim = x.size(-1), rows = x.numel() / dim;
    const int parts = norm_bwd_parts(is_bf16(x), rows, (int)dim);
    const int64_t stats = norm_bwd_stats(is_bf16(x), rows, (int)dim);
    auto dx = torch::empty_like(x);
    auto dwb = torch::empty({2, dim}, x.options());
    auto part = torch::empty({parts * 2 * dim + stats}, x.options().dtype(torch::kFloat32));
    float* sums = part.data_ptr<float>();
    const int rc = launch_norm_bwd(is_bf16(x), x.data_ptr(), ptr(residual), weight.data_ptr(),
                                   dy.data_ptr(), ptr(ds), dx.data_ptr(), sums,
                                   sums + parts * 2 * dim, dwb.data_ptr(), rows, (int)dim, parts,
                                   (float)eps, stream());
    TORCH_CHECK(rc == 0, "layer norm backward launch failed");
    return {dx, dwb};
}

struct LayerNormBackward : Node {
    SavedVariable x, weight, residual;
    double eps;
    std::string name() const override { return "LayerNormBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data();
        weight.reset_data();
        residual.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        check_modes(grads[0], grads.size() > 1 ? grads[1] : Tensor());
        const std::lock_guard<std::mutex> lock(mutex_);
        const Tensor in = x.unpack();
        const OptTensor res = optional(residual);
        const Tensor dy = grads[0].defined() ? contiguous(grads[0]) : torch::zeros_like(in);
        OptTensor ds;
        if (res && grads[1].defined()) ds = contiguous(grads[1]);
        auto [dx, dwb] = layer_norm_bwd(in, res, weight.unpack(), dy, ds, eps);
        return once({dx, should_compute_output(1) ? dwb[0] : Tensor(),
                     should_compute_output(2) ? dwb[1] : Tensor(), res ? dx : Tensor()},
                    "layer_norm");
    }
};

variable_list layer_norm(const Tensor& x, const Tensor& weight, const OptTensor& bias, double eps,
                         const OptTensor& residual) {
    check_modes(x, weight, bias, residual);
    check_first(x, "x");
    const c10::DeviceGuard guard(x.device());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x must have a last axis to normalise, got ",
                      x.sizes());
    const int64_t dim = x.size(-1);
    TORCH_CHECK(dim <= MOST_BLOCKS && x.numel() / dim <= MOST, "x is too large");
    check(weight, "weight", x, x.scalar_type(), {dim});
    if (bias) check(*bias, "bias", x, x.scalar_type(), {dim});
    if (residual) check(*residual, "residual", x, x.scalar_type(), x.sizes());
    const bool track = tracked(x, weight, bias, residual);
    const Tensor in = contiguous(x), w = contiguous(weight);
    const OptTensor b = contiguous(bias), r = contiguous(residual);
    auto [y, s] = layer_norm_fwd(in, w, b, r, eps);
    if (track) {
        auto node = node_of<LayerNormBackward>(in, w, b, r);
        node->x = save(in);
        node->weight = save(w);
        node->residual = save(r);
        node->eps = eps;
        torch::autograd::set_history(y, node);
        if (r) torch::autograd::set_history(s, node);
    }
    return residual ? variable_list{y, s} : variable_list{y};
}

// ---- K10: gated linear recurrence ------------------------------------------
std::tuple<Tensor, Tensor, Tensor> gated_recurrence_fwd(const Tensor& gates, const OptTensor& h0,
                                                        const OptTensor& lengths, bool keep) {
    const int64_t T = gates.size(0), B = gates.size(1), H = gates.size(2) / 3;
    const auto f32 = gates.options().dtype(torch::kFloat32);
    auto y = torch::empty({T, B, H}, gates.options());
    auto hT = torch::empty({B, H}, f32);
    const int64_t chunk = recurrence_chunk(), maps = recurrence_maps((int)T, (int)B, (int)H);
    Tensor kept, work;
    if (keep) kept = torch::empty({(T + chunk - 1) / chunk, B, H}, f32);
    if (maps) work = torch::empty({maps}, f32);
    const int rc = launch_recurrence_fwd(
        is_bf16(gates), gates.data_ptr(), (const float*)ptr(h0), (const int*)ptr(lengths),
        y.data_ptr(), hT.data_ptr<float>(), keep ? kept.data_ptr<float>() : nullptr,
        maps ? work.data_ptr<float>() : nullptr, (int)T, (int)B, (int)H, stream());
    TORCH_CHECK(rc == 0, "gated recurrence launch failed");
    return {y, hT, kept};
}

std::tuple<Tensor, Tensor> gated_recurrence_bwd(const Tensor& gates, const Tensor& kept,
                                                const OptTensor& lengths, const Tensor& dy,
                                                const OptTensor& dhT) {
    const c10::DeviceGuard guard(gates.device());
    const int64_t T = gates.size(0), B = gates.size(1), H = gates.size(2) / 3;
    const int64_t maps = recurrence_maps((int)T, (int)B, (int)H);
    auto dgates = torch::empty_like(gates);
    auto dh0 = torch::empty({B, H}, kept.options());
    Tensor work;
    if (maps) work = torch::empty({maps}, kept.options());
    const int rc = launch_recurrence_bwd(
        is_bf16(gates), gates.data_ptr(), kept.data_ptr<float>(), (const int*)ptr(lengths),
        dy.data_ptr(), (const float*)ptr(dhT), dgates.data_ptr(), dh0.data_ptr<float>(),
        maps ? work.data_ptr<float>() : nullptr, (int)T, (int)B, (int)H, stream());
    TORCH_CHECK(rc == 0, "gated recurrence backward launch failed");
    return {dgates, dh0};
}

struct GatedRecurrenceBackward : Node {
    SavedVariable gates, kept, lengths;
    std::string name() const override { return "GatedRecurrenceBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        gates.reset_data();
        kept.reset_data();
        lengths.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        check_modes(grads[0], grads[1]);
        const std::lock_guard<std::mutex> lock(mutex_);
        const Tensor g = gates.unpack();
        const Tensor dy = grads[0].defined()
            ? contiguous(grads[0])
            : torch::zeros({g.size(0), g.size(1), g.size(2) / 3}, g.options());
        OptTensor dhT;
        if (grads[1].defined()) dhT = contiguous(grads[1]);
        auto [dgates, dh0] = gated_recurrence_bwd(g, kept.unpack(), optional(lengths), dy, dhT);
        return once({dgates, should_compute_output(1) ? dh0 : Tensor()}, "gated_recurrence");
    }
};

std::tuple<Tensor, Tensor> gated_recurrence(const Tensor& gates, const OptTensor& h0,
                                            const OptTensor& lengths) {
    check_modes(gates, h0, lengths);
    check_first(gates, "gates");
    const c10::DeviceGuard guard(gates.device());
    TORCH_CHECK_VALUE(gates.dim() == 3 && gates.size(2) % 3 == 0,
                      "gates must be [T, B, 3H], got ", gates.sizes());
    const int64_t T = gates.size(0), B = gates.size(1), H = gates.size(2) / 3;
    // places in a step are counted in 32 bits, of the whole in 64
    TORCH_CHECK(T <= MOST && B <= MOST && H <= MOST && 3 * B * (H + 1) <= MOST,
                "gates is too large");
    if (h0) check(*h0, "h0 (the state is not rounded)", gates, torch::kFloat32, {B, H});
    if (lengths) check(*lengths, "lengths", gates, torch::kInt32, {B});
    const bool track = tracked(gates, h0);
    const Tensor g = contiguous(gates);
    const OptTensor h = contiguous(h0), n = contiguous(lengths);
    auto [y, hT, kept] = gated_recurrence_fwd(g, h, n, track);
    if (track) {
        auto node = node_of<GatedRecurrenceBackward>(g, h);
        node->gates = save(g);
        node->kept = save(kept);
        node->lengths = save(n);
        torch::autograd::set_history(y, node);
        torch::autograd::set_history(hT, node);
    }
    return {y, hT};
}

// ---- K11: gated linear unit ------------------------------------------------
struct LinearSizes {
    int M, K, F;
    std::vector<int64_t> out;
};

LinearSizes sizes_of(const Tensor& x, const Tensor& weight) {
    auto out = x.sizes().vec();
    int64_t M = 1;
    for (size_t i = 0; i + 1 < out.size(); ++i) M *= out[i];
    const int64_t K = out.back(), F = weight.size(0) / 2;
    out.back() = F;
    return {(int)M, (int)K, (int)F, out};
}

Tensor gated_linear_fwd(const Tensor& x, const Tensor& weight, const OptTensor& bias) {
    const auto n = sizes_of(x, weight);
    auto y = torch::empty(n.out, x.options());
    const int rc = launch_gated_linear_fwd(is_bf16(x), x.data_ptr(), weight.data_ptr(), ptr(bias),
                                           y.data_ptr(), n.M, n.K, n.F, stream());
    TORCH_CHECK(rc == 0, "gated linear launch failed");
    return y;
}

variable_list gated_linear_bwd(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                               const Tensor& dy, bool need_x, bool need_w, bool need_b) {
    const c10::DeviceGuard guard(x.device());
    const auto n = sizes_of(x, weight);
    const int half = is_bf16(x);
    const int64_t rows = need_b ? gated_linear_bias_parts(half, n.M, n.K, n.F) : 0;
    const int64_t splits = gated_linear_split_sums(half, n.M, n.K, n.F, need_x, need_w);
    auto dp = torch::empty({n.M, 2 * (int64_t)n.F}, x.options());
    auto part = torch::empty({splits + rows * 2 * n.F}, x.options().dtype(torch::kFloat32));
    Tensor dx, dw, db;
    if (need_x) dx = torch::empty_like(x);
    if (need_w) dw = torch::empty_like(weight);
    if (need_b) db = torch::empty({2 * (int64_t)n.F}, x.options());
    float* sums = part.data_ptr<float>();  // the splits', 16-byte pieces of them, first
    const int rc = launch_gated_linear_bwd(
        half, x.data_ptr(), weight.data_ptr(), ptr(bias), dy.data_ptr(), dp.data_ptr(),
        need_x ? dx.data_ptr() : nullptr, need_w ? dw.data_ptr() : nullptr,
        need_b ? db.data_ptr() : nullptr, sums + splits, sums, n.M, n.K, n.F, stream());
    TORCH_CHECK(rc == 0, "gated linear backward launch failed");
    return {dx, dw, db};
}

struct GatedLinearBackward : Node {
    SavedVariable x, weight, bias;
    std::string name() const override { return "GatedLinearBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data();
        weight.reset_data();
        bias.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        check_modes(grads[0]);
        const std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        return once(gated_linear_bwd(x.unpack(), weight.unpack(), optional(bias),
                                     contiguous(grads[0]), should_compute_output(0),
                                     should_compute_output(1), should_compute_output(2)),
                    "gated_linear");
    }
};

Tensor gated_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias) {
    check_modes(x, weight, bias);
    check_first(x, "x");
    const c10::DeviceGuard guard(x.device());
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must have a last axis");
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) % 2 == 0,
                      "weight must be [2F, K], got ", weight.sizes());
    const int64_t K = x.size(-1), F = weight.size(0) / 2;
    check(weight, "weight", x, x.scalar_type(), {2 * F, K});
    if (bias) check(*bias, "bias", x, x.scalar_type(), {2 * F});
    int64_t M = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) M *= x.size(i);
    // tiles of 64 by 64 at the least lie on one grid axis
    TORCH_CHECK(M <= MOST && K <= MOST && F <= MOST_BLOCKS, "x or weight is too large");
    const int64_t m = M / 64 + 1, k = K / 64 + 1, f = 2 * F / 64 + 1;
    TORCH_CHECK(m * f <= MOST_BLOCKS && m * k <= MOST_BLOCKS && k * f <= MOST_BLOCKS,
                "x or weight is too large");
    // a tile's places are counted in 32 bits from its first: 256 rows, or a gate's
    // row and its value's
    TORCH_CHECK((F + 256) * K <= MOST && 512 * F <= MOST, "weight is too large");
    const bool track = tracked(x, weight, bias);
    const Tensor in = contiguous(x), w = contiguous(weight);
    const OptTensor b = contiguous(bias);
    auto y = gated_linear_fwd(in, w, b);
    if (track) {
        auto node = node_of<GatedLinearBackward>(in, w, b);
        node->x = save(in);
        node->weight = save(w);
        node->bias = save(b);
        torch::autograd::set_history(y, node);
    }
    return y;
}

// (tile's rows, tile's columns, splits) of the products that make y and dp, dx, and dw.
std::vector<std::tuple<int, int, int>> gated_linear_cuts(bool half, int M, int K, int F) {
    std::vector<std::tuple<int, int, int>> cuts(3);
    for (int i = 0; i < 3; ++i) {
        auto& [bm, bn, splits] = cuts[i];
        gated_linear_cut(half, i, M, K, F, &bm, &bn, &splits);
    }
    return cuts;
}

}  // namespace

void bind_gated(py::module_& m) {
    m.def("layer_norm", &layer_norm, "layer norm, [y] or [y, x + residual] (K9)", py::arg("x"),
          py::arg("weight"), py::arg("bias"), py::arg("eps"), py::arg("residual"));
    m.def("gated_recurrence", &gated_recurrence, "gated linear recurrence, (y, hT) (K10)",
          py::arg("gates"), py::arg("h0"), py::arg("lengths"));
    m.def("gated_linear", &gated_linear, "gated linear unit (K11)", py::arg("x"),
          py::arg("weight"), py::arg("bias"));
    m.def("gated_linear_cuts", &gated_linear_cuts,
          "(tile rows, tile columns, splits) of K11's products for y and dp, dx, dw",
          py::arg("bf16"), py::arg("M"), py::arg("K"), py::arg("F"));
}
