// torch_ops.cpp -- the float operators' calls from torch: checks of the
// arguments, outputs and workspaces, the launch on the tensors' device and
// current stream, and the autograd nodes.
//
// The kernels sit behind the C ABI (include/mi_b200.h); its entry points are
// given to bind() by address, so this file needs no GPU and no CUDA compiler.
// It is native because a call's own cost is what counts for single tokens: the
// same checks and nodes in Python took 15 to 25 us a call and 130 us a backward
// pass, more than their kernels.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <unordered_set>
#include <variant>

#include "../../include/mi_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

#define MI_ENTRIES(X)                                                                                       \
    X(mi_status_string) X(mi_selective_scan) X(mi_selective_scan_checkpoints) X(mi_selective_scan_workspace) \
    X(mi_selective_scan_backward) X(mi_selective_scan_step) X(mi_causal_conv1d) X(mi_causal_conv1d_backward) \
    X(mi_causal_conv1d_backward_workspace) X(mi_causal_conv1d_step) X(mi_rms_norm) X(mi_rms_norm_quant)      \
    X(mi_rms_norm_backward) X(mi_rms_norm_backward_workspace) X(mi_gated_recurrence)                         \
    X(mi_gated_recurrence_checkpoints) X(mi_gated_recurrence_backward)                                       \
    X(mi_gated_recurrence_workspace) X(mi_gated_recurrence_step) X(mi_layer_norm)                   \
    X(mi_layer_norm_backward) X(mi_layer_norm_backward_workspace) X(mi_sample_rows)

struct Entries {
#define X(name) decltype(&::name) name = nullptr;
    MI_ENTRIES(X)
#undef X
} mi;

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
#define X(name) mi.name = reinterpret_cast<decltype(&::name)>(at.at(#name));
    MI_ENTRIES(X)
#undef X
}

// ---------------------------------------------------------------------------
// arguments
// ---------------------------------------------------------------------------
int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MI_DT_F32;
        case at::kBFloat16: return MI_DT_BF16;
        case at::kHalf: return MI_DT_F16;
        default: return -1;
    }
}

void activation(const Tensor& t, const char* name) {
    TORCH_CHECK_TYPE(dtype_code(t) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}

void same_device(const Tensor& t, const Tensor& first, const char* name) {
    TORCH_CHECK_VALUE(t.device() == first.device(), name, " is on ", t.device(), ", the call's other tensors on ",
                      first.device());
}

// Checked last: the other refusals do not need a GPU.
void on_gpu(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor (there is no CPU path)");
}

// An activation of a call whose first one is `first`.
void like(const Tensor& t, const Tensor& first, at::IntArrayRef shape, const char* name) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == first.scalar_type(), name, " must be ", first.scalar_type(),
                     " like the call's other activations, got ", t.scalar_type());
    same_device(t, first, name);
    TORCH_CHECK_VALUE(t.size(-1) <= 1 || t.stride(-1) == 1, name, " must have a unit last stride");
}

// The kernels' grids: sequences, and a convolution's positions.
constexpr int64_t MAX_BATCH = 65535, MAX_CONV_L = 65535 * 128;

// The kernels count positions, channels and rows in 32 bits (offsets in 64).
void countable(const Tensor& t, const char* name) {
    for (const int64_t n : t.sizes()) TORCH_CHECK_VALUE(n <= int64_t(1) << 30, name, " is too long: ", t.sizes());
}

// After a kernel has written to it: saved copies of the tensor are stale.
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Contiguous and on a 16-byte boundary (a copy where it is not).
Tensor aligned(const Tensor& t) {
    Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

void fixed(const Tensor& t, const Tensor& first, at::IntArrayRef shape, at::ScalarType type, const char* name) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
    same_device(t, first, name);
}

// A contiguous operand of a fixed type (parameters, states), undefined if missing.
Tensor plain(const OptTensor& o, const Tensor& first, at::IntArrayRef shape, at::ScalarType type, const char* name) {
    if (!o.has_value()) return Tensor();
    fixed(*o, first, shape, type, name);
    return aligned(*o);
}

void in_place(const Tensor& t, const Tensor& first, at::IntArrayRef shape, at::ScalarType type, const char* name) {
    fixed(t, first, shape, type, name);
    TORCH_CHECK_VALUE(t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name,
                      " is advanced in place: it must be contiguous and start on a 16-byte boundary");
}

Tensor lengths_of(const OptTensor& o, const Tensor& first, int64_t batch) {
    if (!o.has_value()) return Tensor();
    TORCH_CHECK_VALUE(o->scalar_type() == at::kInt && o->dim() == 1 && o->size(0) == batch && o->device() == first.device(),
                      "lengths must be int32 [", batch, "] on ", first.device());
    return o->contiguous();
}

Tensor given(const OptTensor& o) { return o.has_value() ? *o : Tensor(); }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

template <typename... Ts>
bool any_requires_grad(const Ts&... ts) {
    return ((ts.defined() && ts.requires_grad()) || ...);
}

template <typename... Ts>
void no_grad_needed(const Ts&... ts) {
    TORCH_CHECK(!at::GradMode::is_enabled() || !any_requires_grad(ts...),
                "this call has no backward pass: make it under torch.no_grad()");
}

// No formulas for tangents: forward-mode differentiation would lose them.
template <typename... Ts>
void no_tangents(const Ts&... ts) {
    TORCH_CHECK_NOT_IMPLEMENTED(
        !((ts.defined() && ts._fw_grad(/*level=*/0).defined()) || ...) ||
            !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
        "the float operators have no forward-mode derivative: an argument is a dual tensor");
}

// A training call that is being captured.  Where an earlier autograd graph is
// alive over one of its leaves, the leaf's gradient is added on that graph's
// stream; if that is the default stream, which no capture can join, the
// captured backward pass would end the process.
void capturable(c10::ArrayRef<const Tensor*> inputs, c10::Device device) {
    using torch::autograd::Node;
    c10::cuda::CUDAGuard guard(device);
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    std::vector<std::shared_ptr<Node>> todo;
    std::unordered_set<Node*> seen;
    for (const Tensor* t : inputs) {
        if (!t->defined() || !t->requires_grad()) continue;
        todo.push_back(t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t));
    }
    while (!todo.empty()) {
        const std::shared_ptr<Node> node = todo.back();
        todo.pop_back();
        if (!node || !seen.insert(node.get()).second) continue;
        const auto on = node->stream();
        TORCH_CHECK(!on || !on->device().is_cuda() || on->id() != c10::cuda::getDefaultCUDAStream(on->device_index()).id(),
                    "a training step is being captured while an autograd graph made on the default stream is alive over "
                    "one of its leaves: drop that graph's results first");
        for (const auto& edge : node->next_edges()) todo.push_back(edge.function);
    }
}

// `t`, empty, as a result that depends on the others, so that they get their zero gradients
Tensor reached(Tensor t, c10::ArrayRef<const Tensor*> inputs) {
    if (!at::GradMode::is_enabled()) return t;
    for (const Tensor* o : inputs)
        if (o->defined() && o->requires_grad()) t = t + o->sum().to(t.scalar_type());
    return t;
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
int64_t st(const Tensor& t, int64_t d) { return t.defined() ? t.stride(d) : 0; }

// the stream that a call launches on, with its device made the current one
struct Place {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit Place(const Tensor& t)
        : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

void check(int rc, const char* name) {
    TORCH_CHECK(rc == MI_OK, name, " failed: status ", rc, " (", mi.mi_status_string(rc), ")");
}

Tensor workspace(int64_t bytes, const Tensor& like) {
    return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }

// an incoming gradient with a unit last stride
Tensor unit(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

Tensor empty_as(const Tensor& t, bool want = true) {
    return want && t.defined() ? at::empty(t.sizes(), t.options()) : Tensor();
}

// The gradients as backward() returns them: of first order.  Under create_graph
// (`create`: the backward pass was entered with gradients on) they depend on
// what the forward pass saved, whatever came in, so they get a node over all of
// that: a second backward pass that reaches it, by whichever way, is refused.
variable_list once(variable_list grads, bool create, const variable_list& saved, const variable_list& incoming) {
    using namespace torch::autograd;
    if (!create || !(any_variable_requires_grad(saved) || any_variable_requires_grad(incoming))) return grads;
    const auto refusal = std::make_shared<Error>("the float operators have gradients of first order only",
                                                 collect_next_edges(saved, incoming));
    for (auto& t : grads) {
        if (!t.defined()) continue;
        t = t.detach();
        set_history(t, refusal);
    }
    return grads;
}

// ---------------------------------------------------------------------------
// selective scan
// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B,
                                                const Tensor& C, const Tensor& D, const Tensor& z, const Tensor& bias,
                                                const Tensor& h0, const Tensor& lengths, bool softplus, bool keep) {
    const int64_t batch = u.size(0), L = u.size(1), d = u.size(2), N = A.size(1);
    Place place(u);
    Tensor y = at::empty({batch, L, d}, u.options()), h = floats({batch, d, N}, u), ckpt;
    if (keep) ckpt = floats({mi.mi_selective_scan_checkpoints(batch, L, d, N)}, u);
    Tensor ws = workspace(mi.mi_selective_scan_workspace(batch, L, d, N, 0), u);
    check(mi.mi_selective_scan(ptr(u), st(u, 0), st(u, 1), ptr(delta), st(delta, 0), st(delta, 1), fptr(A), ptr(B),
                               st(B, 0), st(B, 1), ptr(C), st(C, 0), st(C, 1), fptr(D), ptr(z), st(z, 0), st(z, 1),
                               fptr(bias), fptr(h0), static_cast<int32_t*>(ptr(lengths)), ptr(y), fptr(h), fptr(ckpt),
                               ptr(ws), batch, L, d, N, softplus, dtype_code(u), place.stream),
          "mi_selective_scan");
    return {y, h, ckpt};
}

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A,
                                 const Tensor& B, const Tensor& C, const OptTensor& D_, const OptTensor& z_,
                                 const OptTensor& bias_, const OptTensor& h0_, const OptTensor& lengths_, bool softplus) {
        const Tensor D = given(D_), z = given(z_), bias = given(bias_), h0 = given(h0_), lengths = given(lengths_);
        auto [y, h, ckpt] = scan_forward(u, delta, A, B, C, D, z, bias, h0, lengths, softplus, true);
        ctx->save_for_backward({u, delta, A, B, C, D, z, bias, lengths, ckpt});
        ctx->saved_data["softplus"] = softplus;
        int64_t need = 0;
        const Tensor* in[] = {&A, &B, &C, &D, &bias, &h0};
        for (int i = 0; i < 6; i++) need |= (int64_t)(in[i]->defined() && in[i]->requires_grad()) << i;
        ctx->saved_data["need"] = need;
        ctx->set_materialize_grads(false);
        return {y, h};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        if (!g[0].defined() && !g[1].defined()) return variable_list(11);
        const auto s = ctx->get_saved_variables();
        const Tensor &u = s[0], &delta = s[1], &A = s[2], &B = s[3], &C = s[4], &D = s[5], &z = s[6], &bias = s[7],
                     &lengths = s[8], &ckpt = s[9];
        const bool softplus = ctx->saved_data["softplus"].toBool();
        const int64_t need = ctx->saved_data["need"].toInt();
        const int64_t batch = u.size(0), L = u.size(1), d = u.size(2), N = A.size(1);
        const bool create = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        Place place(u);
        const Tensor dy = g[0].defined() ? unit(g[0]) : at::zeros({batch, L, d}, u.options());
        const Tensor dh = g[1].defined() ? aligned(g[1]) : Tensor();
        Tensor du = empty_as(u), ddelta = empty_as(delta), dz = empty_as(z);
        Tensor dA = empty_as(A, need & 1), dB = empty_as(B, need & 2), dC = empty_as(C, need & 4);
        Tensor dD = empty_as(D, need & 8), dbias = empty_as(bias, need & 16);
        Tensor dh0 = need & 32 ? floats({batch, d, N}, u) : Tensor();
        Tensor ws = workspace(mi.mi_selective_scan_workspace(batch, L, d, N, 1), u);
        check(mi.mi_selective_scan_backward(
                  ptr(dy), st(dy, 0), st(dy, 1), fptr(dh), ptr(u), st(u, 0), st(u, 1), ptr(delta), st(delta, 0),
                  st(delta, 1), fptr(A), ptr(B), st(B, 0), st(B, 1), ptr(C), st(C, 0), st(C, 1), fptr(D), ptr(z),
                  st(z, 0), st(z, 1), fptr(bias), static_cast<int32_t*>(ptr(lengths)), fptr(ckpt), ptr(du), ptr(ddelta),
                  fptr(dA), ptr(dB), ptr(dC), fptr(dD), ptr(dz), fptr(dbias), fptr(dh0), ptr(ws), batch, L, d, N,
                  softplus, dtype_code(u), place.stream),
              "mi_selective_scan_backward");
        return once({du, ddelta, dA, dB, dC, dD, dz, dbias, dh0, Tensor(), Tensor()}, create, s, g);
    }
};

struct ScanParams {
    Tensor A, D, bias, z;
    int64_t N;
};

// lead: {batch, L} or {batch}
ScanParams scan_arguments(at::IntArrayRef lead, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B,
                          const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& bias) {
    activation(u, "u");
    countable(u, "u");
    const int64_t d = u.size(-1);
    TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == d, "A must be [", d, ", states], got ", A.sizes());
    const int64_t N = A.size(1);
    TORCH_CHECK_VALUE(d > 0 && N >= 1 && N <= 64, "selective scans have 1 to 64 states and at least one channel: A is ",
                      A.sizes());
    c10::SmallVector<int64_t, 3> full(lead.begin(), lead.end()), states(lead.begin(), lead.end());
    full.push_back(d), states.push_back(N);
    like(u, u, full, "u");
    like(delta, u, full, "delta");
    like(B, u, states, "B");
    like(C, u, states, "C");
    if (z.has_value()) like(*z, u, full, "z");
    return {plain(A, u, {d, N}, at::kFloat, "A"), plain(D, u, {d}, at::kFloat, "D"),
            plain(bias, u, {d}, at::kFloat, "delta_bias"), given(z), N};
}

std::tuple<Tensor, Tensor> selective_scan(const Tensor& u, const Tensor& delta, const Tensor& A_, const Tensor& B,
                                          const Tensor& C, const OptTensor& D_, const OptTensor& z_,
                                          const OptTensor& bias_, bool softplus, const OptTensor& h0_,
                                          const OptTensor& lengths_) {
    no_tangents(u, delta, A_, B, C, given(D_), given(z_), given(bias_), given(h0_));
    TORCH_CHECK_VALUE(u.dim() == 3, "u must be [batch, L, channels], got ", u.sizes());
    const int64_t batch = u.size(0), L = u.size(1), d = u.size(2);
    const auto p = scan_arguments({batch, L}, u, delta, A_, B, C, D_, z_, bias_);
    const Tensor h0 = plain(h0_, u, {batch, d, p.N}, at::kFloat, "h0");
    const Tensor lengths = lengths_of(lengths_, u, batch);
    TORCH_CHECK_VALUE(batch <= MAX_BATCH, "at most ", MAX_BATCH, " sequences, got u ", u.sizes());
    on_gpu(u, "u");
    if (batch == 0 || L == 0)  // nothing to scan
        return {reached(u * 1, {&delta, &p.A, &B, &C, &p.D, &p.z, &p.bias, &h0}),
                h0.defined() ? h0 * 1 : at::zeros({batch, d, p.N}, u.options().dtype(at::kFloat))};
    if (at::GradMode::is_enabled() && any_requires_grad(u, delta, p.A, B, C, p.D, p.z, p.bias, h0)) {
        capturable({&u, &delta, &p.A, &B, &C, &p.D, &p.z, &p.bias, &h0}, u.device());
        const auto out = SelectiveScan::apply(u, delta, p.A, B, C, maybe(p.D), maybe(p.z), maybe(p.bias), maybe(h0),
                                              maybe(lengths), softplus);
        return {out[0], out[1]};
    }
    auto [y, h, ckpt] = scan_forward(u, delta, p.A, B, C, p.D, p.z, p.bias, h0, lengths, softplus, false);
    return {y, h};
}

Tensor selective_scan_step(const Tensor& h, const Tensor& u, const Tensor& delta, const Tensor& A_, const Tensor& B,
                           const Tensor& C, const OptTensor& D_, const OptTensor& z_, const OptTensor& bias_,
                           bool softplus) {
    TORCH_CHECK_VALUE(u.dim() == 2, "u must be [batch, channels], got ", u.sizes());
    const int64_t batch = u.size(0), d = u.size(1);
    no_tangents(h, u, delta, A_, B, C, given(D_), given(z_), given(bias_));
    no_grad_needed(h, u, delta, A_, B, C, given(D_), given(z_), given(bias_));
    const auto p = scan_arguments({batch}, u, delta, A_, B, C, D_, z_, bias_);
    in_place(h, u, {batch, d, p.N}, at::kFloat, "h");
    on_gpu(u, "u");
    Place place(u);
    Tensor y = at::empty({batch, d}, u.options());
    check(mi.mi_selective_scan_step(ptr(u), st(u, 0), ptr(delta), st(delta, 0), fptr(p.A), ptr(B), st(B, 0), ptr(C),
                                    st(C, 0), fptr(p.D), ptr(p.z), st(p.z, 0), fptr(p.bias), fptr(h), ptr(y), batch, d,
                                    p.N, softplus, dtype_code(u), place.stream),
          "mi_selective_scan_step");
    written(h);
    return y;
}

// ---------------------------------------------------------------------------
// causal convolution
// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& win,
                                        const Tensor& lengths, bool silu) {
    const int64_t batch = x.size(0), L = x.size(1), d = x.size(2), W = w.size(1);
    Place place(x);
    Tensor y = at::empty({batch, L, d}, x.options()), out = at::empty({batch, W - 1, d}, x.options());
    check(mi.mi_causal_conv1d(ptr(x), st(x, 0), st(x, 1), fptr(w), fptr(bias), ptr(win),
                              static_cast<int32_t*>(ptr(lengths)), ptr(y), ptr(out), batch, L, d, W, silu, dtype_code(x),
                              place.stream),
          "mi_causal_conv1d");
    return {y, out};
}

struct CausalConv1d : torch::autograd::Function<CausalConv1d> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias_,
                                 const OptTensor& win_, const OptTensor& lengths_, bool silu) {
        const Tensor bias = given(bias_), win = given(win_), lengths = given(lengths_);
        auto [y, out] = conv_forward(x, w, bias, win, lengths, silu);
        ctx->save_for_backward({x, w, bias, win, lengths});
        ctx->saved_data["silu"] = silu;
        int64_t need = 0;
        const Tensor* in[] = {&x, &w, &bias, &win};
        for (int i = 0; i < 4; i++) need |= (int64_t)(in[i]->defined() && in[i]->requires_grad()) << i;
        ctx->saved_data["need"] = need;
        ctx->set_materialize_grads(false);
        return {y, out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        if (!g[0].defined() && !g[1].defined()) return variable_list(6);
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &w = s[1], &bias = s[2], &win = s[3], &lengths = s[4];
        const bool silu = ctx->saved_data["silu"].toBool();
        const int64_t need = ctx->saved_data["need"].toInt();
        const int64_t batch = x.size(0), L = x.size(1), d = x.size(2), W = w.size(1);
        const bool create = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        Place place(x);
        const Tensor dy = g[0].defined() ? unit(g[0]) : at::zeros({batch, L, d}, x.options());
        const Tensor dout = g[1].defined() ? aligned(g[1]) : Tensor();
        Tensor dx = empty_as(x, need & 1), dw = empty_as(w, need & 2), dbias = empty_as(bias, need & 4);
        Tensor dwin = empty_as(win, need & 8);
        Tensor ws;
        if (dw.defined() || dbias.defined()) ws = workspace(mi.mi_causal_conv1d_backward_workspace(batch, L, d, W), x);
        check(mi.mi_causal_conv1d_backward(ptr(dy), st(dy, 0), st(dy, 1), ptr(dout), ptr(x), st(x, 0), st(x, 1), fptr(w),
                                           fptr(bias), ptr(win), static_cast<int32_t*>(ptr(lengths)), ptr(dx), fptr(dw),
                                           fptr(dbias), ptr(dwin), ptr(ws), batch, L, d, W, silu, dtype_code(x),
                                           place.stream),
              "mi_causal_conv1d_backward");
        return once({dx, dw, dbias, dwin, Tensor(), Tensor()}, create, s, g);
    }
};

// lead: {batch, L} or {batch}
std::tuple<Tensor, Tensor> conv_arguments(at::IntArrayRef lead, const Tensor& x, const Tensor& weight,
                                          const OptTensor& bias) {
    activation(x, "x");
    countable(x, "x");
    const int64_t d = x.size(-1);
    Tensor w = weight.dim() == 3 && weight.size(1) == 1 ? weight.squeeze(1) : weight;  // nn.Conv1d's [channels, 1, taps]
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == d && d > 0 && w.size(1) >= 2 && w.size(1) <= 4, "weight must be [", d,
                      ", taps] or [", d, ", 1, taps] with 2 to 4 taps, got ", weight.sizes());
    c10::SmallVector<int64_t, 3> full(lead.begin(), lead.end());
    full.push_back(d);
    like(x, x, full, "x");
    return {plain(w, x, {d, w.size(1)}, at::kFloat, "weight"), plain(bias, x, {d}, at::kFloat, "bias")};
}

std::tuple<Tensor, Tensor> causal_conv1d(const Tensor& x, const Tensor& weight, const OptTensor& bias_, bool silu,
                                         const OptTensor& win_, const OptTensor& lengths_) {
    no_tangents(x, weight, given(bias_), given(win_));
    TORCH_CHECK_VALUE(x.dim() == 3, "x must be [batch, L, channels], got ", x.sizes());
    const int64_t batch = x.size(0), L = x.size(1), d = x.size(2);
    const auto [w, bias] = conv_arguments({batch, L}, x, weight, bias_);
    const Tensor win = plain(win_, x, {batch, w.size(1) - 1, d}, x.scalar_type(), "win");
    const Tensor lengths = lengths_of(lengths_, x, batch);
    TORCH_CHECK_VALUE(batch <= MAX_BATCH && L <= MAX_CONV_L, "at most ", MAX_BATCH, " sequences of ", MAX_CONV_L,
                      " positions, got x ", x.sizes());
    on_gpu(x, "x");
    if (batch == 0 || L == 0)
        return {reached(x * 1, {&w, &bias, &win}),
                win.defined() ? win * 1 : at::zeros({batch, w.size(1) - 1, d}, x.options())};
    if (at::GradMode::is_enabled() && any_requires_grad(x, w, bias, win)) {
        capturable({&x, &w, &bias, &win}, x.device());
        const auto out = CausalConv1d::apply(x, w, maybe(bias), maybe(win), maybe(lengths), silu);
        return {out[0], out[1]};
    }
    return conv_forward(x, w, bias, win, lengths, silu);
}

Tensor causal_conv1d_step(const Tensor& x, const Tensor& weight, const Tensor& win, const OptTensor& bias_, bool silu) {
    TORCH_CHECK_VALUE(x.dim() == 2, "x must be [batch, channels], got ", x.sizes());
    const int64_t batch = x.size(0), d = x.size(1);
    no_tangents(x, weight, win, given(bias_));
    no_grad_needed(x, weight, win, given(bias_));
    const auto [w, bias] = conv_arguments({batch}, x, weight, bias_);
    in_place(win, x, {batch, w.size(1) - 1, d}, x.scalar_type(), "win");
    on_gpu(x, "x");
    Place place(x);
    Tensor y = at::empty({batch, d}, x.options());
    check(mi.mi_causal_conv1d_step(ptr(x), st(x, 0), fptr(w), fptr(bias), ptr(win), ptr(y), batch, d, w.size(1), silu,
                                   dtype_code(x), place.stream),
          "mi_causal_conv1d_step");
    written(win);
    return y;
}

// ---------------------------------------------------------------------------
// gated linear recurrence
// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> rec_forward(const Tensor& x, const Tensor& f, const Tensor& z, const Tensor& bias,
                                               const Tensor& h0, const Tensor& lengths, bool convex, bool keep) {
    const int64_t batch = x.size(0), L = x.size(1), d = x.size(2);
    Place place(x);
    Tensor y = at::empty({batch, L, d}, x.options()), h = floats({batch, d}, x), ckpt;
    if (keep) ckpt = floats({mi.mi_gated_recurrence_checkpoints(batch, L, d)}, x);
    Tensor ws = workspace(mi.mi_gated_recurrence_workspace(batch, L, d, 0, dtype_code(x)), x);
    check(mi.mi_gated_recurrence(ptr(x), st(x, 0), st(x, 1), ptr(f), st(f, 0), st(f, 1), ptr(z), st(z, 0), st(z, 1),
                                 fptr(bias), fptr(h0), static_cast<int32_t*>(ptr(lengths)), ptr(y), fptr(h), fptr(ckpt),
                                 ptr(ws), batch, L, d, convex, dtype_code(x), place.stream),
          "mi_gated_recurrence");
    return {y, h, ckpt};
}

struct GatedRecurrence : torch::autograd::Function<GatedRecurrence> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& f, const OptTensor& z_,
                                 const OptTensor& bias_, const OptTensor& h0_, const OptTensor& lengths_, bool convex) {
        const Tensor z = given(z_), bias = given(bias_), h0 = given(h0_), lengths = given(lengths_);
        auto [y, h, ckpt] = rec_forward(x, f, z, bias, h0, lengths, convex, true);
        ctx->save_for_backward({x, f, z, bias, lengths, ckpt});
        ctx->saved_data["convex"] = convex;
        ctx->saved_data["need"] = (int64_t)(bias.defined() && bias.requires_grad()) |
                                  (int64_t)(h0.defined() && h0.requires_grad()) << 1;
        ctx->set_materialize_grads(false);
        return {y, h};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        if (!g[0].defined() && !g[1].defined()) return variable_list(7);
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &f = s[1], &z = s[2], &bias = s[3], &lengths = s[4], &ckpt = s[5];
        const bool convex = ctx->saved_data["convex"].toBool();
        const int64_t need = ctx->saved_data["need"].toInt();
        const int64_t batch = x.size(0), L = x.size(1), d = x.size(2);
        const bool create = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        Place place(x);
        const Tensor dy = g[0].defined() ? unit(g[0]) : at::zeros({batch, L, d}, x.options());
        const Tensor dh = g[1].defined() ? aligned(g[1]) : Tensor();
        Tensor dx = empty_as(x), df = empty_as(f), dz = empty_as(z), dbias = empty_as(bias, need & 1);
        Tensor dh0 = need & 2 ? floats({batch, d}, x) : Tensor();
        Tensor ws = workspace(mi.mi_gated_recurrence_workspace(batch, L, d, 1, dtype_code(x)), x);
        check(mi.mi_gated_recurrence_backward(
                  ptr(dy), st(dy, 0), st(dy, 1), fptr(dh), ptr(x), st(x, 0), st(x, 1), ptr(f), st(f, 0), st(f, 1), ptr(z),
                  st(z, 0), st(z, 1), fptr(bias), static_cast<int32_t*>(ptr(lengths)), fptr(ckpt), ptr(dx), ptr(df),
                  ptr(dz), fptr(dbias), fptr(dh0), ptr(ws), batch, L, d, convex, dtype_code(x), place.stream),
              "mi_gated_recurrence_backward");
        return once({dx, df, dz, dbias, dh0, Tensor(), Tensor()}, create, s, g);
    }
};

// lead: {batch, L} or {batch}; returns the bias
Tensor rec_arguments(at::IntArrayRef lead, const Tensor& x, const Tensor& gate, const OptTensor& z, const OptTensor& bias) {
    activation(x, "x");
    countable(x, "x");
    const int64_t d = x.size(-1);
    TORCH_CHECK_VALUE(d > 0 && d <= 1 << 24, "x must have 1 to ", 1 << 24, " channels, got ", x.sizes());
    c10::SmallVector<int64_t, 3> full(lead.begin(), lead.end());
    full.push_back(d);
    like(x, x, full, "x");
    like(gate, x, full, "gate");
    if (z.has_value()) like(*z, x, full, "z");
    return plain(bias, x, {d}, at::kFloat, "gate_bias");
}

std::tuple<Tensor, Tensor> gated_recurrence(const Tensor& x, const Tensor& gate, const OptTensor& z_,
                                            const OptTensor& bias_, bool convex, const OptTensor& h0_,
                                            const OptTensor& lengths_) {
    const Tensor z = given(z_);
    no_tangents(x, gate, z, given(bias_), given(h0_));
    TORCH_CHECK_VALUE(x.dim() == 3, "x must be [batch, L, channels], got ", x.sizes());
    const int64_t batch = x.size(0), L = x.size(1), d = x.size(2);
    const Tensor bias = rec_arguments({batch, L}, x, gate, z_, bias_);
    const Tensor h0 = plain(h0_, x, {batch, d}, at::kFloat, "h0");
    const Tensor lengths = lengths_of(lengths_, x, batch);
    TORCH_CHECK_VALUE(batch <= MAX_BATCH, "at most ", MAX_BATCH, " sequences, got x ", x.sizes());
    on_gpu(x, "x");
    if (batch == 0 || L == 0)
        return {reached(x * 1, {&gate, &z, &bias, &h0}),
                h0.defined() ? h0 * 1 : at::zeros({batch, d}, x.options().dtype(at::kFloat))};
    if (at::GradMode::is_enabled() && any_requires_grad(x, gate, z, bias, h0)) {
        capturable({&x, &gate, &z, &bias, &h0}, x.device());
        const auto out = GatedRecurrence::apply(x, gate, maybe(z), maybe(bias), maybe(h0), maybe(lengths), convex);
        return {out[0], out[1]};
    }
    auto [y, h, ckpt] = rec_forward(x, gate, z, bias, h0, lengths, convex, false);
    return {y, h};
}

Tensor gated_recurrence_step(const Tensor& h, const Tensor& x, const Tensor& gate, const OptTensor& z_,
                             const OptTensor& bias_, bool convex) {
    const Tensor z = given(z_);
    TORCH_CHECK_VALUE(x.dim() == 2, "x must be [batch, channels], got ", x.sizes());
    const int64_t batch = x.size(0), d = x.size(1);
    no_tangents(h, x, gate, z, given(bias_));
    no_grad_needed(h, x, gate, z, given(bias_));
    const Tensor bias = rec_arguments({batch}, x, gate, z_, bias_);
    in_place(h, x, {batch, d}, at::kFloat, "h");
    TORCH_CHECK_VALUE(batch <= MAX_BATCH, "at most ", MAX_BATCH, " streams, got x ", x.sizes());
    on_gpu(x, "x");
    Place place(x);
    Tensor y = at::empty({batch, d}, x.options());
    if (batch == 0) return y;
    check(mi.mi_gated_recurrence_step(ptr(x), st(x, 0), ptr(gate), st(gate, 0), ptr(z), st(z, 0), fptr(bias), fptr(h),
                                      ptr(y), batch, d, convex, dtype_code(x), place.stream),
          "mi_gated_recurrence_step");
    written(h);
    return y;
}

// ---------------------------------------------------------------------------
// RMS norm
// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> rms_forward(const Tensor& x, const Tensor& w, double eps, const Tensor& r, bool keep) {
    const int64_t T = x.size(0), d = x.size(1);
    Place place(x);
    Tensor y = at::empty({T, d}, x.options()), total = r.defined() ? at::empty({T, d}, r.options()) : Tensor();
    Tensor rstd = keep ? floats({T}, x) : Tensor();
    check(mi.mi_rms_norm(ptr(x), st(x, 0), ptr(r), st(r, 0), fptr(w), ptr(y), ptr(total), fptr(rstd), T, d, eps,
                         dtype_code(x), dtype_code(r.defined() ? r : x), place.stream),
          "mi_rms_norm");
    return {y, total, rstd};
}

struct RMSNorm : torch::autograd::Function<RMSNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& r_, double eps) {
        const Tensor r = given(r_);
        auto [y, total, rstd] = rms_forward(x, w, eps, r, true);
        ctx->save_for_backward({total.defined() ? total : x, w, rstd});
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["need"] =
            (int64_t)x.requires_grad() | (int64_t)w.requires_grad() << 1 | (int64_t)(r.defined() && r.requires_grad()) << 2;
        ctx->set_materialize_grads(false);
        if (total.defined()) return {y, total};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &sum = s[0], &w = s[1], &rstd = s[2];
        const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
        const int64_t need = ctx->saved_data["need"].toInt();
        Tensor dtotal = g.size() > 1 ? g[1] : Tensor();
        if (!g[0].defined()) {
            if (!dtotal.defined()) return variable_list(4);
            return {need & 1 ? dtotal.to(type) : Tensor(), Tensor(), need & 4 ? dtotal : Tensor(), Tensor()};
        }
        const int64_t T = sum.size(0), d = sum.size(1);
        const bool create = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        Place place(sum);
        const Tensor dy = aligned(g[0]);
        if (dtotal.defined()) dtotal = aligned(dtotal);
        const bool same = sum.scalar_type() == type, want_r = need & 4;
        Tensor dx = need & 1 || (same && want_r) ? at::empty({T, d}, sum.options().dtype(type)) : Tensor();
        Tensor dr = want_r && !same ? at::empty({T, d}, sum.options()) : Tensor();
        Tensor dw = need & 2 ? floats({d}, sum) : Tensor();
        Tensor ws = need & 2 ? workspace(mi.mi_rms_norm_backward_workspace(T, d), sum) : Tensor();
        check(mi.mi_rms_norm_backward(ptr(dy), ptr(dtotal), ptr(sum), st(sum, 0), fptr(w), fptr(rstd), ptr(dx), ptr(dr),
                                      fptr(dw), ptr(ws), T, d, dtype_code(dy), dtype_code(sum), place.stream),
              "mi_rms_norm_backward");
        return once({need & 1 ? dx : Tensor(), dw, want_r ? (same ? dx : dr) : Tensor(), Tensor()}, create, s, g);
    }
};

struct Rows {
    Tensor x, w, r, b;
};

Rows norm_arguments(const Tensor& x, const Tensor& weight, const OptTensor& residual, const OptTensor& bias = {}) {
    no_tangents(x, weight, given(residual), given(bias));
    activation(x, "x");
    const int64_t d = x.dim() ? x.size(-1) : 0;
    TORCH_CHECK_VALUE(d >= 1 && d <= 16384, "rows of 1 to 16384 columns, got x ", x.sizes());
    if (residual.has_value()) {
        TORCH_CHECK_VALUE(residual->sizes() == x.sizes(), "residual must be ", x.sizes(), ", got ", residual->sizes());
        TORCH_CHECK_TYPE(residual->scalar_type() == x.scalar_type() || residual->scalar_type() == at::kFloat,
                         "residual must be ", x.scalar_type(), " or float32, got ", residual->scalar_type());
        same_device(*residual, x, "residual");
    }
    const Tensor w = plain(weight, x, {d}, at::kFloat, "weight"), b = plain(bias, x, {d}, at::kFloat, "bias");
    on_gpu(x, "x");
    TORCH_CHECK_VALUE(x.numel() / d <= int64_t(1) << 30, "x has too many rows: ", x.sizes());
    auto rows = [&](const Tensor& t) { return unit(t.dim() == 2 ? t : t.reshape({-1, d})); };
    return {rows(x), w, residual.has_value() ? rows(*residual) : Tensor(), b};
}

std::tuple<Tensor, OptTensor> rms_norm(const Tensor& x, const Tensor& weight, double eps, const OptTensor& residual) {
    const Rows a = norm_arguments(x, weight, residual);
    auto shaped = [&](const Tensor& t) { return x.dim() == 2 ? t : t.view(x.sizes()); };
    if (a.x.size(0) == 0)
        return {reached(x * 1, {&a.w, &a.r}), residual.has_value() ? OptTensor(reached(*residual * 1, {&a.x})) : OptTensor()};
    if (at::GradMode::is_enabled() && any_requires_grad(a.x, a.w, a.r)) {
        capturable({&a.x, &a.w, &a.r}, a.x.device());
        const auto out = RMSNorm::apply(a.x, a.w, maybe(a.r), eps);
        return {shaped(out[0]), out.size() > 1 ? OptTensor(shaped(out[1])) : OptTensor()};
    }
    auto [y, total, rstd] = rms_forward(a.x, a.w, eps, a.r, false);
    return {shaped(y), total.defined() ? OptTensor(shaped(total)) : OptTensor()};
}

std::tuple<Tensor, Tensor, OptTensor> rms_norm_quant(const Tensor& x, const Tensor& weight, double eps,
                                                     const OptTensor& residual) {
    no_grad_needed(x, weight, given(residual));
    const Rows a = norm_arguments(x, weight, residual);
    const int64_t T = a.x.size(0), d = a.x.size(1);
    Place place(a.x);
    Tensor q = at::empty({T, d}, x.options().dtype(at::kChar)), scale = floats({T}, x);
    Tensor total = a.r.defined() ? at::empty({T, d}, a.r.options()) : Tensor();
    if (T)
        check(mi.mi_rms_norm_quant(ptr(a.x), st(a.x, 0), ptr(a.r), st(a.r, 0), fptr(a.w), static_cast<int8_t*>(ptr(q)),
                                   fptr(scale), ptr(total), T, d, eps, dtype_code(x), dtype_code(a.r.defined() ? a.r : x),
                                   place.stream),
              "mi_rms_norm_quant");
    if (x.dim() == 2) return {q, scale, total.defined() ? OptTensor(total) : OptTensor()};
    return {q.view(x.sizes()), scale.view(x.sizes().slice(0, x.dim() - 1)),
            total.defined() ? OptTensor(total.view(x.sizes())) : OptTensor()};
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> ln_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps,
                                              const Tensor& r, bool keep) {
    const int64_t T = x.size(0), d = x.size(1);
    Place place(x);
    Tensor y = at::empty({T, d}, x.options()), total = r.defined() ? at::empty({T, d}, r.options()) : Tensor();
    Tensor stats = keep ? floats({T, 2}, x) : Tensor();
    check(mi.mi_layer_norm(ptr(x), st(x, 0), ptr(r), st(r, 0), fptr(w), fptr(b), ptr(y), ptr(total), fptr(stats), T, d,
                           eps, dtype_code(x), dtype_code(r.defined() ? r : x), place.stream),
          "mi_layer_norm");
    return {y, total, stats};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b_,
                                 const OptTensor& r_, double eps) {
        const Tensor b = given(b_), r = given(r_);
        auto [y, total, stats] = ln_forward(x, w, b, eps, r, true);
        ctx->save_for_backward({total.defined() ? total : x, w, stats});
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["need"] = (int64_t)x.requires_grad() | (int64_t)w.requires_grad() << 1 |
                                  (int64_t)(r.defined() && r.requires_grad()) << 2 |
                                  (int64_t)(b.defined() && b.requires_grad()) << 3;
        ctx->set_materialize_grads(false);
        if (total.defined()) return {y, total};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &sum = s[0], &w = s[1], &stats = s[2];
        const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
        const int64_t need = ctx->saved_data["need"].toInt();
        Tensor dtotal = g.size() > 1 ? g[1] : Tensor();
        if (!g[0].defined()) {
            if (!dtotal.defined()) return variable_list(5);
            return {need & 1 ? dtotal.to(type) : Tensor(), Tensor(), Tensor(), need & 4 ? dtotal : Tensor(), Tensor()};
        }
        const int64_t T = sum.size(0), d = sum.size(1);
        const bool create = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        Place place(sum);
        const Tensor dy = aligned(g[0]);
        if (dtotal.defined()) dtotal = aligned(dtotal);
        const bool same = sum.scalar_type() == type, want_r = need & 4;
        Tensor dx = need & 1 || (same && want_r) ? at::empty({T, d}, sum.options().dtype(type)) : Tensor();
        Tensor dr = want_r && !same ? at::empty({T, d}, sum.options()) : Tensor();
        Tensor dw = need & 2 ? floats({d}, sum) : Tensor(), db = need & 8 ? floats({d}, sum) : Tensor();
        Tensor ws = need & 10 ? workspace(mi.mi_layer_norm_backward_workspace(T, d), sum) : Tensor();
        check(mi.mi_layer_norm_backward(ptr(dy), ptr(dtotal), ptr(sum), st(sum, 0), fptr(w), fptr(stats), ptr(dx),
                                        ptr(dr), fptr(dw), fptr(db), ptr(ws), T, d, dtype_code(dy), dtype_code(sum),
                                        place.stream),
              "mi_layer_norm_backward");
        return once({need & 1 ? dx : Tensor(), dw, db, want_r ? (same ? dx : dr) : Tensor(), Tensor()}, create, s, g);
    }
};

std::tuple<Tensor, OptTensor> layer_norm(const Tensor& x, const Tensor& weight, const OptTensor& bias, double eps,
                                         const OptTensor& residual) {
    const Rows a = norm_arguments(x, weight, residual, bias);
    const Tensor& b = a.b;
    auto shaped = [&](const Tensor& t) { return x.dim() == 2 ? t : t.view(x.sizes()); };
    if (a.x.size(0) == 0)
        return {reached(x * 1, {&a.w, &b, &a.r}),
                residual.has_value() ? OptTensor(reached(*residual * 1, {&a.x})) : OptTensor()};
    if (at::GradMode::is_enabled() && any_requires_grad(a.x, a.w, b, a.r)) {
        capturable({&a.x, &a.w, &b, &a.r}, a.x.device());
        const auto out = LayerNorm::apply(a.x, a.w, maybe(b), maybe(a.r), eps);
        return {shaped(out[0]), out.size() > 1 ? OptTensor(shaped(out[1])) : OptTensor()};
    }
    auto [y, total, stats] = ln_forward(a.x, a.w, b, eps, a.r, false);
    return {shaped(y), total.defined() ? OptTensor(shaped(total)) : OptTensor()};
}

// ---------------------------------------------------------------------------
// the choice of a token
// ---------------------------------------------------------------------------
// A setting of all rows, or of each.
template <typename V>
struct Setting {
    Tensor rows;
    V value{};
    Setting(const std::variant<Tensor, V>& s, const Tensor& logits, at::ScalarType type, const char* name) {
        if (std::holds_alternative<Tensor>(s)) {
            fixed(std::get<Tensor>(s), logits, {logits.size(0)}, type, name);
            rows = std::get<Tensor>(s).contiguous();
        } else {
            value = std::get<V>(s);
        }
    }
};

std::tuple<Tensor, OptTensor> sample_rows(const Tensor& logits, const Tensor& u_, const std::variant<Tensor, double>& t_,
                                          const std::variant<Tensor, int64_t>& k_, const std::variant<Tensor, double>& p_,
                                          const std::variant<Tensor, double>& m_, const OptTensor& out, bool return_prob) {
    const auto rows_of = [](const auto& s) { return std::holds_alternative<Tensor>(s) ? std::get<Tensor>(s) : Tensor(); };
    const Tensor ts = rows_of(t_), ps = rows_of(p_), ms = rows_of(m_);
    no_tangents(logits, u_, ts, ps, ms);
    no_grad_needed(logits, u_, ts, ps, ms);
    activation(logits, "logits");
    TORCH_CHECK_VALUE(logits.dim() == 2 && logits.size(1) >= 1 && logits.size(1) <= 262144,
                      "logits must be [rows, 1 to 262144 tokens], got ", logits.sizes());
    const int64_t rows = logits.size(0), V = logits.size(1);
    like(logits, logits, {rows, V}, "logits");
    TORCH_CHECK_VALUE(rows <= 1 << 27, "logits has too many rows: ", logits.sizes());
    fixed(u_, logits, {rows}, at::kFloat, "u");
    const Tensor u = u_.contiguous();
    const Setting<double> t(t_, logits, at::kFloat, "temperature"), p(p_, logits, at::kFloat, "top_p"),
        m(m_, logits, at::kFloat, "min_p");
    const Setting<int64_t> k(k_, logits, at::kInt, "top_k");
    TORCH_CHECK_VALUE(t.rows.defined() || t.value >= 0, "temperature must be 0 (greedy) or more, got ", t.value);
    TORCH_CHECK_VALUE(k.rows.defined() || k.value >= 0, "top_k must be 0 (off) or more, got ", k.value);
    TORCH_CHECK_VALUE(p.rows.defined() || (p.value >= 0 && p.value <= 1), "top_p must be from 0 to 1, got ", p.value);
    TORCH_CHECK_VALUE(m.rows.defined() || (m.value >= 0 && m.value <= 1), "min_p must be from 0 to 1, got ", m.value);
    if (out.has_value()) {
        TORCH_CHECK_VALUE(out->sizes() == at::IntArrayRef({rows}) && out->is_contiguous(), "out must be contiguous [", rows,
                          "], got ", out->sizes());
        TORCH_CHECK_TYPE(out->scalar_type() == at::kLong, "out must be int64, got ", out->scalar_type());
        same_device(*out, logits, "out");
    }
    on_gpu(logits, "logits");
    Place place(logits);
    Tensor token = out.has_value() ? *out : at::empty({rows}, logits.options().dtype(at::kLong));
    Tensor prob = return_prob ? floats({rows}, logits) : Tensor();
    if (rows == 0) return {token, maybe(prob)};
    check(mi.mi_sample_rows(ptr(logits), st(logits, 0), fptr(u), fptr(t.rows), static_cast<int32_t*>(ptr(k.rows)),
                            fptr(p.rows), fptr(m.rows), t.value, std::min(k.value, V), p.value, m.value,
                            static_cast<int64_t*>(ptr(token)), fptr(prob), rows, V, dtype_code(logits), place.stream),
          "mi_sample_rows");
    if (out.has_value()) written(token);
    return {token, maybe(prob)};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
    m.def("bind", &bind);
    m.def("selective_scan", &selective_scan, free);
    m.def("selective_scan_step", &selective_scan_step, free);
    m.def("causal_conv1d", &causal_conv1d, free);
    m.def("causal_conv1d_step", &causal_conv1d_step, free);
    m.def("sample_rows", &sample_rows, free);
    m.def("layer_norm", &layer_norm, free);
    m.def("gated_recurrence", &gated_recurrence, free);
    m.def("gated_recurrence_step", &gated_recurrence_step, free);
    m.def("rms_norm", &rms_norm, free);
    m.def("rms_norm_quant", &rms_norm_quant, free);
}
