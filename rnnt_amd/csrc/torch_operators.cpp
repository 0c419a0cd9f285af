// torch_operators.cpp — the compiled PyTorch binding of the prediction network's and the decoder's operators (part of
// rnnt_amd/lib/librnnt_amd_torch.so, beside torch_binding.cpp): argument checks, buffers from torch's caching allocator,
// the launch stream from torch's current HIP stream, the backward passes as C++ autograd nodes, and the C ABI of
// include/rnnt_mi355.h underneath.  No kernels and no arithmetic here.
//
// A call on label sequences runs tens of microseconds on the device, and a single-token call a few: the checks are
// made here, once, rather than in Python.  Shapes and types are refused with ValueError / TypeError before the device is
// looked at; tensors that are not on a ROCm device with RuntimeError, as everywhere in this package.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>

#include "../../include/rnnt_mi355.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

void check_status(rnntStatus_t s, const char *what) {
    TORCH_CHECK(s == RNNT_STATUS_SUCCESS, what, ": ", rnntGetStatusString(s), " (rnntStatus_t=", (int)s, ")");
}

rnntDtype_t dtype_code(const Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kFloat: return RNNT_DTYPE_F32;
        case at::kBFloat16: return RNNT_DTYPE_BF16;
        case at::kHalf: return RNNT_DTYPE_F16;
        default: TORCH_CHECK_TYPE(false, name, " must be torch.float32, torch.bfloat16 or torch.float16");
    }
}

Tensor given(const MaybeTensor &t) { return t.has_value() ? *t : Tensor(); }

void check_on_device(const Tensor &x, const char *op) {
    TORCH_CHECK(x.is_cuda(), "rnnt_amd.", op, " computes on MI355X (ROCm device tensors) only; got a tensor on ", x.device(),
                ". There is no CPU path or PyTorch fallback in this package.");
}
void check_same_device(const Tensor &t, const Tensor &x, const char *name) {
    TORCH_CHECK(!t.defined() || t.device() == x.device(), name, " must be on ", x.device(), ", got ", t.device());
}
void check_f32(const Tensor &t, at::IntArrayRef shape, const char *name) {
    if (!t.defined()) return;
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, " must be torch.float32");
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
}
void check_lengths(const Tensor &t, int64_t batch) {
    if (!t.defined()) return;
    TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, "lengths must be torch.int32");
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == batch && t.is_contiguous(), "lengths must be a contiguous [batch] tensor");
}
// rows whose elements are adjacent, at any distance from each other
Tensor rows_of(const Tensor &t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

void *stream_of(const Tensor &x) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.get_device()).stream(); }

template <typename T>
T *pointer(const Tensor &t) {
    return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}
Tensor bytes(size_t n, const Tensor &like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

bool wants_grad(std::initializer_list<const Tensor *> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : inputs)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// There are no forward-mode derivatives here.  An input with a tangent need not require grad, and then no autograd function would
// refuse it: the tangent would be lost without an error.
void check_tangents(std::initializer_list<const Tensor *> inputs, const char *op) {
    for (const Tensor *t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), "rnnt_amd.", op, " has no forward-mode derivative");
}

// Calls without any derivative.  `tensors`: what the call reads, and the buffer it writes: a buffer that autograd follows would keep the
// history of the values that are gone.
void check_no_grad(std::initializer_list<const Tensor *> tensors, const char *op) {
    check_tangents(tensors, op);
    TORCH_CHECK(!wants_grad(tensors), "rnnt_amd.", op, " is for decoding and has no backward: call it under torch.no_grad()");
}

// A call that a graph captures, on a leaf that an eager graph made on the default stream still holds: the backward pass would
// wait for the default stream inside the capture, which ends the process rather than raising.  `inputs` are the caller's own
// tensors, before any is laid out: the copy of a leaf is no leaf.
void check_capture(std::initializer_list<const Tensor *> inputs, const char *op) {
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor *t : inputs) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!accumulator) continue;
        const auto stream = accumulator->stream();
        TORCH_CHECK(!stream || stream->id() != 0 || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None,
                    "rnnt_amd.", op, " cannot be captured while a graph of an eager call on the default stream holds the same leaf: "
                    "drop that call's results, make it on another stream, or capture under torch.no_grad() where no backward pass is captured");
    }
}

// The gradients as they leave a backward node: differentiating them again raises (there is no second derivative here).
variable_list once(variable_list grads, const char *op) {
    if (!at::GradMode::is_enabled()) return grads;
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string("rnnt_amd.") + op + " cannot be differentiated twice",
                                                                (int64_t)grads.size());
    variable_list out;
    for (auto &g : grads) {
        if (g.defined()) g.requires_grad_(true);
        out.push_back(g);
    }
    return (*node)(std::move(out));
}

int as_int(int64_t v, const char *name) {
    TORCH_CHECK_VALUE(v < (1ll << 31), name, " is too large");
    return (int)v;
}

// ---- token embedding -----------------------------------------------------------------------------------------------
Tensor embed_forward(const Tensor &tokens, const Tensor &weight, double scale) {
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(weight.device());
    auto shape = tokens.sizes().vec();
    shape.push_back(weight.size(1));
    Tensor out = at::empty(shape, weight.options());
    check_status(rnnt_token_embedding_forward(tokens.data_ptr(), tokens.scalar_type() == at::kLong, tokens.numel(), weight.data_ptr(),
                                              weight.size(0) == 1 ? weight.size(1) : weight.stride(0), (int)weight.size(0),
                                              (int)weight.size(1), (float)scale, dtype_code(weight, "weight"), out.data_ptr(),
                                              stream_of(weight)),
                 "rnnt_token_embedding_forward");
    return out;
}

class EmbedFunction : public torch::autograd::Function<EmbedFunction> {
public:
    static Tensor forward(AutogradContext *ctx, const Tensor &tokens, const Tensor &weight, double scale, int64_t padding) {
        ctx->save_for_backward({tokens});
        ctx->saved_data["vocab"] = weight.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        return embed_forward(tokens, weight, scale);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const Tensor tokens = ctx->get_saved_variables()[0];
        const int64_t dim = grads[0].size(-1), n = tokens.numel(), vocab = ctx->saved_data["vocab"].toInt();
        Tensor g = grads[0].reshape({n, dim});
        if (dim > 1 && g.stride(1) != 1) g = g.contiguous();
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(g.device());
        Tensor dweight = at::empty({vocab, dim}, g.options());
        size_t need = 0;
        check_status(rnnt_token_embedding_workspace_size(n, (int)vocab, (int)dim, &need), "rnnt_token_embedding_workspace_size");
        const Tensor ws = need ? bytes(need, g) : Tensor();
        check_status(rnnt_token_embedding_backward(tokens.data_ptr(), tokens.scalar_type() == at::kLong, n, g.data_ptr(), g.stride(0),
                                                   (int)vocab, (int)dim, (float)ctx->saved_data["scale"].toDouble(),
                                                   ctx->saved_data["padding"].toInt(), dtype_code(g, "grad"), dweight.data_ptr(),
                                                   pointer<void>(ws), stream_of(g)),
                     "rnnt_token_embedding_backward");
        return once({Tensor(), dweight, Tensor(), Tensor()}, "token_embedding");
    }
};

Tensor token_embedding_op(const Tensor &tokens_in, const Tensor &weight_in, double scale, int64_t padding) {
    TORCH_CHECK_TYPE(tokens_in.scalar_type() == at::kInt || tokens_in.scalar_type() == at::kLong,
                     "tokens must be torch.int32 or torch.int64");
    dtype_code(weight_in, "weight");
    TORCH_CHECK_VALUE(weight_in.dim() == 2 && weight_in.size(0) >= 1 && weight_in.size(1) >= 1, "weight must be a non-empty [vocab, dim] tensor");
    TORCH_CHECK_VALUE(tokens_in.numel() >= 1, "tokens must not be empty");
    TORCH_CHECK_VALUE(padding >= -1 && padding < weight_in.size(0), "padding_idx must be None or a row of weight");
    TORCH_CHECK_VALUE(std::isfinite((float)scale), "scale must be finite in fp32");
    size_t need = 0;
    TORCH_CHECK_VALUE(weight_in.size(0) < (1ll << 31) && weight_in.size(1) < (1ll << 31) &&
                          rnnt_token_embedding_workspace_size(tokens_in.numel(), (int)weight_in.size(0), (int)weight_in.size(1), &need) ==
                              RNNT_STATUS_SUCCESS,
                      "too many tokens (at most 2^30), or too large a weight (2^26 rows, 2^21 columns) for one call");
    check_tangents({&weight_in}, "token_embedding");
    check_on_device(weight_in, "token_embedding");
    check_same_device(tokens_in, weight_in, "tokens");
    check_capture({&weight_in}, "token_embedding");
    const Tensor tokens = tokens_in.contiguous();
    const Tensor weight = weight_in.size(1) == 1 || weight_in.stride(1) == 1 ? weight_in : weight_in.contiguous();
    const bool ordered = weight.size(0) == 1 || weight.stride(0) >= weight.size(1);  // (an expanded weight is laid out first)
    const Tensor w = ordered ? weight : weight.contiguous();
    if (!wants_grad({&w})) return embed_forward(tokens, w, scale);
    return EmbedFunction::apply(tokens, w, scale, padding);
}

// ---- causal convolution -----------------------------------------------------------------------------------------------
rnntConv conv_args(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &initial, const Tensor &lengths, bool silu) {
    rnntConv c = {};
    c.batch = (int)x.size(0);
    c.length = x.dim() == 3 ? (int)x.size(1) : 1;
    c.dim = (int)x.size(-1);
    c.width = (int)weight.size(1);
    c.silu = silu;
    c.dtype = dtype_code(x, "x");
    c.x = x.data_ptr();
    c.x_batch = x.stride(0);
    c.x_time = x.dim() == 3 ? x.stride(1) : 0;
    c.weight = pointer<float>(weight);
    c.bias = pointer<float>(bias);
    c.initial_state = pointer<void>(initial);
    c.lengths = pointer<int>(lengths);
    c.stream = stream_of(x);
    return c;
}

std::tuple<Tensor, Tensor> conv_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &initial,
                                        const Tensor &lengths, bool silu) {
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    rnntConv c = conv_args(x, weight, bias, initial, lengths, silu);
    Tensor y = at::empty(x.sizes(), x.options());
    Tensor final_state = at::empty({x.size(0), weight.size(1) - 1, x.size(2)}, x.options());
    c.y = y.data_ptr();
    c.final_state = final_state.data_ptr();
    check_status(rnnt_causal_conv_forward(&c), "rnnt_causal_conv_forward");
    return {y, final_state};
}

class ConvFunction : public torch::autograd::Function<ConvFunction> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const MaybeTensor &bias,
                                 const MaybeTensor &initial, const MaybeTensor &lengths, bool silu) {
        auto out = conv_forward(x, weight, given(bias), given(initial), given(lengths), silu);
        ctx->save_for_backward({x, weight, given(bias), given(initial), given(lengths)});
        ctx->saved_data["silu"] = silu;
        ctx->set_materialize_grads(false);
        return {std::get<0>(out), std::get<1>(out)};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &initial = saved[3];
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
        rnntConv c = conv_args(x, weight, bias, initial, saved[4], ctx->saved_data["silu"].toBool());
        const Tensor gy = grads[0].defined() ? rows_of(grads[0]) : at::zeros(x.sizes(), x.options());
        const Tensor gf = grads[1].defined() ? grads[1].contiguous() : Tensor();
        Tensor dx = at::empty(x.sizes(), x.options()), dw = at::empty(weight.sizes(), weight.options());
        Tensor db = bias.defined() ? at::empty(bias.sizes(), bias.options()) : Tensor();
        Tensor di = initial.defined() ? at::empty(initial.sizes(), initial.options()) : Tensor();
        size_t need = 0;
        check_status(rnnt_causal_conv_workspace_size(c.batch, c.length, c.dim, c.width, &need), "rnnt_causal_conv_workspace_size");
        const Tensor ws = bytes(need, x);
        c.grad_y = gy.data_ptr();
        c.grad_y_batch = gy.stride(0);
        c.grad_y_time = gy.stride(1);
        c.grad_final = pointer<void>(gf);
        c.grad_x = dx.data_ptr();
        c.grad_weight = pointer<float>(dw);
        c.grad_bias = pointer<float>(db);
        c.grad_initial = pointer<void>(di);
        c.workspace = ws.data_ptr();
        check_status(rnnt_causal_conv_backward(&c), "rnnt_causal_conv_backward");
        return once({dx, dw, db, di, Tensor(), Tensor()}, "causal_conv");
    }
};

void check_conv_weights(const Tensor &weight, const Tensor &bias, int64_t dim) {
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) == dim && weight.size(1) >= 2 && weight.size(1) <= 4,
                      "weight must be [dim, width] with a width of 2, 3 or 4");
    check_f32(weight, weight.sizes(), "weight");
    check_f32(bias, {dim}, "bias");
}
void check_conv_state(const Tensor &state, const Tensor &x, int64_t width, const char *name) {
    if (!state.defined()) return;
    TORCH_CHECK_TYPE(state.scalar_type() == x.scalar_type(), name, " must have x's type");
    TORCH_CHECK_VALUE(state.dim() == 3 && state.size(0) == x.size(0) && state.size(1) == width - 1 && state.size(2) == x.size(-1), name,
                      " must be [batch, width - 1, dim]");
}

std::tuple<Tensor, Tensor> causal_conv_op(const Tensor &x_in, const Tensor &weight_in, const MaybeTensor &bias_in,
                                          const MaybeTensor &initial_in, const MaybeTensor &lengths_in, bool silu) {
    dtype_code(x_in, "x");
    TORCH_CHECK_VALUE(x_in.dim() == 3 && x_in.numel() >= 1, "x must be a non-empty [batch, length, dim] tensor");
    Tensor bias = given(bias_in), initial = given(initial_in);
    const Tensor lengths = given(lengths_in);
    check_conv_weights(weight_in, bias, x_in.size(2));
    check_conv_state(initial, x_in, weight_in.size(1), "initial_state");
    check_lengths(lengths, x_in.size(0));
    size_t need = 0;
    TORCH_CHECK_VALUE(x_in.numel() / x_in.size(2) < (1ll << 31) && x_in.size(2) < (1ll << 28) &&
                          rnnt_causal_conv_workspace_size((int)x_in.size(0), (int)x_in.size(1), (int)x_in.size(2),
                                                          (int)weight_in.size(1), &need) == RNNT_STATUS_SUCCESS,
                      "x is too large for one call");
    check_tangents({&x_in, &weight_in, &bias, &initial}, "causal_conv");
    check_on_device(x_in, "causal_conv");
    check_same_device(weight_in, x_in, "weight");
    check_same_device(bias, x_in, "bias");
    check_same_device(initial, x_in, "initial_state");
    check_same_device(lengths, x_in, "lengths");
    check_capture({&x_in, &weight_in, &bias, &initial}, "causal_conv");
    const Tensor x = rows_of(x_in), weight = weight_in.contiguous();
    if (bias.defined()) bias = bias.contiguous();
    if (initial.defined()) initial = initial.contiguous();
    if (!wants_grad({&x, &weight, &bias, &initial})) return conv_forward(x, weight, bias, initial, lengths, silu);
    const auto out = ConvFunction::apply(x, weight, bias.defined() ? MaybeTensor(bias) : MaybeTensor(),
                                         initial.defined() ? MaybeTensor(initial) : MaybeTensor(), lengths_in, silu);
    return {out[0], out[1]};
}

// A buffer that the caller gives for a result: nothing that the call reads may lie in it (another thread may read it after it
// is written), and autograd learns that it changes.
bool overlap(const Tensor &a, const Tensor &b) {
    auto end = [](const Tensor &t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        return static_cast<const char *>(t.data_ptr()) + (last + 1) * t.element_size();
    };
    return a.data_ptr() < end(b) && b.data_ptr() < end(a);
}
void check_apart(const Tensor &out, std::initializer_list<const Tensor *> inputs, const char *name) {
    for (const Tensor *t : inputs)
        TORCH_CHECK_VALUE(!t->defined() || t->numel() == 0 || !overlap(out, *t), name, " must not overlap another argument of the call");
}
void changed(const Tensor &out) {
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

// a new state beside the old one, or the caller's buffer
Tensor state_buffer(const MaybeTensor &out, const Tensor &state, std::initializer_list<const Tensor *> others) {
    if (!out.has_value()) return at::empty(state.sizes(), state.options());
    TORCH_CHECK_TYPE(out->scalar_type() == state.scalar_type(), "state_out must have the state's type");
    TORCH_CHECK_VALUE(out->sizes() == state.sizes() && out->is_contiguous() && state.is_contiguous(),
                      "state_out must be contiguous and have the state's shape (and the state be contiguous too)");
    TORCH_CHECK(out->device() == state.device(), "state_out must be on ", state.device(), ", got ", out->device());
    // the very buffer or another one: a buffer that overlaps the state by a part would be read after it is written
    const char *a = static_cast<const char *>(out->data_ptr()), *b = static_cast<const char *>(state.data_ptr());
    TORCH_CHECK_VALUE(a == b || a + out->nbytes() <= b || b + state.nbytes() <= a, "state_out must not overlap the state in part");
    check_apart(*out, others, "state_out");
    changed(*out);
    return *out;
}

std::tuple<Tensor, Tensor> causal_conv_step_op(const Tensor &x_in, const Tensor &state_in, const Tensor &weight_in,
                                               const MaybeTensor &bias_in, bool silu, const MaybeTensor &state_out) {
    dtype_code(x_in, "x");
    TORCH_CHECK_VALUE(x_in.dim() == 2 && x_in.numel() >= 1, "x must be a non-empty [batch, dim] tensor");
    Tensor bias = given(bias_in);
    check_conv_weights(weight_in, bias, x_in.size(1));
    check_conv_state(state_in, x_in, weight_in.size(1), "state");
    TORCH_CHECK_VALUE(x_in.numel() < (1ll << 31) && x_in.size(1) < (1ll << 28), "x is too large for one call");
    const Tensor written = given(state_out);
    check_no_grad({&x_in, &state_in, &weight_in, &bias, &written}, "causal_conv_step");
    check_on_device(x_in, "causal_conv_step");
    check_same_device(state_in, x_in, "state");
    check_same_device(weight_in, x_in, "weight");
    check_same_device(bias, x_in, "bias");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
    Tensor out = state_buffer(state_out, state_in, {&x_in, &weight_in, &bias});
    const Tensor x = rows_of(x_in), state = state_in.contiguous(), weight = weight_in.contiguous();
    if (bias.defined()) bias = bias.contiguous();
    Tensor y = at::empty(x.sizes(), x.options());
    rnntConv c = conv_args(x, weight, bias, state, Tensor(), silu);
    c.y = y.data_ptr();
    c.final_state = out.data_ptr();
    check_status(rnnt_causal_conv_step(&c), "rnnt_causal_conv_step");
    return {y, out};
}

// ---- selective scan -----------------------------------------------------------------------------------------------------
struct ScanIn {
    Tensor x, dt, A, B, C, D, z, dt_bias, initial, lengths;
};

rnntScan scan_args(const ScanIn &in) {
    rnntScan a = {};
    const bool seq = in.x.dim() == 3;
    a.batch = (int)in.x.size(0);
    a.length = seq ? (int)in.x.size(1) : 1;
    a.dim = (int)in.x.size(-1);
    a.state = (int)in.A.size(1);
    a.dtype = dtype_code(in.x, "x");
    auto put = [seq](const Tensor &t, const void *&p, long long &batch, long long &time) {
        if (!t.defined()) return;
        p = t.data_ptr();
        batch = t.stride(0);
        time = seq ? t.stride(1) : 0;
    };
    put(in.x, a.x, a.x_batch, a.x_time);
    put(in.dt, a.dt, a.dt_batch, a.dt_time);
    put(in.z, a.z, a.z_batch, a.z_time);
    put(in.B, a.B, a.B_batch, a.B_time);
    put(in.C, a.C, a.C_batch, a.C_time);
    a.A = pointer<float>(in.A);
    a.D = pointer<float>(in.D);
    a.dt_bias = pointer<float>(in.dt_bias);
    a.initial_state = pointer<float>(in.initial);
    a.lengths = pointer<int>(in.lengths);
    a.stream = stream_of(in.x);
    return a;
}

Tensor scan_workspace(const rnntScan &a, int backward, const Tensor &x) {
    size_t need = 0;
    check_status(rnnt_selective_scan_workspace_size(a.batch, a.length, a.dim, a.state, backward, &need),
                 "rnnt_selective_scan_workspace_size");
    return bytes(need, x);
}

std::tuple<Tensor, Tensor, Tensor> scan_forward(const ScanIn &in, bool keep) {
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(in.x.device());
    rnntScan a = scan_args(in);
    Tensor y = at::empty(in.x.sizes(), in.x.options());
    Tensor final_state = at::empty({a.batch, a.dim, a.state}, in.A.options());
    Tensor states;
    if (keep) {
        size_t need = 0;
        check_status(rnnt_selective_scan_states_size(a.batch, a.length, a.dim, a.state, &need), "rnnt_selective_scan_states_size");
        states = at::empty({(int64_t)(need / sizeof(float))}, in.A.options());
    }
    const Tensor ws = scan_workspace(a, 0, in.x);
    a.y = y.data_ptr();
    a.final_state = pointer<float>(final_state);
    a.chunk_states = pointer<float>(states);
    a.workspace = pointer<void>(ws);
    check_status(rnnt_selective_scan_forward(&a), "rnnt_selective_scan_forward");
    return {y, final_state, states};
}

class ScanFunction : public torch::autograd::Function<ScanFunction> {
public:
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B,
                                 const Tensor &C, const MaybeTensor &D, const MaybeTensor &z, const MaybeTensor &dt_bias,
                                 const MaybeTensor &initial, const MaybeTensor &lengths) {
        const ScanIn in = {x, dt, A, B, C, given(D), given(z), given(dt_bias), given(initial), given(lengths)};
        auto out = scan_forward(in, true);
        // (the chunk states begin with the initial state: backward does not read it again)
        ctx->save_for_backward({x, dt, A, B, C, in.D, in.z, in.dt_bias, in.lengths, std::get<2>(out)});
        ctx->saved_data["initial"] = in.initial.defined();
        ctx->set_materialize_grads(false);
        return {std::get<0>(out), std::get<1>(out)};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const ScanIn in = {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], Tensor(), s[8]};
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(in.x.device());
        rnntScan a = scan_args(in);
        const Tensor gy = grads[0].defined() ? rows_of(grads[0]) : at::zeros(in.x.sizes(), in.x.options());
        const Tensor gf = grads[1].defined() ? grads[1].contiguous() : Tensor();
        auto like = [](const Tensor &t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); };
        Tensor dx = like(in.x), ddt = like(in.dt), dA = like(in.A), dB = like(in.B), dC = like(in.C), dD = like(in.D), dz = like(in.z),
               dbias = like(in.dt_bias), dinitial;
        if (ctx->saved_data["initial"].toBool()) dinitial = at::empty({a.batch, a.dim, a.state}, in.A.options());
        const Tensor ws = scan_workspace(a, 1, in.x);
        a.chunk_states = pointer<float>(s[9]);
        a.grad_y = gy.data_ptr();
        a.grad_y_batch = gy.stride(0);
        a.grad_y_time = gy.stride(1);
        a.grad_final = pointer<float>(gf);
        a.grad_x = dx.data_ptr();
        a.grad_dt = ddt.data_ptr();
        a.grad_z = pointer<void>(dz);
        a.grad_B = dB.data_ptr();
        a.grad_C = dC.data_ptr();
        a.grad_A = pointer<float>(dA);
        a.grad_D = pointer<float>(dD);
        a.grad_dt_bias = pointer<float>(dbias);
        a.grad_initial = pointer<float>(dinitial);
        a.workspace = pointer<void>(ws);
        check_status(rnnt_selective_scan_backward(&a), "rnnt_selective_scan_backward");
        return once({dx, ddt, dA, dB, dC, dD, dz, dbias, dinitial, Tensor()}, "selective_scan");
    }
};

ScanIn scan_check(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const MaybeTensor &D,
                  const MaybeTensor &z, const MaybeTensor &dt_bias, const Tensor &state, const MaybeTensor &lengths, bool step,
                  const Tensor &written = Tensor()) {
    ScanIn in = {x, dt, A, B, C, given(D), given(z), given(dt_bias), state, given(lengths)};
    const char *op = step ? "selective_scan_step" : "selective_scan";
    dtype_code(x, "x");
    TORCH_CHECK_VALUE(x.dim() == (step ? 2 : 3) && x.numel() >= 1, "x must be a non-empty ",
                      step ? "[batch, dim] tensor" : "[batch, length, dim] tensor");
    TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == x.size(-1) && (A.size(1) == 8 || A.size(1) == 16 || A.size(1) == 32),
                      "A must be [dim, state] with 8, 16 or 32 states");
    check_f32(A, A.sizes(), "A");
    check_f32(in.D, {x.size(-1)}, "D");
    check_f32(in.dt_bias, {x.size(-1)}, "dt_bias");
    auto same = [&](const Tensor &t, int64_t last, const char *name) {
        if (!t.defined()) return;
        TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " must have x's type");
        bool ok = t.dim() == x.dim() && t.size(-1) == last;
        for (int64_t i = 0; ok && i + 1 < x.dim(); ++i) ok = t.size(i) == x.size(i);
        TORCH_CHECK_VALUE(ok, name, " must agree with x in batch and length and have ", last, " as its last size, got ", t.sizes());
    };
    same(dt, x.size(-1), "dt");
    same(in.z, x.size(-1), "z");
    same(B, A.size(1), "B");
    same(C, A.size(1), "C");
    check_f32(state, {x.size(0), x.size(-1), A.size(1)}, step ? "state" : "initial_state");
    check_lengths(in.lengths, x.size(0));
    size_t need = 0;
    TORCH_CHECK_VALUE(x.numel() / x.size(-1) < (1ll << 31) && x.size(-1) < (1ll << 28) &&
                          rnnt_selective_scan_states_size((int)x.size(0), step ? 1 : (int)x.size(1), (int)x.size(-1), (int)A.size(1),
                                                          &need) == RNNT_STATUS_SUCCESS,
                      "x is too large for one call");
    if (step)
        check_no_grad({&x, &dt, &A, &B, &C, &in.D, &in.z, &in.dt_bias, &in.initial, &written}, op);
    else
        check_tangents({&x, &dt, &A, &B, &C, &in.D, &in.z, &in.dt_bias, &in.initial}, op);
    check_on_device(x, op);
    const Tensor *all[] = {&dt, &A, &B, &C, &in.D, &in.z, &in.dt_bias, &in.initial, &in.lengths};
    const char *names[] = {"dt", "A", "B", "C", "D", "z", "dt_bias", step ? "state" : "initial_state", "lengths"};
    for (int i = 0; i < 9; ++i) check_same_device(*all[i], x, names[i]);
    if (!step) check_capture({&x, &dt, &A, &B, &C, &in.D, &in.z, &in.dt_bias, &in.initial}, op);
    in.x = rows_of(x);
    in.dt = rows_of(dt);
    in.B = rows_of(B);
    in.C = rows_of(C);
    in.A = A.contiguous();
    if (in.z.defined()) in.z = rows_of(in.z);
    if (in.D.defined()) in.D = in.D.contiguous();
    if (in.dt_bias.defined()) in.dt_bias = in.dt_bias.contiguous();
    if (in.initial.defined()) in.initial = in.initial.contiguous();
    return in;
}

std::tuple<Tensor, Tensor> selective_scan_op(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C,
                                             const MaybeTensor &D, const MaybeTensor &z, const MaybeTensor &dt_bias,
                                             const MaybeTensor &initial, const MaybeTensor &lengths) {
    const ScanIn in = scan_check(x, dt, A, B, C, D, z, dt_bias, given(initial), lengths, false);
    if (!wants_grad({&in.x, &in.dt, &in.A, &in.B, &in.C, &in.D, &in.z, &in.dt_bias, &in.initial})) {
        auto out = scan_forward(in, false);
        return {std::get<0>(out), std::get<1>(out)};
    }
    auto maybe = [](const Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
    const auto out = ScanFunction::apply(in.x, in.dt, in.A, in.B, in.C, maybe(in.D), maybe(in.z), maybe(in.dt_bias), maybe(in.initial),
                                         maybe(in.lengths));
    return {out[0], out[1]};
}

std::tuple<Tensor, Tensor> selective_scan_step_op(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C,
                                                  const Tensor &state, const MaybeTensor &D, const MaybeTensor &z,
                                                  const MaybeTensor &dt_bias, const MaybeTensor &state_out) {
    const ScanIn in = scan_check(x, dt, A, B, C, D, z, dt_bias, state, MaybeTensor(), true, given(state_out));
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    Tensor out = state_buffer(state_out, state, {&x, &dt, &A, &B, &C, &in.D, &in.z, &in.dt_bias});
    Tensor y = at::empty(x.sizes(), x.options());
    rnntScan a = scan_args(in);
    a.y = y.data_ptr();
    a.final_state = pointer<float>(out);
    check_status(rnnt_selective_scan_step(&a), "rnnt_selective_scan_step");
    return {y, out};
}

// ---- decoding rules -----------------------------------------------------------------------------------------------------
struct RulesIn {
    Tensor x, bias, allowed, history, history_lens;
    rnntRules r = {};
    int rows = 0, V = 0;
};

RulesIn rules_check(const Tensor &x, const MaybeTensor &bias_in, const MaybeTensor &allowed_in, const MaybeTensor &history_in,
                    const MaybeTensor &history_lens_in, double repetition, double presence, double frequency, const char *op,
                    bool values, const Tensor &written = Tensor()) {
    RulesIn in = {x, given(bias_in), given(allowed_in), given(history_in), given(history_lens_in)};
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) >= 1 && x.size(1) >= 1, "x must be a non-empty [rows, V] tensor");
    dtype_code(x, "x");
    in.rows = as_int(x.size(0), "rows");
    TORCH_CHECK_VALUE(x.size(1) <= (1 << 30), "V is too large");
    in.V = (int)x.size(1);
    size_t need = 0;
    TORCH_CHECK_VALUE(rnnt_row_rules_workspace_size(in.rows, in.V, dtype_code(x, "x"), &need) == RNNT_STATUS_SUCCESS,
                      "x has too many rows for one call");
    int64_t contexts = 1;
    const char *by = nullptr;
    auto agree = [&](const Tensor &t, const char *name) {
        TORCH_CHECK_VALUE(by == nullptr || t.size(0) == contexts, name, " has ", t.size(0), " contexts and ", by, " ", contexts);
        contexts = t.size(0);
        by = name;
    };
    if (in.bias.defined()) {
        TORCH_CHECK_TYPE(in.bias.scalar_type() == at::kFloat, "bias must be torch.float32");
        TORCH_CHECK_VALUE((in.bias.dim() == 1 || in.bias.dim() == 2) && in.bias.size(-1) == in.V, "bias must be [V] or [contexts, V]");
        if (in.bias.dim() == 2) agree(in.bias, "bias");
    }
    const int64_t words = ((int64_t)in.V + 31) / 32;
    if (in.allowed.defined()) {
        TORCH_CHECK_TYPE(in.allowed.scalar_type() == at::kInt, "allowed must be torch.int32 (one bit per token)");
        TORCH_CHECK_VALUE((in.allowed.dim() == 1 || in.allowed.dim() == 2) && in.allowed.size(-1) == words,
                          "allowed must be [(V + 31) // 32] or [contexts, (V + 31) // 32]");
        if (in.allowed.dim() == 2) agree(in.allowed, "allowed");
    }
    TORCH_CHECK_VALUE(!in.history_lens.defined() || in.history.defined(), "history_lens needs history");
    if (in.history.defined()) {
        TORCH_CHECK_TYPE(in.history.scalar_type() == at::kInt, "history must be torch.int32");
        TORCH_CHECK_VALUE(in.history.dim() == 2 && in.history.size(1) <= RNNT_MAX_HISTORY, "history must be [contexts, at most ",
                          RNNT_MAX_HISTORY, " tokens]");
        agree(in.history, "history");
        if (in.history_lens.defined()) {
            TORCH_CHECK_TYPE(in.history_lens.scalar_type() == at::kInt, "history_lens must be torch.int32");
            TORCH_CHECK_VALUE(in.history_lens.dim() == 1 && in.history_lens.size(0) == in.history.size(0), "history_lens must be [contexts]");
        }
    }
    TORCH_CHECK_VALUE(contexts >= 1 && in.rows % contexts == 0, "the rows of x must be a multiple of the contexts (", contexts, ")");
    TORCH_CHECK_VALUE((float)repetition > 0.f && std::isfinite((float)repetition), "repetition_penalty must be positive and finite");
    TORCH_CHECK_VALUE(std::isfinite((float)presence) && std::isfinite((float)frequency),
                      "presence_penalty and frequency_penalty must be finite");
    if (values) check_no_grad({&x, &in.bias, &written}, op);  // (a token alone has no derivative)
    check_on_device(x, op);
    check_same_device(in.bias, x, "bias");
    check_same_device(in.allowed, x, "allowed");
    check_same_device(in.history, x, "history");
    check_same_device(in.history_lens, x, "history_lens");
    in.x = x.contiguous();
    if (in.bias.defined()) in.bias = in.bias.contiguous();
    if (in.allowed.defined()) in.allowed = in.allowed.contiguous();
    if (in.history.defined() && in.history.size(1) == 0) in.history = in.history_lens = Tensor();  // nothing emitted yet
    if (in.history.defined()) in.history = in.history.contiguous();
    if (in.history_lens.defined()) in.history_lens = in.history_lens.contiguous();
    in.r.contexts = (int)contexts;
    in.r.history = pointer<int>(in.history);
    in.r.history_lens = pointer<int>(in.history_lens);
    in.r.history_stride = in.history.defined() ? (int)in.history.size(1) : 0;
    in.r.bias = pointer<float>(in.bias);
    in.r.bias_stride = in.bias.defined() && in.bias.dim() == 2 ? in.V : 0;
    in.r.allowed = pointer<int>(in.allowed);
    in.r.allowed_stride = in.allowed.defined() && in.allowed.dim() == 2 ? words : 0;
    in.r.repetition_penalty = (float)repetition;
    in.r.presence_penalty = (float)presence;
    in.r.frequency_penalty = (float)frequency;
    return in;
}

std::tuple<Tensor, Tensor> row_rules_op(const Tensor &x, const MaybeTensor &bias, const MaybeTensor &allowed, const MaybeTensor &history,
                                        const MaybeTensor &history_lens, double repetition, double presence, double frequency,
                                        bool want_logp) {
    const RulesIn in = rules_check(x, bias, allowed, history, history_lens, repetition, presence, frequency,
                                   want_logp ? "row_max_logp" : "row_argmax", want_logp);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    Tensor token = at::empty({in.rows}, x.options().dtype(at::kInt));
    Tensor logp = at::empty({want_logp ? in.rows : 0}, x.options().dtype(at::kFloat));
    size_t need = 0;
    check_status(rnnt_row_rules_workspace_size(in.rows, in.V, dtype_code(x, "x"), &need), "rnnt_row_rules_workspace_size");
    const Tensor ws = need ? bytes(need, x) : Tensor();
    check_status(rnnt_row_rules(in.x.data_ptr(), in.rows, in.V, dtype_code(x, "x"), &in.r, pointer<int>(token),
                                want_logp ? pointer<float>(logp) : nullptr, pointer<void>(ws), stream_of(x)),
                 "rnnt_row_rules");
    return {token, logp};
}

Tensor process_logits_op(const Tensor &x, const MaybeTensor &bias, const MaybeTensor &allowed, const MaybeTensor &history,
                         const MaybeTensor &history_lens, double repetition, double presence, double frequency,
                         const MaybeTensor &out_in) {
    const RulesIn in = rules_check(x, bias, allowed, history, history_lens, repetition, presence, frequency, "process_logits", true,
                                   given(out_in));
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    Tensor out;
    if (out_in.has_value()) {
        out = *out_in;
        TORCH_CHECK_TYPE(out.scalar_type() == x.scalar_type(), "out must have x's type");
        TORCH_CHECK_VALUE(out.sizes() == x.sizes() && out.is_contiguous(), "out must be contiguous and have x's shape");
        check_same_device(out, x, "out");
        const char *a = static_cast<const char *>(out.data_ptr()), *b = static_cast<const char *>(in.x.data_ptr());
        TORCH_CHECK_VALUE(a == b || a + out.nbytes() <= b || b + in.x.nbytes() <= a, "out must not overlap x in part");
        check_apart(out, {&in.bias, &in.allowed, &in.history, &in.history_lens}, "out");
        changed(out);
    } else {
        out = at::empty(in.x.sizes(), in.x.options());
    }
    check_status(rnnt_process_logits(in.x.data_ptr(), in.rows, in.V, dtype_code(x, "x"), &in.r, out.data_ptr(), stream_of(x)),
                 "rnnt_process_logits");
    return out;
}

}  // namespace

// (a caller's result buffer is declared as written: a compiled graph would drop a call whose returned tensors it does not use)
TORCH_LIBRARY_FRAGMENT(rnnt_amd, m) {
    m.def("token_embedding(Tensor tokens, Tensor weight, float scale, int padding_idx) -> Tensor", &token_embedding_op);
    m.def("causal_conv(Tensor x, Tensor weight, Tensor? bias, Tensor? initial_state, Tensor? lengths, bool silu) -> (Tensor, Tensor)",
          &causal_conv_op);
    m.def("causal_conv_step(Tensor x, Tensor state, Tensor weight, Tensor? bias, bool silu, Tensor(a!)? state_out) -> (Tensor, Tensor(a!))",
          &causal_conv_step_op);
    m.def("selective_scan(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, "
          "Tensor? initial_state, Tensor? lengths) -> (Tensor, Tensor)",
          &selective_scan_op);
    m.def("selective_scan_step(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor state, Tensor? D, Tensor? z, "
          "Tensor? dt_bias, Tensor(a!)? state_out) -> (Tensor, Tensor(a!))",
          &selective_scan_step_op);
    m.def("row_rules(Tensor x, Tensor? bias, Tensor? allowed, Tensor? history, Tensor? history_lens, float repetition_penalty, "
          "float presence_penalty, float frequency_penalty, bool want_logp) -> (Tensor, Tensor)",
          &row_rules_op);
    m.def("process_logits(Tensor x, Tensor? bias, Tensor? allowed, Tensor? history, Tensor? history_lens, float repetition_penalty, "
          "float presence_penalty, float frequency_penalty, Tensor(a!)? out) -> Tensor(a!)",
          &process_logits_op);
}
