// The sequence operators as PyTorch dispatcher ops (torch.ops.unetmi.seq_conv, .ssm_scan, .block_norm and their _bwd and
// _step forms): checks of arguments, outputs, workspaces, autograd, and the calls of libunetmi.so's C entry points
// (include/unetmi.h).  The other ops of this package are registered from Python.  These are called once per token and
// layer, where Python's share of a call was several times the kernel's (a single stream's scan: 13.5 us a call from Python,
// 6.6 from here, of which the kernel takes 4), and in backward passes, which autograd runs on a thread of its own (a small
// convolution forward and backward: 114 us from Python, 70 from here, of which the engine itself takes about 45).
//
// Outputs are dense; an output that a call does not have is an empty tensor.  Scratch memory is taken from torch's caching
// allocator call by call (under graph capture: from the graph's own pool), never from a buffer that calls share.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>
#include <torch/types.h>

#include "../../include/unetmi.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

// the entry points of the library that unet_amd._lib loaded
struct Entries {
    void (*last_error)(char*, size_t);
    decltype(&unetmi_seq_conv_fwd) conv_fwd;
    decltype(&unetmi_seq_conv_bwd_workspace_bytes) conv_bwd_bytes;
    decltype(&unetmi_seq_conv_bwd) conv_bwd;
    decltype(&unetmi_seq_conv_step) conv_step;
    decltype(&unetmi_ssm_scan_marks_bytes) scan_marks_bytes;
    decltype(&unetmi_ssm_scan_fwd_workspace_bytes) scan_fwd_bytes;
    decltype(&unetmi_ssm_scan_fwd) scan_fwd;
    decltype(&unetmi_ssm_scan_bwd_workspace_bytes) scan_bwd_bytes;
    decltype(&unetmi_ssm_scan_bwd) scan_bwd;
    decltype(&unetmi_ssm_scan_step) scan_step;
    decltype(&unetmi_block_norm_fwd) norm_fwd;
    decltype(&unetmi_block_norm_bwd_workspace_bytes) norm_bwd_bytes;
    decltype(&unetmi_block_norm_bwd) norm_bwd;
} lib;

void check(int code, const char* what) {
    if (code == UNETMI_OK) return;
    char text[512] = "";
    lib.last_error(text, sizeof text);
    TORCH_CHECK(false, what, " failed (", code, "): ", text);
}

// the library counts in 32 bits, and refuses what is larger than it takes itself
int32_t count(int64_t n, const char* op) {
    TORCH_CHECK_VALUE(n <= INT32_MAX, "unetmi::", op, ": an axis of ", n, " elements is too long");
    return (int32_t)n;
}

int32_t kind(const Tensor& x, const char* op, int64_t axes) {
    TORCH_CHECK_VALUE(x.is_cuda() && (x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16), "unetmi::", op,
                      ": x must be a float32 or bfloat16 device tensor, got ", x.scalar_type(), " on ", x.device());
    TORCH_CHECK_VALUE(x.dim() == axes, "unetmi::", op, ": x must have ", axes, " axes, got shape ", x.sizes());
    return x.scalar_type() == at::kBFloat16 ? UNETMI_DTYPE_BF16 : UNETMI_DTYPE_F32;
}

void same(const Tensor& t, const char* name, const char* op, at::ScalarType type, const Tensor& like, at::IntArrayRef shape) {
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == like.device() && t.sizes() == shape, "unetmi::", op, ": ", name, " must be a ",
                      type, " tensor of shape ", shape, " on ", like.device(), ", got ", t.scalar_type(), " of shape ", t.sizes(), " on ",
                      t.device());
}
void dense(const Tensor& t, const char* name, const char* op, at::ScalarType type, const Tensor& like, at::IntArrayRef shape) {
    same(t, name, op, type, like, shape);
    TORCH_CHECK_VALUE(t.is_contiguous(), "unetmi::", op, ": ", name, " must be contiguous");
}
void dense(const Maybe& t, const char* name, const char* op, at::ScalarType type, const Tensor& like, at::IntArrayRef shape) {
    if (t) dense(*t, name, op, type, like, shape);
}

// elements between two entries of an axis; a single entry's stride may be anything and means nothing
int64_t apart(const Tensor& t, int64_t axis) { return t.size(axis) > 1 ? t.stride(axis) : 0; }

// the last axis dense and steps not too far apart: a copy where they are not
Tensor rows(const Tensor& t) {
    const int64_t n = t.dim();
    const bool ok = (t.stride(n - 1) == 1 || t.size(n - 1) <= 1) && (n < 3 || apart(t, 1) <= UNETMI_SEQ_MAX_STEP);
    return ok ? t : t.contiguous();
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
float* f32(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }
float* f32(const Maybe& t) { return t ? static_cast<float*>(t->data_ptr()) : nullptr; }
const int32_t* i32(const Maybe& t) { return t ? static_cast<const int32_t*>(t->data_ptr()) : nullptr; }

Tensor empty(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options()); }
Tensor empty(at::IntArrayRef shape, const Tensor& like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type)); }
Tensor scratch(size_t bytes, const Tensor& like) { return empty({(int64_t)(bytes ? bytes : 16)}, like, at::kByte); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

// The kernel wrote the tensor through its pointer: what autograd saved of it is stale from here on.
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---------------------------------------------------------------------------------------------------------------------
// the causal convolution
// ---------------------------------------------------------------------------------------------------------------------
UnetmiSeqConvDesc conv_desc(const char* op, const Tensor& x, const Tensor& weight, const Maybe& bias, const Maybe& state, const Maybe& lengths, bool silu) {
    UnetmiSeqConvDesc d = {};
    d.dtype = kind(x, op, 3);
    TORCH_CHECK_VALUE(weight.dim() == 2, "unetmi::", op, ": weight must be [channels, taps]");
    const int64_t B = x.size(0), D = x.size(2), K = weight.size(1);
    dense(weight, "weight", op, at::kFloat, x, {D, K});
    dense(bias, "bias", op, at::kFloat, x, {D});
    dense(state, "state", op, x.scalar_type(), x, {B, K - 1, D});
    dense(lengths, "lengths", op, at::kInt, x, {B});
    d.batch = count(B, op); d.length = count(x.size(1), op); d.channels = count(D, op); d.taps = count(K, op);
    d.act = silu ? UNETMI_ACT_SILU : UNETMI_ACT_NONE;
    return d;
}

std::tuple<Tensor, Tensor> seq_conv(const Tensor& x0, const Tensor& weight, const Maybe& bias, const Maybe& state, const Maybe& lengths, bool silu,
                                    bool want_state) {
    UnetmiSeqConvDesc d = conv_desc("seq_conv", x0, weight, bias, state, lengths, silu);
    const Tensor x = rows(x0);
    d.x_stride[0] = apart(x, 0); d.x_stride[1] = apart(x, 1);
    const c10::DeviceGuard guard(x.device());
    const Tensor y = empty(x.sizes(), x);
    const Tensor out = want_state ? empty({d.batch, d.taps - 1, d.channels}, x) : empty({0}, x);
    check(lib.conv_fwd(&d, ptr(x), f32(weight), f32(bias), ptr(state), i32(lengths), ptr(y), want_state ? ptr(out) : nullptr, stream_of(x)),
          "unetmi_seq_conv_fwd");
    return {y, out};
}

// (dx, dweight, dbias, dstate or empty)
std::tuple<Tensor, Tensor, Tensor, Tensor> seq_conv_bwd(const Tensor& x0, const Tensor& weight, const Maybe& bias, const Maybe& state,
                                                        const Maybe& lengths, bool silu, const Tensor& dy0, const Maybe& dstate_out) {
    const char* op = "seq_conv_bwd";
    UnetmiSeqConvDesc d = conv_desc(op, x0, weight, bias, state, lengths, silu);
    same(dy0, "dy", op, x0.scalar_type(), x0, x0.sizes());
    dense(dstate_out, "dstate_out", op, x0.scalar_type(), x0, {d.batch, d.taps - 1, d.channels});
    const Tensor x = rows(x0), dy = rows(dy0);
    d.x_stride[0] = apart(x, 0); d.x_stride[1] = apart(x, 1);
    d.dy_stride[0] = apart(dy, 0); d.dy_stride[1] = apart(dy, 1);
    const c10::DeviceGuard guard(x.device());
    const Tensor dx = empty(x.sizes(), x), dw = empty(weight.sizes(), weight), db = empty({d.channels}, weight);
    const Tensor dstate = state ? empty(state->sizes(), x) : empty({0}, x);
    if (d.batch == 0) {
        dw.zero_();
        db.zero_();
        return {dx, dw, db, dstate};
    }
    const Tensor ws = scratch(lib.conv_bwd_bytes(&d), x);
    check(lib.conv_bwd(&d, ptr(x), f32(weight), f32(bias), ptr(state), i32(lengths), ptr(dy), ptr(dstate_out), ptr(dx), f32(dw), f32(db),
                       state ? ptr(dstate) : nullptr, ptr(ws), ws.numel(), stream_of(x)), "unetmi_seq_conv_bwd");
    return {dx, dw, db, dstate};
}

Tensor seq_conv_step(const Tensor& x0, const Tensor& weight, const Maybe& bias, const Tensor& state, const Maybe& slots, bool silu) {
    const char* op = "seq_conv_step";
    UnetmiSeqConvDesc d = {};
    d.dtype = kind(x0, op, 2);
    TORCH_CHECK_VALUE(weight.dim() == 2 && state.dim() == 3, "unetmi::", op, ": weight must be [channels, taps], state [slots, taps-1, channels]");
    const int64_t B = x0.size(0), D = x0.size(1), K = weight.size(1);
    dense(weight, "weight", op, at::kFloat, x0, {D, K});
    dense(bias, "bias", op, at::kFloat, x0, {D});
    dense(state, "state", op, x0.scalar_type(), x0, {state.size(0), K - 1, D});
    dense(slots, "slots", op, at::kInt, x0, {B});
    const int32_t slot_count = count(state.size(0), op);
    d.batch = count(B, op); d.length = 1; d.channels = count(D, op); d.taps = count(K, op);
    const Tensor x = rows(x0);
    d.act = silu ? UNETMI_ACT_SILU : UNETMI_ACT_NONE;
    d.x_stride[0] = apart(x, 0);
    const c10::DeviceGuard guard(x.device());
    const Tensor y = empty(x.sizes(), x);
    check(lib.conv_step(&d, ptr(x), f32(weight), f32(bias), i32(slots), slot_count, ptr(state), ptr(y), stream_of(x)), "unetmi_seq_conv_step");
    written(state);
    return y;
}

// ---------------------------------------------------------------------------------------------------------------------
// the scan
// ---------------------------------------------------------------------------------------------------------------------
struct ScanIn {
    UnetmiScanDesc d = {};
    Tensor x, dt, B, C;
    Maybe z;
    ScanIn(const char* op, const Tensor& x0, const Tensor& dt0, const Tensor& A, const Tensor& B0, const Tensor& C0, const Maybe& D, const Maybe& z0,
           const Maybe& dt_bias, bool softplus, int64_t axes) {
        d.dtype = kind(x0, op, axes);
        const at::ScalarType type = x0.scalar_type();
        same(dt0, "dt", op, type, x0, x0.sizes());
        if (z0) same(*z0, "z", op, type, x0, x0.sizes());
        TORCH_CHECK_VALUE(A.dim() == 2, "unetmi::", op, ": A must be [channels, state]");
        const int64_t channels = x0.size(axes - 1), N = A.size(1);
        const bool grouped = B0.dim() == axes + 1;                    // else one group: [.., state]
        c10::SmallVector<int64_t, 4> bc(x0.sizes().begin(), x0.sizes().end() - 1);
        if (grouped) bc.push_back(B0.size(axes - 1));
        bc.push_back(N);
        same(B0, "B", op, type, x0, bc);
        same(C0, "C", op, type, x0, bc);
        dense(A, "A", op, at::kFloat, x0, {channels, N});
        dense(D, "D", op, at::kFloat, x0, {channels});
        dense(dt_bias, "dt_bias", op, at::kFloat, x0, {channels});
        d.batch = count(x0.size(0), op); d.length = axes == 3 ? count(x0.size(1), op) : 1; d.channels = count(channels, op); d.state = count(N, op);
        d.groups = grouped ? count(B0.size(axes - 1), op) : 1;
        x = rows(x0); dt = rows(dt0); B = rows(B0); C = rows(C0);
        if (z0) z = rows(*z0);
        d.softplus = softplus;
        for (int64_t i = 0; i < axes - 1; ++i) {
            d.x_stride[i] = apart(x, i); d.dt_stride[i] = apart(dt, i); d.z_stride[i] = z ? apart(*z, i) : 0;
            d.b_stride[i] = apart(B, i); d.c_stride[i] = apart(C, i);
        }
        if (grouped) { d.b_stride[2] = apart(B, axes - 1); d.c_stride[2] = apart(C, axes - 1); }
    }
};

// (y, final state [B, channels, N] or empty, the states the backward call needs or empty)
std::tuple<Tensor, Tensor, Tensor> ssm_scan(const Tensor& x0, const Tensor& dt0, const Tensor& A, const Tensor& B0, const Tensor& C0, const Maybe& D,
                                            const Maybe& z0, const Maybe& dt_bias, const Maybe& state, const Maybe& lengths, bool softplus,
                                            bool want_state, bool want_marks) {
    const char* op = "ssm_scan";
    const ScanIn in(op, x0, dt0, A, B0, C0, D, z0, dt_bias, softplus, 3);
    const UnetmiScanDesc& d = in.d;
    const Tensor& x = in.x;
    dense(state, "state", op, at::kFloat, x, {d.batch, d.channels, d.state});
    dense(lengths, "lengths", op, at::kInt, x, {d.batch});
    const c10::DeviceGuard guard(x.device());
    const Tensor y = empty(x.sizes(), x);
    const Tensor out = want_state ? empty({d.batch, d.channels, d.state}, A) : empty({0}, A);
    const Tensor marks = empty({want_marks ? (int64_t)(lib.scan_marks_bytes(&d) / sizeof(float)) : 0}, A);
    const size_t need = lib.scan_fwd_bytes(&d, lengths.has_value());
    Tensor ws;
    if (need) ws = scratch(need, x);
    check(lib.scan_fwd(&d, ptr(x), ptr(in.dt), f32(A), ptr(in.B), ptr(in.C), f32(D), ptr(in.z), f32(dt_bias), f32(state), i32(lengths), ptr(y),
                       want_state ? f32(out) : nullptr, want_marks ? f32(marks) : nullptr, need ? ptr(ws) : nullptr, need, stream_of(x)),
          "unetmi_ssm_scan_fwd");
    return {y, out, marks};
}

// (dx, ddt, dA, dB, dC, dD, dz or empty, ddt_bias, dstate or empty)
typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> Nine;
Nine ssm_scan_bwd(const Tensor& x0, const Tensor& dt0, const Tensor& A, const Tensor& B0, const Tensor& C0, const Maybe& D, const Maybe& z0,
                  const Maybe& dt_bias, const Maybe& lengths, bool softplus, const Tensor& marks, const Tensor& dy0, const Maybe& dstate_out,
                  bool want_dstate) {
    const char* op = "ssm_scan_bwd";
    ScanIn in(op, x0, dt0, A, B0, C0, D, z0, dt_bias, softplus, 3);
    UnetmiScanDesc& d = in.d;
    const Tensor& x = in.x;
    same(dy0, "dy", op, x.scalar_type(), x, x.sizes());
    dense(lengths, "lengths", op, at::kInt, x, {d.batch});
    dense(dstate_out, "dstate_out", op, at::kFloat, x, {d.batch, d.channels, d.state});
    dense(marks, "marks", op, at::kFloat, x, {(int64_t)(lib.scan_marks_bytes(&d) / sizeof(float))});
    const Tensor dy = rows(dy0);
    d.dy_stride[0] = apart(dy, 0); d.dy_stride[1] = apart(dy, 1);
    const c10::DeviceGuard guard(x.device());
    const Tensor dx = empty(x.sizes(), x), ddt = empty(x.sizes(), x), dB = empty(in.B.sizes(), x), dC = empty(in.B.sizes(), x);
    const Tensor dz = in.z ? empty(x.sizes(), x) : empty({0}, x);
    const Tensor dA = empty(A.sizes(), A), dD = empty({d.channels}, A), dbias = empty({d.channels}, A);
    const Tensor dstate = want_dstate ? empty({d.batch, d.channels, d.state}, A) : empty({0}, A);
    if (d.batch == 0) {
        dA.zero_();
        dD.zero_();
        dbias.zero_();
    } else {
        const Tensor ws = scratch(lib.scan_bwd_bytes(&d, lengths.has_value()), x);
        check(lib.scan_bwd(&d, ptr(x), ptr(in.dt), f32(A), ptr(in.B), ptr(in.C), f32(D), ptr(in.z), f32(dt_bias), i32(lengths), f32(marks), ptr(dy),
                           f32(dstate_out), ptr(dx), ptr(ddt), f32(dA), ptr(dB), ptr(dC), f32(dD), f32(dbias), in.z ? ptr(dz) : nullptr,
                           want_dstate ? f32(dstate) : nullptr, ptr(ws), ws.numel(), stream_of(x)), "unetmi_ssm_scan_bwd");
    }
    return {dx, ddt, dA, dB, dC, dD, dz, dbias, dstate};
}

Tensor ssm_scan_step(const Tensor& x0, const Tensor& dt0, const Tensor& A, const Tensor& B0, const Tensor& C0, const Maybe& D, const Maybe& z0,
                     const Maybe& dt_bias, const Tensor& state, const Maybe& slots, bool softplus) {
    const char* op = "ssm_scan_step";
    const ScanIn in(op, x0, dt0, A, B0, C0, D, z0, dt_bias, softplus, 2);
    const UnetmiScanDesc& d = in.d;
    const Tensor& x = in.x;
    TORCH_CHECK_VALUE(state.dim() == 3, "unetmi::", op, ": state must be [slots, channels, state]");
    dense(state, "state", op, at::kFloat, x, {state.size(0), d.channels, d.state});
    dense(slots, "slots", op, at::kInt, x, {d.batch});
    const int32_t slot_count = count(state.size(0), op);
    const c10::DeviceGuard guard(x.device());
    const Tensor y = empty(x.sizes(), x);
    check(lib.scan_step(&d, ptr(x), ptr(in.dt), f32(A), ptr(in.B), ptr(in.C), f32(D), ptr(in.z), f32(dt_bias), i32(slots), slot_count, f32(state),
                        ptr(y), stream_of(x)), "unetmi_ssm_scan_step");
    written(state);
    return y;
}

// ---------------------------------------------------------------------------------------------------------------------
// the block norm
// ---------------------------------------------------------------------------------------------------------------------
struct NormIn {
    UnetmiNormDesc d = {};
    Tensor x;
    Maybe gate, residual;
    NormIn(const char* op, const Tensor& x0, const Maybe& gate0, const Maybe& post, const Maybe& residual0, const Maybe& scale, const Maybe& pre,
           double eps, at::ScalarType residual_type) {
        d.dtype = kind(x0, op, 2);
        const at::IntArrayRef shape = x0.sizes();
        dense(post, "post_weight", op, at::kFloat, x0, {shape[1]});
        dense(scale, "scale", op, at::kFloat, x0, {shape[1]});
        dense(pre, "pre_weight", op, at::kFloat, x0, {shape[1]});
        x = rows(x0);
        if (gate0) {
            same(*gate0, "gate", op, x0.scalar_type(), x0, shape);
            gate = rows(*gate0);
            d.gate_stride = apart(*gate, 0);
        }
        if (residual0) {
            residual_type = residual0->scalar_type() == at::kFloat ? at::kFloat : x0.scalar_type();
            same(*residual0, "residual", op, residual_type, x0, shape);
            residual = rows(*residual0);
            d.residual_stride = apart(*residual, 0);
        }
        d.rows = shape[0]; d.channels = count(shape[1], op); d.eps = eps; d.x_stride = apart(x, 0);
        d.residual_dtype = residual_type == at::kBFloat16 ? UNETMI_DTYPE_BF16 : UNETMI_DTYPE_F32;
    }
};

// (r, n) with a residual (n empty without pre_weight), else (p, empty); and the row statistics the backward call needs or empty
std::tuple<Tensor, Tensor, Tensor> block_norm(const Tensor& x0, const Maybe& gate, const Maybe& post, const Maybe& residual, const Maybe& scale,
                                              const Maybe& pre, double eps, bool want_stats) {
    TORCH_CHECK_VALUE(residual || (!scale && !pre), "unetmi::block_norm: scale and pre_weight belong to a residual stream");
    const NormIn in("block_norm", x0, gate, post, residual, scale, pre, eps, x0.scalar_type());
    const Tensor& x = in.x;
    const c10::DeviceGuard guard(x.device());
    const Tensor out = in.residual ? empty(x.sizes(), *in.residual) : empty(x.sizes(), x);
    const Tensor out_n = pre ? empty(x.sizes(), x) : empty({0}, x);
    const Tensor stats = want_stats ? empty({x.size(0), 2}, x, at::kFloat) : empty({0}, x, at::kFloat);
    check(lib.norm_fwd(&in.d, ptr(x), ptr(in.gate), f32(post), ptr(in.residual), f32(scale), f32(pre), ptr(out), pre ? ptr(out_n) : nullptr,
                       want_stats ? f32(stats) : nullptr, stream_of(x)), "unetmi_block_norm_fwd");
    return {out, out_n, stats};
}

// (dx, dgate or empty, dresidual or empty, [dpost_weight, dscale, dpre_weight])
std::tuple<Tensor, Tensor, Tensor, Tensor> block_norm_bwd(const Tensor& x0, const Maybe& gate, const Maybe& post, const Maybe& residual, const Maybe& scale,
                                                          const Maybe& pre, double eps, const Tensor& stats, const Maybe& d_out, const Maybe& d_norm, bool has_residual,
                                                          bool residual_f32) {
    const char* op = "block_norm_bwd";
    const at::ScalarType rtype = residual_f32 ? at::kFloat : x0.scalar_type();
    const NormIn in(op, x0, gate, post, residual, scale, pre, eps, rtype);
    const Tensor& x = in.x;
    dense(stats, "stats", op, at::kFloat, x, {x.size(0), 2});
    dense(d_out, "d_out", op, has_residual ? rtype : x.scalar_type(), x, x.sizes());
    dense(d_norm, "d_norm", op, x.scalar_type(), x, x.sizes());
    const c10::DeviceGuard guard(x.device());
    const Tensor dx = empty(x.sizes(), x), dgate = gate ? empty(x.sizes(), x) : empty({0}, x);
    const Tensor dres = has_residual ? empty(x.sizes(), x, rtype) : empty({0}, x, rtype);
    const Tensor dw = empty({3, x.size(1)}, x, at::kFloat);
    if (x.size(0) == 0) {
        dw.zero_();
        return {dx, dgate, dres, dw};
    }
    const Tensor ws = scratch(lib.norm_bwd_bytes(&in.d), x);
    check(lib.norm_bwd(&in.d, ptr(x), ptr(in.gate), f32(post), ptr(in.residual), f32(scale), f32(pre), f32(stats), ptr(d_out), ptr(d_norm), ptr(dx),
                       gate ? ptr(dgate) : nullptr, has_residual ? ptr(dres) : nullptr, f32(dw), ptr(ws), ws.numel(), stream_of(x)),
          "unetmi_block_norm_bwd");
    return {dx, dgate, dres, dw};
}

// ---------------------------------------------------------------------------------------------------------------------
// autograd: the ops above below the dispatcher's autograd key, their _bwd ops as the nodes' backward
// ---------------------------------------------------------------------------------------------------------------------
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor value(const Maybe& t) { return t ? *t : Tensor(); }
// Which gradients are wanted, asked in the order of the forward call's tensors: the node counts those that were given.
struct Wanted {
    AutogradContext* ctx;
    size_t edge = 0;
    bool next(bool given = true) { return given && ctx->needs_input_grad(edge++); }
    Tensor next(const Tensor& gradient, bool given = true) { return next(given) ? gradient : Tensor(); }
};

// The gradients are values, no functions of the inputs: under create_graph they carry a node that says so when a second
// derivative is asked for.
variable_list once(const char* what, variable_list gradients) {
    if (!at::GradMode::is_enabled()) return gradients;
    for (Tensor& t : gradients)
        if (t.defined()) t = t.detach().requires_grad_();
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string("unet_amd: ") + what + " can be differentiated once only", gradients.size());
    return (*node)(std::move(gradients));
}

// A captured backward pass cannot hand its gradients to a node that lives on the default stream, as the leaves' nodes do
// while an eager graph of the same leaves is alive: waiting on that stream breaks the capture, and ends the process later.
// Said here, before that wait.
void joins_capture(const char* what, const Tensor& x) {
    if (!x.is_cuda()) return;                                         // no stream (kernels that stand in on the CPU)
    const auto here = c10::hip::getCurrentHIPStream();
    if (here.id() == 0) return;                                       // the default stream is never captured
    const auto node = torch::autograd::get_current_node();
    if (!node || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        const auto& to = node->next_edge(i).function;
        const auto stream = to && node->task_should_compute_output(i) ? to->stream() : std::nullopt;
        TORCH_CHECK(!stream || stream->id() != 0, "unet_amd: the backward pass of ", what, " is being captured into a graph, but an input's gradient "
                    "belongs to an eager graph on the default stream: free that graph (its outputs) before the capture, or run it on another stream");
    }
}

// whether autograd records a call on these tensors
bool recorded(std::initializer_list<const Tensor*> given, std::initializer_list<const Maybe*> optional) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : given)
        if (t->requires_grad()) return true;
    for (const Maybe* t : optional)
        if (*t && (*t)->requires_grad()) return true;
    return false;
}

template <class F>
auto typed(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// Forward-mode derivatives are not built.  A tensor that carries a tangent need not require a gradient, so every op asks by
// itself, before the kernel would drop the tangent without a word.
template <class T>
void no_tangent(const char*, const T&) {}
void no_tangent(const char* what, const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "unet_amd: ", what, " has no forward-mode derivative");
}
void no_tangent(const char* what, const Maybe& t) {
    if (t) no_tangent(what, *t);
}
template <class... A>
void no_tangents(const char* what, const A&... args) {
    if (torch::autograd::ForwardADLevel::try_get_by_idx(0)) (no_tangent(what, args), ...);         // tangents live inside a level
}
// the _bwd and _step ops below the autograd key: they record nothing
template <const auto& Name, auto Kernel>
struct Below;
template <const auto& Name, class R, class... A, R (*Kernel)(A...)>
struct Below<Name, Kernel> {
    static R call(c10::DispatchKeySet keys, A... args) {
        no_tangents(Name, args...);
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = typed<R(A...)>(Name);
        return op.redispatch(keys & c10::after_ADInplaceOrView_keyset, args...);
    }
};
constexpr char kConvBwd[] = "unetmi::seq_conv_bwd", kScanBwd[] = "unetmi::ssm_scan_bwd", kNormBwd[] = "unetmi::block_norm_bwd",
               kConvStep[] = "unetmi::seq_conv_step", kScanStep[] = "unetmi::ssm_scan_step";

// The token ops write the cache through its pointer and have no gradients.  Where autograd would record the call they say so:
// a result without a history would cut a training program's gradients off unseen.
void inference_only(const char* what, std::initializer_list<const Tensor*> given, std::initializer_list<const Maybe*> optional) {
    TORCH_CHECK(!recorded(given, optional), "unet_amd: ", what, " is inference only, but an input, a parameter or the cache requires a gradient: "
                "call it under torch.no_grad() or torch.inference_mode(), or on detached tensors");
}
Tensor seq_conv_step_autograd(c10::DispatchKeySet keys, const Tensor& x, const Tensor& weight, const Maybe& bias, const Tensor& state,
                              const Maybe& slots, bool silu) {
    inference_only("causal_conv_step", {&x, &weight, &state}, {&bias});
    return Below<kConvStep, seq_conv_step>::call(keys, x, weight, bias, state, slots, silu);
}
Tensor ssm_scan_step_autograd(c10::DispatchKeySet keys, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                              const Maybe& D, const Maybe& z, const Maybe& dt_bias, const Tensor& state, const Maybe& slots, bool softplus) {
    inference_only("selective_scan_step", {&x, &dt, &A, &B, &C, &state}, {&D, &z, &dt_bias});
    return Below<kScanStep, ssm_scan_step>::call(keys, x, dt, A, B, C, D, z, dt_bias, state, slots, softplus);
}

struct ConvNode : torch::autograd::Function<ConvNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias, const Maybe& state,
                                 const Maybe& lengths, bool silu, bool want_state) {
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = typed<decltype(seq_conv)>("unetmi::seq_conv");
        auto [y, out] = op.call(x, weight, bias, state, lengths, silu, want_state);
        ctx->save_for_backward({x, weight, value(bias), value(state), value(lengths)});
        ctx->saved_data["silu"] = silu;
        ctx->set_materialize_grads(false);
        return {y, out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(7);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const variable_list s = ctx->get_saved_variables();
        joins_capture("causal_conv", s[0]);
        const Tensor dy = grads[0].defined() ? grads[0] : at::zeros_like(s[0], at::MemoryFormat::Contiguous);
        const Maybe dout = grads[1].defined() && grads[1].dim() == 3 ? Maybe(grads[1].contiguous()) : Maybe();
        static auto op = typed<decltype(seq_conv_bwd)>("unetmi::seq_conv_bwd");
        auto [dx, dw, db, ds] = op.call(s[0], s[1], maybe(s[2]), maybe(s[3]), maybe(s[4]), ctx->saved_data["silu"].toBool(), dy, dout);
        Wanted wanted{ctx};
        out[0] = wanted.next(dx);
        out[1] = wanted.next(dw);
        out[2] = wanted.next(db, s[2].defined());
        out[3] = wanted.next(ds, s[3].defined());
        return once("causal_conv", std::move(out));
    }
};
std::tuple<Tensor, Tensor> seq_conv_autograd(const Tensor& x, const Tensor& weight, const Maybe& bias, const Maybe& state, const Maybe& lengths,
                                             bool silu, bool want_state) {
    no_tangents("causal_conv", x, weight, bias, state);
    if (!recorded({&x, &weight}, {&bias, &state})) {
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = typed<decltype(seq_conv)>("unetmi::seq_conv");
        return op.call(x, weight, bias, state, lengths, silu, want_state);
    }
    const variable_list r = ConvNode::apply(x, weight, bias, state, lengths, silu, want_state);
    return {r[0], r[1]};
}

struct ScanNode : torch::autograd::Function<ScanNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                                 const Maybe& D, const Maybe& z, const Maybe& dt_bias, const Maybe& state, const Maybe& lengths, bool softplus,
                                 bool want_state) {
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = typed<decltype(ssm_scan)>("unetmi::ssm_scan");
        auto [y, out, marks] = op.call(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, true);
        ctx->save_for_backward({x, dt, A, B, C, value(D), value(z), value(dt_bias), value(lengths), marks});
        ctx->saved_data["softplus"] = softplus;
        ctx->saved_data["state"] = state.has_value();
        ctx->set_materialize_grads(false);
        return {y, out};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(12);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const variable_list s = ctx->get_saved_variables();
        joins_capture("selective_scan", s[0]);
        const Tensor dy = grads[0].defined() ? grads[0] : at::zeros_like(s[0], at::MemoryFormat::Contiguous);
        const Maybe dout = grads[1].defined() && grads[1].dim() == 3 ? Maybe(grads[1].contiguous()) : Maybe();
        Wanted wanted{ctx};
        bool want[9];
        for (int i = 0; i < 5; ++i) want[i] = wanted.next();
        for (int i = 5; i < 8; ++i) want[i] = wanted.next(s[i].defined());
        want[8] = wanted.next(ctx->saved_data["state"].toBool());
        static auto op = typed<decltype(ssm_scan_bwd)>("unetmi::ssm_scan_bwd");
        const Nine r = op.call(s[0], s[1], s[2], s[3], s[4], maybe(s[5]), maybe(s[6]), maybe(s[7]), maybe(s[8]), ctx->saved_data["softplus"].toBool(),
                               s[9], dy, dout, want[8]);
        const Tensor all[9] = {std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r), std::get<4>(r),
                               std::get<5>(r), std::get<6>(r), std::get<7>(r), std::get<8>(r)};
        for (int i = 0; i < 9; ++i)
            if (want[i]) out[i] = all[i];
        return once("selective_scan", std::move(out));
    }
};
std::tuple<Tensor, Tensor, Tensor> ssm_scan_autograd(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                                                     const Maybe& D, const Maybe& z, const Maybe& dt_bias, const Maybe& state, const Maybe& lengths,
                                                     bool softplus, bool want_state, bool want_marks) {
    no_tangents("selective_scan", x, dt, A, B, C, D, z, dt_bias, state);
    if (!recorded({&x, &dt, &A, &B, &C}, {&D, &z, &dt_bias, &state})) {       // no node, and no states saved for one
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = typed<decltype(ssm_scan)>("unetmi::ssm_scan");
        return op.call(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, want_marks);
    }
    const variable_list r = ScanNode::apply(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state);
    return {r[0], r[1], at::empty({0}, A.options())};
}

struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& gate, const Maybe& post, const Maybe& residual,
                                 const Maybe& scale, const Maybe& pre, double eps) {
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = typed<decltype(block_norm)>("unetmi::block_norm");
        auto [out, out_n, stats] = op.call(x, gate, post, residual, scale, pre, eps, true);
        ctx->save_for_backward({x, value(gate), value(post), value(scale), value(pre), pre ? *residual : Tensor(), stats});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["residual"] = residual.has_value();
        ctx->saved_data["f32"] = residual && residual->scalar_type() == at::kFloat;
        ctx->set_materialize_grads(false);
        return {out, out_n};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(7);
        const variable_list s = ctx->get_saved_variables();
        joins_capture("block_norm", s[0]);
        const Maybe d_out = grads[0].defined() ? Maybe(grads[0].contiguous()) : Maybe();
        const Maybe d_norm = s[4].defined() && grads[1].defined() ? Maybe(grads[1].contiguous()) : Maybe();
        if (!d_out && !d_norm) return out;
        const bool has = ctx->saved_data["residual"].toBool();
        static auto op = typed<decltype(block_norm_bwd)>("unetmi::block_norm_bwd");
        auto [dx, dgate, dres, dw] = op.call(s[0], maybe(s[1]), maybe(s[2]), maybe(s[5]), maybe(s[3]), maybe(s[4]), ctx->saved_data["eps"].toDouble(),
                                             s[6], d_out, d_norm, has, ctx->saved_data["f32"].toBool());
        Wanted wanted{ctx};
        out[0] = wanted.next(dx);
        out[1] = wanted.next(dgate, s[1].defined());
        if (wanted.next(s[2].defined())) out[2] = dw.select(0, 0);
        out[3] = wanted.next(dres, has);
        if (wanted.next(s[3].defined())) out[4] = dw.select(0, 1);
        if (wanted.next(s[4].defined())) out[5] = dw.select(0, 2);
        return once("block_norm", std::move(out));
    }
};
std::tuple<Tensor, Tensor, Tensor> block_norm_autograd(const Tensor& x, const Maybe& gate, const Maybe& post, const Maybe& residual,
                                                       const Maybe& scale, const Maybe& pre, double eps, bool want_stats) {
    no_tangents("block_norm", x, gate, post, residual, scale, pre);
    if (!recorded({&x}, {&gate, &post, &residual, &scale, &pre})) {
        at::AutoDispatchBelowADInplaceOrView below;
        static auto op = typed<decltype(block_norm)>("unetmi::block_norm");
        return op.call(x, gate, post, residual, scale, pre, eps, want_stats);
    }
    const variable_list r = NormNode::apply(x, gate, post, residual, scale, pre, eps);
    return {r[0], r[1], at::empty({0}, x.options().dtype(at::kFloat))};
}

}  // namespace

// The library whose entry points the ops call, by the path it was loaded from: 0, or -1 if one is missing.
extern "C" int unetmi_torch_bind(const char* path) {
    void* so = dlopen(path, RTLD_NOW | RTLD_NOLOAD);
    if (!so) return -1;
    bool ok = true;
    auto get = [&](auto& f, const char* name) {
        f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(so, name));
        ok = ok && f;
    };
    get(lib.last_error, "unetmi_last_error");
    get(lib.conv_fwd, "unetmi_seq_conv_fwd");
    get(lib.conv_bwd_bytes, "unetmi_seq_conv_bwd_workspace_bytes");
    get(lib.conv_bwd, "unetmi_seq_conv_bwd");
    get(lib.conv_step, "unetmi_seq_conv_step");
    get(lib.scan_marks_bytes, "unetmi_ssm_scan_marks_bytes");
    get(lib.scan_fwd_bytes, "unetmi_ssm_scan_fwd_workspace_bytes");
    get(lib.scan_fwd, "unetmi_ssm_scan_fwd");
    get(lib.scan_bwd_bytes, "unetmi_ssm_scan_bwd_workspace_bytes");
    get(lib.scan_bwd, "unetmi_ssm_scan_bwd");
    get(lib.scan_step, "unetmi_ssm_scan_step");
    get(lib.norm_fwd, "unetmi_block_norm_fwd");
    get(lib.norm_bwd_bytes, "unetmi_block_norm_bwd_workspace_bytes");
    get(lib.norm_bwd, "unetmi_block_norm_bwd");
    return ok ? 0 : -1;
}

TORCH_LIBRARY_FRAGMENT(unetmi, m) {
    m.def("seq_conv(Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu, bool want_state) -> (Tensor, Tensor)");
    m.def("seq_conv_bwd(Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu, Tensor dy, Tensor? dstate_out) "
          "-> (Tensor, Tensor, Tensor, Tensor)");
    m.def("seq_conv_step(Tensor x, Tensor weight, Tensor? bias, Tensor(a!) state, Tensor? slots, bool silu) -> Tensor");
    m.def("ssm_scan(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, Tensor? state, Tensor? lengths, "
          "bool softplus, bool want_state, bool want_marks) -> (Tensor, Tensor, Tensor)");
    m.def("ssm_scan_bwd(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, Tensor? lengths, bool softplus, "
          "Tensor marks, Tensor dy, Tensor? dstate_out, bool want_dstate) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("ssm_scan_step(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, Tensor(a!) state, "
          "Tensor? slots, bool softplus) -> Tensor");
    m.def("block_norm(Tensor x, Tensor? gate, Tensor? post_weight, Tensor? residual, Tensor? scale, Tensor? pre_weight, float eps, "
          "bool want_stats) -> (Tensor, Tensor, Tensor)");
    m.def("block_norm_bwd(Tensor x, Tensor? gate, Tensor? post_weight, Tensor? residual, Tensor? scale, Tensor? pre_weight, float eps, "
          "Tensor stats, Tensor? d_out, Tensor? d_norm, bool has_residual, bool residual_f32) -> (Tensor, Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(unetmi, CUDA, m) {                                 // ROCm tensors dispatch here
    m.impl("seq_conv", seq_conv);
    m.impl("seq_conv_bwd", seq_conv_bwd);
    m.impl("seq_conv_step", seq_conv_step);
    m.impl("ssm_scan", ssm_scan);
    m.impl("ssm_scan_bwd", ssm_scan_bwd);
    m.impl("ssm_scan_step", ssm_scan_step);
    m.impl("block_norm", block_norm);
    m.impl("block_norm_bwd", block_norm_bwd);
}
TORCH_LIBRARY_IMPL(unetmi, Autograd, m) {
    m.impl("seq_conv", seq_conv_autograd);
    m.impl("ssm_scan", ssm_scan_autograd);
    m.impl("block_norm", block_norm_autograd);
    m.impl("seq_conv_bwd", Below<kConvBwd, seq_conv_bwd>::call);
    m.impl("ssm_scan_bwd", Below<kScanBwd, ssm_scan_bwd>::call);
    m.impl("block_norm_bwd", Below<kNormBwd, block_norm_bwd>::call);
    m.impl("seq_conv_step", seq_conv_step_autograd);
    m.impl("ssm_scan_step", ssm_scan_step_autograd);
}
