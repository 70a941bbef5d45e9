// dense_host.cpp -- the host part of the dense layers' ordinary calls, without Python in it.
//
// A short call's time is its host time: argument checks, allocations and packing in Python take two
// to four times what the launches do, and a Python autograd node adds some 60 us a training step.
// Each function here takes the calls that need no copy and no refusal (contiguous, 16-byte aligned,
// one device, that device current, supported types and sizes), allocates through torch and calls the
// C entry point; for any other call it returns None and vaayu_b200/dense.py, which checks, copies and
// refuses, carries on.  The kernels are the same ones, through the same C ABI.
#include <ATen/ATen.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>
#include <tuple>

#include "../../include/vaayu_b200.h"

namespace {

using at::Tensor;

// The C entry points, bound once from the loaded library.
struct Entries {
    decltype(&vy_last_error) last_error;
    decltype(&vy_gated_ffn_saved_floats) ffn_saved;
    decltype(&vy_gated_ffn_workspace_size) ffn_workspace;
    decltype(&vy_gated_ffn_forward) ffn_forward;
    decltype(&vy_gated_ffn_backward) ffn_backward;
    decltype(&vy_int8_quantize) quantize;
    decltype(&vy_int8_linear) linear;
    decltype(&vy_int8_gated_ffn_workspace_size) int8_ffn_workspace;
    decltype(&vy_int8_gated_ffn) int8_ffn;
};
Entries g{};

void bind(const std::vector<uintptr_t>& a) {
    TORCH_CHECK(a.size() == 9, "nine entry points");
    g.last_error = reinterpret_cast<decltype(g.last_error)>(a[0]);
    g.ffn_saved = reinterpret_cast<decltype(g.ffn_saved)>(a[1]);
    g.ffn_workspace = reinterpret_cast<decltype(g.ffn_workspace)>(a[2]);
    g.ffn_forward = reinterpret_cast<decltype(g.ffn_forward)>(a[3]);
    g.ffn_backward = reinterpret_cast<decltype(g.ffn_backward)>(a[4]);
    g.quantize = reinterpret_cast<decltype(g.quantize)>(a[5]);
    g.linear = reinterpret_cast<decltype(g.linear)>(a[6]);
    g.int8_ffn_workspace = reinterpret_cast<decltype(g.int8_ffn_workspace)>(a[7]);
    g.int8_ffn = reinterpret_cast<decltype(g.int8_ffn)>(a[8]);
}

void check(int status, const char* what) {
    TORCH_CHECK(status == VY_OK, what, " failed (status ", status, "): ", g.last_error());
}

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return VY_BF16;
        case at::kHalf: return VY_F16;
        case at::kFloat: return VY_F32;
        default: return -1;
    }
}

// A tensor with a forward-mode tangent, which the kernels would drop.
bool dual(const Tensor& t) { return t._fw_grad(0).defined(); }
// Gradients are wanted for an operand of a call that has none: dense.py marks its result.
bool cut_off(const Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }
// A plain CUDA tensor whose memory the kernels can take as it is.
bool plain(const Tensor& t, int device) {
    if (!t.is_cuda() || t.get_device() != device || !t.is_contiguous() || t.is_neg() || dual(t)) return false;
    const auto keys = t.unsafeGetTensorImpl()->key_set();
    return !keys.has(c10::DispatchKey::Python) && !keys.has(c10::DispatchKey::FuncTorchBatched) &&
           !keys.has(c10::DispatchKey::FuncTorchGradWrapper) && !keys.has(c10::DispatchKey::Functionalize);
}
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }
bool is16(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// [inter, hidden], [inter, hidden], [hidden, inter] around x's last dimension.
bool ffn_shapes(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t unit) {
    if (x.dim() < 1 || wg.dim() != 2 || wu.dim() != 2 || wd.dim() != 2) return false;
    const int64_t h = x.size(-1), i = wg.size(0);
    return wg.size(1) == h && wu.size(0) == i && wu.size(1) == h && wd.size(0) == h && wd.size(1) == i && h % unit == 0 &&
           i % unit == 0 && h > 0 && i > 0 && h < 131072 && i < 131072 && x.numel() > 0;
}

vy_ffn_call ffn_call(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
    vy_ffn_call c{};
    c.act_dtype = code_of(x.scalar_type());
    c.activation = static_cast<int32_t>(act);
    c.hidden = static_cast<int32_t>(x.size(-1));
    c.inter = static_cast<int32_t>(wg.size(0));
    c.n_tokens = x.numel() / c.hidden;
    c.x = x.const_data_ptr();
    c.x_row_stride = c.hidden;
    c.w_gate = wg.const_data_ptr();
    c.w_up = wu.const_data_ptr();
    c.w_down = wd.const_data_ptr();
    return c;
}

Tensor scratch(size_t bytes, const Tensor& like) {
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// (out, saved): saved is undefined unless asked for.
std::tuple<Tensor, Tensor> ffn_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act,
                                       bool save) {
    vy_ffn_call c = ffn_call(x, wg, wu, wd, act);
    Tensor out = at::empty_like(x), saved;
    c.out = out.mutable_data_ptr();
    c.out_row_stride = c.hidden;
    c.workspace_bytes = g.ffn_workspace(&c, 0);
    const Tensor ws = scratch(c.workspace_bytes, x);
    c.workspace = ws.mutable_data_ptr();
    if (save) {
        saved = at::empty({g.ffn_saved(c.n_tokens, c.inter)}, x.options().dtype(at::kFloat));
        c.saved = saved.mutable_data_ptr<float>();
    }
    check(g.ffn_forward(&c, stream_of(x.get_device())), "gated_ffn");
    return {out, saved};
}

// A tensor of the backward pass as the kernels take it.  What a hook on saved tensors gives back, or a
// node called by hand is given, may be anything: it is checked before its address is used.
Tensor backward_operand(const Tensor& t, at::ScalarType type, int device, const char* what) {
    TORCH_CHECK(t.is_cuda() && t.get_device() == device && t.scalar_type() == type, "gated_ffn backward: ", what,
                " is not on cuda:", device, " in ", type);
    TORCH_CHECK_NOT_IMPLEMENTED(!dual(t), "gated_ffn backward: no forward-mode derivatives (", what, " is a dual tensor)");
    if (t.is_contiguous() && !t.is_neg() && aligned(t)) return t;
    const Tensor c = t.resolve_neg().contiguous();
    return aligned(c) ? c : c.clone();
}

struct GatedFfn : torch::autograd::Function<GatedFfn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                          const Tensor& wd, int64_t act) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [out, saved] = ffn_forward(x, wg, wu, wd, act, true);
        ctx->save_for_backward({x, wg, wu, wd, saved});
        ctx->saved_data["act"] = act;
        return out;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        auto v = ctx->get_saved_variables();
        const bool again = at::GradMode::is_enabled();      // create_graph
        torch::autograd::variable_list out(5);
        {
            at::AutoDispatchBelowADInplaceOrView below;
            TORCH_CHECK(v[0].is_cuda() && is16(v[0]), "gated_ffn backward: x is not a 16-bit CUDA tensor");
            const at::ScalarType type = v[0].scalar_type();
            const int device = v[0].get_device();
            const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
            const char* const names[5] = {"x", "w_gate", "w_up", "w_down", "what the forward call saved"};
            for (int i = 0; i < 5; ++i) v[i] = backward_operand(v[i], i < 4 ? type : at::kFloat, device, names[i]);
            const Tensor dy = backward_operand(grads[0], type, device, "the incoming gradient");
            TORCH_CHECK(ffn_shapes(v[0], v[1], v[2], v[3], 8) && dy.sizes() == v[0].sizes() &&
                            v[4].numel() == g.ffn_saved(v[0].numel() / v[0].size(-1), static_cast<int32_t>(v[1].size(0))),
                        "gated_ffn backward: tensors of other sizes than the forward call's");
            vy_ffn_call c = ffn_call(v[0], v[1], v[2], v[3], ctx->saved_data["act"].toInt());
            for (int i = 0; i < 4; ++i)
                if (ctx->needs_input_grad(i)) out[i] = at::empty_like(v[i]);
            c.saved = v[4].mutable_data_ptr<float>();
            c.d_out = dy.const_data_ptr();
            c.d_out_row_stride = c.d_x_row_stride = c.hidden;
            void** const to[4] = {&c.d_x, &c.d_w_gate, &c.d_w_up, &c.d_w_down};
            for (int i = 0; i < 4; ++i)
                if (out[i].defined()) *to[i] = out[i].mutable_data_ptr();
            c.workspace_bytes = g.ffn_workspace(&c, 1);
            const Tensor ws = scratch(c.workspace_bytes, dy);
            c.workspace = ws.mutable_data_ptr();
            check(g.ffn_backward(&c, stream_of(dy.get_device())), "gated_ffn backward");
        }
        if (again) {      // the gradients are not differentiable again: say so when it is tried
            torch::autograd::variable_list wanted;
            for (const Tensor& t : out)
                if (t.defined()) {
                    Tensor d = t.detach();
                    d.set_requires_grad(true);
                    wanted.push_back(d);
                }
            auto fn = std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice a function that was marked with @once_differentiable",
                static_cast<int64_t>(wanted.size()));
            wanted = (*fn)(std::move(wanted));
            size_t n = 0;
            for (Tensor& t : out)
                if (t.defined()) t = wanted[n++];
        }
        return out;
    }
};

std::optional<Tensor> gated_ffn(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
    if (!x.is_cuda() || !ffn_shapes(x, wg, wu, wd, 8) || !is16(x)) return std::nullopt;
    const int device = c10::cuda::current_device();
    for (const Tensor* t : {&x, &wg, &wu, &wd})
        if (t->scalar_type() != x.scalar_type() || !plain(*t, device) || !aligned(*t)) return std::nullopt;
    if (at::GradMode::is_enabled() &&
        (x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad()))
        return GatedFfn::apply(x, wg, wu, wd, act);
    at::AutoDispatchBelowADInplaceOrView below;
    return std::get<0>(ffn_forward(x, wg, wu, wd, act, false));
}

std::optional<std::tuple<Tensor, Tensor>> quantize(const Tensor& x) {
    const int code = code_of(x.scalar_type());
    if (!x.is_cuda() || code < 0 || x.dim() < 1 || x.numel() == 0) return std::nullopt;
    const int device = c10::cuda::current_device();
    if (!plain(x, device) || cut_off(x)) return std::nullopt;
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    if (rows > 0x7FFFFFFF) return std::nullopt;
    Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
    auto shape = x.sizes().vec();
    shape.back() = 1;
    Tensor scale = at::empty(shape, x.options().dtype(at::kFloat));
    check(g.quantize(x.const_data_ptr(), code, cols, rows, cols, codes.mutable_data_ptr<int8_t>(),
                     scale.mutable_data_ptr<float>(), stream_of(device)),
          "quantize_int8");
    return std::make_tuple(codes, scale);
}

// fp32 scales of `n` rows.
bool plain_scales(const Tensor& s, int64_t n, int device) {
    return s.scalar_type() == at::kFloat && s.numel() == n && plain(s, device) && !cut_off(s);
}

std::optional<Tensor> int8_linear(const Tensor& codes, const Tensor& scale, const Tensor& w, const Tensor& ws,
                                  const std::optional<Tensor>& bias, int64_t out_code) {
    if (!codes.is_cuda() || codes.scalar_type() != at::kChar || w.scalar_type() != at::kChar || codes.dim() < 1 || w.dim() != 2 ||
        codes.numel() == 0 || w.size(1) != codes.size(-1) || out_code < 0 || out_code > VY_F32)
        return std::nullopt;
    const int device = c10::cuda::current_device();
    vy_int8_linear_call c{};
    const int64_t k = w.size(1), n = w.size(0), rows = codes.numel() / k;
    if (k % 16 || k >= 131072 || n == 0 || n > 0x7FFFFF00 || !plain(codes, device) || !plain(w, device) || !aligned(codes) ||
        !aligned(w) || !plain_scales(scale, rows, device) || !plain_scales(ws, n, device))
        return std::nullopt;
    if (bias.has_value()) {
        if (bias->dim() != 1 || bias->size(0) != n || code_of(bias->scalar_type()) < 0 || !plain(*bias, device) ||
            cut_off(*bias))
            return std::nullopt;
        c.bias = bias->const_data_ptr();
        c.bias_dtype = code_of(bias->scalar_type());
    }
    at::AutoDispatchBelowADInplaceOrView below;
    const at::ScalarType type = out_code == VY_BF16 ? at::kBFloat16 : out_code == VY_F16 ? at::kHalf : at::kFloat;
    auto shape = codes.sizes().vec();
    shape.back() = n;
    Tensor out = at::empty(shape, codes.options().dtype(type));
    c.n_tokens = rows;
    c.k = static_cast<int32_t>(k);
    c.n = static_cast<int32_t>(n);
    c.codes = codes.const_data_ptr<int8_t>();
    c.codes_row_stride = k;
    c.scales = scale.const_data_ptr<float>();
    c.weight = w.const_data_ptr<int8_t>();
    c.weight_scales = ws.const_data_ptr<float>();
    c.out_dtype = static_cast<int32_t>(out_code);
    c.out = out.mutable_data_ptr();
    c.out_row_stride = n;
    check(g.linear(&c, stream_of(device)), "int8_linear");
    return out;
}

std::optional<Tensor> int8_gated_ffn(const Tensor& x, const Tensor& wg, const Tensor& sg, const Tensor& wu, const Tensor& su,
                                     const Tensor& wd, const Tensor& sd, int64_t act) {
    if (!x.is_cuda() || !ffn_shapes(x, wg, wu, wd, 16) || !is16(x)) return std::nullopt;
    const int device = c10::cuda::current_device();
    if (!plain(x, device) || cut_off(x)) return std::nullopt;
    for (const Tensor* t : {&wg, &wu, &wd})
        if (t->scalar_type() != at::kChar || !plain(*t, device) || !aligned(*t)) return std::nullopt;
    vy_int8_ffn_call c{};
    c.hidden = static_cast<int32_t>(x.size(-1));
    c.inter = static_cast<int32_t>(wg.size(0));
    if (!plain_scales(sg, c.inter, device) || !plain_scales(su, c.inter, device) || !plain_scales(sd, c.hidden, device))
        return std::nullopt;
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor out = at::empty_like(x);
    c.act_dtype = code_of(x.scalar_type());
    c.activation = static_cast<int32_t>(act);
    c.n_tokens = x.numel() / c.hidden;
    c.x = x.const_data_ptr();
    c.x_row_stride = c.out_row_stride = c.hidden;
    c.w_gate = wg.const_data_ptr<int8_t>();
    c.w_up = wu.const_data_ptr<int8_t>();
    c.w_down = wd.const_data_ptr<int8_t>();
    c.gate_scales = sg.const_data_ptr<float>();
    c.up_scales = su.const_data_ptr<float>();
    c.down_scales = sd.const_data_ptr<float>();
    c.out = out.mutable_data_ptr();
    c.workspace_bytes = g.int8_ffn_workspace(&c);
    const Tensor ws = scratch(c.workspace_bytes, x);
    c.workspace = ws.mutable_data_ptr();
    check(g.int8_ffn(&c, stream_of(device)), "int8_gated_ffn");
    return out;
}

}  // namespace

PYBIND11_MODULE(_dense_host, m) {
    using Free = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("bind", &bind);
    m.def("gated_ffn", &gated_ffn, Free());
    m.def("quantize_int8", &quantize, Free());
    m.def("int8_linear", &int8_linear, Free());
    m.def("int8_gated_ffn", &int8_gated_ffn, Free());
}
