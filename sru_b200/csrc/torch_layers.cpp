// Torch operators of the parts around the recurrent layers, with their autograd: one native call per forward and per
// backward pass (a call costs 8 us on the host).  linear_recurrence.py, embedding.py and orthogonalize.py call these; a timer or
// NVTX ranges see them through hooks on their graph nodes, so that what is profiled is what runs otherwise.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>
#include <torch/types.h>

#include <algorithm>

#include "../../include/sru_b200.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return SRU_F32;
        case at::kHalf: return SRU_F16;
        case at::kBFloat16: return SRU_BF16;
        default: TORCH_CHECK(false, "float32, float16 or bfloat16 expected, got ", t);
    }
    return -1;
}

void check(int rc) { TORCH_CHECK(rc == 0, "sru_b200 call failed (", rc, "): ", sru_b200_last_error()); }

void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *floats(const Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// A dual tensor need not require grad, and its tangent would be dropped without a word.
void refuse_tangent(const OptTensor &t, const char *name, const char *op) {
    TORCH_CHECK(!t.has_value() || !t->defined() || !t->_fw_grad(0).defined(), op, " has no forward-mode derivative, and ", name,
                " carries a tangent");
}

// What a backward pass returns under create_graph: the gradients, with an error where they are differentiated again.
variable_list once(variable_list grads, const char *name) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is differentiable once", (int64_t)grads.size());
    variable_list live;
    for (auto &g : grads)
        if (g.defined()) live.push_back(g.requires_grad() ? g : g.detach().requires_grad_());
    variable_list out = (*error)(std::move(live));
    size_t k = 0;
    for (auto &g : grads)
        if (g.defined()) g = out[k++];
    return grads;
}

// ---- gated linear recurrence ----------------------------------------------------------------------------------------
// (L, B, n) with unit stride in the last dimension and every group of `unit` elements aligned to its size
Tensor rows(const Tensor &t, int64_t unit) {
    if (t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % (unit * t.element_size()) == 0 &&
        t.stride(0) % unit == 0 && t.stride(1) % unit == 0)
        return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

Tensor small(const OptTensor &t) {
    if (!t.has_value() || !t->defined()) return Tensor();
    return t->detach().to(at::kFloat).contiguous();
}

void check_like(const Tensor &u, const OptTensor &t, const char *name, at::IntArrayRef shape, bool floating) {
    if (!t.has_value() || !t->defined()) return;
    TORCH_CHECK(t->device() == u.device(), name, " is on ", t->device(), ", u on ", u.device());
    TORCH_CHECK(t->sizes() == shape, name, " must have shape ", shape, ", got ", t->sizes());
    TORCH_CHECK(!floating || t->is_floating_point(), name, " must be a floating-point tensor, got ", t->scalar_type());
}

struct Scanned { Tensor h, last, states; };

Scanned scan(const Tensor &u, const Tensor &c0, const Tensor &bias, const Tensor &mask, bool reverse, bool need_states) {
    const int64_t L = u.size(0), B = u.size(1), d = u.size(2) / 2;
    Scanned s;
    s.h = at::empty({L, B, d}, u.options());
    if (L == 0 || B == 0) {
        s.last = c0.defined() ? c0.clone() : at::zeros({B, d}, u.options().dtype(at::kFloat));
        return s;
    }
    s.last = at::empty({B, d}, u.options().dtype(at::kFloat));
    if (need_states)
        s.states = at::empty({(int64_t)(sru_b200_linear_recurrence_states_bytes(L, B, d) / 4)}, u.options().dtype(at::kFloat));
    check(sru_b200_linear_recurrence_forward(s.h.data_ptr(), floats(s.last), pointer(s.states), u.data_ptr(), floats(bias),
                                             floats(c0), static_cast<const uint8_t *>(pointer(mask)), L, B, d, u.stride(0),
                                             u.stride(1), reverse, code_of(u.scalar_type()),
                                             at::cuda::getCurrentCUDAStream().stream()));
    return s;
}

class GatedLinearRecurrence : public torch::autograd::Function<GatedLinearRecurrence> {
  public:
    static variable_list forward(AutogradContext *ctx, const Tensor &u, const OptTensor &c0, const OptTensor &bias,
                                 const OptTensor &mask, bool reverse) {
        ctx->set_materialize_grads(false);
        const bool single = u.dim() == 2;
        const Tensor r = rows(single ? u.detach().unsqueeze(0) : u.detach(), 2), b = small(bias), m = mask.has_value() ? *mask : Tensor();
        Scanned s = scan(r, small(c0), b, m, reverse, true);
        ctx->save_for_backward({r, b, m, s.states});
        ctx->saved_data["single"] = single;
        ctx->saved_data["reverse"] = reverse;
        ctx->saved_data["u"] = u.requires_grad();
        ctx->saved_data["c0"] = c0.has_value() && c0->requires_grad() ? (int64_t)c0->scalar_type() : (int64_t)-1;
        ctx->saved_data["bias"] = bias.has_value() && bias->requires_grad() ? (int64_t)bias->scalar_type() : (int64_t)-1;
        return {single ? s.h.squeeze(0) : s.h, s.last};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const bool single = ctx->saved_data["single"].toBool();
        const auto saved = ctx->get_saved_variables();
        const Tensor &u = saved[0], &bias = saved[1], &mask = saved[2], &states = saved[3];
        const int64_t c0_type = ctx->saved_data["c0"].toInt(), bias_type = ctx->saved_data["bias"].toInt();
        c10::cuda::CUDAGuard guard(u.device());
        const int64_t L = u.size(0), B = u.size(1), d = u.size(2) / 2;
        const auto f32 = u.options().dtype(at::kFloat);
        Tensor gu = at::empty({L, B, 2 * d}, u.options()), gb, gi, gl, gh;
        if (bias_type >= 0) gb = at::empty({d}, f32);
        if (c0_type >= 0) gi = at::empty({B, d}, f32);
        if (grads[1].defined()) gl = grads[1].detach().to(at::kFloat).contiguous();
        if (L == 0 || B == 0) {
            if (gb.defined()) gb.zero_();
            if (gi.defined()) gl.defined() ? gi.copy_(gl) : gi.zero_();
        } else {
            if (grads[0].defined()) gh = rows((single ? grads[0].detach().unsqueeze(0) : grads[0].detach()).to(u.scalar_type()), 1);
            const size_t bytes = gb.defined() ? sru_b200_linear_recurrence_backward_workspace_bytes(L, B, d, code_of(u.scalar_type())) : 0;
            Tensor ws;
            if (bytes) ws = at::empty({(int64_t)bytes}, u.options().dtype(at::kByte));
            check(sru_b200_linear_recurrence_backward(
                gu.data_ptr(), floats(gb), floats(gi), u.data_ptr(), floats(bias), pointer(states),
                static_cast<const uint8_t *>(pointer(mask)), pointer(gh), floats(gl), L, B, d, u.stride(0), u.stride(1),
                gh.defined() ? gh.stride(0) : 0, gh.defined() ? gh.stride(1) : 0, ctx->saved_data["reverse"].toBool(),
                code_of(u.scalar_type()), pointer(ws), bytes, at::cuda::getCurrentCUDAStream().stream()));
        }
        if (gi.defined()) gi = gi.to((at::ScalarType)c0_type);
        if (gb.defined()) gb = gb.to((at::ScalarType)bias_type);
        if (!ctx->saved_data["u"].toBool()) gu = Tensor();
        else if (single) gu = gu.squeeze(0);
        return once({gu, gi, gb, Tensor(), Tensor()}, "gated_linear_recurrence");
    }
};

std::tuple<Tensor, Tensor> gated_linear_recurrence(const Tensor &u, const OptTensor &c0, const OptTensor &bias,
                                                   const OptTensor &mask_pad, bool reverse) {
    TORCH_CHECK(u.is_cuda(), "sru_b200 has no CPU path: u must be a CUDA tensor");
    code_of(u.scalar_type());
    TORCH_CHECK((u.dim() == 2 || u.dim() == 3) && u.size(-1) >= 2 && u.size(-1) % 2 == 0,
                "u must be (length, batch, 2 * hidden) or (batch, 2 * hidden), got ", u.sizes());
    const bool single = u.dim() == 2;
    const int64_t B = u.size(-2), d = u.size(-1) / 2;
    check_like(u, c0, "c0", {B, d}, true);
    check_like(u, bias, "bias", {d}, true);
    if (single) check_like(u, mask_pad, "mask_pad", {B}, false);
    else check_like(u, mask_pad, "mask_pad", {u.size(0), B}, false);
    refuse_tangent(u, "u", "gated_linear_recurrence");
    refuse_tangent(c0, "c0", "gated_linear_recurrence");
    refuse_tangent(bias, "bias", "gated_linear_recurrence");
    c10::cuda::CUDAGuard guard(u.device());
    OptTensor mask;
    if (mask_pad.has_value() && mask_pad->defined()) mask = mask_pad->to(at::kBool).contiguous();      // one step: (B) as (1, B)
    auto learns = [](const OptTensor &t) { return t.has_value() && t->requires_grad(); };
    if (at::GradMode::is_enabled() && (u.requires_grad() || learns(c0) || learns(bias))) {
        variable_list out = GatedLinearRecurrence::apply(u, c0, bias, mask, reverse);
        return {out[0], out[1]};
    }
    const Tensor r = rows(single ? u.detach().unsqueeze(0) : u.detach(), 2);
    Scanned s = scan(r, small(c0), small(bias), mask.has_value() ? *mask : Tensor(), reverse, false);
    return {single ? s.h.squeeze(0) : s.h, s.last};
}

// ---- embedding ------------------------------------------------------------------------------------------------------
Tensor lookup(const Tensor &tokens, const Tensor &table, double scale, at::ScalarType out) {
    const int64_t n = tokens.numel(), d = table.size(1);
    Tensor y = at::empty({n, d}, table.options().dtype(out));
    if (n)
        check(sru_b200_embedding_forward(y.data_ptr(), tokens.data_ptr(), table.data_ptr(), n, table.size(0), d, table.stride(0),
                                         scale, (int)tokens.element_size(), code_of(table.scalar_type()), code_of(out),
                                         at::cuda::getCurrentCUDAStream().stream()));
    return y;
}

class EmbeddingLookup : public torch::autograd::Function<EmbeddingLookup> {
  public:
    static Tensor forward(AutogradContext *ctx, const Tensor &tokens, const Tensor &table, double scale, int64_t padding,
                          at::ScalarType out) {
        ctx->save_for_backward({tokens});
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["hidden"] = table.size(1);
        ctx->saved_data["type"] = (int64_t)table.scalar_type();
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        return lookup(tokens, table.detach(), scale, out);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const Tensor tokens = ctx->get_saved_variables()[0];
        const int64_t v = ctx->saved_data["rows"].toInt(), d = ctx->saved_data["hidden"].toInt(), n = tokens.numel();
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        c10::cuda::CUDAGuard guard(tokens.device());
        const Tensor dy = grads[0].detach().contiguous();
        Tensor out = at::empty({v, d}, dy.options().dtype(type));
        const size_t bytes = sru_b200_embedding_backward_workspace_bytes(n, v, d);
        Tensor ws = at::empty({(int64_t)bytes}, dy.options().dtype(at::kByte));
        check(sru_b200_embedding_backward(out.data_ptr(), tokens.data_ptr(), dy.data_ptr(), n, v, d, ctx->saved_data["padding"].toInt(),
                                          ctx->saved_data["scale"].toDouble(), (int)tokens.element_size(), code_of(type),
                                          code_of(dy.scalar_type()), ws.data_ptr(), bytes,
                                          at::cuda::getCurrentCUDAStream().stream()));
        return once({Tensor(), out, Tensor(), Tensor(), Tensor()}, "embedding_lookup");
    }
};

Tensor embedding_lookup(const Tensor &tokens, const Tensor &weight, double scale, c10::optional<int64_t> padding,
                        c10::optional<at::ScalarType> out_type) {
    TORCH_CHECK(weight.is_cuda() && tokens.is_cuda(), "sru_b200 has no CPU path: tokens and weight must be CUDA tensors");
    TORCH_CHECK(tokens.device() == weight.device(), "tokens are on ", tokens.device(), ", weight on ", weight.device());
    TORCH_CHECK(tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong, "tokens must be int32 or int64, got ", tokens.scalar_type());
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0, "weight must be (vocabulary, hidden), got ", weight.sizes());
    const at::ScalarType type = weight.scalar_type(), out_dtype = out_type.value_or(type);
    code_of(type);
    TORCH_CHECK(out_dtype == type || (type == at::kFloat && (out_dtype == at::kHalf || out_dtype == at::kBFloat16)),
                "a ", type, " table cannot be read into ", out_dtype);
    int64_t padding_idx = -1;
    if (padding.has_value()) {
        const int64_t v = weight.size(0);
        TORCH_CHECK(*padding >= -v && *padding < v, "padding_idx ", *padding, " is outside a table of ", v, " rows");
        padding_idx = *padding < 0 ? *padding + v : *padding;
    }
    refuse_tangent(weight, "weight", "embedding_lookup");
    c10::cuda::CUDAGuard guard(weight.device());
    const Tensor table = weight.stride(1) == 1 && weight.stride(0) >= weight.size(1) ? weight : weight.contiguous();
    const Tensor flat = tokens.detach().reshape({-1}).contiguous();
    Tensor y = at::GradMode::is_enabled() && table.requires_grad() ? EmbeddingLookup::apply(flat, table, scale, padding_idx, out_dtype)
                                                                   : lookup(flat, table.detach(), scale, out_dtype);
    std::vector<int64_t> shape = tokens.sizes().vec();
    shape.push_back(weight.size(1));
    return y.view(shape);
}

// ---- orthogonalised update -------------------------------------------------------------------------------------------
Tensor orthogonalize(const Tensor &grad, int64_t steps, double a, double b, double c, double eps, c10::optional<at::ScalarType> out_type) {
    TORCH_CHECK(grad.is_cuda(), "sru_b200 has no CPU path: grad must be a CUDA tensor");
    TORCH_CHECK(grad.dim() == 2 || grad.dim() == 3, "grad must be (rows, cols) or (batch, rows, cols), got ", grad.sizes());
    const at::ScalarType type = grad.scalar_type(), out_dtype = out_type.value_or(type == at::kFloat ? at::kBFloat16 : type);
    const int code = code_of(type);
    TORCH_CHECK(out_dtype == at::kHalf || out_dtype == at::kBFloat16, "the result is float16 or bfloat16, got ", out_dtype);
    c10::cuda::CUDAGuard guard(grad.device());
    Tensor out = at::empty(grad.sizes(), grad.options().dtype(out_dtype));
    Tensor g = grad.detach();
    if (g.numel() > 0 && g.stride(-1) != 1 && g.stride(-2) != 1) g = g.contiguous();
    const int64_t batch = g.dim() == 3 ? g.size(0) : 1, rows = g.size(-2), cols = g.size(-1);
    const size_t bytes = sru_b200_orthogonalize_workspace_bytes_for(batch, rows, cols, code_of(out_dtype));
    Tensor ws = at::empty({(int64_t)bytes}, g.options().dtype(at::kByte));
    check(sru_b200_orthogonalize(out.data_ptr(), g.data_ptr(), batch, rows, cols, g.dim() == 3 ? g.stride(0) : 0, g.stride(-2),
                                 g.stride(-1), (int)std::min<int64_t>(std::max<int64_t>(steps, -1), 1 << 30), a, b, c, eps, code,
                                 code_of(out_dtype), ws.data_ptr(), bytes, at::cuda::getCurrentCUDAStream().stream()));
    return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sru_b200, m) {
    m.def("orthogonalize(Tensor grad, int steps=5, float a=3.4445, float b=-4.7750, float c=2.0315, float eps=1e-7, "
          "ScalarType? out_dtype=None) -> Tensor",
          &orthogonalize);
    m.def("gated_linear_recurrence(Tensor u, Tensor? c0=None, Tensor? bias=None, Tensor? mask_pad=None, bool reverse=False) "
          "-> (Tensor, Tensor)",
          &gated_linear_recurrence);
    m.def("embedding_lookup(Tensor tokens, Tensor weight, float scale=1.0, int? padding_idx=None, ScalarType? out_dtype=None) -> Tensor",
          &embedding_lookup);
}
