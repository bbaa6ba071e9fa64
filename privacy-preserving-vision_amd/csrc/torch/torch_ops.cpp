// Autograd nodes and the optimiser's list in C++, on top of the C ABI (ppv_hip.h): lib/ppv_torch.so.
//
// Why not in Python like the other modules: these operators take 5 to 50 us on the GPU.  As torch.autograd.Function classes over ctypes a layer norm's
// forward and backward cost 120 us of interpreter time, an attention's 150 us, an AdamW step over 333 tensors 430 us; a C++ node runs in
// the engine's thread without the interpreter.  Arguments are checked in Python (nn_ops.layer_norm, attention.multihead_attention,
// optim.AdamW); here is what happens after that.  The library's entry points come from the loaded libppv_hip.so by address (bind), so that
// there is one copy of it.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include <algorithm>
#include <unordered_set>

#include "ppv_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct {
    decltype(&ppv_layernorm_fwd) layernorm_fwd;
    decltype(&ppv_layernorm_bwd) layernorm_bwd;
    decltype(&ppv_layernorm_bwd_workspace_bytes) layernorm_ws;
    decltype(&ppv_attention_fwd) attention_fwd;
    decltype(&ppv_attention_fwd_workspace_bytes) attention_fwd_ws;
    decltype(&ppv_attention_bwd) attention_bwd;
    decltype(&ppv_attention_bwd_workspace_bytes) attention_bwd_ws;
    decltype(&ppv_adamw_multi) adamw_multi;
} abi = {};

void bind(const std::vector<std::pair<std::string, size_t>>& entries) {
    for (const auto& [name, at] : entries) {
        if (name == "ppv_layernorm_fwd") abi.layernorm_fwd = reinterpret_cast<decltype(abi.layernorm_fwd)>(at);
        else if (name == "ppv_layernorm_bwd") abi.layernorm_bwd = reinterpret_cast<decltype(abi.layernorm_bwd)>(at);
        else if (name == "ppv_layernorm_bwd_workspace_bytes") abi.layernorm_ws = reinterpret_cast<decltype(abi.layernorm_ws)>(at);
        else if (name == "ppv_attention_fwd") abi.attention_fwd = reinterpret_cast<decltype(abi.attention_fwd)>(at);
        else if (name == "ppv_attention_fwd_workspace_bytes") abi.attention_fwd_ws = reinterpret_cast<decltype(abi.attention_fwd_ws)>(at);
        else if (name == "ppv_attention_bwd") abi.attention_bwd = reinterpret_cast<decltype(abi.attention_bwd)>(at);
        else if (name == "ppv_attention_bwd_workspace_bytes") abi.attention_bwd_ws = reinterpret_cast<decltype(abi.attention_bwd_ws)>(at);
        else if (name == "ppv_adamw_multi") abi.adamw_multi = reinterpret_cast<decltype(abi.adamw_multi)>(at);
        else TORCH_CHECK(false, "ppv_torch: unknown entry point ", name);
    }
}

void check(int status, const char* what) { TORCH_CHECK(status == 0, "libppv_hip: ", what, " failed with status ", status); }

ppv_stream_t stream() { return reinterpret_cast<ppv_stream_t>(c10::hip::getCurrentHIPStream().stream()); }

int code(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2; }

template <class P> P* data(const Tensor& t) { return t.defined() ? static_cast<P*>(t.data_ptr()) : nullptr; }

constexpr c10::DispatchKeySet stand_ins({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::BatchedNestedTensor,
                                         c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched, c10::DispatchKey::Functionalize});

// A tensor whose memory holds its values: not a negation that is still to be done (z.conj().imag), nor zeros without memory.
bool is_plain(const Tensor& t) { return !t.is_neg() && !t._is_zerotensor(); }
Tensor plain(const Tensor& t) { return is_plain(t) ? t : t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_neg(); }

// A saved tensor as the backward pass finds it: saved-tensor hooks may have moved it away and back (other strides are read as they are), but what
// the kernels read by address has to be of this size, type and device.
Tensor saved_as(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
    TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.sizes() == sizes && t.scalar_type() == type && t.device() == device &&
                    !t.key_set().has_any(stand_ins),
                "ppv_amd: a saved tensor came back from its hooks with another size, type or device");
    return plain(t);
}

// The kernels go by addresses, out of sight of torch's dispatcher.  What it does besides computing would be missing from the result without a word;
// the arguments of both operators, and the gradients that come back to them, are looked over for it: forward-mode tangents, and whoever records the
// dispatched calls to run them again (torch.jit.trace, make_fx) or to run them without data: the record would be the allocation of the result alone;
// tensors that stand for others (functorch's, subclasses with a dispatch of their own).
void refuse_unseen(const char* name, std::initializer_list<const Tensor*> ts) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), "ppv_amd ", name, ": torch.jit.trace does not see the kernel");
    TORCH_CHECK_NOT_IMPLEMENTED(!TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) && !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) &&
                                    !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL) &&
                                    !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch),
                                "ppv_amd ", name, ": a tracing mode (make_fx, fake tensors, functionalization) does not see the kernel");
    const bool tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const Tensor* t : ts) {
        if (!t->defined()) continue;
        TORCH_CHECK_NOT_IMPLEMENTED(!t->key_set().has_any(stand_ins), "ppv_amd ", name,
                                    ": tensors under torch.func / vmap and subclasses with a __torch_dispatch__ do not reach the kernel");
        TORCH_CHECK_NOT_IMPLEMENTED(!tangents || !t->_fw_grad(0).defined(), "ppv_amd ", name, ": forward-mode derivatives are not implemented");
    }
}

// Gradients of a node that is differentiable once: where a graph of the backward pass is asked for, differentiating through it is an error.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (const auto& g : grads) in.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
    torch::autograd::DelayedError error("trying to differentiate twice a function of ppv_amd that is differentiable once", (int64_t)grads.size());
    return error(std::move(in));
}

// A backward pass that is captured into a graph must not go on to a node of the default stream: the engine would make that stream wait for the
// captured one, which no capture allows, and the broken capture ends the process when its graph is destroyed.  Such a node is the accumulation of a
// leaf whose eager graph still lives, possibly some views away.
void refuse_capture_of_eager_graph() {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto* wanted = torch::autograd::get_current_graph_task_exec_info();              // (empty: all of the graph)
    auto runs = [&](torch::autograd::Node* n) {
        if (!wanted || wanted->empty()) return true;
        const auto at = wanted->find(n);
        return at != wanted->end() && at->second.should_execute();
    };
    const auto node = torch::autograd::get_current_node();
    std::vector<torch::autograd::Node*> todo{node.get()};
    std::unordered_set<torch::autograd::Node*> seen{node.get()};
    while (!todo.empty()) {
        torch::autograd::Node* n = todo.back();
        todo.pop_back();
        for (const auto& e : n->next_edges())
            if (e.function && runs(e.function.get()) && seen.insert(e.function.get()).second) {
                const auto s = e.function->stream();
                TORCH_CHECK(!s || s->id() != 0, "ppv_amd: this backward pass is being captured into a graph, but ", e.function->name(),
                            " belongs to an eager graph of the default stream; drop that graph (or make it on a side stream) first");
                todo.push_back(e.function.get());
            }
    }
}

// ------------------------------------------------------------------------------------------------------------------------- layer norm

Tensor rows_of(const Tensor& t, int64_t C) {
    Tensor r = plain(t);
    if (t.dim() != 2) r = r.reshape({-1, C});
    return C == 1 || r.stride(1) == 1 ? r : r.contiguous();
}
long row_stride(const Tensor& r) { return r.size(0) == 1 ? 0 : r.stride(0); }

std::pair<Tensor, Tensor> norm_forward(const Tensor& x2, const Tensor& w, const Tensor& b, double eps, bool keep) {
    const int64_t rows = x2.size(0), C = x2.size(1);
    Tensor y = at::empty({rows, C}, x2.options()), stats;
    if (keep) stats = at::empty({2, rows}, x2.options().dtype(at::kFloat));
    if (rows) {
        float* s = data<float>(stats);
        check(abi.layernorm_fwd(x2.data_ptr(), row_stride(x2), data<void>(w), data<void>(b), y.data_ptr(), s, s ? s + rows : nullptr, rows, (int)C,
                                code(x2.scalar_type()), w.defined() ? code(w.scalar_type()) : b.defined() ? code(b.scalar_type()) : 0, (float)eps, stream()),
              "ppv_layernorm_fwd");
    }
    return {y, stats};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
        c10::DeviceGuard guard(x.device());
        const Tensor x2 = rows_of(x, x.size(-1));
        const Tensor w = weight ? plain(weight->contiguous()) : Tensor(), b = bias ? plain(bias->contiguous()) : Tensor();
        auto [y, stats] = norm_forward(x2, w, b, eps, true);
        ctx->save_for_backward({x2, w, stats});
        const auto& par = w.defined() ? w : b;
        ctx->saved_data["has"] = (int64_t)(w.defined() + 2 * b.defined());
        ctx->saved_data["par"] = par.defined() ? (int64_t)par.scalar_type() : (int64_t)at::kFloat;
        return x.dim() == 2 ? y : y.view(x.sizes());
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list r;
        {
            at::NoGradGuard off;
            refuse_unseen("layer_norm", {&grads[0]});
            refuse_capture_of_eager_graph();
            const auto saved = ctx->get_saved_variables();
            const Tensor& g = grads[0];
            c10::DeviceGuard guard(g.device());
            const int64_t C = g.size(-1), rows = g.numel() / C;
            const auto par = (at::ScalarType)ctx->saved_data["par"].toInt();
            const int64_t has = ctx->saved_data["has"].toInt();                             // (a node's edges are those of the tensors it was given)
            const Tensor g2 = rows_of(g, C), x2 = rows_of(saved_as(saved[0], {rows, C}, g.scalar_type(), g.device()), C);
            const Tensor w = has & 1 ? saved_as(saved[1], {C}, par, g.device()).contiguous() : Tensor();
            const Tensor stats = saved_as(saved[2], {2, rows}, at::kFloat, g.device()).contiguous();
            const bool want_w = (has & 1) && ctx->needs_input_grad(1), want_b = (has & 2) && ctx->needs_input_grad(1 + (has & 1));
            Tensor dx = at::empty({rows, C}, x2.options()), dw, db, ws;
            if (want_w) dw = at::empty({C}, x2.options().dtype(par));
            if (want_b) db = at::empty({C}, x2.options().dtype(par));
            if (rows) {
                const int dt = code(x2.scalar_type());
                if (want_w || want_b) ws = at::empty({(int64_t)abi.layernorm_ws(rows, (int)C, dt)}, x2.options().dtype(at::kByte));
                float* s = data<float>(stats);
                check(abi.layernorm_bwd(g2.data_ptr(), row_stride(g2), x2.data_ptr(), row_stride(x2), data<void>(w), s, s + rows, dx.data_ptr(),
                                        data<void>(dw), data<void>(db), data<void>(ws), rows, (int)C, dt, code(par), stream()),
                      "ppv_layernorm_bwd");
            } else {
                if (want_w) dw.zero_();
                if (want_b) db.zero_();
            }
            r = {ctx->needs_input_grad(0) ? (g.dim() == 2 ? dx : dx.view(g.sizes())) : Tensor(), dw, db, Tensor()};
        }
        return once(std::move(r));
    }
};

bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    refuse_unseen("layer_norm", {&x, &w, &b});
    if (wants_grad({&x, &w, &b})) return LayerNorm::apply(x, weight, bias, eps);
    at::NoGradGuard off;
    c10::DeviceGuard guard(x.device());
    const Tensor y = norm_forward(rows_of(x, x.size(-1)), w.defined() ? plain(w.contiguous()) : w, b.defined() ? plain(b.contiguous()) : b, eps, false).first;
    return x.dim() == 2 ? y : y.view(x.sizes());
}

// -------------------------------------------------------------------------------------------------------------------------- attention

// t [B,T,H,D] as the kernels read it: unit last stride, every other stride and the address multiples of 16 bytes, D padded to Dp.  A view
// that is already so is taken as it is, any other is copied (zeros behind D add nothing to a product).
Tensor operand(const Tensor& t, int64_t Dp) {
    const int64_t v = 16 / t.element_size();
    if (!is_plain(t)) return operand(plain(t), Dp);
    bool fits = t.size(3) == Dp && t.stride(3) == 1 && reinterpret_cast<size_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) fits = fits && (t.size(i) == 1 || t.stride(i) % v == 0);
    if (fits && (t.size(1) == 1 || t.stride(1) <= 1 << 22)) return t;
    Tensor p = at::empty({t.size(0), t.size(1), t.size(2), Dp}, t.options());
    if (Dp != t.size(3)) p.narrow(3, t.size(3), Dp - t.size(3)).zero_();
    p.narrow(3, 0, t.size(3)).copy_(t);
    return p;
}
// ... and as they write it: without gaps, from a multiple of 16 bytes
Tensor packed(const Tensor& t) {
    return t.is_contiguous() && reinterpret_cast<size_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}
long stride_of(const Tensor& t, int i) { return t.size(i) == 1 ? 0 : t.stride(i); }

PpvAttention describe(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lo, const Tensor& lse, const Tensor& ql,
                      const Tensor& kl, bool causal, double scale) {
    PpvAttention a = {};
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.out = out.data_ptr();
    a.out_lo = data<void>(lo);
    a.lse = data<float>(lse);
    a.q_lens = data<int>(ql);
    a.k_lens = data<int>(kl);
    a.sqb = stride_of(q, 0); a.sqt = stride_of(q, 1); a.sqh = stride_of(q, 2);
    a.skb = stride_of(k, 0); a.skt = stride_of(k, 1); a.skh = stride_of(k, 2);
    a.svb = stride_of(v, 0); a.svt = stride_of(v, 1); a.svh = stride_of(v, 2);
    a.B = (int)q.size(0); a.Tq = (int)q.size(1); a.H = (int)q.size(2); a.D = (int)q.size(3);
    a.Tk = (int)k.size(1); a.Hkv = (int)k.size(2);
    a.dtype = code(q.scalar_type());
    a.causal = causal;
    a.scale = (float)scale;
    return a;
}

struct Forward { Tensor q, k, v, out, lo, lse; };

// keep: for a backward pass (whose rowsum(dO O) would carry the rounding of a 16-bit O into every score's gradient: `lo` is what it took)
Forward attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& ql, const Tensor& kl, bool causal, double scale, bool keep) {
    const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), D = q.size(3), w = 16 / q.element_size(), Dp = (D + w - 1) / w * w;
    Forward f{operand(q, Dp), operand(k, Dp), operand(v, Dp), at::empty({B, Tq, H, Dp}, q.options()), Tensor(), Tensor()};
    if (keep) {
        f.lse = at::empty({B, H, Tq}, q.options().dtype(at::kFloat));
        if (q.scalar_type() != at::kFloat) f.lo = at::empty_like(f.out);
    }
    if (f.out.numel() == 0) return f;
    if (k.numel() == 0) {                                      // no keys at all: every row is empty
        f.out.zero_();
        return f;
    }
    PpvAttention a = describe(f.q, f.k, f.v, f.out, f.lo, f.lse, ql, kl, causal, scale);
    Tensor ws;
    if (const size_t n = abi.attention_fwd_ws(a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.dtype)) {
        ws = at::empty({(int64_t)n}, q.options().dtype(at::kByte));
        a.workspace = ws.data_ptr();
    }
    check(abi.attention_fwd(&a, stream()), "ppv_attention_fwd");
    return f;
}
Tensor unpadded(const Tensor& t, int64_t D) { return t.size(3) == D ? t : t.narrow(3, 0, D).contiguous(); }

struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& q_lens,
                          const std::optional<Tensor>& k_lens, bool causal, double scale) {
        c10::DeviceGuard guard(q.device());
        const Tensor ql = q_lens.value_or(Tensor()), kl = k_lens.value_or(Tensor());
        Forward f = attention_forward(q, k, v, ql, kl, causal, scale, true);
        ctx->save_for_backward({f.q, f.k, f.v, f.out, f.lo, f.lse, ql, kl});
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        return unpadded(f.out, q.size(3));
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list r(7);
        {
            at::NoGradGuard off;
            refuse_unseen("multihead_attention", {&grads[0]});
            refuse_capture_of_eager_graph();
            const auto saved = ctx->get_saved_variables();
            const Tensor& go = grads[0];
            c10::DeviceGuard guard(go.device());
            const auto type = go.scalar_type();
            const auto on = go.device();
            const int64_t B = go.size(0), Tq = go.size(1), H = go.size(2), D = go.size(3), w = 16 / go.element_size(), Dp = (D + w - 1) / w * w;
            const Tensor q = operand(saved_as(saved[0], {B, Tq, H, Dp}, type, on), Dp);
            TORCH_CHECK(saved[1].dim() == 4, "ppv_amd: a saved tensor came back from its hooks with another size, type or device");
            const int64_t Tk = saved[1].size(1), Hkv = saved[1].size(2);
            const Tensor k = operand(saved_as(saved[1], {B, Tk, Hkv, Dp}, type, on), Dp), v = operand(saved_as(saved[2], {B, Tk, Hkv, Dp}, type, on), Dp);
            TORCH_CHECK(Hkv > 0 && H % Hkv == 0, "ppv_amd: a saved tensor came back from its hooks with another size, type or device");
            const Tensor out = packed(saved_as(saved[3], {B, Tq, H, Dp}, type, on)), lse = saved_as(saved[5], {B, H, Tq}, at::kFloat, on).contiguous();
            const Tensor lo = type == at::kFloat ? Tensor() : packed(saved_as(saved[4], {B, Tq, H, Dp}, type, on));
            const auto lens = [&](const Tensor& t) { return t.defined() ? saved_as(t, {B}, at::kInt, on).contiguous() : Tensor(); };
            const Tensor ql = lens(saved[6]), kl = lens(saved[7]);
            Tensor d[3] = {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options()), at::empty(k.sizes(), k.options())};
            if (q.numel() == 0 || k.numel() == 0) {
                for (auto& t : d) t.zero_();
            } else {
                PpvAttention a = describe(q, k, v, out, lo, lse, ql, kl, ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
                const Tensor g = operand(go, Dp);
                a.dout = g.data_ptr();
                a.sgb = stride_of(g, 0); a.sgt = stride_of(g, 1); a.sgh = stride_of(g, 2);
                a.dq = d[0].data_ptr(); a.dk = d[1].data_ptr(); a.dv = d[2].data_ptr();
                const Tensor ws = at::empty({(int64_t)abi.attention_bwd_ws(a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.dtype)}, q.options().dtype(at::kByte));
                a.workspace = ws.data_ptr();
                check(abi.attention_bwd(&a, stream()), "ppv_attention_bwd");
            }
            for (int i = 0; i < 3; ++i)
                if (ctx->needs_input_grad(i)) r[i] = unpadded(d[i], D);
        }
        return once(std::move(r));
    }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& q_lens, const std::optional<Tensor>& k_lens,
                 bool causal, double scale) {
    const Tensor ql = q_lens.value_or(Tensor()), kl = k_lens.value_or(Tensor());
    refuse_unseen("multihead_attention", {&q, &k, &v, &ql, &kl});
    if (wants_grad({&q, &k, &v})) return Attention::apply(q, k, v, q_lens, k_lens, causal, scale);
    at::NoGradGuard off;
    c10::DeviceGuard guard(q.device());
    return unpadded(attention_forward(q, k, v, ql, kl, causal, scale, false).out, q.size(3));
}

// ------------------------------------------------------------------------------------------------------------------------------ AdamW

// A list of parameters with their moments (ms, vs undefined: 32 bits) whose gradients are taken as they are at each step.  The descriptor table on
// the device is made again whenever one of the addresses it holds, or the stream, is another one.
struct AdamWList {
    std::vector<Tensor> p, m, v, ms, vs, rest;                 // rest: the group's parameters that had no gradient
    std::vector<int64_t> place, key;
    static constexpr int WORDS = 11;                           // of the key for each parameter: six addresses, its size, what its moments are
    std::vector<std::pair<int64_t, int64_t>> spans;            // what a step writes, in order: addresses [from, to)
    Tensor table;
    int records = 0, blocks = 0;

    AdamWList(std::vector<Tensor> p_, std::vector<Tensor> m_, std::vector<Tensor> v_, const std::vector<std::optional<Tensor>>& ms_,
              const std::vector<std::optional<Tensor>>& vs_, std::vector<int64_t> place_)
        : p(std::move(p_)), m(std::move(m_)), v(std::move(v_)), place(std::move(place_)) {
        for (const auto& t : ms_) ms.push_back(t.value_or(Tensor()));
        for (const auto& t : vs_) vs.push_back(t.value_or(Tensor()));
    }

    // every parameter of the list has a gradient, none of the others has
    bool complete() const {
        for (const auto& t : p)
            if (!t.grad().defined()) return false;
        for (const auto& t : rest)
            if (t.grad().defined()) return false;
        return true;
    }

    void step(double lr, double b1, double b2, double eps, double wd, double number, uint32_t seed) {
        const auto dev = p[0].device();
        c10::DeviceGuard guard(dev);
        const ppv_stream_t st = stream();
        std::vector<int64_t> now;
        now.reserve(p.size() * WORDS + 1);
        now.push_back(reinterpret_cast<int64_t>(st));
        for (size_t i = 0; i < p.size(); ++i) {
            const Tensor& g = p[i].grad();
            TORCH_CHECK_NOT_IMPLEMENTED(g.defined() && g.layout() == at::kStrided && g.scalar_type() == at::kFloat && g.is_contiguous() &&
                                            g.device() == dev && is_plain(g) && is_plain(p[i]) && p[i].scalar_type() == at::kFloat &&
                                            p[i].is_contiguous() && p[i].device() == dev && dev.is_cuda() && g.numel() == p[i].numel(),
                                        "ppv_amd.optim.AdamW: contiguous f32 parameters and gradients on one GPU only");
            const Tensor* held[] = {&p[i], &g, &m[i], &v[i], &ms[i], &vs[i]};
            for (const Tensor* t : held) now.push_back(t->defined() ? reinterpret_cast<int64_t>(t->data_ptr()) : 0);
            now.push_back(p[i].numel());
            for (int k = 2; k < 6; ++k)                         // (another tensor, a shorter one, may lie where the old one lay)
                now.push_back(held[k]->defined() ? held[k]->numel() * 128 + (int64_t)held[k]->scalar_type() * 2 + held[k]->is_contiguous() : 0);
        }
        if (now != key) {
            describe(now);
            key = std::move(now);
        }
        if (!records) return;
        check(abi.adamw_multi(table.data_ptr(), records, blocks, lr, b1, b2, eps, wd, number, seed, st), "ppv_adamw_multi");
        for (const auto* list : {&p, &m, &v, &ms, &vs})
            for (const Tensor& t : *list) written(t);
    }

    // The kernel writes through addresses.  What goes by a tensor's version has to be told: autograd's check of saved tensors, and every cache
    // of a weight's layout (nn_ops._layouts: the convolutions would stay with the weights of the first step).  (Inference tensors have no version.)
    static void written(const Tensor& t) {
        if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }

    void describe(const std::vector<int64_t>& now) {
        struct Record { int64_t at[6], numel; int32_t blk0; uint32_t place; };
        static_assert(sizeof(Record) == 64, "include/ppv_hip.h ppv_adamw_multi");
        int count = 0;                                         // (a list that is refused stays as it was: its key does, too)
        int64_t blk = 0;
        Tensor host = at::empty({(int64_t)(p.size() * sizeof(Record))}, at::TensorOptions().dtype(at::kByte).pinned_memory(true));
        auto* r = static_cast<Record*>(host.data_ptr());
        for (size_t i = 0; i < p.size(); ++i) {
            const int64_t* at = now.data() + 1 + i * WORDS;
            auto fits = [&](const Tensor& t, at::ScalarType kind, int64_t n) {
                return t.scalar_type() == kind && t.numel() == n && t.is_contiguous() && t.device() == p[i].device();
            };
            const bool small = ms[i].defined();                // (`.data` of a tensor that is kept may have become another one)
            const auto kind = small ? at::kFloat8_e4m3fn : at::kFloat;
            TORCH_CHECK_VALUE(fits(m[i], kind, at[6]) && fits(v[i], kind, at[6]) &&
                                  (!small || (fits(ms[i], at::kFloat, (at[6] + 255) / 256) && fits(vs[i], at::kFloat, (at[6] + 255) / 256))),
                              "ppv_amd.optim.AdamW: a parameter's state does not belong to it (type, size, device or layout)");
            if (at[6] == 0) continue;
            Record& x = r[count++];
            std::copy(at, at + 6, x.at);
            x.numel = at[6];
            x.blk0 = (int32_t)blk;
            x.place = (uint32_t)place[i];
            blk += (at[6] + 4095) / 4096;
        }
        auto apart = spans_of(now);
        TORCH_CHECK(blk <= INT32_MAX, "ppv_amd.optim.AdamW: too many elements in one group");
        // pinned and non-blocking: a list whose gradients move every step does not wait for the device
        table = count ? host.to(p[0].device(), at::kByte, /*non_blocking=*/true) : Tensor();
        records = count;
        blocks = (int)blk;
        spans = std::move(apart);
    }

    // The launch's workgroups write in any order: nothing they write may overlap, and no gradient may lie in it but a parameter's own (every
    // element is read before it is written).
    std::vector<std::pair<int64_t, int64_t>> spans_of(const std::vector<int64_t>& now) const {
        bool moved = key.size() != now.size();
        for (size_t i = 0; i < p.size() && !moved; ++i)
            for (int k = 0; k < 7 && !moved; ++k) moved = k != 1 && key[1 + i * WORDS + k] != now[1 + i * WORDS + k];
        std::vector<std::pair<int64_t, int64_t>> r = spans;
        auto end = [&](int64_t from, const Tensor& t) { return from + (int64_t)t.nbytes(); };
        if (moved) {
            r.clear();
            for (size_t i = 0; i < p.size(); ++i) {
                const int64_t* at = now.data() + 1 + i * WORDS;
                const Tensor* held[] = {&p[i], nullptr, &m[i], &v[i], &ms[i], &vs[i]};
                for (int k = 0; k < 6; ++k)
                    if (held[k] && held[k]->defined() && held[k]->numel()) r.emplace_back(at[k], end(at[k], *held[k]));
            }
            std::sort(r.begin(), r.end());
            for (size_t i = 1; i < r.size(); ++i)
                TORCH_CHECK_VALUE(r[i - 1].second <= r[i].first, "ppv_amd.optim.AdamW: parameters or moments of one group share memory");
        }
        for (size_t i = 0; i < p.size(); ++i) {
            const int64_t* at = now.data() + 1 + i * WORDS;
            if (at[6] == 0 || at[1] == at[0]) continue;
            const auto next = std::upper_bound(r.begin(), r.end(), std::make_pair(at[1], INT64_MAX));
            TORCH_CHECK_VALUE((next == r.end() || end(at[1], p[i]) <= next->first) && (next == r.begin() || std::prev(next)->second <= at[1]),
                              "ppv_amd.optim.AdamW: a gradient and what the step writes share memory");
        }
        return r;
    }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
    namespace py = pybind11;
    using release = py::call_guard<py::gil_scoped_release>;
    mod.def("bind", &bind);
    // what this file was compiled against: _lib.torch_ops() compares it with what is loaded
    mod.attr("abi_version") = PPV_ABI_VERSION;
    mod.attr("attention_bytes") = sizeof(PpvAttention);
    mod.attr("torch_version") = TORCH_VERSION;
    mod.def("layer_norm", &layer_norm, release());
    mod.def("attention", &attention, release());
    py::class_<AdamWList>(mod, "AdamWList")
        .def(py::init<std::vector<Tensor>, std::vector<Tensor>, std::vector<Tensor>, const std::vector<std::optional<Tensor>>&,
                      const std::vector<std::optional<Tensor>>&, std::vector<int64_t>>())
        .def("without", [](AdamWList& a, std::vector<Tensor> rest) { a.rest = std::move(rest); })
        .def("complete", &AdamWList::complete)
        .def("step", &AdamWList::step, release());
}
