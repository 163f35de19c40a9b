// The operator's autograd functions as native torch nodes (Python module theseus._native).
//
// theseus/wkv7.py's _WKV, theseus/gdn.py's _GDN and theseus/vocab.py's _Loss do the same through Python: contiguous
// inputs, the checks of kernels/wkv7_state.cpp:10-15, outputs and workspace from torch's
// allocator, one C-ABI call on the current stream.  For few tokens that host work is the
// call: a forward+backward through the Python functions takes 225 us of host time (B=1, T=64,
// H=2, bf16), a good part of it the engine's device thread taking the interpreter lock for
// the backward; here it takes 49 us.  Python keeps its functions for what these do not cover
// (functorch transforms, tensor subclasses).
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include <cstdlib>
#include <cstring>
#include <limits>
#include <unordered_set>

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include "../../include/theseus_embed.h"
#include "../../include/theseus_gdn_ex.h"
#include "../../include/theseus_vocab.h"
#include "../../include/theseus_wkv7.h"

namespace py = pybind11;
using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

void raise_status(int st, const char* who) {
    TORCH_CHECK(st == 0, who, ": ", theseus_wkv7_error_string(st));
}
hipStream_t stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
Tensor scratch(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(torch::kUInt8)) : Tensor();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }

// check() of kernels/wkv7_state.cpp:10-15, the same messages
void check(const Tensor& r, std::initializer_list<Tensor> xs) {
    TORCH_CHECK(r.is_cuda() && r.is_contiguous() && r.dim() == 4, "expected contiguous CUDA [B,T,H,N]");
    TORCH_CHECK(r.size(1) > 0 && r.size(3) >= 2 && r.size(3) <= 128, "invalid T or head size (2..128)");
    TORCH_CHECK(r.scalar_type() == torch::kBFloat16 || r.scalar_type() == torch::kFloat32, "expected BF16 or FP32");
    for (const Tensor& x : xs)
        TORCH_CHECK(x.device() == r.device() && x.sizes() == r.sizes() && x.scalar_type() == r.scalar_type() &&
                        x.is_contiguous(),
                    "input mismatch");
}
struct Dims {
    int B, T, H, N, dt;
    explicit Dims(const Tensor& r)
        : B((int)r.size(0)), T((int)r.size(1)), H((int)r.size(2)), N((int)r.size(3)),
          dt(r.scalar_type() == torch::kBFloat16 ? THESEUS_WKV7_BF16 : THESEUS_WKV7_FP32) {}
    std::vector<int64_t> saved() const { return {B, H, (int64_t)theseus_wkv7_checkpoint_count(T), N, N}; }
    int family() const { return theseus_wkv7_kernel_family(B, T, H, N, dt); }
};
bool env_is_1(const char* name) {
    const char* e = std::getenv(name);
    return e && std::strcmp(e, "1") == 0;
}
// Extension._warn_fallback: a warning (or, THESEUS_WKV7_STRICT=1, an error) when a call runs
// on the step-serial kernels without having asked for them.  The warning names the caller of
// theseus.wkv7.wkv7 (three frames up: this function, wkv7, the caller).
void warn_fallback(const Dims& d, int family) {
    if (family != THESEUS_WKV7_FAMILY_FP32 && family != THESEUS_WKV7_FAMILY_HEAD_SIZE &&
        family != THESEUS_WKV7_FAMILY_SIZE)
        return;
    py::gil_scoped_acquire gil;
    py::module_::import("theseus.wkv7").attr("extension")().attr("_warn_fallback")(d.B, d.T, d.H, d.N, d.dt, 3);
}
// THESEUS_WKV7_CHECK_WAITS=1 (Extension._check_waits)
void check_waits() {
    if (!env_is_1("THESEUS_WKV7_CHECK_WAITS")) return;
    unsigned int n = 0;
    raise_status(theseus_wkv7_wait_timeouts(&n, 1), "theseus_wkv7");
    TORCH_CHECK(n == 0, "theseus_wkv7: ", n,
                " bounded wait(s) timed out in the chunked kernels; the outputs hold NaN where they depended on them");
}

struct Fwd {
    Tensor y, end, saved;
};
Fwd wkv7_forward(const std::array<Tensor, 6>& x, const Tensor& s0, bool save) {
    const auto& [r, w, k, v, a, b] = x;
    check(r, {w, k, v, a, b});
    const Dims d(r);
    TORCH_CHECK(s0.device() == r.device() && s0.scalar_type() == torch::kFloat32 && s0.is_contiguous(),
                "s0 must be contiguous CUDA FP32");
    TORCH_CHECK(s0.sizes() == at::IntArrayRef({d.B, d.H, d.N, d.N}), "invalid s0 shape");
    c10::OptionalDeviceGuard guard(r.device());
    Fwd o{at::empty_like(r), at::empty_like(s0), Tensor()};
    if (save) o.saved = at::empty(d.saved(), s0.options());
    if (d.T > 1 || save) warn_fallback(d, d.family());
    const size_t need = theseus_wkv7_forward_best_workspace_size(d.B, d.T, d.H, d.N, d.dt, save);
    const Tensor ws = scratch(need, r);
    raise_status(theseus_wkv7_forward(d.B, d.T, d.H, d.N, d.dt, ptr(r), ptr(w), ptr(k), ptr(v), ptr(a), ptr(b), fptr(s0),
                                      ptr(o.y), fptr(o.end), fptr(o.saved), ptr(ws), need, stream_of(r)),
                 "theseus_wkv7");
    check_waits();
    return o;
}

Tensor float_rows(const Tensor& t) { return t.to(torch::kFloat32).contiguous(); }

struct Wkv7 : torch::autograd::Function<Wkv7> {
    static variable_list forward(AutogradContext* ctx, const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v,
                                 const Tensor& a, const Tensor& b, const Tensor& state) {
        ctx->set_materialize_grads(false);
        const std::array<Tensor, 6> x{r.contiguous(), w.contiguous(), k.contiguous(),
                                      v.contiguous(), a.contiguous(), b.contiguous()};
        const Fwd o = wkv7_forward(x, float_rows(state), true);
        ctx->save_for_backward({x[0], x[1], x[2], x[3], x[4], x[5], o.saved});
        // the saved states' order is the chunked kernels' (family 0) or [value][key]
        ctx->saved_data["tiled"] = Dims(x[0]).family() == THESEUS_WKV7_FAMILY_CHUNKED;
        return {o.y, o.end};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &r = s[0], &saved = s[6];
        const Tensor dy = g[0].defined() ? g[0].to(r.scalar_type()).contiguous() : at::zeros_like(r);
        const Tensor dend = g[1].defined() ? float_rows(g[1]) : Tensor();
        check(r, {s[1], s[2], s[3], s[4], s[5], dy});
        const Dims d(r);
        const int family = d.family();
        TORCH_CHECK(ctx->saved_data["tiled"].toBool() == (family == THESEUS_WKV7_FAMILY_CHUNKED),
                    "saved states were written by the other kernel family (their order differs); run the backward with "
                    "the forward's THESEUS_WKV7_FAMILY");
        TORCH_CHECK(saved.device() == r.device() && saved.scalar_type() == torch::kFloat32 && saved.is_contiguous() &&
                        saved.sizes() == at::IntArrayRef(d.saved()),
                    "invalid history");
        TORCH_CHECK(!dend.defined() ||
                        (dend.device() == r.device() && dend.sizes() == at::IntArrayRef({d.B, d.H, d.N, d.N})),
                    "invalid dend");
        c10::OptionalDeviceGuard guard(r.device());
        variable_list o(7);
        for (int i = 0; i < 6; i++) o[i] = at::empty_like(r);
        o[6] = at::empty({d.B, d.H, d.N, d.N}, saved.options());
        // (the forward of these sizes has warned, and the engine's thread has no caller to name)
        if (env_is_1("THESEUS_WKV7_STRICT")) warn_fallback(d, family);
        const size_t need = theseus_wkv7_backward_workspace_size(d.B, d.T, d.H, d.N, d.dt);
        const Tensor ws = scratch(need, r);
        raise_status(theseus_wkv7_backward(d.B, d.T, d.H, d.N, d.dt, ptr(r), ptr(s[1]), ptr(s[2]), ptr(s[3]), ptr(s[4]),
                                           ptr(s[5]), fptr(saved), ptr(dy), fptr(dend), ptr(o[0]), ptr(o[1]), ptr(o[2]),
                                           ptr(o[3]), ptr(o[4]), ptr(o[5]), fptr(o[6]), ptr(ws), need, stream_of(r)),
                     "theseus_wkv7");
        check_waits();
        return o;
    }
};

std::pair<Tensor, Tensor> wkv7(const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a,
                               const Tensor& b, const Tensor& state) {
    py::gil_scoped_release free;
    bool grad = false;
    if (at::GradMode::is_enabled())
        for (const Tensor* t : {&r, &w, &k, &v, &a, &b, &state}) grad = grad || t->requires_grad();
    if (grad) {
        const variable_list o = Wkv7::apply(r, w, k, v, a, b, state);
        return {o[0], o[1]};
    }
    const std::array<Tensor, 6> x{r.contiguous(), w.contiguous(), k.contiguous(),
                                  v.contiguous(), a.contiguous(), b.contiguous()};
    const Fwd o = wkv7_forward(x, float_rows(state), false);
    return {o.y, o.end};
}

// Extension._gdn_check
void gdn_check(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const Tensor& s0) {
    TORCH_CHECK(q.scalar_type() == torch::kBFloat16 || q.scalar_type() == torch::kFloat32,
                "theseus_gdn: expected bfloat16 or float32 q, k, v");
    for (const Tensor* x : {&q, &k, &v})
        TORCH_CHECK(x->is_cuda() && x->scalar_type() == q.scalar_type() && x->is_contiguous() && x->dim() == 4 &&
                        x->sizes() == q.sizes() && x->device() == q.device(),
                    "theseus_gdn: expected contiguous CUDA q, k, v [B,T,H,N] of one dtype");
    for (const Tensor* x : {&g, &beta})
        TORCH_CHECK(x->device() == q.device() && x->scalar_type() == torch::kFloat32 && x->is_contiguous() &&
                        x->sizes() == q.sizes().slice(0, 3),
                    "theseus_gdn: expected contiguous float32 g, beta [B,T,H]");
    TORCH_CHECK(!s0.defined() || (s0.device() == q.device() && s0.scalar_type() == torch::kFloat32 && s0.is_contiguous() &&
                                  s0.sizes() == at::IntArrayRef({q.size(0), q.size(2), q.size(3), q.size(3)})),
                "theseus_gdn: expected contiguous float32 state [B,H,N,N]");
}

struct Gdn : torch::autograd::Function<Gdn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                 const Tensor& beta, const Tensor& s0, bool qk_l2norm) {
        ctx->set_materialize_grads(false);
        gdn_check(q, k, v, g, beta, s0);
        const Dims d(q);
        c10::OptionalDeviceGuard guard(q.device());
        const Tensor o = at::empty_like(q), sT = at::empty_like(s0), saved = at::empty(d.saved(), s0.options());
        const size_t need = theseus_gdn_forward_best_workspace_size(d.B, d.T, d.H, d.N, 1);
        const Tensor ws = scratch(need, q);
        raise_status(theseus_gdn_forward_train_ex(d.B, d.T, d.H, d.N, d.dt, qk_l2norm, ptr(q), ptr(k), ptr(v), fptr(g),
                                                  fptr(beta), fptr(s0), ptr(o), fptr(sT), fptr(saved), ptr(ws), need,
                                                  stream_of(q)),
                     "theseus_wkv7");
        ctx->save_for_backward({q, k, v, g, beta, saved});
        ctx->saved_data["qk_l2norm"] = qk_l2norm;
        return {o, sT};
    }
    static variable_list backward(AutogradContext* ctx, variable_list gr) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &g = s[3], &beta = s[4], &saved = s[5];
        const Tensor dout = gr[0].defined() ? gr[0].to(q.scalar_type()).contiguous() : at::zeros_like(q);
        const Tensor dsT = gr[1].defined() ? float_rows(gr[1]) : Tensor();
        gdn_check(q, k, v, g, beta, dsT);
        const Dims d(q);
        TORCH_CHECK(dout.sizes() == q.sizes() && dout.device() == q.device(),
                    "theseus_gdn: expected a contiguous output gradient like q");
        TORCH_CHECK(saved.scalar_type() == torch::kFloat32 && saved.is_contiguous() && saved.device() == q.device() &&
                        saved.sizes() == at::IntArrayRef(d.saved()),
                    "theseus_gdn: invalid saved states");
        c10::OptionalDeviceGuard guard(q.device());
        variable_list o{at::empty_like(q), at::empty_like(q), at::empty_like(q), at::empty_like(g), at::empty_like(beta),
                        at::empty({d.B, d.H, d.N, d.N}, saved.options())};
        const size_t need = theseus_gdn_backward_workspace_size(d.B, d.T, d.H, d.N);
        const Tensor ws = scratch(need, q);
        raise_status(theseus_gdn_backward_ex(d.B, d.T, d.H, d.N, d.dt, ctx->saved_data["qk_l2norm"].toBool(), ptr(q),
                                             ptr(k), ptr(v), fptr(g), fptr(beta), fptr(saved), ptr(dout), fptr(dsT),
                                             ptr(o[0]), ptr(o[1]), ptr(o[2]), fptr(o[3]), fptr(o[4]), fptr(o[5]), ptr(ws),
                                             need, stream_of(q)),
                     "theseus_wkv7");
        o.emplace_back();  // (qk_l2norm)
        return o;
    }
};

std::pair<Tensor, Tensor> gdn(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                              const Tensor& s0, bool qk_l2norm) {
    py::gil_scoped_release free;
    const variable_list o = Gdn::apply(q, k, v, g, beta, s0, qk_l2norm);
    return {o[0], o[1]};
}

// theseus.vocab's losses: the arguments as theseus/vocab.py's _loss has checked and laid them out
// (h [M][D] and w [V][D] with rows apart, the others contiguous).
struct VocabLoss : torch::autograd::Function<VocabLoss> {
    using Opt = std::optional<Tensor>;
    static constexpr const char *INDEX = "labels (or top_indices)", *TOP = "top_values", *LSE = "teacher_lse", *WEIGHT = "token_weight";
    static void* optr(const Opt& t) { return t ? t->data_ptr() : nullptr; }
    static void call(const Tensor& h, const Tensor& w, const Tensor& index, const Opt& top, const Opt& lse, const Opt& weight,
                     int64_t ignore, double T, int64_t reduction, int64_t piece, const Tensor& loss, const Tensor& row_grad,
                     const Tensor& dh, const Tensor& dw, Tensor* kept = nullptr) {
        theseus_vocab_loss_args a{};
        a.rows = h.size(0), a.vocab = w.size(0), a.width = (int)h.size(1), a.targets = top ? (int)top->size(1) : 1;
        a.hidden = h.data_ptr(), a.weight = w.data_ptr();
        a.hidden_stride = std::max(h.stride(0), h.size(1)), a.weight_stride = std::max(w.stride(0), w.size(1));
        a.index = index.data_ptr<int64_t>(), a.top_values = optr(top);
        a.top_dtype = top && top->scalar_type() == torch::kFloat32 ? THESEUS_VOCAB_FP32 : THESEUS_VOCAB_BF16;
        a.reduction = (int)reduction, a.teacher_lse = static_cast<float*>(optr(lse)), a.row_weight = static_cast<float*>(optr(weight));
        a.ignore_index = ignore, a.temperature = (float)T, a.loss = fptr(loss), a.row_grad = fptr(row_grad);
        a.dhidden = ptr(dh), a.dweight = ptr(dw), a.piece_rows = piece;
        if (kept) {  // an empty tensor: the forward, into what it can keep; else the gradients from it
            a.phase = kept->defined() ? THESEUS_VOCAB_GRADIENTS : THESEUS_VOCAB_FORWARD;
            if (!kept->defined()) {
                *kept = scratch(theseus_vocab_loss_kept_size(&a), h);
                if (!kept->defined()) a.phase = THESEUS_VOCAB_ALL;
            }
            a.kept = ptr(*kept);
        }
        const size_t need = theseus_vocab_loss_workspace_size(&a);
        const Tensor ws = scratch(need, h);
        raise_status(theseus_vocab_loss(&a, ptr(ws), need, stream_of(h)), "theseus_vocab");
    }
    static Tensor new_loss(const Tensor& h, int64_t reduction) {
        const auto f = h.options().dtype(torch::kFloat32);
        return reduction == THESEUS_VOCAB_NONE ? at::empty({h.size(0)}, f) : at::empty({}, f);
    }
    // What a backward that forms the logits again reads of the targets, and that it was not changed since: the
    // others (gradients made with the loss, kept exponentials) do not look at these, so they are not saved
    // variables, whose unpacking would ask of every backward what only this one needs.  Tensors of inference
    // mode have no version: a copy.
    static void hold(AutogradContext* ctx, const char* name, const Opt& t) {
        if (!t) return;
        const Tensor own = t->is_inference() ? t->clone() : *t;
        ctx->saved_data[name] = own;
        ctx->saved_data[std::string(name) + " version"] = (int64_t)own._version();
    }
    static Opt held(AutogradContext* ctx, const char* name) {
        const auto at = ctx->saved_data.find(name);
        if (at == ctx->saved_data.end()) return Opt();
        const Tensor t = at->second.toTensor();
        TORCH_CHECK((int64_t)t._version() == ctx->saved_data[std::string(name) + " version"].toInt(), "theseus_vocab: the ", name,
                    " have been modified by an inplace operation after the loss whose gradients need them");
        return t;
    }
    static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& index, const Opt& top, const Opt& lse,
                          const Opt& weight, int64_t ignore, double T, int64_t reduction, int64_t piece) {
        c10::OptionalDeviceGuard guard(h.device());
        const Tensor loss = new_loss(h, reduction);
        Tensor dh, dw, kept;
        if (reduction != THESEUS_VOCAB_NONE) {
            if (h.requires_grad()) dh = at::empty(h.sizes(), h.options());
            if (w.requires_grad()) dw = at::empty(w.sizes(), w.options());
            ctx->saved_data["made"] = true;
            ctx->saved_data["dh"] = dh.defined() ? at::IValue(dh) : at::IValue();
            ctx->saved_data["dw"] = dw.defined() ? at::IValue(dw) : at::IValue();
        } else {
            ctx->saved_data["made"] = false;
        }
        call(h, w, index, top, lse, weight, ignore, T, reduction, piece, loss, Tensor(), dh, dw,
             reduction == THESEUS_VOCAB_NONE ? &kept : nullptr);
        ctx->saved_data["kept"] = kept.defined() ? at::IValue(kept) : at::IValue();
        ctx->save_for_backward({h, w});
        hold(ctx, INDEX, index), hold(ctx, TOP, top), hold(ctx, LSE, lse), hold(ctx, WEIGHT, weight);
        ctx->saved_data["ignore"] = ignore, ctx->saved_data["T"] = T, ctx->saved_data["reduction"] = reduction;
        ctx->saved_data["piece"] = piece;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        auto& d = ctx->saved_data;
        auto tensor = [](at::IValue& v) { return v.isTensor() ? v.toTensor() : Tensor(); };
        Tensor dh, dw;
        const Tensor grad = float_rows(g[0]);
        const int64_t reduction = d["reduction"].toInt();
        c10::OptionalDeviceGuard guard(grad.device());
        const bool made = d["made"].toBool();
        if (made) {  // the gradients of upstream gradient 1, handed out once
            dh = tensor(d["dh"]), dw = tensor(d["dw"]);
            d["made"] = false, d["dh"] = at::IValue(), d["dw"] = at::IValue();
        } else {
            const variable_list s = ctx->get_saved_variables();
            if (ctx->needs_input_grad(0)) dh = at::empty(s[0].sizes(), s[0].options());
            if (ctx->needs_input_grad(1)) dw = at::empty(s[1].sizes(), s[1].options());
            Tensor kept = tensor(d["kept"]);
            d["kept"] = at::IValue();
            auto target = [&](const char* name) {  // (with exponentials, their targets were kept too)
                if (!kept.defined()) return held(ctx, name);
                const auto at = d.find(name);
                return at == d.end() ? Opt() : Opt(at->second.toTensor());
            };
            call(s[0], s[1], *target(INDEX), target(TOP), target(LSE), target(WEIGHT), d["ignore"].toInt(), d["T"].toDouble(),
                 reduction, d["piece"].toInt(), Tensor(), reduction == THESEUS_VOCAB_NONE ? grad : Tensor(), dh, dw, kept.defined() ? &kept : nullptr);
        }
        if (reduction != THESEUS_VOCAB_NONE)
            raise_status(theseus_vocab_scale(ptr(dh), dh.defined() ? dh.numel() : 0, ptr(dw), dw.defined() ? dw.numel() : 0, fptr(grad),
                                             stream_of(grad)),
                         "theseus_vocab");
        variable_list o{dh, dw};
        if (at::GradMode::is_enabled()) {  // (create_graph: a later derivative through these raises)
            for (Tensor& t : o)
                if (t.defined()) t.requires_grad_();
            o = (*std::make_shared<torch::autograd::DelayedError>("theseus_vocab: the losses are differentiable once", 2))(std::move(o));
        }
        o.resize(10);
        return o;
    }
};

Tensor vocab_loss(const Tensor& h, const Tensor& w, const Tensor& index, const std::optional<Tensor>& top, const std::optional<Tensor>& lse,
                  const std::optional<Tensor>& weight, int64_t ignore, double T, int64_t reduction, int64_t piece) {
    py::gil_scoped_release free;
    if (at::GradMode::is_enabled() && (h.requires_grad() || w.requires_grad()))
        return VocabLoss::apply(h, w, index, top, lse, weight, ignore, T, reduction, piece);
    c10::OptionalDeviceGuard guard(h.device());
    const Tensor loss = VocabLoss::new_loss(h, reduction);
    VocabLoss::call(h, w, index, top, lse, weight, ignore, T, reduction, piece, loss, Tensor(), Tensor(), Tensor());
    return loss;
}

// theseus.vocab.top_logits for x [M][V], checked there: values, indices, lse of M rows
std::tuple<Tensor, Tensor, Tensor> vocab_top(const Tensor& x, int64_t k, double T) {
    py::gil_scoped_release free;
    c10::OptionalDeviceGuard guard(x.device());
    const int64_t M = x.size(0), V = x.size(1);
    const int dt = x.scalar_type() == torch::kBFloat16 ? THESEUS_VOCAB_BF16 : THESEUS_VOCAB_FP32;
    const Tensor values = at::empty({M, k}, x.options()), indices = at::empty({M, k}, x.options().dtype(torch::kInt64)),
                 lse = at::empty({M}, x.options().dtype(torch::kFloat32));
    const size_t need = theseus_vocab_top_workspace_size(M, V, (int)k, dt);
    const Tensor ws = scratch(need, x);
    raise_status(theseus_vocab_top(M, V, (int)k, dt, (float)T, x.data_ptr(), std::max(x.stride(0), V), values.data_ptr(),
                                   indices.data_ptr<int64_t>(), fptr(lse), ptr(ws), need, stream_of(x)),
                 "theseus_vocab");
    return {values, indices, lse};
}

// theseus.vocab.embedding.  A node of its own: a short call's host time is mostly the engine's, and
// torch::autograd::Function adds its dictionary to it.
int embed_type(const Tensor& t) { return t.scalar_type() == torch::kBFloat16 ? THESEUS_EMBED_BF16 : THESEUS_EMBED_FP32; }
struct EmbeddingGrad : torch::autograd::Node {
    torch::autograd::SavedVariable ids;
    int64_t V, D, skip;
    float scale;
    bool fp32;
    std::string name() const override { return "EmbeddingBackward"; }
    void release_variables() override { ids.reset_data(); }
    variable_list apply(variable_list&& g) override {
        if (!g[0].defined()) return {Tensor()};
        const Tensor at = ids.unpack();
        const int64_t M = at.numel();
        Tensor dw;
        {
            at::NoGradGuard no_grad;
            Tensor grad = g[0].dim() == 2 ? g[0] : g[0].reshape({M, D});
            if (grad.scalar_type() != torch::kBFloat16) grad = grad.to(torch::kFloat32);
            if (grad.stride(1) != 1 || (grad.stride(0) < D && grad.stride(0) != 0)) grad = grad.contiguous();
            c10::OptionalDeviceGuard guard(grad.device());
            dw = at::empty({V, D}, grad.options().dtype(fp32 ? torch::kFloat32 : torch::kBFloat16));
            const size_t need = theseus_embed_grad_workspace_size(M, V, (int)D);
            const Tensor ws = scratch(need, grad);
            raise_status(theseus_embed_grad(M, V, (int)D, embed_type(grad), embed_type(dw), at.data_ptr<int64_t>(), skip, grad.data_ptr(),
                                            grad.stride(0), scale, dw.data_ptr(), ptr(ws), need, stream_of(grad)),
                         "theseus_vocab");
        }
        variable_list o{dw};
        if (at::GradMode::is_enabled()) {  // (create_graph: a later derivative through this raises)
            o[0].requires_grad_();
            o = (*std::make_shared<torch::autograd::DelayedError>("theseus_vocab: embedding is differentiable once", 1))(std::move(o));
        }
        return o;
    }
};

// A captured backward runs each node on the stream that the node was made on: one that was made outside of the capture
// would draw its stream into it, and end the process.  Such are the nodes of a weight that was computed there, and of each
// leaf below the accumulator of an eager graph that lives.
void check_capture(const Tensor& w) {
    const auto held = w.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(w) : w.grad_fn();
    if (!held) return;
    hipStreamCaptureStatus now = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream_of(w), &now) != hipSuccess || now == hipStreamCaptureStatusNone) return;
    const auto here = c10::impl::VirtualGuardImpl(w.device().type()).getStream(w.device());
    std::vector<torch::autograd::Node*> nodes{held.get()};
    std::unordered_set<torch::autograd::Node*> seen{held.get()};
    while (!nodes.empty()) {
        torch::autograd::Node* const node = nodes.back();
        nodes.pop_back();
        const auto made_on = node->stream();
        TORCH_CHECK(!made_on || *made_on == here,
                    "theseus_vocab: embedding is captured into a graph while an autograd graph of its weight from another stream lives: free "
                    "that one (its outputs and losses) first");
        for (const auto& edge : node->next_edges())
            if (edge.function && seen.insert(edge.function.get()).second) nodes.push_back(edge.function.get());
    }
}

// Nothing where an argument is not as the kernels take it: theseus/vocab.py then lays it out or says what is wrong.
std::optional<Tensor> embedding(const Tensor& ids, const Tensor& w, double scale, std::optional<int64_t> padding_idx, std::optional<at::ScalarType> dtype) {
    auto known = [](at::ScalarType t) { return t == torch::kBFloat16 || t == torch::kFloat32; };
    if (!w.is_cuda() || w.layout() != at::kStrided || w.dim() != 2 || !known(w.scalar_type()) || !ids.is_cuda() || ids.layout() != at::kStrided ||
        ids.scalar_type() != torch::kInt64 || ids.device() != w.device() || !ids.is_contiguous() || !known(dtype.value_or(w.scalar_type())))
        return {};
    const int64_t M = ids.numel(), V = w.size(0), D = w.size(1);
    const int64_t skip = !padding_idx ? -1 : *padding_idx < 0 ? *padding_idx + V : *padding_idx;
    if (V < 1 || D < 1 || V > 1 << 22 || D > 1 << 17 || M > 1 << 30 || (D > 1 && w.stride(1) != 1) || (V > 1 && w.stride(0) < D) ||
        (padding_idx && (skip < 0 || skip >= V)) || !(std::abs(scale) <= std::numeric_limits<float>::max()))
        return {};
    py::gil_scoped_release free;
    c10::OptionalDeviceGuard guard(w.device());
    const bool differentiable = at::GradMode::is_enabled() && w.requires_grad();
    if (differentiable) check_capture(w);
    at::DimVector sizes(ids.sizes());
    sizes.push_back(D);
    const Tensor out = at::empty(sizes, w.options().dtype(dtype.value_or(w.scalar_type())));
    raise_status(theseus_embed_lookup(M, V, (int)D, embed_type(w), embed_type(out), ids.data_ptr<int64_t>(), w.data_ptr(), std::max(w.stride(0), D),
                                      (float)scale, out.data_ptr(), stream_of(w)),
                 "theseus_vocab");
    if (differentiable) {
        const std::shared_ptr<EmbeddingGrad> node(new EmbeddingGrad(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(w));
        // (tokens of inference mode have no version: a copy)
        node->ids = torch::autograd::SavedVariable(ids.is_inference() ? ids.clone() : ids, false);
        node->V = V, node->D = D, node->skip = skip, node->scale = (float)scale, node->fp32 = embed_type(w) == THESEUS_EMBED_FP32;
        torch::autograd::set_history(out, node);
    }
    return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("wkv7", &wkv7, "(y, end state) of the recurrence, differentiable");
    m.def("gdn", &gdn, "(o, end state) of the gated delta rule with gradients, differentiable", py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("g"), py::arg("beta"), py::arg("s0"), py::arg("qk_l2norm") = false);
    m.def("vocab_loss", &vocab_loss, "a vocabulary loss, differentiable in h and w");
    m.def("embedding", &embedding, "rows of a table by index, differentiable in the table");
    m.def("vocab_top", &vocab_top, "(values, indices, log-sum-exp) of the top logits");
}
