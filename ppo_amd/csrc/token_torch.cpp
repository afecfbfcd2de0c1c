// ppo_amd.tokens below its documentation: argument checks, allocation and autograd nodes over the C ABI of the losses
// over a large vocabulary (include/ppo_hip.h).  A call on a few rows is host time and little else: the same steps in
// Python and ctypes took 25 us for the policy loss with its gradient and 120 us for a forward and a backward pass.
//
// The library is the one that ppo_amd._lib has loaded; its functions' addresses are handed over at import.
#include <ATen/core/Tensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/ppo_hip.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------------------------------------ the library
#define LIBRARY(F) \
    F(ppo_token_workspace_bytes) F(ppo_token_logprobs) F(ppo_token_logprobs_backward) F(ppo_policy_loss) \
    F(ppo_preference_loss) F(ppo_distillation_loss) F(ppo_distillation_backward) F(ppo_hip_strerror)
struct Library {
#define MEMBER(name) decltype(&::name) name = nullptr;
    LIBRARY(MEMBER)
#undef MEMBER
};
static Library lib;

static void bind(const std::map<std::string, uintptr_t>& address) {
#define SET(name) lib.name = reinterpret_cast<decltype(&::name)>(address.at(#name));
    LIBRARY(SET)
#undef SET
}

static void done(int code) {
    TORCH_CHECK(code == 0, "libppo_hip call failed (", code, "): ", lib.ppo_hip_strerror(code));
}

// ------------------------------------------------------------------------------------------ arguments
static const char* type_name(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kDouble: return "torch.float64";
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kLong: return "torch.int64";
        case at::kInt: return "torch.int32";
        case at::kBool: return "torch.bool";
        case at::kByte: return "torch.uint8";
        default: return c10::toString(t);
    }
}

static int type_code(at::ScalarType t) {
    return t == at::kFloat ? PPO_F32 : t == at::kBFloat16 ? PPO_BF16 : t == at::kHalf ? PPO_F16 : -1;
}

// Outputs carry no forward-mode derivative, and one that is missing would be taken for zero.
static void no_tangent(const Tensor& t, const char* name) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name, ": the losses over a vocabulary have no forward-mode derivative");
}

static at::IntArrayRef check_logits(const Tensor& x) {
    no_tangent(x, "logits");
    TORCH_CHECK_VALUE(x.dim() == 2 || x.dim() == 3,
                      "logits must be a tensor [sequences, tokens, vocabulary] or [tokens, vocabulary]");
    TORCH_CHECK_VALUE(type_code(x.scalar_type()) >= 0, "logits of type ", type_name(x.scalar_type()),
                      ": float32, bfloat16 and float16 are supported");
    TORCH_CHECK_VALUE(!x.is_neg(), "logits that torch has yet to negate (a lazy view): resolve_neg() them first");
    TORCH_CHECK_VALUE(x.size(-1) > 0, "logits over an empty vocabulary");
    TORCH_CHECK_VALUE(x.size(-1) == 1 || x.stride(-1) == 1, "the vocabulary must be the contiguous dimension of the logits");
    return x.sizes().slice(0, x.dim() - 1);
}

enum class Kind { INTEGERS, MASK, FLOATS, LOGITS };

// A tensor beside the logits: of its types, of this shape, where the logits are, without a gradient of its own.
static void check(const Tensor& x, const Tensor& t, const char* name, Kind kind, at::IntArrayRef shape) {
    TORCH_CHECK_VALUE(t.defined() && t.device() == x.device(), name, " must be a tensor on ", x.device(), ", where the logits are");
    no_tangent(t, name);
    TORCH_CHECK_VALUE(!t.requires_grad(), name, " requires grad, but gradients are computed with respect to the logits only: detach it");
    const auto d = t.scalar_type();
    switch (kind) {
        case Kind::INTEGERS:
            TORCH_CHECK_VALUE(d == at::kLong || d == at::kInt, name, " of type ", type_name(d), ": int64 and int32 are supported");
            break;
        case Kind::MASK:
            TORCH_CHECK_VALUE(d == at::kBool || d == at::kByte, name, " of type ", type_name(d), ": bool and uint8 are supported");
            break;
        case Kind::FLOATS:
            TORCH_CHECK_VALUE(type_code(d) >= 0 || d == at::kDouble, name, " of type ", type_name(d), ": floating point is expected");
            break;
        case Kind::LOGITS:
            TORCH_CHECK_VALUE(type_code(d) >= 0, name, " of type ", type_name(d), ": float32, bfloat16 and float16 are supported");
            break;
    }
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " of shape ", t.sizes(), ", expected ", shape);
}

static Tensor integers(const Tensor& x, const Tensor& t, const char* name, at::IntArrayRef shape) {
    check(x, t, name, Kind::INTEGERS, shape);
    return t.contiguous();
}
static Tensor mask_of(const Tensor& x, const OptTensor& t, at::IntArrayRef shape) {
    if (!t) return Tensor();
    check(x, *t, "mask", Kind::MASK, shape);
    return t->contiguous();
}
// The numbers themselves, where complex arithmetic has left a view that torch has yet to negate.
static Tensor resolved(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
static Tensor floats(const Tensor& x, const Tensor& t, const char* name, at::IntArrayRef shape) {
    check(x, t, name, Kind::FLOATS, shape);
    return resolved(t.scalar_type() == at::kFloat ? t : t.to(at::kFloat));
}

static double inverse(double temperature) {
    TORCH_CHECK_VALUE(temperature >= 1e-6 && temperature <= 1e6, "temperature ", temperature, ": between 1e-6 and 1e6 is expected");
    return 1.0 / temperature;
}

struct Strides {
    int64_t seq, tok;
};
static Strides row_strides(const Tensor& t) {   // of a tensor of one number a row
    return t.dim() == 2 ? Strides{t.stride(0), t.stride(1)} : Strides{0, t.stride(0)};
}

// Address range of a tensor's elements.
static std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
    int64_t last = t.numel() ? 0 : -1;
    if (t.numel())
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    const auto at = (uintptr_t)t.data_ptr();
    return {at, at + (last + 1) * t.element_size()};
}

// The place for a gradient that the caller gave: of the logits' kind, rows apart, over nothing but the logits themselves.
static Tensor check_out(const Tensor& out, const Tensor& x, std::initializer_list<std::pair<const char*, Tensor>> others) {
    TORCH_CHECK_VALUE(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && out.device() == x.device(),
                      "out must have the shape, the type and the device of the logits");
    no_tangent(out, "out");
    TORCH_CHECK_VALUE(!out.is_neg(), "out is a view that torch has yet to negate");
    TORCH_CHECK_VALUE(out.size(-1) == 1 || out.stride(-1) == 1, "the vocabulary must be the contiguous dimension of out");
    int64_t order[2] = {out.dim() - 2, 0}, reach = out.size(-1);     // the rows' dimensions, the closer rows first
    if (out.dim() == 3 && out.size(0) > 1 && out.size(1) > 1 && out.stride(0) < out.stride(1)) std::swap(order[0], order[1]);
    for (int64_t k = 0; k < out.dim() - 1; ++k) {
        const int64_t d = order[k];
        if (out.size(d) <= 1) continue;
        TORCH_CHECK_VALUE(out.stride(d) >= reach, "rows of out overlap");
        reach += (out.size(d) - 1) * out.stride(d);
    }
    const auto [lo, hi] = span(out);
    const auto [xlo, xhi] = span(x);
    TORCH_CHECK_VALUE(xlo >= hi || lo >= xhi || (xlo == lo && out.strides() == x.strides()),
                      "out shares memory with the logits: only the logits themselves can be overwritten");
    for (const auto& [name, t] : others) {
        if (!t.defined()) continue;
        const auto [a, b] = span(t);
        TORCH_CHECK_VALUE(a >= hi || lo >= b, "out shares memory with ", name);
    }
    return out.detach();
}

// Storage for the gradient: the logits' own row strides and alignment where that wastes little memory (16-byte accesses
// then fall on the same boundaries in both), dense rows otherwise.
static Tensor grad_like(const Tensor& x) {
    if (x.is_contiguous()) return at::empty_like(x);
    int64_t reach = x.size(-1);
    bool follow = x.numel() > 0;
    for (int64_t d = x.dim() - 2; d >= 0 && follow; --d) {
        if (x.size(d) > 1 && x.stride(d) < reach) follow = false;   // broadcast or reordered rows
        reach += (x.size(d) - 1) * x.stride(d);
    }
    if (!follow || (double)reach > 1.25 * (double)x.numel() + 64) return at::empty_like(x, {}, at::MemoryFormat::Contiguous);
    const int64_t lead = (int64_t)((uintptr_t)x.data_ptr() % 16 / x.element_size());
    return at::empty({reach + lead}, x.options()).as_strided(x.sizes(), x.strides(), lead);
}

static ppo_token_logits rows_of(const Tensor& x, double inv_t, const Tensor& grad = Tensor()) {
    ppo_token_logits r{};
    const bool three = x.dim() == 3;
    r.data = x.data_ptr();
    r.seq_stride = three ? x.stride(0) : 0;
    r.tok_stride = x.stride(-2);
    if (grad.defined()) {
        r.grad_seq_stride = three ? grad.stride(0) : 0;
        r.grad_tok_stride = grad.stride(-2);
    }
    r.n_seq = three ? x.size(0) : 1;
    r.n_tok = x.size(-2);
    r.vocab = x.size(-1);
    r.dtype = type_code(x.scalar_type());
    r.inv_temperature = inv_t;
    return r;
}

// ------------------------------------------------------------------------------------------ calls
struct Call {                 // the logits' device is the current one; the stream is its current stream
    c10::OptionalDeviceGuard guard;
    void* stream;
    explicit Call(const Tensor& x) {
        TORCH_CHECK(x.is_cuda(), "ppo_amd: logits on ", x.device(), "; the HIP engine has no CPU fallback");
        guard.reset_device(x.device());
        stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream();
    }
};

template <typename T> static T* at_of(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
static bool is_i64(const Tensor& t) { return t.scalar_type() == at::kLong; }

static Tensor new_floats(const Tensor& x, at::IntArrayRef shape) { return at::empty(shape, x.options().dtype(at::kFloat)); }

// Scratch of one call, and `floats` a row behind it that a backward call reads.
struct Scratch {
    Tensor memory;
    int64_t need;
    char* at() const { return (char*)memory.data_ptr(); }
    float* behind() const { return (float*)(at() + need); }
};
static Scratch scratch(const Tensor& x, at::IntArrayRef rows, int64_t floats) {
    const int64_t n_seq = rows.size() == 2 ? rows[0] : 1, n_tok = rows.back();
    const int64_t need = (int64_t)lib.ppo_token_workspace_bytes(n_seq, n_tok);
    return {at::empty({need + 4 * floats * n_seq * n_tok}, x.options().dtype(at::kByte)), need};
}

// A gradient that comes into a backward call, or none.
static Tensor incoming(const Tensor& g) {
    if (g.defined()) no_tangent(g, "a gradient");
    return resolved(g);
}

static bool wants_grad(const Tensor& x) { return at::GradMode::is_enabled() && x.requires_grad(); }

// A gradient that is itself differentiated raises, and not before.
static Tensor once(const Tensor& grad) {
    if (!at::GradMode::is_enabled()) return grad;
    auto error = std::make_shared<torch::autograd::DelayedError>("ppo_amd: the losses over a vocabulary can be differentiated once", 1);
    return (*error)({grad.detach().requires_grad_(true)})[0];
}

static Tensor backward_call(const Tensor& x, const Tensor& tokens, const Tensor& mask, double inv_t, const float* stats,
                            const float* g_lp, Strides lp, const float* g_ent, Strides ent, const Tensor& factor) {
    const Call call(x);
    const Tensor grad = grad_like(x);
    const ppo_token_logits r = rows_of(x, inv_t, grad);
    done(lib.ppo_token_logprobs_backward(&r, tokens.data_ptr(), is_i64(tokens), at_of<uint8_t>(mask), stats, g_lp, lp.seq,
                                         lp.tok, g_ent, ent.seq, ent.tok, at_of<float>(factor), grad.data_ptr(), call.stream));
    return once(grad);
}

// ------------------------------------------------------------------------------------------ log-probabilities
struct Logprobs : torch::CustomClassHolder {
    Tensor tokens, mask;
    double inv_t = 1.0;
    bool entropy = true;
};

static std::pair<Tensor, Tensor> logprobs_call(const Tensor& x, const Logprobs& p, const Tensor& stats) {
    const Call call(x);
    const Tensor lp = new_floats(x, p.tokens.sizes()), ent = p.entropy ? at::empty_like(lp) : Tensor();
    const ppo_token_logits r = rows_of(x, p.inv_t);
    const bool few_long = p.tokens.numel() <= PPO_TOKEN_CUT_ROWS && x.size(-1) * x.element_size() >= PPO_TOKEN_CUT_BYTES;
    const Scratch ws = few_long ? scratch(x, p.tokens.sizes(), 0) : Scratch{Tensor(), 0};
    done(lib.ppo_token_logprobs(&r, p.tokens.data_ptr(), is_i64(p.tokens), at_of<uint8_t>(p.mask), at_of<float>(lp),
                                at_of<float>(ent), at_of<float>(stats), at_of<void>(ws.memory), (size_t)ws.need, call.stream));
    return {lp, ent};
}

struct LogprobsNode : torch::autograd::Function<LogprobsNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const c10::intrusive_ptr<Logprobs>& p) {
        const Tensor stats = new_floats(x, {p->tokens.numel(), 4});
        const auto [lp, ent] = logprobs_call(x, *p, stats);
        ctx->saved_data["inv_t"] = p->inv_t;
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, p->tokens, p->mask, stats});
        if (p->entropy) return {lp, ent};
        return {lp};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const Tensor g_lp = incoming(g[0]), g_ent = g.size() > 1 ? incoming(g[1]) : Tensor();
        if (!g_lp.defined() && !g_ent.defined()) return variable_list(2);
        const auto s = ctx->get_saved_variables();
        const Strides none{0, 0};
        return {backward_call(s[0], s[1], s[2], ctx->saved_data["inv_t"].toDouble(), at_of<float>(s[3]),
                              at_of<float>(g_lp), g_lp.defined() ? row_strides(g_lp) : none, at_of<float>(g_ent),
                              g_ent.defined() ? row_strides(g_ent) : none, Tensor()),
                Tensor()};
    }
};

static std::pair<Tensor, OptTensor> token_logprobs(const Tensor& x, const Tensor& tokens, const OptTensor& mask,
                                                   double temperature, bool entropy) {
    const auto shape = check_logits(x);
    auto p = c10::make_intrusive<Logprobs>();
    p->tokens = integers(x, tokens, "tokens", shape);
    p->mask = mask_of(x, mask, shape);
    p->inv_t = inverse(temperature);
    p->entropy = entropy;
    if (wants_grad(x)) {
        const auto out = LogprobsNode::apply(x, p);
        return {out[0], entropy ? OptTensor(out[1]) : OptTensor()};
    }
    const auto [lp, ent] = logprobs_call(x, *p, Tensor());
    return {lp, entropy ? OptTensor(ent) : OptTensor()};
}

// ------------------------------------------------------------------------------------------ clipped policy loss
struct Policy : torch::CustomClassHolder {
    Tensor tokens, mask, old_lp, adv, ref;
    Strides adv_strides{};
    ppo_policy_terms terms{};
    double inv_t = 1.0;
};

static c10::intrusive_ptr<Policy> policy_args(const Tensor& x, const Tensor& tokens, const Tensor& old_lp, const Tensor& adv,
                                              const OptTensor& mask, const OptTensor& ref, double eps_clip,
                                              std::optional<double> eps_high, double kl, double ent, double temperature,
                                              int reduction, double scale) {
    auto p = c10::make_intrusive<Policy>();
    const auto shape = check_logits(x);
    p->tokens = integers(x, tokens, "tokens", shape);
    p->mask = mask_of(x, mask, shape);
    p->old_lp = floats(x, old_lp, "old_logprobs", shape).contiguous();
    const int64_t n_seq = shape.size() == 2 ? shape[0] : 1;
    const bool per_sequence = adv.sizes() != shape &&
        ((adv.dim() == 1 && adv.size(0) == n_seq) || (adv.dim() == 2 && adv.size(0) == n_seq && adv.size(1) == 1));
    p->adv = floats(x, adv, "advantages", per_sequence ? adv.sizes() : shape);
    p->adv_strides = per_sequence ? Strides{p->adv.stride(0), 0} : row_strides(p->adv);
    TORCH_CHECK_VALUE(ref || kl == 0.0, "kl_coef without ref_logprobs");
    if (ref) p->ref = floats(x, *ref, "ref_logprobs", shape).contiguous();
    const double high = eps_high.value_or(eps_clip);
    TORCH_CHECK_VALUE(eps_clip >= 0.0 && eps_clip <= 1.0 && high >= 0.0, "clip range [1 - ", eps_clip, ", 1 + ", high,
                      "]: 0 <= eps_clip <= 1 and eps_clip_high >= 0 are expected");
    p->terms = {(float)eps_clip, (float)high, (float)kl, (float)ent, (float)scale, reduction};
    p->inv_t = inverse(temperature);
    return p;
}

struct PolicyOut {
    Tensor loss, lp, ent;
    Scratch ws;
};

// Statistics and seeds for a backward call lie behind the scratch: 4 floats a row, then dloss/dlogprob, then dloss/dentropy.
static PolicyOut policy_call(const Tensor& x, const Policy& p, const Tensor& grad, bool seeds) {
    const Call call(x);
    PolicyOut o{new_floats(x, {}), at::empty_like(p.old_lp), at::empty_like(p.old_lp), scratch(x, p.old_lp.sizes(), seeds ? 6 : 0)};
    const ppo_token_logits r = rows_of(x, p.inv_t, grad);
    float* stats = seeds ? o.ws.behind() : nullptr;
    done(lib.ppo_policy_loss(&r, p.tokens.data_ptr(), is_i64(p.tokens), at_of<uint8_t>(p.mask), at_of<float>(p.old_lp),
                             at_of<float>(p.adv), p.adv_strides.seq, p.adv_strides.tok, at_of<float>(p.ref), &p.terms,
                             at_of<float>(o.loss), at_of<float>(o.lp), at_of<float>(o.ent), stats,
                             seeds ? stats + 4 * p.old_lp.numel() : nullptr, at_of<void>(grad), o.ws.at(), (size_t)o.ws.need,
                             call.stream));
    return o;
}

struct PolicyNode : torch::autograd::Function<PolicyNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const c10::intrusive_ptr<Policy>& p) {
        const PolicyOut o = policy_call(x, *p, Tensor(), true);
        ctx->saved_data["offset"] = o.ws.need;
        ctx->saved_data["inv_t"] = p->inv_t;
        ctx->saved_data["entropy"] = p->terms.entropy_coef != 0.0f;
        ctx->mark_non_differentiable({o.lp, o.ent});
        ctx->set_materialize_grads(false);    // else two launches fill zeros that nobody reads
        ctx->save_for_backward({x, p->tokens, p->mask, o.ws.memory});
        return {o.loss, o.lp, o.ent};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        if (!g[0].defined()) return variable_list(2);
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &tokens = s[1];
        const float* stats = (const float*)((const char*)s[3].data_ptr() + ctx->saved_data["offset"].toInt());
        const float* g_lp = stats + 4 * tokens.numel();
        const Strides dense = row_strides(tokens);
        return {backward_call(x, tokens, s[2], ctx->saved_data["inv_t"].toDouble(), stats, g_lp, dense,
                              ctx->saved_data["entropy"].toBool() ? g_lp + tokens.numel() : nullptr, dense, incoming(g[0])),
                Tensor()};
    }
};

using Policy3 = std::tuple<Tensor, Tensor, Tensor>;
static Policy3 policy_loss(const Tensor& x, const Tensor& tokens, const Tensor& old_lp, const Tensor& adv, const OptTensor& mask,
                           const OptTensor& ref, double eps_clip, std::optional<double> eps_high, double kl, double ent,
                           double temperature, int reduction, double scale) {
    const auto p = policy_args(x, tokens, old_lp, adv, mask, ref, eps_clip, eps_high, kl, ent, temperature, reduction, scale);
    if (wants_grad(x)) {
        const auto out = PolicyNode::apply(x, p);
        return {out[0], out[1], out[2]};
    }
    const PolicyOut o = policy_call(x, *p, Tensor(), false);
    return {o.loss, o.lp, o.ent};
}

// The logits of a call that gives their gradient itself.
static Tensor values_of(const Tensor& x) {
    no_tangent(x, "logits");      // (detach leaves it behind)
    return x.detach();
}

// The version counter of overwritten memory moves, so that autograd notices a use of old values.
static void overwritten(const OptTensor& out, const Tensor& x) {
    if (!out) return;         // (tensors of inference mode have no counter)
    if (!out->is_inference()) torch::autograd::impl::bump_version(*out);
    if (out->data_ptr() == x.data_ptr() && !x.is_inference()) torch::autograd::impl::bump_version(x);
}

static std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss_and_grad(
    const Tensor& x_, const Tensor& tokens, const Tensor& old_lp, const Tensor& adv, const OptTensor& mask, const OptTensor& ref,
    double eps_clip, std::optional<double> eps_high, double kl, double ent, double temperature, int reduction, double scale,
    const OptTensor& out) {
    const at::NoGradGuard off;
    const Tensor x = values_of(x_);
    const auto p = policy_args(x, tokens, old_lp, adv, mask, ref, eps_clip, eps_high, kl, ent, temperature, reduction, scale);
    const Tensor grad = out ? check_out(*out, x, {{"tokens", p->tokens}, {"mask", p->mask}, {"old_logprobs", p->old_lp},
                                                  {"advantages", p->adv}, {"ref_logprobs", p->ref}})
                            : grad_like(x);
    const PolicyOut o = policy_call(x, *p, grad, false);
    overwritten(out, x_);
    return {o.loss, grad, o.lp, o.ent};
}

// ------------------------------------------------------------------------------------------ preference loss
struct Preference : torch::CustomClassHolder {
    Tensor tokens, mask, ref;
    double beta = 0, smoothing = 0, scale = 1;
};

static c10::intrusive_ptr<Preference> preference_args(const Tensor& x, const Tensor& tokens, const Tensor& ref,
                                                      const OptTensor& mask, double beta, double smoothing, double scale) {
    auto p = c10::make_intrusive<Preference>();
    const auto shape = check_logits(x);
    TORCH_CHECK_VALUE(x.dim() == 3 && x.size(0) >= 2 && x.size(0) % 2 == 0,
                      "preference losses need logits [2 * pairs, tokens, vocabulary]: the preferred sequences, then the rejected "
                      "ones in the same order; got ", x.sizes());
    p->tokens = integers(x, tokens, "tokens", shape);
    p->mask = mask_of(x, mask, shape);
    p->ref = floats(x, ref, "ref_logprobs", shape.slice(0, 1)).contiguous();
    TORCH_CHECK_VALUE(smoothing >= 0.0 && smoothing < 1.0, "label_smoothing ", smoothing, ": 0 <= label_smoothing < 1 is expected");
    p->beta = beta;
    p->smoothing = smoothing;
    p->scale = scale;
    return p;
}

struct PreferenceOut {
    Tensor loss, rewards, seeds;   // seeds: dloss/dlogprob of each sequence's tokens
    Scratch ws;                    // the rows' statistics behind it
};

static PreferenceOut preference_call(const Tensor& x, const Preference& p, const Tensor& grad, bool seeds) {
    const Call call(x);
    PreferenceOut o{new_floats(x, {}), at::empty_like(p.ref), seeds ? at::empty_like(p.ref) : Tensor(),
                    scratch(x, p.tokens.sizes(), seeds ? 4 : 0)};
    const ppo_token_logits r = rows_of(x, 1.0, grad);
    done(lib.ppo_preference_loss(&r, p.tokens.data_ptr(), is_i64(p.tokens), at_of<uint8_t>(p.mask), at_of<float>(p.ref), p.beta,
                                 p.smoothing, p.scale, at_of<float>(o.loss), at_of<float>(o.rewards),
                                 seeds ? o.ws.behind() : nullptr, at_of<float>(o.seeds), at_of<void>(grad), o.ws.at(),
                                 (size_t)o.ws.need, call.stream));
    return o;
}

struct PreferenceNode : torch::autograd::Function<PreferenceNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const c10::intrusive_ptr<Preference>& p) {
        const PreferenceOut o = preference_call(x, *p, Tensor(), true);
        ctx->saved_data["offset"] = o.ws.need;
        ctx->mark_non_differentiable({o.rewards});
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, p->tokens, p->mask, o.ws.memory, o.seeds});
        return {o.loss, o.rewards};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        if (!g[0].defined()) return variable_list(2);
        const auto s = ctx->get_saved_variables();
        const float* stats = (const float*)((const char*)s[3].data_ptr() + ctx->saved_data["offset"].toInt());
        return {backward_call(s[0], s[1], s[2], 1.0, stats, at_of<float>(s[4]), {1, 0}, nullptr, {0, 0}, incoming(g[0])), Tensor()};
    }
};

static std::pair<Tensor, Tensor> preference_loss(const Tensor& x, const Tensor& tokens, const Tensor& ref, const OptTensor& mask,
                                                 double beta, double smoothing, double scale) {
    const auto p = preference_args(x, tokens, ref, mask, beta, smoothing, scale);
    if (wants_grad(x)) {
        const auto out = PreferenceNode::apply(x, p);
        return {out[0], out[1]};
    }
    const PreferenceOut o = preference_call(x, *p, Tensor(), false);
    return {o.loss, o.rewards};
}

static Policy3 preference_loss_and_grad(const Tensor& x_, const Tensor& tokens, const Tensor& ref, const OptTensor& mask,
                                        double beta, double smoothing, double scale, const OptTensor& out) {
    const at::NoGradGuard off;
    const Tensor x = values_of(x_);
    const auto p = preference_args(x, tokens, ref, mask, beta, smoothing, scale);
    const Tensor grad = out ? check_out(*out, x, {{"tokens", p->tokens}, {"mask", p->mask}, {"ref_logprobs", p->ref}}) : grad_like(x);
    const PreferenceOut o = preference_call(x, *p, grad, false);
    overwritten(out, x_);
    return {o.loss, grad, o.rewards};
}

// ------------------------------------------------------------------------------------------ distillation
struct Teacher : torch::CustomClassHolder {
    Tensor index, logits, mask;
    double inv_t = 1.0;
    float scale = 1.0f;
    int reduction = 0;
};

static c10::intrusive_ptr<Teacher> teacher_args(const Tensor& x, const Tensor& index, const Tensor& values, const OptTensor& mask,
                                                double temperature, int reduction, double scale) {
    auto p = c10::make_intrusive<Teacher>();
    const auto shape = check_logits(x);
    TORCH_CHECK_VALUE(index.dim() == x.dim() && index.size(-1) >= 1 && index.size(-1) <= PPO_MAX_TEACHER_TOP,
                      "teacher_tokens must be ", shape, " by 1 to ", PPO_MAX_TEACHER_TOP, " entries");
    std::vector<int64_t> full(shape.begin(), shape.end());
    full.push_back(index.size(-1));
    p->index = integers(x, index, "teacher_tokens", full);
    check(x, values, "teacher_logits", Kind::LOGITS, full);
    p->logits = resolved(values).contiguous();
    p->mask = mask_of(x, mask, shape);
    p->inv_t = inverse(temperature);
    p->reduction = reduction;
    p->scale = (float)scale;
    return p;
}

struct TeacherOut {
    Tensor loss, each;
    Scratch ws;               // the rows' statistics behind it
};

static TeacherOut teacher_call(const Tensor& x, const Teacher& p, const Tensor& grad, bool seeds) {
    const Call call(x);
    const auto shape = x.sizes().slice(0, x.dim() - 1);
    TeacherOut o{new_floats(x, {}), new_floats(x, shape), scratch(x, shape, seeds ? 4 : 0)};
    const ppo_token_logits r = rows_of(x, p.inv_t, grad);
    done(lib.ppo_distillation_loss(&r, p.index.data_ptr(), is_i64(p.index), p.logits.data_ptr(), type_code(p.logits.scalar_type()),
                                   (int)p.index.size(-1), at_of<uint8_t>(p.mask), p.reduction, p.scale, at_of<float>(o.loss),
                                   at_of<float>(o.each), seeds ? o.ws.behind() : nullptr, at_of<void>(grad), o.ws.at(),
                                   (size_t)o.ws.need, call.stream));
    return o;
}

struct TeacherNode : torch::autograd::Function<TeacherNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const c10::intrusive_ptr<Teacher>& p) {
        const TeacherOut o = teacher_call(x, *p, Tensor(), true);
        ctx->saved_data["offset"] = o.ws.need;
        ctx->saved_data["inv_t"] = p->inv_t;
        ctx->mark_non_differentiable({o.each});
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, p->index, p->logits, p->mask, o.ws.memory});
        return {o.loss, o.each};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        if (!g[0].defined()) return variable_list(2);
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &index = s[1], &values = s[2];
        const float* stats = (const float*)((const char*)s[4].data_ptr() + ctx->saved_data["offset"].toInt());
        const Call call(x);
        const Tensor factor = incoming(g[0]), grad = grad_like(x);
        const ppo_token_logits r = rows_of(x, ctx->saved_data["inv_t"].toDouble(), grad);
        done(lib.ppo_distillation_backward(&r, index.data_ptr(), is_i64(index), values.data_ptr(), type_code(values.scalar_type()),
                                           (int)index.size(-1), at_of<uint8_t>(s[3]), stats, at_of<float>(factor), grad.data_ptr(),
                                           call.stream));
        return {once(grad), Tensor()};
    }
};

static std::pair<Tensor, Tensor> distillation_loss(const Tensor& x, const Tensor& index, const Tensor& values, const OptTensor& mask,
                                                   double temperature, int reduction, double scale) {
    const auto p = teacher_args(x, index, values, mask, temperature, reduction, scale);
    if (wants_grad(x)) {
        const auto out = TeacherNode::apply(x, p);
        return {out[0], out[1]};
    }
    const TeacherOut o = teacher_call(x, *p, Tensor(), false);
    return {o.loss, o.each};
}

static Policy3 distillation_loss_and_grad(const Tensor& x_, const Tensor& index, const Tensor& values, const OptTensor& mask,
                                          double temperature, int reduction, double scale, const OptTensor& out) {
    const at::NoGradGuard off;
    const Tensor x = values_of(x_);
    const auto p = teacher_args(x, index, values, mask, temperature, reduction, scale);
    const Tensor grad = out ? check_out(*out, x, {{"teacher_tokens", p->index}, {"teacher_logits", p->logits}, {"mask", p->mask}})
                            : grad_like(x);
    const TeacherOut o = teacher_call(x, *p, grad, false);
    overwritten(out, x_);
    return {o.loss, grad, o.each};
}

PYBIND11_MODULE(_token_ops, m) {
    m.def("bind", &bind);
    m.def("grad_like", &grad_like);
    m.attr("MAX_TEACHER_TOP") = PPO_MAX_TEACHER_TOP;
    m.attr("REDUCTIONS") = std::map<std::string, int>{{"sum", PPO_REDUCE_SUM}, {"token_mean", PPO_REDUCE_TOKEN_MEAN},
                                                      {"sequence_mean", PPO_REDUCE_SEQUENCE_MEAN}};
#define DEF(name) m.def(#name, &name, pybind11::call_guard<pybind11::gil_scoped_release>())
    DEF(token_logprobs);
    DEF(policy_loss);
    DEF(policy_loss_and_grad);
    DEF(preference_loss);
    DEF(preference_loss_and_grad);
    DEF(distillation_loss);
    DEF(distillation_loss_and_grad);
#undef DEF
}
