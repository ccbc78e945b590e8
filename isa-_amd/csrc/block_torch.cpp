// torch's side of libisa_block_hip.so (include/isa_block.h): the public operators of
// isa.kernels.transformer_block with their checks, allocations and gradients.
//
// It is native because these operators are called for a few microseconds of work each, dozens of
// times in a token or a training step: the same calls made from Python (ctypes, and gradients
// that take the interpreter's lock on autograd's own thread) took 18 us a call without gradients
// and 75 to 150 us a step, several times what their kernels run.
//
// Every call checks on the host what the kernels assume, allocates outputs and workspace with
// torch's caching allocator and enqueues on the current stream of the tensors' device.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <array>
#include <cmath>
#include <functional>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <tuple>

#include "isa_block.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
    std::ostringstream s;
    (s << ... << parts);
    throw std::runtime_error(s.str());
}

void check(int rc, const char* what) {
    if (rc != 0) refuse(what, " failed (", rc, "): ", isa_block_last_error());
}

std::string type_name(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        case at::kDouble: return "torch.float64";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        default: return c10::toString(t.scalar_type());
    }
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return ISA_BLOCK_F32;
        case at::kBFloat16: return ISA_BLOCK_BF16;
        case at::kHalf: return ISA_BLOCK_F16;
        default: return -1;
    }
}

// A trace would hold the allocation of a result and not what fills it.
void not_traced() {
    using namespace c10::impl;
    if (torch::jit::tracer::isTracing() || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) ||
        TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE))
        refuse("the operators of isa.kernels.transformer_block cannot be traced");
}

void require(const Tensor& t, const char* name) {
    if (!t.is_cuda()) refuse(name, " must be a CUDA tensor");
    if (type_of(t) < 0) refuse(name, " must be float32, bfloat16 or float16, got ", type_name(t));
}

void require(const Tensor& t, const char* name, const Tensor& like) {
    require(t, name);
    if (t.device() != like.device()) refuse(name, " must be on ", like.device(), ", got ", t.device());
}

void* stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor bytes(size_t n, const Tensor& like) {
    return n ? at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte)) : Tensor();
}

bool tracked(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// A tangent that a tensor carries would be lost: whether or not it requires a gradient.
template <typename Tensors>
void no_tangents(const Tensors& tensors) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor& t : tensors)
        if (t.defined() && t._fw_grad(/*level=*/0).defined())
            refuse("the operators of isa.kernels.transformer_block have no forward-mode derivatives");
}

void first_derivatives_only(const variable_list& grads) {
    if (at::GradMode::is_enabled())
        refuse("the operators of isa.kernels.transformer_block have first derivatives only (create_graph is set)");
    no_tangents(grads);
    not_traced();
}

// t's elements as they lie in memory: a view that stands for its negative (the imaginary part of a
// conjugate) is written out, which contiguous() alone does not.
Tensor plain(const Tensor& t) { return t.defined() ? t.resolve_neg() : t; }
Tensor packed(const Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }

// t as [rows, dim] with adjacent elements in a row: a copy only where no view does it.
Tensor rows_of(const Tensor& t_) {
    const Tensor t = plain(t_);
    const int64_t dim = t.size(-1);
    Tensor r = t.dim() == 2 ? t : t.numel() ? t.reshape({-1, dim}) : t.reshape({t.numel() / dim, dim});
    return r.stride(1) == 1 || dim == 1 ? r : r.contiguous();
}

// ---- layer norm ---------------------------------------------------------------------------

void check_norm(const Tensor* x, const Tensor& residual, const Tensor& weight, const Tensor& bias) {
    const char* name = x ? "residual" : "x";
    require(residual, name);
    if (residual.dim() < 1 || residual.size(-1) < 1 || residual.size(-1) > ISA_BLOCK_NORM_MAX_DIM)
        refuse(name, "'s last dimension must be 1 to ", ISA_BLOCK_NORM_MAX_DIM, ", got shape ", residual.sizes());
    const auto dtype = residual.scalar_type();
    if (x) {
        require(*x, "x", residual);
        if (x->sizes() != residual.sizes())
            refuse("x and residual must have one shape, got ", x->sizes(), " and ", residual.sizes());
        if (x->scalar_type() != dtype && dtype != at::kFloat)
            refuse("x must be ", type_name(residual), " as residual is (or residual torch.float32), got ", type_name(*x));
    }
    require(weight, "weight", residual);
    if (weight.scalar_type() != dtype && weight.scalar_type() != at::kFloat)
        refuse("weight must be ", type_name(residual), " or torch.float32, got ", type_name(weight));
    if (weight.dim() != 1 || weight.size(0) != residual.size(-1))
        refuse("weight must be [", residual.size(-1), "], got ", weight.sizes());
    if (bias.defined()) {
        require(bias, "bias", residual);
        if (bias.scalar_type() != weight.scalar_type() || bias.sizes() != weight.sizes())
            refuse("bias must have weight's type and shape");
    }
}

isa_block_norm norm_of(const Tensor& rows, int x_type, const Tensor& weight, const Tensor& bias, double eps) {
    isa_block_norm n{};
    n.type = type_of(rows);
    n.x_type = x_type;
    n.weight_type = type_of(weight);
    n.rows = rows.size(0);
    n.dim = rows.size(1);
    n.eps = static_cast<float>(eps);
    n.weight = weight.data_ptr();
    n.bias = pointer(bias);
    return n;
}

// y, h (undefined without x) and, if asked for, stats [2, rows]: mean, rstd.
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor* x, const Tensor& residual, const Tensor& weight,
                                                const Tensor& bias, double eps, bool with_stats) {
    const Tensor r = rows_of(residual), xs = x ? rows_of(*x) : Tensor();
    const Tensor w = packed(weight), b = packed(bias);
    const c10::DeviceGuard guard(r.device());
    const isa_block_norm n = norm_of(r, x ? type_of(*x) : type_of(r), w, b, eps);
    Tensor y = at::empty(residual.sizes(), residual.options()), h, stats;
    if (x) h = at::empty(residual.sizes(), residual.options());
    if (with_stats) stats = at::empty({2, n.rows}, residual.options().dtype(at::kFloat));
    float* mean = static_cast<float*>(pointer(stats));
    check(isa_block_norm_forward(&n, pointer(xs), x ? xs.stride(0) : 0, r.data_ptr(), r.stride(0), y.data_ptr(),
                                 pointer(h), mean, mean ? mean + n.rows : nullptr, stream_of(r)),
          "isa_block_norm_forward");
    return {y, h, stats};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    // without x: y of residual; else y and h
    static variable_list forward(AutogradContext* ctx, const Tensor& residual, const Tensor& weight, const Maybe& bias,
                                 const Maybe& x, double eps) {
        ctx->set_materialize_grads(false);
        auto [y, h, stats] = norm_forward(x ? &*x : nullptr, residual, weight, bias.value_or(Tensor()), eps, true);
        ctx->saved_data["x_type"] = static_cast<int64_t>((x ? *x : residual).scalar_type());
        ctx->saved_data["has_bias"] = bias.has_value();
        ctx->saved_data["has_x"] = x.has_value();
        ctx->save_for_backward({x ? h : residual, weight, stats});
        return x ? variable_list{y, h} : variable_list{y};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &stats = saved[2];
        const auto x_type = static_cast<at::ScalarType>(ctx->saved_data["x_type"].toInt());
        const Tensor rows = rows_of(h), weight = packed(saved[1]);
        const c10::DeviceGuard guard(h.device());
        const Tensor dy = grads[0].defined() ? packed(grads[0]) : at::zeros(h.sizes(), h.options());
        const Tensor dh = grads.size() > 1 ? packed(grads[1]) : Tensor();
        const bool separate = x_type != h.scalar_type();
        Tensor dr = at::empty(h.sizes(), h.options()), dx, dw, db, workspace;
        if (separate) dx = at::empty(h.sizes(), h.options().dtype(x_type));
        // counted over the tensors that were there
        const bool has_bias = ctx->saved_data["has_bias"].toBool(), has_x = ctx->saved_data["has_x"].toBool();
        const bool need_r = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        const bool need_b = has_bias && ctx->needs_input_grad(2), need_x = has_x && ctx->needs_input_grad(2 + has_bias);
        if (need_w || need_b) {
            dw = at::empty({rows.size(1)}, weight.options());
            if (need_b) db = at::empty({rows.size(1)}, weight.options());
            workspace = bytes(isa_block_norm_backward_workspace(rows.size(0), rows.size(1)), h);
        }
        const isa_block_norm n = norm_of(rows, separate ? type_of(dx) : type_of(h), weight, Tensor(), 0.0);
        const float* mean = static_cast<const float*>(stats.data_ptr());
        check(isa_block_norm_backward(&n, dy.data_ptr(), pointer(dh), rows.data_ptr(), rows.stride(0), mean,
                                      mean + n.rows, pointer(dx), dr.data_ptr(), pointer(dw), pointer(db),
                                      pointer(workspace), workspace.defined() ? workspace.numel() : 0, stream_of(h)),
              "isa_block_norm_backward");
        return {need_r ? dr : Tensor(), need_w ? dw : Tensor(), need_b ? db : Tensor(),
                need_x ? (separate ? dx : dr) : Tensor(), Tensor()};
    }
};

Tensor layer_norm(const Tensor& x, const Tensor& weight, const Maybe& bias, double eps) {
    not_traced();
    const Tensor b = bias.value_or(Tensor());
    check_norm(nullptr, x, weight, b);
    no_tangents(std::array{std::cref(x), std::cref(weight), std::cref(b)});
    if (tracked({&x, &weight, &b})) return LayerNorm::apply(x, weight, bias, Maybe(), eps)[0];
    return std::get<0>(norm_forward(nullptr, x, weight, b, eps, false));
}

std::tuple<Tensor, Tensor> add_layer_norm(const Tensor& x, const Tensor& residual, const Tensor& weight,
                                          const Maybe& bias, double eps) {
    not_traced();
    const Tensor b = bias.value_or(Tensor());
    check_norm(&x, residual, weight, b);
    no_tangents(std::array{std::cref(x), std::cref(residual), std::cref(weight), std::cref(b)});
    if (tracked({&x, &residual, &weight, &b})) {
        const auto r = LayerNorm::apply(residual, weight, bias, Maybe(x), eps);
        return {r[0], r[1]};
    }
    auto [y, h, stats] = norm_forward(&x, residual, weight, b, eps, false);
    return {y, h};
}

// ---- attention ------------------------------------------------------------------------------

constexpr int64_t kLongest = int64_t{1} << 30, kFar = int64_t{1} << 24;  // tokens, bytes between tokens

// Strides of batch, token and head; a dimension of one element has none that matters.
void strides_of(const Tensor& t, int64_t (&s)[3]) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// t, or a copy where its heads' elements are apart, 16-byte loads would not be aligned or tokens
// overlap (as broadcast ones do) or lie too far apart.
Tensor attention_operand(const Tensor& t_) {
    const Tensor t = plain(t_);
    if (t.numel() == 0) return at::empty(t.sizes(), t.options());  // whatever its strides
    int64_t s[3];
    strides_of(t, s);
    const bool tokens = t.size(1) < 2 || (s[1] >= t.size(3) && s[1] * t.element_size() < kFar);
    if (t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (s[0] | s[1] | s[2]) % 8 == 0 && tokens)
        return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

struct How {
    int64_t window, sinks;  // window 0: none
    double scale;
};

isa_block_attention attention_of(const Tensor& q, const Tensor& k, const Tensor& v, const How& how,
                                 const Tensor& lengths) {
    isa_block_attention a{};
    a.type = type_of(q);
    a.batch = q.size(0);
    a.queries = q.size(1);
    a.heads = q.size(2);
    a.head_dim = q.size(3);
    a.keys = k.size(1);
    a.kv_heads = k.size(2);
    a.window = std::min(how.window, kLongest);  // past the longest sequence: no window
    a.sinks = std::min(how.sinks, kLongest);
    a.scale = static_cast<float>(how.scale);
    a.key_lengths = static_cast<const int32_t*>(pointer(lengths));
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    strides_of(q, a.q_strides);
    strides_of(k, a.k_strides);
    strides_of(v, a.v_strides);
    return a;
}

// out and, for a backward call, rest (16-bit types: what out's rounding left) and lse.
std::tuple<Tensor, Tensor, Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const How& how,
                                                     const Tensor& lengths, bool for_backward) {
    const c10::DeviceGuard guard(q.device());
    const isa_block_attention a = attention_of(q, k, v, how, lengths);
    Tensor out = at::empty(q.sizes(), q.options()), rest, lse;
    if (for_backward) {
        lse = at::empty({a.batch, a.heads, a.queries, 2}, q.options().dtype(at::kFloat));
        if (a.type != ISA_BLOCK_F32) rest = at::empty(q.sizes(), q.options());
    }
    const Tensor workspace = bytes(isa_block_attention_forward_workspace(&a), q);
    check(isa_block_attention_forward(&a, out.data_ptr(), pointer(rest), static_cast<float*>(pointer(lse)),
                                      pointer(workspace), workspace.defined() ? workspace.numel() : 0, stream_of(q)),
          "isa_block_attention_forward");
    return {out, rest, lse};
}

struct WindowAttention : torch::autograd::Function<WindowAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t window,
                          int64_t sinks, double scale, const Maybe& key_lengths) {
        const Tensor lengths = key_lengths.value_or(Tensor()), q = attention_operand(q_), k = attention_operand(k_), v = attention_operand(v_);
        auto [out, rest, lse] = attention_forward(q, k, v, {window, sinks, scale}, lengths, true);
        ctx->save_for_backward({q, k, v, out, rest, lse, lengths});
        ctx->saved_data["window"] = window;
        ctx->saved_data["sinks"] = sinks;
        ctx->saved_data["scale"] = scale;
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only(grads);
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2];
        const How how{ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt(),
                      ctx->saved_data["scale"].toDouble()};
        const c10::DeviceGuard guard(q.device());
        const isa_block_attention a = attention_of(q, k, v, how, s[6]);
        const Tensor dout = attention_operand(grads[0]);
        int64_t by[3];
        strides_of(dout, by);
        const bool need_q = ctx->needs_input_grad(0), need_k = ctx->needs_input_grad(1),
                   need_v = ctx->needs_input_grad(2);
        Tensor dq, dk, dv;
        if (need_q) dq = at::empty(q.sizes(), q.options());
        if (need_k || need_v) {
            dk = at::empty(k.sizes(), k.options());
            dv = at::empty(v.sizes(), v.options());
        }
        const Tensor workspace = bytes(isa_block_attention_backward_workspace(&a), q);
        check(isa_block_attention_backward(&a, s[3].data_ptr(), pointer(s[4]), static_cast<const float*>(pointer(s[5])),
                                           dout.data_ptr(), by, pointer(dq), pointer(dk), pointer(dv),
                                           pointer(workspace), workspace.defined() ? workspace.numel() : 0, stream_of(q)),
              "isa_block_attention_backward");
        return {dq, need_k ? dk : Tensor(), need_v ? dv : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor window_attention(const Tensor& q, const Tensor& k, const Tensor& v, std::optional<int64_t> window, int64_t sinks,
                        std::optional<double> scale, const Maybe& key_lengths) {
    not_traced();
    require(q, "q");
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{k, "k"}, {v, "v"}}) {
        require(t, name, q);
        if (t.scalar_type() != q.scalar_type())
            refuse(name, " must be ", type_name(q), " as q is, got ", type_name(t));
    }
    if (q.dim() != 4 || k.dim() != 4 || k.sizes() != v.sizes())
        refuse("q must be [batch, queries, heads, head_dim], k and v [batch, keys, kv_heads, head_dim]; got ", q.sizes(),
               ", ", k.sizes(), " and ", v.sizes());
    if (q.size(0) != k.size(0) || q.size(3) != k.size(3))
        refuse("batch and head_dim of q ", q.sizes(), " and k ", k.sizes(), " differ");
    if (k.size(2) < 1 || q.size(2) < 1 || q.size(2) % k.size(2))
        refuse("heads (", q.size(2), ") must be a multiple of kv_heads (", k.size(2), ")");
    if (q.size(3) % 8 || q.size(3) < 8 || q.size(3) > ISA_BLOCK_ATTENTION_MAX_DIM)
        refuse("head_dim must be a multiple of 8 up to ", ISA_BLOCK_ATTENTION_MAX_DIM, ", got ", q.size(3));
    if (window && *window < 1) refuse("window must be None or at least 1, got ", *window);
    if (sinks < 0) refuse("sinks must not be negative, got ", sinks);
    const double by = scale.value_or(1.0 / std::sqrt(static_cast<double>(q.size(3))));
    if (!(by > 0.0) || std::isinf(by)) refuse("scale must be positive and finite, got ", by);
    Tensor lengths;
    if (key_lengths) {
        lengths = *key_lengths;
        const auto type = lengths.scalar_type();
        if ((type != at::kInt && type != at::kLong) || lengths.dim() != 1 || lengths.size(0) != q.size(0))
            refuse("key_lengths must be int32 or int64 [", q.size(0), "], got ", type_name(lengths), " ", lengths.sizes());
        if (lengths.device() != q.device()) refuse("key_lengths must be on ", q.device(), ", got ", lengths.device());
        if (type == at::kLong) lengths = lengths.clamp(0, kLongest).to(at::kInt);
        lengths = packed(lengths);
    }
    no_tangents(std::array{std::cref(q), std::cref(k), std::cref(v)});
    if (tracked({&q, &k, &v}))
        return WindowAttention::apply(q, k, v, window.value_or(0), sinks, by, lengths.defined() ? Maybe(lengths) : Maybe());
    return std::get<0>(attention_forward(attention_operand(q), attention_operand(k), attention_operand(v),
                                         {window.value_or(0), sinks, by}, lengths, false));
}

// ---- cross-entropy ------------------------------------------------------------------------

void check_loss(const Tensor& logits, const Tensor& targets) {
    require(logits, "logits");
    if (logits.dim() < 1 || logits.size(-1) < 1) refuse("logits must be [..., vocab], got ", logits.sizes());
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    if (targets.scalar_type() != at::kLong || targets.sizes() != lead)
        refuse("targets must be int64 ", lead, ", got ", type_name(targets), " ", targets.sizes());
    if (targets.device() != logits.device()) refuse("targets must be on ", logits.device(), ", got ", targets.device());
}

int reduction_of(const std::string& name) {
    if (name == "mean") return ISA_BLOCK_MEAN;
    if (name == "sum") return ISA_BLOCK_SUM;
    if (name == "none") return ISA_BLOCK_NONE;
    refuse("reduction must be mean, none or sum, got ", name);
}

isa_block_loss loss_of(const Tensor& rows, const Tensor& targets, int64_t ignore) {
    isa_block_loss l{};
    l.type = type_of(rows);
    l.rows = rows.size(0);
    l.vocab = rows.size(1);
    l.ignore_index = ignore;
    l.logits = rows.data_ptr();
    l.logits_stride = rows.stride(0);
    l.targets = static_cast<const int64_t*>(targets.data_ptr());
    return l;
}

// A new tensor as t [rows, vocab]. Where that adds an eighth at most, rows of both are aligned alike: as far
// apart (a padded vocabulary, whose rows then stay on whole cache lines), or by the same remainder of 16 bytes.
Tensor like_rows(const Tensor& t) {
    const int64_t vocab = t.size(1), apart = t.stride(0);
    if (t.size(0) < 2 || apart <= vocab) return at::empty(t.sizes(), t.options());
    const int64_t extra = apart - vocab, odd = extra % (16 / t.element_size()), most = vocab / 8;
    return at::empty_strided(t.sizes(), {vocab + (extra <= most ? extra : odd <= most ? odd : 0), 1}, t.options());
}

Tensor shaped(const Tensor& rows, at::IntArrayRef sizes) { return rows.sizes() == sizes ? rows : rows.reshape(sizes); }

std::tuple<Tensor, Tensor, Tensor> loss_forward(const Tensor& rows, const Tensor& targets, int64_t ignore, int reduction,
                                                bool with_stats) {
    const c10::DeviceGuard guard(rows.device());
    const isa_block_loss l = loss_of(rows, targets, ignore);
    const auto f32 = rows.options().dtype(at::kFloat);
    Tensor out = reduction == ISA_BLOCK_NONE ? at::empty({l.rows}, f32) : at::empty({}, f32), stats, count;
    if (with_stats) {
        stats = at::empty({l.rows, 2}, f32);
        count = at::empty({1}, f32);
    }
    const Tensor workspace = bytes(isa_block_loss_workspace(&l), rows);
    check(isa_block_loss_forward(&l, reduction, static_cast<float*>(out.data_ptr()), static_cast<float*>(pointer(stats)),
                                 static_cast<float*>(pointer(count)), pointer(workspace), workspace.numel(),
                                 stream_of(rows)),
          "isa_block_loss_forward");
    return {out, stats, count};
}

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t ignore,
                          int64_t reduction) {
        const Tensor rows = rows_of(logits), t = packed(targets.reshape({-1}));
        auto [out, stats, count] = loss_forward(rows, t, ignore, static_cast<int>(reduction), true);
        ctx->save_for_backward({rows, t, stats, count});
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["reduction"] = reduction;
        ctx->saved_data["shape"] = logits.sizes().vec();
        return reduction == ISA_BLOCK_NONE ? shaped(out, targets.sizes()) : out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only(grads);
        const auto s = ctx->get_saved_variables();
        const Tensor& rows = s[0];
        const c10::DeviceGuard guard(rows.device());
        const isa_block_loss l = loss_of(rows, s[1], ctx->saved_data["ignore"].toInt());
        const Tensor grad = like_rows(rows), up = packed(grads[0].to(at::kFloat));
        check(isa_block_loss_backward(&l, static_cast<int>(ctx->saved_data["reduction"].toInt()),
                                      static_cast<const float*>(s[2].data_ptr()),
                                      static_cast<const float*>(s[3].data_ptr()),
                                      static_cast<const float*>(up.data_ptr()), grad.data_ptr(), grad.stride(0),
                                      stream_of(rows)),
              "isa_block_loss_backward");
        return {shaped(grad, ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor(), Tensor()};
    }
};

Tensor cross_entropy(const Tensor& logits, const Tensor& targets, int64_t ignore, const std::string& reduction_name) {
    not_traced();
    const int reduction = reduction_of(reduction_name);
    check_loss(logits, targets);
    no_tangents(std::array{std::cref(logits)});
    if (tracked({&logits})) return CrossEntropy::apply(logits, targets, ignore, static_cast<int64_t>(reduction));
    const Tensor out =
        std::get<0>(loss_forward(rows_of(logits), packed(targets.reshape({-1})), ignore, reduction, false));
    return reduction == ISA_BLOCK_NONE ? shaped(out, targets.sizes()) : out;
}

std::tuple<Tensor, Tensor> cross_entropy_with_grad(const Tensor& logits, const Tensor& targets, int64_t ignore,
                                                   double grad_scale) {
    not_traced();
    check_loss(logits, targets);
    no_tangents(std::array{std::cref(logits)});
    const at::NoGradGuard untracked;
    const Tensor rows = rows_of(logits.detach()), t = packed(targets.reshape({-1}));
    const c10::DeviceGuard guard(rows.device());
    const isa_block_loss l = loss_of(rows, t, ignore);
    const Tensor out = at::empty({}, rows.options().dtype(at::kFloat)), grad = like_rows(rows);
    const Tensor workspace = bytes(isa_block_loss_workspace(&l), rows);
    check(isa_block_loss_with_grad(&l, static_cast<float>(grad_scale), static_cast<float*>(out.data_ptr()),
                                   grad.data_ptr(), grad.stride(0), pointer(workspace), workspace.numel(),
                                   stream_of(rows)),
          "isa_block_loss_with_grad");
    return {out, shaped(grad, logits.sizes())};
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
    // the interpreter's lock is not needed past the arguments
    using Free = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("abi_version", &isa_block_abi_version);
    m.attr("ABI_VERSION") = ISA_BLOCK_ABI_VERSION;
    m.def("layer_norm", &layer_norm, Free());
    m.def("add_layer_norm", &add_layer_norm, Free());
    m.def("window_attention", &window_attention, Free());
    m.def("cross_entropy", &cross_entropy, Free());
    m.def("cross_entropy_with_grad", &cross_entropy_with_grad, Free());
}
