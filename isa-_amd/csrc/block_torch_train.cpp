// torch's side of include/isa_train.h: embeddings, dropout and the losses of tuning, with their gradients.
#include "block_torch.hpp"

#include <c10/hip/HIPGraphsC10Utils.h>

namespace {

// Autograd keeps a leaf's accumulator, with the stream it was made on, as long as a graph of that leaf lives. One of
// the default stream would take part in a capture, which the runtime answers with an error in autograd's threads,
// where it ends the process.
bool captured() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

void leaf_can_be_captured(const Tensor& t) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = node ? node->stream() : std::nullopt;
    if (stream && stream->id() == c10::hip::getDefaultHIPStream(t.device().index()).id())
        refuse("a graph of a leaf lives that was made on the default stream: free it (the results that hold it), or "
               "make it on another stream, before a step with that leaf is captured");
}

bool recorded(std::initializer_list<const Tensor*> tensors) {
    if (!tracked(tensors)) return false;
    if (captured())
        for (const Tensor* t : tensors) leaf_can_be_captured(*t);
    return true;
}

// For a model that calls the operators unchecked: called in its backward pass, before that reaches a leaf.
void leaves_can_be_captured(const std::vector<Tensor>& leaves) {
    if (captured())
        for (const Tensor& t : leaves) leaf_can_be_captured(t);
}

// Integer indices as contiguous int64.
Tensor indices(const Tensor& t, const char* name, const Tensor& like) {
    if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
        refuse(name, " must be int64 or int32, got ", type_name(t));
    if (t.device() != like.device()) refuse(name, " must be on ", like.device(), ", got ", t.device());
    return packed(t.scalar_type() == at::kLong ? t : t.to(at::kLong));
}

// ---- embedding ------------------------------------------------------------------------------

void check_table(const Tensor& t, const char* name, int64_t least_rows) {
    if (t.dim() != 2 || t.size(1) < 1 || t.size(1) > ISA_TRAIN_EMBEDDING_MAX_DIM || t.size(0) < least_rows ||
        t.size(0) > ISA_TRAIN_EMBEDDING_MAX_ROWS)
        refuse(name, " must be [rows, dim] of ", least_rows, " to ", ISA_TRAIN_EMBEDDING_MAX_ROWS, " rows and 1 to ",
               ISA_TRAIN_EMBEDDING_MAX_DIM, " columns, got ", t.sizes());
}

// ids and place_ids: contiguous int64; without place_ids a second table's rows are taken in turn along ids' last dimension.
struct Lookup {
    Tensor ids, place_ids;
    double scale;
    int64_t padding;  // -1: none
};

int64_t period_of(const Tensor& ids) { return ids.dim() ? std::max<int64_t>(ids.size(-1), 1) : 1; }

isa_train_embedding embedding_of(const Lookup& how, int type, int64_t dim, int64_t vocab, int64_t places) {
    isa_train_embedding e{};
    e.type = type;
    e.tokens = how.ids.numel();
    e.dim = dim;
    e.vocab = vocab;
    e.ids = static_cast<const int64_t*>(how.ids.data_ptr());
    e.scale = static_cast<float>(how.scale);
    e.places = places;
    e.place_ids = static_cast<const int64_t*>(pointer(how.place_ids));
    e.period = period_of(how.ids);
    return e;
}

// y and, for a backward call, the lists of the tables that learn.
std::tuple<Tensor, Tensor> lookup(const Tensor& weight, const Tensor& places, const Lookup& how, bool learns,
                                  bool places_learn) {
    const c10::DeviceGuard guard(weight.device());
    const Tensor w = rows_of(weight), p = places.defined() ? rows_of(places) : Tensor();
    isa_train_embedding e = embedding_of(how, type_of(w), w.size(1), w.size(0), p.defined() ? p.size(0) : 0);
    e.weight = w.data_ptr();
    e.weight_stride = w.stride(0);
    if (p.defined()) {
        e.place_weight = p.data_ptr();
        e.places_stride = p.stride(0);
    }
    std::vector<int64_t> shape = how.ids.sizes().vec();
    shape.push_back(e.dim);
    Tensor y = at::empty(shape, weight.options());
    const Tensor lists = bytes(isa_train_embedding_lists(&e, learns, places_learn), w);
    check(isa_train_embedding_forward(&e, y.data_ptr(), learns, places_learn, how.padding, pointer(lists),
                                      lists.defined() ? lists.numel() : 0, stream_of(w)),
          "isa_train_embedding_forward");
    return {y, lists};
}

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, const Maybe& places,
                          const Maybe& place_ids, double scale, int64_t padding) {
        const Lookup how{ids, place_ids.value_or(Tensor()), scale, padding};
        const bool learns = weight.requires_grad(), places_learn = places && places->requires_grad();
        auto [y, lists] = lookup(weight, places.value_or(Tensor()), how, learns, places_learn);
        ctx->save_for_backward({ids, how.place_ids, lists});
        ctx->saved_data["learns"] = learns;
        ctx->saved_data["places_learn"] = places_learn;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        ctx->saved_data["rows"] = weight.size(0);
        ctx->saved_data["places"] = places ? places->size(0) : int64_t{-1};
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only(grads);
        const auto s = ctx->get_saved_variables();
        const Tensor dy = packed(grads[0]);
        const c10::DeviceGuard guard(dy.device());
        const int64_t places = ctx->saved_data["places"].toInt();
        const Lookup how{s[0], s[1], ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt()};
        const isa_train_embedding e =
            embedding_of(how, type_of(dy), dy.size(-1), ctx->saved_data["rows"].toInt(), std::max<int64_t>(places, 0));
        Tensor dw, dp;
        if (ctx->needs_input_grad(0)) dw = at::empty({e.vocab, e.dim}, dy.options());
        // counted over the tensors that were there
        if (places >= 0 && ctx->needs_input_grad(2)) dp = at::empty({places, e.dim}, dy.options());
        const Tensor workspace = bytes(isa_train_embedding_backward_workspace(&e, dw.defined(), dp.defined()), dy);
        check(isa_train_embedding_backward(&e, pointer(s[2]), s[2].defined() ? s[2].numel() : 0, dy.data_ptr(), pointer(dw),
                                           pointer(dp), ctx->saved_data["learns"].toBool(),
                                           ctx->saved_data["places_learn"].toBool(), pointer(workspace),
                                           workspace.defined() ? workspace.numel() : 0, stream_of(dy)),
              "isa_train_embedding_backward");
        return {dw, Tensor(), dp, Tensor(), Tensor(), Tensor()};
    }
};

// unchecked: the caller answers for a backward pass that is captured (leaves_can_be_captured).
Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, const Maybe& positions,
                 const Maybe& position_weight, std::optional<int64_t> padding_index, bool unchecked) {
    not_traced();
    require(weight, "weight");
    check_table(weight, "weight", 0);
    if (!std::isfinite(static_cast<float>(scale))) refuse("scale must be finite in float32, got ", scale);
    if (padding_index && (*padding_index < 0 || *padding_index >= weight.size(0)))
        refuse("padding_index must be None or a row of weight (0 to ", weight.size(0) - 1, "), got ", *padding_index);
    const Tensor places = position_weight.value_or(Tensor());
    Tensor place_ids;
    if (places.defined()) {
        require(places, "position_weight", weight);
        check_table(places, "position_weight", 1);
        if (places.scalar_type() != weight.scalar_type() || places.size(1) != weight.size(1))
            refuse("position_weight must be ", type_name(weight), " [rows, ", weight.size(1), "] as weight is, got ",
                   type_name(places), " ", places.sizes());
        if (!positions && ids.numel() && period_of(ids) > places.size(0))
            refuse(ids.size(-1), " tokens do not fit a table of ", places.size(0), " positions");
    }
    const Tensor tokens = indices(ids, "ids", weight);
    if (positions) {
        if (!places.defined()) refuse("positions need position_weight");
        place_ids = indices(*positions, "positions", weight);
        if (place_ids.sizes() != tokens.sizes()) {
            if (!at::is_expandable_to(place_ids.sizes(), tokens.sizes()))
                refuse("positions ", place_ids.sizes(), " must broadcast to ids ", tokens.sizes());
            place_ids = place_ids.expand(tokens.sizes()).contiguous();
        }
    }
    no_tangents(std::array{std::cref(weight), std::cref(places)});
    const int64_t padding = padding_index.value_or(-1);
    if (unchecked ? tracked({&weight, &places}) : recorded({&weight, &places}))
        return Embedding::apply(weight, tokens, position_weight, place_ids.defined() ? Maybe(place_ids) : Maybe(), scale,
                                padding);
    return std::get<0>(lookup(weight, places, {tokens, place_ids, scale, padding}, false, false));
}

// ---- dropout --------------------------------------------------------------------------------

int threshold_of(double p) {
    if (!(p >= 0.0 && p <= 1.0)) refuse("p must be 0 to 1, got ", p);
    return static_cast<int>(std::nearbyint(p * 65536.0));
}

Tensor seed_of(const Tensor& seed, const Tensor& like) {
    if (seed.scalar_type() != at::kLong || seed.dim() != 1 || seed.size(0) != 2)
        refuse("seed must be int64 [2], got ", type_name(seed), " ", seed.sizes());
    if (seed.device() != like.device()) refuse("seed must be on ", like.device(), ", got ", seed.device());
    return packed(seed);
}

isa_train_dropout dropout_of(const Tensor& seed, int64_t site, int64_t threshold) {
    return {static_cast<const int64_t*>(seed.data_ptr()), site, static_cast<int>(threshold)};
}

Tensor dropped(const Tensor& x, const Tensor& seed, int64_t site, int64_t threshold) {
    Tensor y = at::empty(x.sizes(), x.options());
    if (x.numel() == 0) return y;
    const c10::DeviceGuard guard(x.device());
    const Tensor rows = rows_of(x);
    const isa_train_dropout d = dropout_of(seed, site, threshold);
    check(isa_train_dropout_apply(&d, type_of(rows), rows.size(0), rows.size(1), rows.data_ptr(), rows.stride(0),
                                  y.data_ptr(), stream_of(rows)),
          "isa_train_dropout_apply");
    return y;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& seed, int64_t site, int64_t threshold) {
        ctx->save_for_backward({seed});
        ctx->saved_data["site"] = site;
        ctx->saved_data["threshold"] = threshold;
        return dropped(x, seed, site, threshold);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only(grads);
        const auto s = ctx->get_saved_variables();
        return {dropped(grads[0], s[0], ctx->saved_data["site"].toInt(), ctx->saved_data["threshold"].toInt()), Tensor(),
                Tensor(), Tensor()};
    }
};

Tensor dropout(const Tensor& x, double p, const Tensor& seed_, int64_t site) {
    not_traced();
    require(x, "x");
    if (x.dim() < 1 || x.size(-1) > (int64_t{1} << 30)) refuse("x must be [..., dim], dim up to 2^30, got ", x.sizes());
    const int64_t threshold = threshold_of(p);
    const Tensor seed = seed_of(seed_, x);
    no_tangents(std::array{std::cref(x)});
    if (recorded({&x})) return DropoutFunction::apply(x, seed, site, threshold);
    return dropped(x, seed, site, threshold);
}

// y, h and, if asked for, stats [2, rows]: mean, rstd.
std::tuple<Tensor, Tensor, Tensor> dropout_norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight,
                                                        const Tensor& bias, const Tensor& seed, int64_t site,
                                                        int64_t threshold, double eps, bool with_stats) {
    const Tensor r = rows_of(residual), xs = rows_of(x), w = packed(weight), b = packed(bias);
    const c10::DeviceGuard guard(r.device());
    const isa_block_norm n = norm_of(r, type_of(xs), w, b, eps);
    const isa_train_dropout d = dropout_of(seed, site, threshold);
    Tensor y = at::empty(residual.sizes(), residual.options()), h = at::empty(residual.sizes(), residual.options()), stats;
    if (with_stats) stats = at::empty({2, n.rows}, residual.options().dtype(at::kFloat));
    float* mean = static_cast<float*>(pointer(stats));
    check(isa_train_dropout_norm_forward(&n, &d, xs.data_ptr(), xs.stride(0), r.data_ptr(), r.stride(0), y.data_ptr(),
                                         h.data_ptr(), mean, mean ? mean + n.rows : nullptr, stream_of(r)),
          "isa_train_dropout_norm_forward");
    return {y, h, stats};
}

struct DropoutLayerNorm : torch::autograd::Function<DropoutLayerNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& weight,
                                 const Tensor& seed, const Maybe& bias, int64_t site, int64_t threshold, double eps) {
        ctx->set_materialize_grads(false);
        auto [y, h, stats] = dropout_norm_forward(x, residual, weight, bias.value_or(Tensor()), seed, site, threshold, eps, true);
        ctx->saved_data["x_type"] = static_cast<int64_t>(x.scalar_type());
        ctx->saved_data["has_bias"] = bias.has_value();
        ctx->saved_data["site"] = site;
        ctx->saved_data["threshold"] = threshold;
        ctx->save_for_backward({h, weight, stats, seed});
        return {y, h};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &stats = saved[2];
        const auto x_type = static_cast<at::ScalarType>(ctx->saved_data["x_type"].toInt());
        const Tensor rows = rows_of(h), weight = packed(saved[1]);
        const c10::DeviceGuard guard(h.device());
        const Tensor dy = grads[0].defined() ? packed(grads[0]) : at::zeros(h.sizes(), h.options());
        const Tensor dh = packed(grads[1]);
        Tensor dr = at::empty(h.sizes(), h.options()), dx = at::empty(h.sizes(), h.options().dtype(x_type)), dw, db, workspace;
        // counted over the tensors that were there
        const bool need_b = ctx->saved_data["has_bias"].toBool() && ctx->needs_input_grad(4);
        if (ctx->needs_input_grad(2) || need_b) {
            dw = at::empty({rows.size(1)}, weight.options());
            if (need_b) db = at::empty({rows.size(1)}, weight.options());
            workspace = bytes(isa_block_norm_backward_workspace(rows.size(0), rows.size(1)), h);
        }
        const isa_block_norm n = norm_of(rows, type_of(dx), weight, Tensor(), 0.0);
        const isa_train_dropout d = dropout_of(saved[3], ctx->saved_data["site"].toInt(), ctx->saved_data["threshold"].toInt());
        const float* mean = static_cast<const float*>(stats.data_ptr());
        check(isa_train_dropout_norm_backward(&n, &d, dy.data_ptr(), pointer(dh), rows.data_ptr(), rows.stride(0), mean,
                                              mean + n.rows, dx.data_ptr(), dr.data_ptr(), pointer(dw), pointer(db),
                                              pointer(workspace), workspace.defined() ? workspace.numel() : 0,
                                              stream_of(h)),
              "isa_train_dropout_norm_backward");
        return {ctx->needs_input_grad(0) ? dx : Tensor(), ctx->needs_input_grad(1) ? dr : Tensor(),
                ctx->needs_input_grad(2) ? dw : Tensor(), Tensor(), need_b ? db : Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> dropout_add_layer_norm(const Tensor& x, const Tensor& residual, const Tensor& weight,
                                                  const Maybe& bias, double eps, double p, const Tensor& seed_,
                                                  int64_t site) {
    not_traced();
    const Tensor b = bias.value_or(Tensor());
    check_norm(&x, residual, weight, b);
    const int64_t threshold = threshold_of(p);
    const Tensor seed = seed_of(seed_, residual);
    no_tangents(std::array{std::cref(x), std::cref(residual), std::cref(weight), std::cref(b)});
    if (recorded({&x, &residual, &weight, &b})) {
        const auto r = DropoutLayerNorm::apply(x, residual, weight, seed, bias, site, threshold, eps);
        return {r[0], r[1]};
    }
    auto [y, h, stats] = dropout_norm_forward(x, residual, weight, b, seed, site, threshold, eps, false);
    return {y, h};
}

// ---- losses ---------------------------------------------------------------------------------

// An input that is held fixed: float32 of a shape, contiguous.
Tensor fixed(const Tensor& t, const char* name, at::IntArrayRef shape, const Tensor& like) {
    if (t.scalar_type() != at::kFloat || t.sizes() != shape)
        refuse(name, " must be torch.float32 ", shape, ", got ", type_name(t), " ", t.sizes());
    if (t.device() != like.device()) refuse(name, " must be on ", like.device(), ", got ", t.device());
    if (at::GradMode::is_enabled() && t.requires_grad()) refuse(name, " takes no gradient: detach it");
    return packed(t);
}

struct Policy {
    Tensor old_logp, advantages, ref_logp;
    double low, high, kl;
    int64_t ignore;
};

isa_train_policy policy_of(const Tensor& rows, const Tensor& actions, const Policy& how) {
    isa_train_policy p{};
    p.loss = loss_of(rows, actions, how.ignore);
    p.old_logp = static_cast<const float*>(how.old_logp.data_ptr());
    p.advantages = static_cast<const float*>(how.advantages.data_ptr());
    p.ref_logp = static_cast<const float*>(pointer(how.ref_logp));
    p.low = static_cast<float>(how.low);
    p.high = static_cast<float>(how.high);
    p.kl = static_cast<float>(how.kl);
    return p;
}

Policy checked_policy(const Tensor& logits, const Tensor& actions, const Tensor& old_logp, const Tensor& advantages,
                      const Maybe& ref_logp, double clip_low, double clip_high, double kl, int64_t ignore) {
    check_loss(logits, actions, "actions");
    if (!(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0))
        refuse("clip must be (0 to 1, 0 or more), got (", clip_low, ", ", clip_high, ")");
    if (!(kl >= 0.0) || std::isinf(static_cast<float>(kl))) refuse("kl must be finite and not negative, got ", kl);
    if (kl > 0.0 && !ref_logp) refuse("kl needs ref_logp");
    Policy how{fixed(old_logp, "old_logp", actions.sizes(), logits),
               fixed(advantages, "advantages", actions.sizes(), logits),
               Tensor(), 1.0 - clip_low, 1.0 + clip_high, kl, ignore};
    if (ref_logp) how.ref_logp = fixed(*ref_logp, "ref_logp", actions.sizes(), logits);
    no_tangents(std::array{std::cref(logits), std::cref(old_logp), std::cref(advantages), std::cref(how.ref_logp)});
    return how;
}

// loss, logp, stats, slope, count (the last three undefined unless asked for)
std::array<Tensor, 5> policy_forward(const Tensor& rows, const Tensor& actions, const Policy& how, int reduction,
                                     bool for_backward) {
    const c10::DeviceGuard guard(rows.device());
    const isa_train_policy p = policy_of(rows, actions, how);
    const auto f32 = rows.options().dtype(at::kFloat);
    const int64_t n = p.loss.rows;
    Tensor out = reduction == ISA_BLOCK_NONE ? at::empty({n}, f32) : at::empty({}, f32), logp = at::empty({n}, f32);
    Tensor stats, slope, count;
    if (for_backward) {
        stats = at::empty({n, 2}, f32);
        slope = at::empty({n}, f32);
        count = at::empty({1}, f32);
    }
    const Tensor workspace = bytes(isa_block_loss_workspace(&p.loss), rows);
    check(isa_train_policy_forward(&p, reduction, static_cast<float*>(out.data_ptr()), static_cast<float*>(logp.data_ptr()),
                                   static_cast<float*>(pointer(stats)), static_cast<float*>(pointer(slope)),
                                   static_cast<float*>(pointer(count)), pointer(workspace), workspace.numel(),
                                   stream_of(rows)),
          "isa_train_policy_forward");
    return {out, logp, stats, slope, count};
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& actions, const Policy& how,
                                 int64_t reduction) {
        ctx->set_materialize_grads(false);
        const Tensor rows = rows_of(logits), t = packed(actions.reshape({-1}));
        auto [out, logp, stats, slope, count] = policy_forward(rows, t, how, static_cast<int>(reduction), true);
        ctx->save_for_backward({rows, t, stats, slope, count});
        ctx->saved_data["ignore"] = how.ignore;
        ctx->saved_data["reduction"] = reduction;
        ctx->saved_data["shape"] = logits.sizes().vec();
        logp = shaped(logp, actions.sizes());
        ctx->mark_non_differentiable({logp});
        return {reduction == ISA_BLOCK_NONE ? shaped(out, actions.sizes()) : out, logp};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only(grads);
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const auto s = ctx->get_saved_variables();
        const Tensor& rows = s[0];
        const c10::DeviceGuard guard(rows.device());
        const isa_block_loss l = loss_of(rows, s[1], ctx->saved_data["ignore"].toInt());
        const Tensor grad = like_rows(rows), up = packed(grads[0].to(at::kFloat));
        check(isa_train_policy_backward(&l, static_cast<int>(ctx->saved_data["reduction"].toInt()),
                                        static_cast<const float*>(s[2].data_ptr()),
                                        static_cast<const float*>(s[3].data_ptr()),
                                        static_cast<const float*>(s[4].data_ptr()),
                                        static_cast<const float*>(up.data_ptr()), grad.data_ptr(), grad.stride(0),
                                        stream_of(rows)),
              "isa_train_policy_backward");
        return {shaped(grad, ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& actions, const Tensor& old_logp,
                                       const Tensor& advantages, const Maybe& ref_logp, double clip_low,
                                       double clip_high, double kl, int64_t ignore, const std::string& reduction_name) {
    not_traced();
    const int reduction = reduction_of(reduction_name);
    const Policy how = checked_policy(logits, actions, old_logp, advantages, ref_logp, clip_low, clip_high, kl, ignore);
    if (recorded({&logits})) {
        const auto r = PolicyLoss::apply(logits, actions, how, static_cast<int64_t>(reduction));
        return {r[0], r[1]};
    }
    const auto r = policy_forward(rows_of(logits), packed(actions.reshape({-1})), how, reduction, false);
    return {reduction == ISA_BLOCK_NONE ? shaped(r[0], actions.sizes()) : r[0], shaped(r[1], actions.sizes())};
}

std::tuple<Tensor, Tensor, Tensor> policy_loss_with_grad(const Tensor& logits, const Tensor& actions,
                                                         const Tensor& old_logp, const Tensor& advantages,
                                                         const Maybe& ref_logp, double clip_low, double clip_high,
                                                         double kl, int64_t ignore, double grad_scale) {
    not_traced();
    const at::NoGradGuard untracked;
    const Policy how = checked_policy(logits, actions, old_logp, advantages, ref_logp, clip_low, clip_high, kl, ignore);
    const Tensor rows = rows_of(logits.detach()), t = packed(actions.reshape({-1}));
    const c10::DeviceGuard guard(rows.device());
    const isa_train_policy p = policy_of(rows, t, how);
    const auto f32 = rows.options().dtype(at::kFloat);
    const Tensor out = at::empty({}, f32), logp = at::empty(actions.sizes(), f32), grad = like_rows(rows);
    const Tensor workspace = bytes(isa_block_loss_workspace(&p.loss), rows);
    check(isa_train_policy_with_grad(&p, static_cast<float>(grad_scale), static_cast<float*>(out.data_ptr()),
                                     static_cast<float*>(logp.data_ptr()), grad.data_ptr(), grad.stride(0),
                                     pointer(workspace), workspace.numel(), stream_of(rows)),
          "isa_train_policy_with_grad");
    return {out, shaped(grad, logits.sizes()), logp};
}

struct Preference {
    Tensor ref_logp;
    double beta;
    int64_t ignore;
};

isa_train_preference preference_of(const Tensor& rows, const Tensor& targets, const Preference& how) {
    isa_train_preference p{};
    p.loss = loss_of(rows, targets, how.ignore);
    p.pairs = targets.size(0) / 2;
    p.tokens = targets.size(1);
    p.ref_logp = static_cast<const float*>(pointer(how.ref_logp));
    p.beta = static_cast<float>(how.beta);
    return p;
}

Preference checked_preference(const Tensor& logits, const Tensor& targets, const Tensor& ref_logp, double beta,
                              int64_t ignore) {
    check_loss(logits, targets);
    if (logits.dim() != 3 || logits.size(0) % 2)
        refuse("logits must be [2 pairs, tokens, vocab], chosen sequences first, got ", logits.sizes());
    if (!(beta > 0.0) || std::isinf(static_cast<float>(beta)) || static_cast<float>(beta) == 0.0f)
        refuse("beta must be positive and finite, got ", beta);
    const Preference how{fixed(ref_logp, "ref_logp", logits.sizes().slice(0, 1), logits), beta, ignore};
    no_tangents(std::array{std::cref(logits), std::cref(ref_logp)});
    return how;
}

// loss, logp, stats, slope (the last two undefined unless asked for)
std::array<Tensor, 4> preference_forward(const Tensor& rows, const Tensor& targets, const Preference& how, int reduction,
                                         bool for_backward) {
    const c10::DeviceGuard guard(rows.device());
    const isa_train_preference p = preference_of(rows, targets, how);
    const auto f32 = rows.options().dtype(at::kFloat);
    Tensor out = reduction == ISA_BLOCK_NONE ? at::empty({p.pairs}, f32) : at::empty({}, f32);
    Tensor logp = at::empty({2 * p.pairs}, f32), stats, slope;
    if (for_backward) {
        stats = at::empty({p.loss.rows, 2}, f32);
        slope = at::empty({2 * p.pairs}, f32);
    }
    const Tensor workspace = bytes(isa_train_preference_workspace(&p), rows);
    check(isa_train_preference_forward(&p, reduction, static_cast<float*>(out.data_ptr()),
                                       static_cast<float*>(logp.data_ptr()), static_cast<float*>(pointer(stats)),
                                       static_cast<float*>(pointer(slope)), pointer(workspace),
                                       workspace.defined() ? workspace.numel() : 0, stream_of(rows)),
          "isa_train_preference_forward");
    return {out, logp, stats, slope};
}

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, const Preference& how,
                                 int64_t reduction) {
        ctx->set_materialize_grads(false);
        const Tensor rows = rows_of(logits), t = packed(targets);
        auto [out, logp, stats, slope] = preference_forward(rows, t, how, static_cast<int>(reduction), true);
        ctx->save_for_backward({rows, t, stats, slope, how.ref_logp});
        ctx->saved_data["ignore"] = how.ignore;
        ctx->saved_data["beta"] = how.beta;
        ctx->saved_data["reduction"] = reduction;
        ctx->saved_data["shape"] = logits.sizes().vec();
        ctx->mark_non_differentiable({logp});
        return {out, logp};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        first_derivatives_only(grads);
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const auto s = ctx->get_saved_variables();
        const Tensor& rows = s[0];
        const c10::DeviceGuard guard(rows.device());
        const isa_train_preference p =
            preference_of(rows, s[1], {s[4], ctx->saved_data["beta"].toDouble(), ctx->saved_data["ignore"].toInt()});
        const Tensor grad = like_rows(rows), up = packed(grads[0].to(at::kFloat));
        check(isa_train_preference_backward(&p, static_cast<int>(ctx->saved_data["reduction"].toInt()),
                                            static_cast<const float*>(s[2].data_ptr()),
                                            static_cast<const float*>(s[3].data_ptr()),
                                            static_cast<const float*>(up.data_ptr()), grad.data_ptr(), grad.stride(0),
                                            stream_of(rows)),
              "isa_train_preference_backward");
        return {shaped(grad, ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> preference_loss(const Tensor& logits, const Tensor& targets, const Tensor& ref_logp,
                                           double beta, int64_t ignore, const std::string& reduction_name) {
    not_traced();
    const int reduction = reduction_of(reduction_name);
    const Preference how = checked_preference(logits, targets, ref_logp, beta, ignore);
    if (recorded({&logits})) {
        const auto r = PreferenceLoss::apply(logits, targets, how, static_cast<int64_t>(reduction));
        return {r[0], r[1]};
    }
    const auto r = preference_forward(rows_of(logits), packed(targets), how, reduction, false);
    return {r[0], r[1]};
}

std::tuple<Tensor, Tensor, Tensor> preference_loss_with_grad(const Tensor& logits, const Tensor& targets,
                                                             const Tensor& ref_logp, double beta, int64_t ignore,
                                                             double grad_scale) {
    not_traced();
    const at::NoGradGuard untracked;
    const Preference how = checked_preference(logits, targets, ref_logp, beta, ignore);
    const Tensor rows = rows_of(logits.detach()), t = packed(targets);
    const c10::DeviceGuard guard(rows.device());
    const isa_train_preference p = preference_of(rows, t, how);
    const auto f32 = rows.options().dtype(at::kFloat);
    const Tensor out = at::empty({}, f32), logp = at::empty({2 * p.pairs}, f32), grad = like_rows(rows);
    const Tensor workspace = bytes(isa_train_preference_workspace(&p), rows);
    check(isa_train_preference_with_grad(&p, static_cast<float>(grad_scale), static_cast<float*>(out.data_ptr()),
                                         static_cast<float*>(logp.data_ptr()), grad.data_ptr(), grad.stride(0),
                                         pointer(workspace), workspace.defined() ? workspace.numel() : 0, stream_of(rows)),
          "isa_train_preference_with_grad");
    return {out, shaped(grad, logits.sizes()), logp};
}

}  // namespace

void bind_training(pybind11::module_& m) {
    // the interpreter's lock is not needed past the arguments
    using Free = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("train_abi_version", &isa_train_abi_version);
    m.attr("TRAIN_ABI_VERSION") = ISA_TRAIN_ABI_VERSION;
    m.def("embedding", &embedding, Free());
    m.def("leaves_can_be_captured", &leaves_can_be_captured, Free());
    m.def("dropout", &dropout, Free());
    m.def("dropout_add_layer_norm", &dropout_add_layer_norm, Free());
    m.def("policy_loss", &policy_loss, Free());
    m.def("policy_loss_with_grad", &policy_loss_with_grad, Free());
    m.def("preference_loss", &preference_loss, Free());
    m.def("preference_loss_with_grad", &preference_loss_with_grad, Free());
}
