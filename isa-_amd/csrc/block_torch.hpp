// What the parts of torch's binding to libisa_block_hip.so share: checks of tensors, views, allocations.
#pragma once

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
#include "isa_train.h"

// One of each in every part that includes this: some use only a few.
#pragma GCC diagnostic ignored "-Wunused-function"
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

// ---- norms and losses ---------------------------------------------------------------------

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

void check_loss(const Tensor& logits, const Tensor& targets, const char* name = "targets") {
    require(logits, "logits");
    if (logits.dim() < 1 || logits.size(-1) < 1) refuse("logits must be [..., vocab], got ", logits.sizes());
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    if (targets.scalar_type() != at::kLong || targets.sizes() != lead)
        refuse(name, " must be int64 ", lead, ", got ", type_name(targets), " ", targets.sizes());
    if (targets.device() != logits.device()) refuse(name, " must be on ", logits.device(), ", got ", targets.device());
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

}  // namespace

// The operators of block_torch_train.cpp.
void bind_training(pybind11::module_& m);
