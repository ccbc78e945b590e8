// Cross-entropy and its gradient: the C entries.
#include "block_loss.hpp"

using namespace isa_block;

// One count, then a loss for each row.
extern "C" size_t isa_block_loss_workspace(const isa_block_loss* l) {
    if (!l || l->rows < 0 || l->rows > kMaxRows) return 0;
    return (static_cast<size_t>(l->rows) + 64) * sizeof(float);
}

extern "C" int isa_block_loss_forward(const isa_block_loss* l, int reduction, float* out, float* stats, float* count,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(l)) return rc;
    if (reduction < ISA_BLOCK_MEAN || reduction > ISA_BLOCK_NONE) return fail("unknown reduction %d", reduction);
    if (reduction == ISA_BLOCK_NONE && l->rows == 0) return 0;
    if (!out) return fail("out is null");
    if (int rc = check_workspace(l, workspace, workspace_bytes)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(workspace);
    if (!count) count = ws;
    if (reduction == ISA_BLOCK_MEAN) {
        loss_count_kernel<<<1, kMostThreads, 0, s>>>(l->targets, l->rows, l->ignore_index, count);
        if (int rc = launched("loss_count_kernel")) return rc;
    }
    LossArgs a = args_of(l);
    a.row_loss = reduction == ISA_BLOCK_NONE ? out : ws + 64;
    a.stats = stats;
    if (l->rows) run_rows<Of::kCrossEntropy>(l->type, a, s);
    if (int rc = launched("loss_kernel")) return rc;
    if (reduction == ISA_BLOCK_NONE) return 0;
    loss_sum_kernel<<<1, kMostThreads, 0, s>>>(ws + 64, l->rows, reduction == ISA_BLOCK_MEAN ? count : nullptr, out);
    return launched("loss_sum_kernel");
}

extern "C" int isa_block_loss_backward(const isa_block_loss* l, int reduction, const float* stats, const float* count,
                                       const float* grad_out, void* grad, int64_t grad_stride, void* stream) {
    if (int rc = check(l)) return rc;
    if (reduction < ISA_BLOCK_MEAN || reduction > ISA_BLOCK_NONE) return fail("unknown reduction %d", reduction);
    if (l->rows == 0) return 0;
    if (!stats || !grad_out || !grad || (reduction == ISA_BLOCK_MEAN && !count))
        return fail("stats, grad_out, grad_logits and a mean's count must be set");
    if (!aligned(grad, type_bytes(l->type))) return fail("grad_logits is not aligned to its type");
    LossArgs a = args_of(l);
    a.stats = const_cast<float*>(stats);
    a.count = reduction == ISA_BLOCK_MEAN ? count : nullptr;
    a.scale_by = grad_out;
    a.scale_step = reduction == ISA_BLOCK_NONE;
    a.grad = grad;
    a.grad_stride = grad_stride;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    run_backward<false>(l->type, a, s);
    return launched("loss_backward_kernel");
}

extern "C" int isa_block_loss_with_grad(const isa_block_loss* l, float grad_scale, float* out, void* grad,
                                        int64_t grad_stride, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(l)) return rc;
    if (!out || (l->rows && !grad)) return fail("out and grad_logits must be set");
    if (l->rows && !aligned(grad, type_bytes(l->type))) return fail("grad_logits is not aligned to its type");
    if (int rc = check_workspace(l, workspace, workspace_bytes)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(workspace);
    loss_count_kernel<<<1, kMostThreads, 0, s>>>(l->targets, l->rows, l->ignore_index, ws);
    if (int rc = launched("loss_count_kernel")) return rc;
    LossArgs a = args_of(l);
    a.row_loss = ws + 64;
    a.count = ws;
    a.scale = grad_scale;
    a.grad = grad;
    a.grad_stride = grad_stride;
    if (l->rows) run_rows<Of::kCrossEntropy>(l->type, a, s);
    if (int rc = launched("loss_kernel")) return rc;
    loss_sum_kernel<<<1, kMostThreads, 0, s>>>(ws + 64, l->rows, ws, out);
    return launched("loss_sum_kernel");
}
