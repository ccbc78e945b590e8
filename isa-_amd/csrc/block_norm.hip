// Layer norm with the residual add: the C entries.
#include "block_norm.hpp"

using namespace isa_block;

extern "C" int isa_block_norm_forward(const isa_block_norm* n, const void* x, int64_t x_stride, const void* residual,
                                      int64_t residual_stride, void* y, void* h, float* mean, float* rstd,
                                      void* stream) {
    return run_forward<Plain>(n, Dropout{}, x, x_stride, residual, residual_stride, y, h, mean, rstd, stream);
}

extern "C" size_t isa_block_norm_backward_workspace(int64_t rows, int64_t dim) {
    if (rows < 0 || dim < 1 || dim > ISA_BLOCK_NORM_MAX_DIM) return 0;
    return static_cast<size_t>(backward_blocks(rows, dim)) * 2 * dim * sizeof(float);
}

extern "C" int isa_block_norm_backward(const isa_block_norm* n, const void* dy, const void* dh, const void* h,
                                       int64_t h_stride, const float* mean, const float* rstd, void* dx,
                                       void* dresidual, void* dweight, void* dbias, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    // (the other checks of n follow, before anything runs)
    if (n && n->rows > 0 && dy && h && mean && rstd && dresidual && (dx != nullptr) != (n->x_type != n->type))
        return fail("grad_x is written where x's type is not the residual's, and only there");
    return run_backward<Plain>(n, Dropout{}, dy, dh, h, h_stride, mean, rstd, dx, dresidual, dweight, dbias, workspace,
                               workspace_bytes, stream);
}
