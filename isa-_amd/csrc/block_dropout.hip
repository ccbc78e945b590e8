// Dropout from a counter-based generator, alone and in the norm's residual add, for gfx950.
//
//   y = keep ? x 65536 / (65536 - t) : 0,  keep iff the element's 16-bit number >= t
//
// No mask is stored: the backward makes the numbers again from the counter. Bound by HBM, one read and one write
// of each element; a thread takes eight adjacent elements, the numbers of one call of the generator.
#include "block_norm.hpp"

namespace isa_block {
namespace {

constexpr int kMaxDropoutBlocks = 4096;

struct DropoutArgs {
    Dropout drop;
    const void* x;
    void* y;
    int64_t x_stride, groups;  // of eight elements, in all rows
    int dim, per_row;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs a) {
    const DropoutKey key(a.drop);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < a.groups; i += step) {
        const int64_t r = i / a.per_row;
        const int at = static_cast<int>(i - r * a.per_row) * 8, left = a.dim - at;
        Pack<T, 8> p;
        load_loose(p, static_cast<const T*>(a.x) + r * a.x_stride + at, left);
        const DropoutNumbers n(key, static_cast<uint64_t>(i));
#pragma unroll
        for (int e = 0; e < 8; ++e) p.v[e] = static_cast<T>(dropped(static_cast<float>(p.v[e]), n.number(e), a.drop));
        store_loose(static_cast<T*>(a.y) + r * a.dim + at, p, left);
    }
}

template <typename T>
void launch_dropout(const DropoutArgs& a, hipStream_t s) {
    const int64_t blocks = std::min<int64_t>(ceil_div(a.groups, kThreads), kMaxDropoutBlocks);
    dropout_kernel<T><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s>>>(a);
}

}  // namespace
}  // namespace isa_block

using namespace isa_block;

extern "C" int isa_train_dropout_apply(const isa_train_dropout* drop, int type, int64_t rows, int64_t dim,
                                       const void* x, int64_t x_stride, void* y, void* stream) {
    if (int rc = check(drop)) return rc;
    if (!known_type(type)) return fail("unknown element type %d", type);
    if (rows < 0 || dim < 0 || dim > (int64_t{1} << 30) || rows > (int64_t{1} << 60) / std::max<int64_t>(dim, 1))
        return fail("rows must not be negative and dim be 0 to 2^30, got %lld and %lld", static_cast<long long>(rows),
                    static_cast<long long>(dim));
    if (rows == 0 || dim == 0) return 0;
    if (!x || !y) return fail("x and y must be set");
    if (!aligned(x, type_bytes(type)) || !aligned(y, type_bytes(type))) return fail("x or y is not aligned to its type");
    DropoutArgs a{};
    a.drop = dropout_of(*drop);
    a.x = x;
    a.y = y;
    a.x_stride = x_stride;
    a.dim = static_cast<int>(dim);
    a.per_row = static_cast<int>(ceil_div(dim, 8));
    a.groups = rows * a.per_row;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == ISA_BLOCK_F32) launch_dropout<float>(a, s);
    else if (type == ISA_BLOCK_BF16) launch_dropout<bf16>(a, s);
    else launch_dropout<f16>(a, s);
    return launched("dropout_kernel");
}

extern "C" int isa_train_dropout_norm_forward(const isa_block_norm* n, const isa_train_dropout* drop, const void* x,
                                              int64_t x_stride, const void* residual, int64_t residual_stride, void* y,
                                              void* h, float* mean, float* rstd, void* stream) {
    if (int rc = check(drop)) return rc;
    if (n && n->rows > 0 && !x) return fail("x must be set");
    return run_forward<Dropped>(n, dropout_of(*drop), x, x_stride, residual, residual_stride, y, h, mean, rstd, stream);
}

extern "C" int isa_train_dropout_norm_backward(const isa_block_norm* n, const isa_train_dropout* drop, const void* dy,
                                               const void* dh, const void* h, int64_t h_stride, const float* mean,
                                               const float* rstd, void* dx, void* dresidual, void* dweight,
                                               void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(drop)) return rc;
    if (n && n->rows > 0 && !dx) return fail("grad_x must be set");
    return run_backward<Dropped>(n, dropout_of(*drop), dy, dh, h, h_stride, mean, rstd, dx, dresidual, dweight, dbias,
                                 workspace, workspace_bytes, stream);
}
