// Layer norm with the residual add, forward and backward, for gfx950.
//
//   h = round(x + r),  n = (h - mean) rstd,  y = n w + b
//   dn = dy w,  dh = rstd (dn - mean(dn) - n mean(dn n)) + dh_in,  dw = sum dy n,  db = sum dy
//
// Both directions are bound by HBM: some 10 operations per element that is moved. A row lives in
// the registers of one wave (up to 2048 columns) or one block (up to 16384), so it is read once:
// mean and variance are two passes over registers, each a wave sum. The backward's threads keep
// their columns' dw and db in registers over all rows that they take; blocks leave one partial
// row each, which a second kernel sums in a fixed order (no atomics).
#include "block_common.hpp"

#include <algorithm>

namespace isa_block {
namespace {

constexpr int kThreads = 256;
constexpr int kReduceThreads = 1024;
constexpr int kMaxForwardBlocks = 2048;
constexpr int kMaxBackwardBlocks = 512;

struct NormArgs {
    const void *x, *residual, *weight, *bias;
    void *y, *h;
    float *mean, *rstd;
    int64_t rows, x_stride, residual_stride;
    int dim;
    float eps;
};

struct NormGradArgs {
    const void *dy, *dh, *h, *weight;
    const float *mean, *rstd;
    void *dx, *dresidual;
    float* partial;  // [blocks][2][dim], or null
    int64_t rows, h_stride;
    int dim;
};

// Which columns a thread of a row's `TPR` threads holds: chunk c's VEC adjacent ones with vector
// loads, single ones TPR apart where rows or pointers are not aligned for those.
template <int TPR, int VEC, bool ALIGNED>
__device__ __forceinline__ int column(int lane, int c, int e) {
    return ALIGNED ? (c * TPR + lane) * VEC + e : (c * VEC + e) * TPR + lane;
}

template <typename T, int TPR, int E, int VEC, bool ALIGNED>
__device__ __forceinline__ void load_row(const T* row, int lane, int dim, float (&out)[E]) {
#pragma unroll
    for (int c = 0; c < E / VEC; ++c) {
        if constexpr (ALIGNED) {
            const int at = column<TPR, VEC, true>(lane, c, 0);
            Pack<T, VEC> p{};
            if (at < dim) p = *reinterpret_cast<const Pack<T, VEC>*>(row + at);
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[c * VEC + e] = static_cast<float>(p.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int at = column<TPR, VEC, false>(lane, c, e);
                out[c * VEC + e] = at < dim ? static_cast<float>(row[at]) : 0.0f;
            }
        }
    }
}

template <typename T, int TPR, int E, int VEC, bool ALIGNED>
__device__ __forceinline__ void store_row(T* row, int lane, int dim, const float (&in)[E]) {
#pragma unroll
    for (int c = 0; c < E / VEC; ++c) {
        if constexpr (ALIGNED) {
            const int at = column<TPR, VEC, true>(lane, c, 0);
            Pack<T, VEC> p;
#pragma unroll
            for (int e = 0; e < VEC; ++e) p.v[e] = static_cast<T>(in[c * VEC + e]);
            if (at < dim) *reinterpret_cast<Pack<T, VEC>*>(row + at) = p;
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int at = column<TPR, VEC, false>(lane, c, e);
                if (at < dim) row[at] = static_cast<T>(in[c * VEC + e]);
            }
        }
    }
}

// The sum over a row's threads. `slot`: four floats of LDS that the row's next two sums leave alone.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* slot) {
    x = wave_sum(x);
    if constexpr (TPR == kWave) return x;
    if (threadIdx.x % kWave == 0) slot[threadIdx.x / kWave] = x;
    __syncthreads();
    return (slot[0] + slot[1]) + (slot[2] + slot[3]);
}

// Two sums with one barrier: the next two take other slots.
template <int TPR>
__device__ __forceinline__ void row_sums(float& x, float& y, float (*slots)[4]) {
    x = wave_sum(x);
    y = wave_sum(y);
    if constexpr (TPR == kWave) return;
    if (threadIdx.x % kWave == 0) {
        slots[0][threadIdx.x / kWave] = x;
        slots[1][threadIdx.x / kWave] = y;
    }
    __syncthreads();
    x = (slots[0][0] + slots[0][1]) + (slots[0][2] + slots[0][3]);
    y = (slots[1][0] + slots[1][1]) + (slots[1][2] + slots[1][3]);
}

template <typename X, typename S, typename W, int TPR, int E, int VEC, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void norm_forward_kernel(NormArgs a) {
    constexpr int kRows = kThreads / TPR;
    __shared__ float slots[2][4];
    const int lane = threadIdx.x % TPR, dim = a.dim;
    const float inv = 1.0f / static_cast<float>(dim);
    float w[E], b[E];
    load_row<W, TPR, E, VEC, ALIGNED>(static_cast<const W*>(a.weight), lane, dim, w);
    if (a.bias)
        load_row<W, TPR, E, VEC, ALIGNED>(static_cast<const W*>(a.bias), lane, dim, b);
    else
#pragma unroll
        for (int e = 0; e < E; ++e) b[e] = 0.0f;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    // a row is its TPR threads' alone: with whole-block rows all threads make the same turns
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR; r < a.rows; r += step) {
        float h[E];
        load_row<S, TPR, E, VEC, ALIGNED>(static_cast<const S*>(a.residual) + r * a.residual_stride, lane, dim, h);
        if (a.x) {
            float x[E];
            load_row<X, TPR, E, VEC, ALIGNED>(static_cast<const X*>(a.x) + r * a.x_stride, lane, dim, x);
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] = static_cast<float>(static_cast<S>(h[e] + x[e]));
            store_row<S, TPR, E, VEC, ALIGNED>(static_cast<S*>(a.h) + r * dim, lane, dim, h);
        }
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) sum += h[e];  // columns past the row's end hold 0
        const float mean = row_sum<TPR>(sum, slots[0]) * inv;
        float square = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            h[e] = column<TPR, VEC, ALIGNED>(lane, e / VEC, e % VEC) < dim ? h[e] - mean : 0.0f;
            square = fmaf(h[e], h[e], square);
        }
        const float rstd = 1.0f / sqrtf(fmaf(row_sum<TPR>(square, slots[1]), inv, a.eps));
        if (a.mean && lane == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) h[e] = fmaf(h[e] * rstd, w[e], b[e]);
        store_row<S, TPR, E, VEC, ALIGNED>(static_cast<S*>(a.y) + r * dim, lane, dim, h);
    }
}

template <typename X, typename S, typename W, int TPR, int E, int VEC, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(NormGradArgs a) {
    constexpr int kRows = kThreads / TPR;
    __shared__ float slots[2][2][4];
    const int lane = threadIdx.x % TPR, dim = a.dim;
    const float inv = 1.0f / static_cast<float>(dim);
    float w[E], dw[E], db[E];
    load_row<W, TPR, E, VEC, ALIGNED>(static_cast<const W*>(a.weight), lane, dim, w);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.0f;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int turn = 0;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR; r < a.rows; r += step, turn ^= 1) {
        float n[E], g[E], dh[E];
        load_row<S, TPR, E, VEC, ALIGNED>(static_cast<const S*>(a.h) + r * a.h_stride, lane, dim, n);
        load_row<S, TPR, E, VEC, ALIGNED>(static_cast<const S*>(a.dy) + r * dim, lane, dim, g);
        if (a.dh)
            load_row<S, TPR, E, VEC, ALIGNED>(static_cast<const S*>(a.dh) + r * dim, lane, dim, dh);
        else
#pragma unroll
            for (int e = 0; e < E; ++e) dh[e] = 0.0f;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            n[e] = (n[e] - mean) * rstd;  // past the row's end dy is 0, and so is all that n is multiplied by
            db[e] += g[e];
            dw[e] = fmaf(g[e], n[e], dw[e]);
            g[e] *= w[e];
            s1 += g[e];
            s2 = fmaf(g[e], n[e], s2);
        }
        row_sums<TPR>(s1, s2, slots[turn]);
        const float m1 = s1 * inv, m2 = s2 * inv;
#pragma unroll
        for (int e = 0; e < E; ++e) dh[e] = fmaf(rstd, g[e] - m1 - n[e] * m2, dh[e]);
        store_row<S, TPR, E, VEC, ALIGNED>(static_cast<S*>(a.dresidual) + r * dim, lane, dim, dh);
        if constexpr (!std::is_same_v<X, S>)
            store_row<X, TPR, E, VEC, ALIGNED>(static_cast<X*>(a.dx) + r * dim, lane, dim, dh);
    }
    if (!a.partial) return;
    float* mine = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * dim;
    if constexpr (TPR == kWave) {  // the block's waves hold the same columns: one adds to the other
        __shared__ float sums[2][E * kWave];
        for (int k = 0; k < kRows; ++k) {
            if (static_cast<int>(threadIdx.x / kWave) == k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    sums[0][e * kWave + lane] = k ? sums[0][e * kWave + lane] + dw[e] : dw[e];
                    sums[1][e * kWave + lane] = k ? sums[1][e * kWave + lane] + db[e] : db[e];
                }
            __syncthreads();
        }
        if (threadIdx.x < kWave)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dw[e] = sums[0][e * kWave + lane];
                db[e] = sums[1][e * kWave + lane];
            }
        else
            return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int at = column<TPR, VEC, ALIGNED>(lane, e / VEC, e % VEC);
        if (at < dim) {
            mine[at] = dw[e];
            mine[dim + at] = db[e];
        }
    }
}

// grad_weight and grad_bias from the blocks' partial rows: a block takes 64 of the 2 dim columns,
// its waves every 16th partial row.
template <typename W>
__global__ __launch_bounds__(kReduceThreads) void norm_reduce_kernel(const float* partial, int blocks, int dim,
                                                                     W* dweight, W* dbias) {
    constexpr int kWaves = kReduceThreads / kWave;
    __shared__ float sums[kWaves][kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int at = blockIdx.x * kWave + lane;
    float s = 0.0f;
    if (at < 2 * dim)
#pragma unroll 8
        for (int k = wave; k < blocks; k += kWaves) s += partial[static_cast<int64_t>(k) * 2 * dim + at];
    sums[wave][lane] = s;
    __syncthreads();
    if (wave || at >= 2 * dim) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) s += sums[k][lane];
    if (at < dim)
        dweight[at] = static_cast<W>(s);
    else if (dbias)
        dbias[at - dim] = static_cast<W>(s);
}

int64_t forward_blocks(int64_t rows, int rows_per_block) {
    return std::min<int64_t>(ceil_div(rows, rows_per_block), kMaxForwardBlocks);
}

bool wide_row(int64_t dim) { return dim > 32 * kWave; }  // a row takes a whole block

// A wave's row leaves a block with four rows at a time; two turns of it or more pay for the
// block's partial row of dw and db.
int64_t backward_blocks(int64_t rows, int64_t dim) {
    const int per_block = wide_row(dim) ? 1 : kThreads / kWave;
    return std::min<int64_t>(ceil_div(rows, 2 * per_block), kMaxBackwardBlocks);
}

struct Launch {
    bool backward;
    NormArgs f;
    NormGradArgs g;
    hipStream_t stream;
};

template <typename X, typename S, typename W, int TPR, int E, int VEC, bool ALIGNED>
void launch(const Launch& l) {
    if (l.backward) {
        const int64_t blocks = backward_blocks(l.g.rows, l.g.dim);
        norm_backward_kernel<X, S, W, TPR, E, VEC, ALIGNED>
            <<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, l.stream>>>(l.g);
    } else {
        const int64_t blocks = forward_blocks(l.f.rows, kThreads / TPR);
        norm_forward_kernel<X, S, W, TPR, E, VEC, ALIGNED>
            <<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, l.stream>>>(l.f);
    }
}

template <typename X, typename S, typename W>
void pick(const Launch& l, int64_t dim, bool aligned) {
    if (!aligned) {
        if (dim <= 8 * 64) return launch<X, S, W, 64, 8, 1, false>(l);
        if (dim <= 32 * 64) return launch<X, S, W, 64, 32, 1, false>(l);
        if (dim <= 16 * 256) return launch<X, S, W, 256, 16, 1, false>(l);
        return launch<X, S, W, 256, 64, 1, false>(l);
    }
    if constexpr (sizeof(S) == 4) {  // 16 bytes of the stream a load
        if (dim <= 4 * 64) return launch<X, S, W, 64, 4, 4, true>(l);
        if (dim <= 8 * 64) return launch<X, S, W, 64, 8, 4, true>(l);
        if (dim <= 12 * 64) return launch<X, S, W, 64, 12, 4, true>(l);
        if (dim <= 16 * 64) return launch<X, S, W, 64, 16, 4, true>(l);
        if (dim <= 32 * 64) return launch<X, S, W, 64, 32, 4, true>(l);
        if (dim <= 16 * 256) return launch<X, S, W, 256, 16, 4, true>(l);
        if (dim <= 32 * 256) return launch<X, S, W, 256, 32, 4, true>(l);
        return launch<X, S, W, 256, 64, 4, true>(l);
    } else {
        if (dim <= 8 * 64) return launch<X, S, W, 64, 8, 8, true>(l);
        if (dim <= 16 * 64) return launch<X, S, W, 64, 16, 8, true>(l);
        if (dim <= 32 * 64) return launch<X, S, W, 64, 32, 8, true>(l);
        if (dim <= 16 * 256) return launch<X, S, W, 256, 16, 8, true>(l);
        if (dim <= 32 * 256) return launch<X, S, W, 256, 32, 8, true>(l);
        return launch<X, S, W, 256, 64, 8, true>(l);
    }
}

void dispatch(const isa_block_norm& n, const Launch& l, bool aligned) {
    if (n.type == ISA_BLOCK_F32) {
        if (n.x_type == ISA_BLOCK_F32) return pick<float, float, float>(l, n.dim, aligned);
        if (n.x_type == ISA_BLOCK_BF16) return pick<bf16, float, float>(l, n.dim, aligned);
        return pick<f16, float, float>(l, n.dim, aligned);
    }
    if (n.type == ISA_BLOCK_BF16) {
        if (n.weight_type == ISA_BLOCK_F32) return pick<bf16, bf16, float>(l, n.dim, aligned);
        return pick<bf16, bf16, bf16>(l, n.dim, aligned);
    }
    if (n.weight_type == ISA_BLOCK_F32) return pick<f16, f16, float>(l, n.dim, aligned);
    return pick<f16, f16, f16>(l, n.dim, aligned);
}

int check(const isa_block_norm* n) {
    if (!n) return fail("norm is null");
    if (!known_type(n->type) || !known_type(n->x_type) || !known_type(n->weight_type))
        return fail("unknown element type (%d, %d, %d)", n->type, n->x_type, n->weight_type);
    if (n->x_type != n->type && n->type != ISA_BLOCK_F32)
        return fail("x has the residual's type, or 16 bits beside a residual of 32");
    if (n->weight_type != n->type && n->weight_type != ISA_BLOCK_F32)
        return fail("weight has the residual's type or 32 bits");
    if (n->rows < 0) return fail("negative rows %lld", static_cast<long long>(n->rows));
    if (n->dim < 1 || n->dim > ISA_BLOCK_NORM_MAX_DIM)
        return fail("dim must be 1 to %d, got %lld", ISA_BLOCK_NORM_MAX_DIM, static_cast<long long>(n->dim));
    if (!(n->eps >= 0.0f)) return fail("eps must not be negative");
    if (n->rows && !n->weight) return fail("weight is null");
    return 0;
}

// Whether each row of a tensor can be read `n` elements at a time.
bool vector_rows(const void* p, int64_t stride, int n, size_t bytes) {
    return !p || (aligned(p, n * bytes) && stride % n == 0);
}

}  // namespace
}  // namespace isa_block

using namespace isa_block;

extern "C" int isa_block_norm_forward(const isa_block_norm* n, const void* x, int64_t x_stride, const void* residual,
                                      int64_t residual_stride, void* y, void* h, float* mean, float* rstd,
                                      void* stream) {
    if (int rc = check(n)) return rc;
    if (n->rows == 0) return 0;
    if (!residual || !y) return fail("residual and y must be set");
    if ((x == nullptr) != (h == nullptr)) return fail("x and h go together");
    if ((mean == nullptr) != (rstd == nullptr)) return fail("mean and rstd go together");
    if (!x && n->x_type != n->type) return fail("without x its type is the residual's");
    const int v = n->type == ISA_BLOCK_F32 ? 4 : 8;
    const size_t s = type_bytes(n->type), w = type_bytes(n->weight_type);
    const bool vectors = n->dim % v == 0 && vector_rows(x, x_stride, v, type_bytes(n->x_type)) &&
                         vector_rows(residual, residual_stride, v, s) && vector_rows(y, n->dim, v, s) &&
                         vector_rows(h, n->dim, v, s) && vector_rows(n->weight, 0, v, w) &&
                         vector_rows(n->bias, 0, v, w);
    Launch l{};
    l.f = {x, residual, n->weight, n->bias, y, h, mean, rstd, n->rows, x_stride, residual_stride,
           static_cast<int>(n->dim), n->eps};
    l.stream = static_cast<hipStream_t>(stream);
    dispatch(*n, l, vectors);
    return launched("norm_forward_kernel");
}

extern "C" size_t isa_block_norm_backward_workspace(int64_t rows, int64_t dim) {
    if (rows < 0 || dim < 1 || dim > ISA_BLOCK_NORM_MAX_DIM) return 0;
    return static_cast<size_t>(backward_blocks(rows, dim)) * 2 * dim * sizeof(float);
}

extern "C" int isa_block_norm_backward(const isa_block_norm* n, const void* dy, const void* dh, const void* h,
                                       int64_t h_stride, const float* mean, const float* rstd, void* dx,
                                       void* dresidual, void* dweight, void* dbias, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    if (int rc = check(n)) return rc;
    if (n->rows && (!dy || !h || !mean || !rstd || !dresidual))
        return fail("grad_y, h, mean, rstd and grad_residual must be set");
    if (n->rows && (dx != nullptr) != (n->x_type != n->type))
        return fail("grad_x is written where x's type is not the residual's, and only there");
    if (!dweight && dbias) return fail("grad_bias needs grad_weight");
    const int64_t blocks = backward_blocks(n->rows, n->dim);
    if (dweight && n->rows) {
        if (workspace_bytes < isa_block_norm_backward_workspace(n->rows, n->dim))
            return fail("workspace too small: %zu bytes", workspace_bytes);
        if (!workspace || !aligned(workspace, 256)) return fail("workspace must be 256-byte aligned");
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (n->rows) {
        const int v = n->type == ISA_BLOCK_F32 ? 4 : 8;
        const size_t b = type_bytes(n->type);
        const bool vectors = n->dim % v == 0 && vector_rows(dy, n->dim, v, b) && vector_rows(dh, n->dim, v, b) &&
                             vector_rows(h, h_stride, v, b) && vector_rows(dresidual, n->dim, v, b) &&
                             vector_rows(dx, n->dim, v, type_bytes(n->x_type)) &&
                             vector_rows(n->weight, 0, v, type_bytes(n->weight_type));
        Launch l{};
        l.backward = true;
        l.g = {dy, dh, h, n->weight, mean, rstd, dx, dresidual, dweight ? static_cast<float*>(workspace) : nullptr,
               n->rows, h_stride, static_cast<int>(n->dim)};
        l.stream = s;
        dispatch(*n, l, vectors);
        if (int rc = launched("norm_backward_kernel")) return rc;
    }
    if (!dweight) return 0;
    const dim3 grid(static_cast<unsigned>(ceil_div(2 * n->dim, kWave)));
    const float* partial = static_cast<const float*>(workspace);
    const int count = static_cast<int>(blocks), dim = static_cast<int>(n->dim);
    if (n->weight_type == ISA_BLOCK_F32)
        norm_reduce_kernel<<<grid, dim3(kReduceThreads), 0, s>>>(partial, count, dim, static_cast<float*>(dweight),
                                                                static_cast<float*>(dbias));
    else if (n->weight_type == ISA_BLOCK_BF16)
        norm_reduce_kernel<<<grid, dim3(kReduceThreads), 0, s>>>(partial, count, dim, static_cast<bf16*>(dweight),
                                                                static_cast<bf16*>(dbias));
    else
        norm_reduce_kernel<<<grid, dim3(kReduceThreads), 0, s>>>(partial, count, dim, static_cast<f16*>(dweight),
                                                                static_cast<f16*>(dbias));
    return launched("norm_reduce_kernel");
}
