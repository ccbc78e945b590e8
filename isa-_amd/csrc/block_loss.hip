// Cross-entropy and its gradient, for gfx950.
//
//   loss_r = log(sum_j exp(x_rj - top_r)) + top_r - x_rt
//   dx_rj  = (exp(x_rj - top_r) / sum - [j == t]) share_r
//
// Bound by HBM: a row of logits is read once and its gradient written once. One block takes a
// row and holds it in registers, as the 16-byte chunks that were loaded, between the maximum,
// the sum and the gradient; rows too long for that are read again from the caches.
#include "block_common.hpp"

#include <algorithm>

namespace isa_block {
namespace {

constexpr int kMostThreads = 1024;
constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct LossArgs {
    const void* logits;
    const int64_t* targets;
    int64_t rows, stride, grad_stride, ignore;
    int vocab;
    float* row_loss;      // [rows], or null
    float* stats;         // [rows][2], or null
    void* grad;           // or null
    const float* count;   // rows that count, or null: no division by it
    const float* scale_by;  // gradient's factor, or null: `scale`
    int scale_step;       // 0: one factor, 1: one a row
    float scale;
};

template <int THREADS>
__device__ __forceinline__ float block_max(float x, float* slots) {
    x = wave_max(x);
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = x;
    __syncthreads();
    x = slots[0];
#pragma unroll
    for (int k = 1; k < THREADS / kWave; ++k) x = fmaxf(x, slots[k]);
    return x;
}

template <int THREADS>
__device__ __forceinline__ float block_sum(float x, float* slots) {
    x = wave_sum(x);
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0.0f;
#pragma unroll
    for (int k = 0; k < THREADS / kWave; ++k) x += slots[k];
    return x;
}

// A row as 16-byte chunks at aligned addresses: chunk c holds elements c N - skip and on. The
// first and the last may hold fewer than N of the row's elements; the others' places get `fill`.
template <typename T>
struct Row {
    static constexpr int N = 16 / sizeof(T);
    using Chunk = Pack<T, N>;
    const T* p;
    int skip, vocab;

    __device__ Row(const T* row, int n) : p(row), vocab(n) {
        skip = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
    }
    __device__ int chunks() const { return (vocab + skip + N - 1) / N; }
    __device__ __forceinline__ void load(Chunk& r, int c, T fill) const {
        const int at = c * N - skip;
        if (at >= 0 && at + N <= vocab) {
            using V = vec<T, N>;
            const V x = *reinterpret_cast<const V*>(p + at);
#pragma unroll
            for (int e = 0; e < N; ++e) r.v[e] = x[e];
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) r.v[e] = at + e >= 0 && at + e < vocab ? p[at + e] : fill;
        }
    }
    __device__ void store(T* out, int c, const Chunk& r) const {
        const int at = c * N - skip;
        // the gradient's rows may be aligned otherwise than the logits'
        if (at >= 0 && at + N <= vocab && reinterpret_cast<uintptr_t>(out + at) % 16 == 0) {
            *reinterpret_cast<Chunk*>(out + at) = r;
            return;
        }
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (at + e >= 0 && at + e < vocab) out[at + e] = r.v[e];
    }
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> gradient(const Pack<T, N>& x, int at, int target, float top, float factor,
                                               float share) {
    Pack<T, N> g;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        // exp as one correctly scaled difference: the rounding of x - top is relative to what remains
        float p = __builtin_amdgcn_exp2f((static_cast<float>(x.v[e]) - top) * kLog2E) * factor;
        if (at + e == target) p -= share;
        g.v[e] = static_cast<T>(p);
    }
    return g;
}

__device__ __forceinline__ float share_of(const LossArgs& a, int64_t r) {
    float share = a.scale_by ? a.scale_by[r * a.scale_step] : a.scale;
    if (a.count) share /= a.count[0];
    return share;
}

// The row that a block takes, in a grid of two dimensions: one may hold less than 2^32 threads, which a block a row
// passes at 2^22 rows of 1024.
__device__ __forceinline__ int64_t block_row() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

dim3 grid_of(int64_t rows) {
    constexpr int64_t kWide = int64_t{1} << 21;
    const int64_t wide = std::min(rows, kWide);
    return dim3(static_cast<unsigned>(wide), static_cast<unsigned>(ceil_div(rows, wide)));
}

// C > 0: a thread holds C chunks of the row. C == 0: the row is read once for the statistics,
// with a running maximum, and once more for the gradient.
template <typename T, int C, int THREADS>
__global__ __launch_bounds__(THREADS) void loss_kernel(LossArgs a) {
    using R = Row<T>;
    constexpr int N = R::N;
    __shared__ float slots[2][THREADS / kWave];
    const int64_t r = block_row();
    if (r >= a.rows) return;  // (a whole block)
    const R row(static_cast<const T*>(a.logits) + r * a.stride, a.vocab);
    const int chunks = row.chunks();
    const int64_t target = a.targets[r];
    T* grad = a.grad ? static_cast<T*>(a.grad) + r * a.grad_stride : nullptr;
    if (target == a.ignore) {
        if (threadIdx.x == 0) {
            if (a.row_loss) a.row_loss[r] = 0.0f;
            if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.0f;
        }
        if (grad)
            for (int c = threadIdx.x; c < chunks; c += THREADS) row.store(grad, c, typename R::Chunk{});
        return;
    }
    const T low = static_cast<T>(-INFINITY);
    float top = -INFINITY, sum = 0.0f;
    typename R::Chunk held[C ? C : 1];
    if constexpr (C > 0) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = threadIdx.x + i * THREADS;
            if (c < chunks) row.load(held[i], c, low);
            else
#pragma unroll
                for (int e = 0; e < N; ++e) held[i].v[e] = low;
        }
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) top = fmaxf(top, static_cast<float>(held[i].v[e]));
        top = block_max<THREADS>(top, slots[0]);
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e)
                sum += __builtin_amdgcn_exp2f((static_cast<float>(held[i].v[e]) - top) * kLog2E);
    } else {
        for (int c = threadIdx.x; c < chunks; c += THREADS) {
            typename R::Chunk x;
            row.load(x, c, low);
            float t = top;
#pragma unroll
            for (int e = 0; e < N; ++e) t = fmaxf(t, static_cast<float>(x.v[e]));
            const float base = t == -INFINITY ? 0.0f : t;
            sum *= __builtin_amdgcn_exp2f((top - base) * kLog2E);
#pragma unroll
            for (int e = 0; e < N; ++e)
                sum += __builtin_amdgcn_exp2f((static_cast<float>(x.v[e]) - base) * kLog2E);
            top = t;
        }
        const float mine = top;
        top = block_max<THREADS>(top, slots[0]);
        const float base = top == -INFINITY ? 0.0f : top;
        sum *= __builtin_amdgcn_exp2f((mine - base) * kLog2E);
    }
    sum = block_sum<THREADS>(sum, slots[1]);
    const bool inside = target >= 0 && target < a.vocab;
    if (threadIdx.x == 0) {
        const float log_sum = logf(sum);
        if (a.row_loss) a.row_loss[r] = inside ? log_sum + (top - static_cast<float>(row.p[target])) : NAN;
        if (a.stats) {
            a.stats[2 * r] = top;
            a.stats[2 * r + 1] = log_sum;
        }
    }
    if (!grad) return;
    const float share = inside ? share_of(a, r) : NAN, factor = share / sum;
    const int hot = inside ? static_cast<int>(target) : -1;
    if constexpr (C > 0) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = threadIdx.x + i * THREADS;
            if (c < chunks) row.store(grad, c, gradient<T, N>(held[i], c * N - row.skip, hot, top, factor, share));
        }
    } else {
        for (int c = threadIdx.x; c < chunks; c += THREADS) {
            typename R::Chunk x;
            row.load(x, c, low);
            row.store(grad, c, gradient<T, N>(x, c * N - row.skip, hot, top, factor, share));
        }
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void loss_backward_kernel(LossArgs a) {
    using R = Row<T>;
    constexpr int N = R::N;
    const int64_t r = block_row();
    if (r >= a.rows) return;  // (a whole block)
    const R row(static_cast<const T*>(a.logits) + r * a.stride, a.vocab);
    const int chunks = row.chunks();
    const int64_t target = a.targets[r];
    T* grad = static_cast<T*>(a.grad) + r * a.grad_stride;
    if (target == a.ignore) {
        for (int c = threadIdx.x; c < chunks; c += THREADS) row.store(grad, c, typename R::Chunk{});
        return;
    }
    const bool inside = target >= 0 && target < a.vocab;
    const float top = a.stats[2 * r], share = inside ? share_of(a, r) : NAN;
    const float factor = share * __builtin_amdgcn_exp2f(-a.stats[2 * r + 1] * kLog2E);
    const int hot = inside ? static_cast<int>(target) : -1;
    for (int c = threadIdx.x; c < chunks; c += THREADS) {
        typename R::Chunk x;
        row.load(x, c, static_cast<T>(-INFINITY));
        row.store(grad, c, gradient<T, N>(x, c * N - row.skip, hot, top, factor, share));
    }
}

// The rows that count, as a float (exact to 2^24 rows; the rows' number is held to that).
__global__ __launch_bounds__(kMostThreads) void loss_count_kernel(const int64_t* targets, int64_t rows, int64_t ignore,
                                                              float* count) {
    __shared__ float slots[kMostThreads / kWave];
    float n = 0.0f;
    for (int64_t r = threadIdx.x; r < rows; r += kMostThreads) n += targets[r] != ignore ? 1.0f : 0.0f;
    n = block_sum<kMostThreads>(n, slots);
    if (threadIdx.x == 0) count[0] = n;
}

__global__ __launch_bounds__(kMostThreads) void loss_sum_kernel(const float* row_loss, int64_t rows, const float* count,
                                                            float* out) {
    __shared__ float slots[kMostThreads / kWave];
    float s = 0.0f;
    for (int64_t r = threadIdx.x; r < rows; r += kMostThreads) s += row_loss[r];
    s = block_sum<kMostThreads>(s, slots);
    if (threadIdx.x == 0) out[0] = count ? s / count[0] : s;
}

template <typename T, int C, int THREADS>
void launch(const LossArgs& a, hipStream_t s) {
    loss_kernel<T, C, THREADS><<<grid_of(a.rows), dim3(THREADS), 0, s>>>(a);
}

// Chunks of the longest row, one more where rows start inside a chunk.
template <typename T>
int64_t chunks_of(const LossArgs& a) {
    return ceil_div(a.vocab, 16 / sizeof(T)) + 1;
}

// Blocks of 256 threads where those hold a row in four chunks each, so that several rows share a
// compute unit (1023 rows of 5003 in bf16: 7.6 us, in blocks of 1024 11.3); larger rows take 1024.
template <typename T>
void launch_rows(const LossArgs& a, hipStream_t s) {
    const int64_t chunks = chunks_of<T>(a), few = ceil_div(chunks, 256), each = ceil_div(chunks, 1024);
    if (!a.grad) return few <= 4 ? launch<T, 0, 256>(a, s) : launch<T, 0, 1024>(a, s);  // nothing is read twice
    if (few <= 1) return launch<T, 1, 256>(a, s);
    if (few <= 2) return launch<T, 2, 256>(a, s);
    if (few <= 3) return launch<T, 3, 256>(a, s);
    if (few <= 4) return launch<T, 4, 256>(a, s);
    if (each <= 2) return launch<T, 2, 1024>(a, s);
    if (each <= 4) return launch<T, 4, 1024>(a, s);
    if (each <= 7) return launch<T, 7, 1024>(a, s);
    if (each <= 10) return launch<T, 10, 1024>(a, s);
    if (each <= 13) return launch<T, 13, 1024>(a, s);
    if (each <= 16) return launch<T, 16, 1024>(a, s);
    launch<T, 0, 1024>(a, s);
}

template <typename T>
void launch_backward(const LossArgs& a, hipStream_t s) {
    const dim3 grid = grid_of(a.rows);
    if (chunks_of<T>(a) <= 1024)
        loss_backward_kernel<T, 256><<<grid, 256, 0, s>>>(a);
    else
        loss_backward_kernel<T, 1024><<<grid, 1024, 0, s>>>(a);
}

void run_rows(int type, const LossArgs& a, hipStream_t s) {
    if (type == ISA_BLOCK_F32) launch_rows<float>(a, s);
    else if (type == ISA_BLOCK_BF16) launch_rows<bf16>(a, s);
    else launch_rows<f16>(a, s);
}

constexpr int64_t kMaxRows = int64_t{1} << 24;

int check(const isa_block_loss* l) {
    if (!l) return fail("loss is null");
    if (!known_type(l->type)) return fail("unknown element type %d", l->type);
    if (l->rows < 0 || l->rows > kMaxRows)
        return fail("rows must be 0 to %lld, got %lld", static_cast<long long>(kMaxRows),
                    static_cast<long long>(l->rows));
    if (l->vocab < 1 || l->vocab > (int64_t{1} << 30))
        return fail("vocab must be 1 to 2^30, got %lld", static_cast<long long>(l->vocab));
    if (l->rows && (!l->logits || !l->targets)) return fail("logits and targets must be set");
    if (l->rows && !aligned(l->logits, type_bytes(l->type))) return fail("logits are not aligned to their type");
    return 0;
}

int check_workspace(const isa_block_loss* l, const void* workspace, size_t bytes) {
    if (bytes < isa_block_loss_workspace(l)) return fail("workspace too small: %zu bytes", bytes);
    if (!workspace || !aligned(workspace, 256)) return fail("workspace must be 256-byte aligned");
    return 0;
}

LossArgs args_of(const isa_block_loss* l) {
    LossArgs a{};
    a.logits = l->logits;
    a.targets = l->targets;
    a.rows = l->rows;
    a.stride = l->logits_stride;
    a.ignore = l->ignore_index;
    a.vocab = static_cast<int>(l->vocab);
    return a;
}

}  // namespace
}  // namespace isa_block

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
    if (l->rows) run_rows(l->type, a, s);
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
    if (l->type == ISA_BLOCK_F32) launch_backward<float>(a, s);
    else if (l->type == ISA_BLOCK_BF16) launch_backward<bf16>(a, s);
    else launch_backward<f16>(a, s);
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
    if (l->rows) run_rows(l->type, a, s);
    if (int rc = launched("loss_kernel")) return rc;
    loss_sum_kernel<<<1, kMostThreads, 0, s>>>(ws + 64, l->rows, ws, out);
    return launched("loss_sum_kernel");
}
