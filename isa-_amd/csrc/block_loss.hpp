// Losses of a softmax over logits and their gradients, for gfx950: the kernels over rows.
//
//   l_r   = x_rt - top_r - log(sum_j exp(x_rj - top_r))
//   dx_rj = (exp(x_rj - top_r) / sum - [j == t]) share_r
//
// The cross-entropy is -l_r; other losses are functions of l_r, whose negative slope joins the share.
//
// Bound by HBM: a row of logits is read once and its gradient written once. One block takes a
// row and holds it in registers, as the 16-byte chunks that were loaded, between the maximum,
// the sum and the gradient. Rows too long for that, of more than 16 chunks a thread (65500 elements of fp32, 131000 of
// 16 bits), are read again, in part from the last cache: 4096 x 128256 in fp32 1012 us, 6.2 TB/s of three transfers.
#pragma once

#include "block_common.hpp"

#include "isa_train.h"

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
    // losses of l: rows r tokens .. (r + 1) tokens - 1 share slope[r] (and factor r mod pairs, if any has one)
    const float* slope;  // backward: dloss / dl, or null: -1
    int64_t tokens, pairs;
    bool backwards;      // backward: the last rows first
    const float *old_logp, *advantages, *ref_logp;  // [rows]
    float low, high, kl;
    float* logp;      // [rows]
    float* row_slope;  // [rows], or null
    double* row_logp;  // [rows], statistics alone: l, 0 in ignored rows
    bool count_here;   // each block counts the rows that are not ignored, for its gradient
    bool past;         // the gradient is written past the caches
};

// What a row's loss is of its l.
enum class Of { kCrossEntropy, kPolicy, kStats };  // kStats: l and the statistics alone

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

// The rows that are not ignored, by a block (a float: exact to 2^24 rows, which the rows' number is held to).
template <int THREADS>
__device__ __forceinline__ float block_count(const int64_t* targets, int64_t rows, int64_t ignore, float* slots) {
    float n = 0.0f;
    for (int64_t r = threadIdx.x; r < rows; r += THREADS) n += targets[r] != ignore ? 1.0f : 0.0f;
    return block_sum<THREADS>(n, slots);
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
    __device__ void store(T* out, int c, const Chunk& r, bool past = false) const {
        const int at = c * N - skip;
        // the gradient's rows may be aligned otherwise than the logits'
        if (at >= 0 && at + N <= vocab && reinterpret_cast<uintptr_t>(out + at) % 16 == 0) {
            if (past) {
                using V = vec<uint32_t, 4>;
                asm volatile("");  // two stores of one value to one place become one, of the ordinary kind: not with these between
                __builtin_nontemporal_store(__builtin_bit_cast(V, r), reinterpret_cast<V*>(out + at));
                asm volatile("");
            } else {
                *reinterpret_cast<Chunk*>(out + at) = r;
            }
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

// The same with the slope of a loss of l.
__device__ __forceinline__ float sloped_share_of(const LossArgs& a, int64_t r) {
    const int64_t s = r / a.tokens;
    float share = a.scale_by ? a.scale_by[a.scale_step ? s % a.pairs : 0] : 1.0f;
    share *= a.scale;
    if (a.count) share /= a.count[0];
    return -a.slope[s] * share;
}

// The policy loss of a row and its slope by l.
__device__ __forceinline__ float policy(const LossArgs& a, int64_t r, float l, float& slope) {
    const float moved = l - a.old_logp[r], ratio = expf(moved), by = a.advantages[r];
    // (without an advantage 0, also of a ratio past fp32's largest number)
    const float free = by == 0.0f && fabsf(moved) < INFINITY ? 0.0f : ratio * by, held = fminf(fmaxf(ratio, a.low), a.high) * by;
    float loss = -fminf(free, held);
    slope = free <= held ? -free : 0.0f;
    if (free != free) loss = slope = free;  // (the minimum of NaN and a number is the number)
    if (a.kl != 0.0f) {
        const float gap = a.ref_logp[r] - l, e = expm1f(gap);
        loss = fmaf(a.kl, e - gap, loss);
        slope = fmaf(-a.kl, e, slope);
    }
    return loss;
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
template <typename T, int C, int THREADS, Of OF>
__global__ __launch_bounds__(THREADS) void loss_kernel(LossArgs a) {
    using R = Row<T>;
    constexpr int N = R::N;
    __shared__ float slots[2][THREADS / kWave];
    [[maybe_unused]] __shared__ float count_slots[OF == Of::kPolicy ? THREADS / kWave : 1];
    const int64_t r = block_row();
    if (r >= a.rows) return;  // (a whole block)
    const R row(static_cast<const T*>(a.logits) + r * a.stride, a.vocab);
    const int chunks = row.chunks();
    const int64_t target = a.targets[r];
    [[maybe_unused]] float count = 1.0f;
    T* grad = a.grad ? static_cast<T*>(a.grad) + r * a.grad_stride : nullptr;
    if (target == a.ignore) {
        if (threadIdx.x == 0) {
            if (a.row_loss) a.row_loss[r] = 0.0f;
            if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.0f;
            if constexpr (OF == Of::kPolicy) {
                a.logp[r] = 0.0f;
                if (a.row_slope) a.row_slope[r] = 0.0f;
            }
            if constexpr (OF == Of::kStats) a.row_logp[r] = 0.0;
        }
        if (grad)
            for (int c = threadIdx.x; c < chunks; c += THREADS) row.store(grad, c, typename R::Chunk{}, OF == Of::kPolicy && a.past);
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
        if constexpr (OF == Of::kPolicy)  // while the row is on its way
            if (a.count_here) count = block_count<THREADS>(a.targets, a.rows, a.ignore, count_slots);
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
        if constexpr (OF == Of::kPolicy)
            if (a.count_here) count = block_count<THREADS>(a.targets, a.rows, a.ignore, count_slots);
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
    [[maybe_unused]] float slope = 0.0f;
    if constexpr (OF == Of::kPolicy) {
        const float l = inside ? (static_cast<float>(row.p[target]) - top) - logf(sum) : NAN;
        const float loss = policy(a, r, l, slope);
        if (threadIdx.x == 0) {
            a.row_loss[r] = loss;
            a.logp[r] = l;
            if (a.row_slope) a.row_slope[r] = slope;
        }
    }
    if (threadIdx.x == 0) {
        const float log_sum = logf(sum);
        if (OF == Of::kCrossEntropy && a.row_loss)
            a.row_loss[r] = inside ? log_sum + (top - static_cast<float>(row.p[target])) : NAN;
        // sums of it over a long sequence need more than its own rounding leaves (for the statistics alone: a logarithm of
        // 64 bits takes registers, and 16 more than 64 leave a compute unit to one row of the others)
        if constexpr (OF == Of::kStats)
            a.row_logp[r] = inside ? static_cast<double>(static_cast<float>(row.p[target])) - top - log(static_cast<double>(sum))
                                   : NAN;
        if (a.stats) {
            a.stats[2 * r] = top;
            a.stats[2 * r + 1] = log_sum;
        }
    }
    if (!grad) return;
    float share = inside ? share_of(a, r) : NAN;
    if constexpr (OF == Of::kPolicy) share = share / count * -slope;  // (as where the count is an input)
    const float factor = share / sum;
    const int hot = inside ? static_cast<int>(target) : -1;
    if constexpr (C > 0) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = threadIdx.x + i * THREADS;
            if (c < chunks) row.store(grad, c, gradient<T, N>(held[i], c * N - row.skip, hot, top, factor, share),
                                      OF == Of::kPolicy && a.past);
        }
    } else {
        for (int c = threadIdx.x; c < chunks; c += THREADS) {
            typename R::Chunk x;
            row.load(x, c, low);
            row.store(grad, c, gradient<T, N>(x, c * N - row.skip, hot, top, factor, share), OF == Of::kPolicy && a.past);
        }
    }
}

// A row's gradient from its statistics, by a block; share(): its factor, asked for where the row counts.
template <typename T, int THREADS, typename Share>
__device__ __forceinline__ void row_gradient(const LossArgs& a, int64_t r, bool past, Share share_of_row) {
    using R = Row<T>;
    constexpr int N = R::N;
    const R row(static_cast<const T*>(a.logits) + r * a.stride, a.vocab);
    const int chunks = row.chunks();
    const int64_t target = a.targets[r];
    T* grad = static_cast<T*>(a.grad) + r * a.grad_stride;
    if (target == a.ignore) {
        for (int c = threadIdx.x; c < chunks; c += THREADS) row.store(grad, c, typename R::Chunk{}, past);
        return;
    }
    const bool inside = target >= 0 && target < a.vocab;
    const float top = a.stats[2 * r], share = inside ? share_of_row() : NAN;
    const float factor = share * __builtin_amdgcn_exp2f(-a.stats[2 * r + 1] * kLog2E);
    const int hot = inside ? static_cast<int>(target) : -1;
    for (int c = threadIdx.x; c < chunks; c += THREADS) {
        typename R::Chunk x;
        row.load(x, c, static_cast<T>(-INFINITY));
        row.store(grad, c, gradient<T, N>(x, c * N - row.skip, hot, top, factor, share), past);
    }
}

template <typename T, int THREADS, bool SLOPED>
__global__ __launch_bounds__(THREADS) void loss_backward_kernel(LossArgs a) {
    int64_t r = block_row();
    if (r >= a.rows) return;  // (a whole block)
    if (SLOPED && a.backwards) r = a.rows - 1 - r;
    row_gradient<T, THREADS>(a, r, SLOPED && a.past, [&] { return SLOPED ? sloped_share_of(a, r) : share_of(a, r); });
}

__global__ __launch_bounds__(kMostThreads) void loss_count_kernel(const int64_t* targets, int64_t rows, int64_t ignore,
                                                              float* count) {
    __shared__ float slots[kMostThreads / kWave];
    const float n = block_count<kMostThreads>(targets, rows, ignore, slots);
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

template <typename T, int C, int THREADS, Of OF>
void launch(const LossArgs& a, hipStream_t s) {
    loss_kernel<T, C, THREADS, OF><<<grid_of(a.rows), dim3(THREADS), 0, s>>>(a);
}

// Chunks of the longest row, one more where rows start inside a chunk.
template <typename T>
int64_t chunks_of(const LossArgs& a) {
    return ceil_div(a.vocab, 16 / sizeof(T)) + 1;
}

// Blocks of 256 threads where those hold a row in four chunks each, so that several rows share a
// compute unit (1023 rows of 5003 in bf16: 7.6 us, in blocks of 1024 11.3); larger rows take 1024.
//
// The losses of l take blocks of 256 up to 2304 chunks and of 512 up to 4096 (16-bit types, or passes that hold no row): one
// of 1024, whose rows of few chunks a thread end at its slowest wave, leaves the compute unit to one row. Policy calls
// of 8192 rows, us of 256 / 512 / 1024 threads: 5003 in fp32 60 / 60 / 74, 8500 101 / 98 / 108, 10000 115 / 114 / 111,
// 8200 in bf16 57 / 60 / 79, 16384 109 / 117 / 148, 24000 149 / 153 / 179, 28000 228 / 175 / 199; 4096 rows of 33333
// 240 / 161 / 142. Preference calls of 8192 rows: 5003 in fp32 71 / 74 / 95, 12000 155 / 148 / 156, 50304 729 / 699 / 677.
template <typename T, Of OF>
bool launch_smaller_rows(const LossArgs& a, int64_t chunks, hipStream_t s) {
    const int64_t few = ceil_div(chunks, 256), some = ceil_div(chunks, 512);
    if (few > 4 && few <= 9) {
        if (!a.grad) launch<T, 0, 256, OF>(a, s);
        else if (few <= 5) launch<T, 5, 256, OF>(a, s);
        else if (few <= 7) launch<T, 7, 256, OF>(a, s);
        else launch<T, 9, 256, OF>(a, s);
        return true;
    }
    if (few > 9 && some <= 8 && (!a.grad || sizeof(T) == 2)) {
        if (!a.grad) launch<T, 0, 512, OF>(a, s);
        else if (some <= 6) launch<T, 6, 512, OF>(a, s);
        else launch<T, 8, 512, OF>(a, s);
        return true;
    }
    return false;
}

template <typename T, Of OF>
void launch_rows(const LossArgs& a, hipStream_t s) {
    const int64_t chunks = chunks_of<T>(a), few = ceil_div(chunks, 256), each = ceil_div(chunks, 1024);
    if constexpr (OF != Of::kCrossEntropy)
        if (launch_smaller_rows<T, OF>(a, chunks, s)) return;
    if (!a.grad) return few <= 4 ? launch<T, 0, 256, OF>(a, s) : launch<T, 0, 1024, OF>(a, s);  // nothing is read twice
    if (few <= 1) return launch<T, 1, 256, OF>(a, s);
    if (few <= 2) return launch<T, 2, 256, OF>(a, s);
    if (few <= 3) return launch<T, 3, 256, OF>(a, s);
    if (few <= 4) return launch<T, 4, 256, OF>(a, s);
    if (each <= 2) return launch<T, 2, 1024, OF>(a, s);
    if (each <= 4) return launch<T, 4, 1024, OF>(a, s);
    if (each <= 7) return launch<T, 7, 1024, OF>(a, s);
    if (each <= 10) return launch<T, 10, 1024, OF>(a, s);
    if (each <= 13) return launch<T, 13, 1024, OF>(a, s);
    if (each <= 16) return launch<T, 16, 1024, OF>(a, s);
    launch<T, 0, 1024, OF>(a, s);
}

template <typename T, bool SLOPED>
void launch_backward(const LossArgs& a, hipStream_t s) {
    const dim3 grid = grid_of(a.rows);
    const int64_t chunks = chunks_of<T>(a);
    if constexpr (SLOPED)
        if (chunks > 2304 && chunks <= 4096) {
            loss_backward_kernel<T, 512, SLOPED><<<grid, 512, 0, s>>>(a);
            return;
        }
    if (chunks <= (SLOPED ? 2304 : 1024))
        loss_backward_kernel<T, 256, SLOPED><<<grid, 256, 0, s>>>(a);
    else
        loss_backward_kernel<T, 1024, SLOPED><<<grid, 1024, 0, s>>>(a);
}

template <Of OF>
void run_rows(int type, const LossArgs& a, hipStream_t s) {
    if (type == ISA_BLOCK_F32) launch_rows<float, OF>(a, s);
    else if (type == ISA_BLOCK_BF16) launch_rows<bf16, OF>(a, s);
    else launch_rows<f16, OF>(a, s);
}

template <bool SLOPED>
void run_backward(int type, const LossArgs& a, hipStream_t s) {
    if (type == ISA_BLOCK_F32) launch_backward<float, SLOPED>(a, s);
    else if (type == ISA_BLOCK_BF16) launch_backward<bf16, SLOPED>(a, s);
    else launch_backward<f16, SLOPED>(a, s);
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
