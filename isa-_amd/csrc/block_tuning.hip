// Losses of tuning a model by rewards or by pairs of answers, and their gradients: the C entries.
//
// The policy loss is a function of each row's l alone: one pass over the logits, as the cross-entropy's, bound by
// HBM. The preference loss's slope needs the sums of whole sequences: one pass reads the logits for l and the
// rows' statistics, a block a pair makes the slopes, a second pass reads them again and writes the gradient, last rows
// first. 8192 x 50304 in fp32: policy 527 us (2.9 GB without the ignored quarter's rows, 5.5 TB/s), preference 58 + 344 (40%
// of its rows count; the first pass finds the rest of the last call's in the cache).
#include "block_loss.hpp"

namespace isa_block {
namespace {

constexpr int kPairThreads = 256;

// Up to so many rows each row's block counts those that are not ignored: 8 KiB of targets, read beside its logits,
// instead of a launch before (a call of 1023 x 5003 in bf16: 10.7 us, with the launch 13.8; of 2048 x 5003 17.0 and 16.3).
constexpr int64_t kCountHere = 1024;

// Up to so many rows one block takes all pairs and their sum (a call of 8192 x 5003 in bf16: 52.2 us, with a block a
// pair and one for the sum 53.8; of 16384 x 1000 in 32 pairs 45.6 and 40.9).
constexpr int64_t kPairsHere = 8192;

// Up to so many rows of so many bytes and pairs each row's block of 256 makes its pair's slope from the pair's l, which saves
// a launch: a call of 2 x 512 x 1000 in bf16 10.2 us, else 15.0; of 6 x 171 x 5003 in fp16 14.8 and 17.8; of 32 x 32 x
// 5003 in bf16 17.6 and 17.9; of 2 x 1024 x 5003 21.5 and 21.4, of 64 x 32 x 1000 22.5 and 17.3, of 8 x 128 x 50304 in
// fp32 133 and 101.
constexpr int64_t kFewRows = 1536, kFewPairs = 16, kFewBytes = 2304 * 16;

// Gradients of so many bytes are written past the caches.
constexpr size_t kGradientPast = size_t{128} << 20;

struct PairArgs {
    const double* row_logp;  // [2 pairs][tokens]
    const float* ref;
    int64_t pairs, tokens;
    float *loss, *logp, *slope;  // [pairs], [2 pairs], [2 pairs] or null
    float beta;
};

// The mean over the rows that are not ignored, which are counted here.
__global__ __launch_bounds__(kMostThreads) void loss_mean_kernel(const float* row_loss, const int64_t* targets,
                                                             int64_t rows, int64_t ignore, float* out) {
    __shared__ float slots[2][kMostThreads / kWave];
    float s = 0.0f;
    for (int64_t r = threadIdx.x; r < rows; r += kMostThreads) s += row_loss[r];
    const float n = block_count<kMostThreads>(targets, rows, ignore, slots[0]);
    s = block_sum<kMostThreads>(s, slots[1]);
    if (threadIdx.x == 0) out[0] = s / n;
}

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) x += __shfl_xor(x, by);
    return x;
}

__device__ __forceinline__ double pair_margin(const PairArgs& a, int64_t p, double chosen, double other) {
    return a.beta * ((chosen - a.ref[p]) - (other - a.ref[a.pairs + p]));
}

// The slope of a pair's loss by its chosen sequence's sum; by the other one's it is the negative.
__device__ __forceinline__ float pair_slope(const PairArgs& a, double margin) {
    return static_cast<float>(-a.beta / (1.0 + exp(margin)));
}

// A pair's loss and slopes from the sums of its sequences.
__device__ __forceinline__ float pair_loss(const PairArgs& a, int64_t p, double chosen, double other) {
    const double m = pair_margin(a, p, chosen, other);
    a.logp[p] = static_cast<float>(chosen);
    a.logp[a.pairs + p] = static_cast<float>(other);
    if (a.slope) {
        a.slope[p] = pair_slope(a, m);
        a.slope[a.pairs + p] = -a.slope[p];
    }
    return static_cast<float>((m < 0.0 ? -m : 0.0) + log1p(exp(-fabs(m))));
}

template <int THREADS>
__device__ __forceinline__ double block_sum64(double x, double* slots) {
    x = wave_sum64(x);
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0.0;
    for (int k = 0; k < THREADS / kWave; ++k) x += slots[k];
    return x;
}

// The sums of pair p's sequences, in all threads of a block. `slots` are free again after the block's next barrier.
template <int THREADS>
__device__ __forceinline__ void pair_sums(const PairArgs& a, int64_t p, double (&slots)[2][THREADS / kWave],
                                          double (&sums)[2]) {
    double s[2] = {0.0, 0.0};
    for (int64_t i = threadIdx.x; i < a.tokens; i += THREADS) {
        s[0] += a.row_logp[p * a.tokens + i];
        s[1] += a.row_logp[(a.pairs + p) * a.tokens + i];
    }
    for (int k = 0; k < 2; ++k) sums[k] = block_sum64<THREADS>(s[k], slots[k]);
}

// A block a pair.
__global__ __launch_bounds__(kPairThreads) void preference_pair_kernel(PairArgs a) {
    __shared__ double slots[2][kPairThreads / kWave];
    for (int64_t p = blockIdx.x; p < a.pairs; p += gridDim.x) {
        double sums[2];
        pair_sums<kPairThreads>(a, p, slots, sums);
        if (threadIdx.x == 0) a.loss[p] = pair_loss(a, p, sums[0], sums[1]);
        __syncthreads();
    }
}

// All pairs, a wave each, and the sum or mean of their losses.
template <int THREADS>
__device__ __forceinline__ void all_pairs(const PairArgs& a, int mean, float* out) {
    __shared__ double slots[THREADS / kWave];
    const int lane = threadIdx.x % kWave;
    double all = 0.0;
    for (int64_t p = threadIdx.x / kWave; p < a.pairs; p += THREADS / kWave) {
        double sums[2];
        for (int k = 0; k < 2; ++k) {
            const double* rows = a.row_logp + (k * a.pairs + p) * a.tokens;
            double s = 0.0;
#pragma unroll 8
            for (int64_t i = lane; i < a.tokens; i += kWave) s += rows[i];
            sums[k] = wave_sum64(s);
        }
        if (lane == 0) all += pair_loss(a, p, sums[0], sums[1]);
    }
    all = block_sum64<THREADS>(all, slots);
    if (threadIdx.x == 0) out[0] = static_cast<float>(mean ? all / a.pairs : all);
}

__global__ __launch_bounds__(kMostThreads) void preference_pairs_kernel(PairArgs a, int mean, float* out) {
    all_pairs<kMostThreads>(a, mean, out);
}

// The gradients of few rows, each of whose blocks makes its pair's slope, and by one block more the pairs' losses.
template <typename T>
__global__ __launch_bounds__(kPairThreads) void preference_rows_kernel(LossArgs a, PairArgs b, float* out) {
    __shared__ double slots[2][kPairThreads / kWave];
    const int64_t r = blockIdx.x;
    if (r == a.rows) return all_pairs<kPairThreads>(b, 1, out);
    row_gradient<T, kPairThreads>(a, r, false, [&] {
        const int64_t sequence = r / b.tokens, p = sequence % b.pairs;
        double sums[2];
        pair_sums<kPairThreads>(b, p, slots, sums);
        const float slope = pair_slope(b, pair_margin(b, p, sums[0], sums[1]));
        return (sequence < b.pairs ? -slope : slope) * a.scale;
    });
}

__global__ __launch_bounds__(kPairThreads) void preference_sum_kernel(const float* loss, int64_t pairs, int mean,
                                                                      float* out) {
    __shared__ double slots[kPairThreads / kWave];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < pairs; i += kPairThreads) s += loss[i];
    s = block_sum64<kPairThreads>(s, slots);
    if (threadIdx.x == 0) out[0] = static_cast<float>(mean ? s / pairs : s);
}

bool past_caches(const isa_block_loss& l) {
    return static_cast<size_t>(l.rows) * l.vocab * type_bytes(l.type) >= kGradientPast;
}

int check(const isa_train_policy* p) {
    if (!p) return fail("policy is null");
    if (int rc = check(&p->loss)) return rc;
    if (p->loss.rows && (!p->old_logp || !p->advantages)) return fail("old_logp and advantages must be set");
    if (!(p->low >= 0.0f && p->high >= p->low)) return fail("the ratio's bounds must be 0 <= low <= high");
    if (!(p->kl >= 0.0f)) return fail("kl must not be negative");
    if (p->loss.rows && p->kl != 0.0f && !p->ref_logp) return fail("kl needs ref_logp");
    return 0;
}

LossArgs args_of(const isa_train_policy* p) {
    LossArgs a = args_of(&p->loss);
    a.old_logp = p->old_logp;
    a.advantages = p->advantages;
    a.ref_logp = p->ref_logp;
    a.low = p->low;
    a.high = p->high;
    a.kl = p->kl;
    return a;
}

int check(const isa_train_preference* p) {
    if (!p) return fail("preference is null");
    if (int rc = check(&p->loss)) return rc;
    if (p->pairs < 0 || p->tokens < 0 || p->pairs > kMaxRows || p->tokens > kMaxRows ||
        p->loss.rows != 2 * p->pairs * p->tokens)
        return fail("rows must be 2 pairs tokens");
    if (p->pairs && !p->ref_logp) return fail("ref_logp must be set");
    if (!(p->beta > 0.0f) || p->beta > 3e38f) return fail("beta must be positive and finite");
    return 0;
}

// The workspace's parts: rows' l, their statistics, the pairs' losses, the sequences' slopes.
struct PreferenceSpace {
    size_t stats, loss, slope, bytes;
    explicit PreferenceSpace(const isa_train_preference* p) {
        stats = static_cast<size_t>(p->loss.rows) * sizeof(double);
        loss = stats + static_cast<size_t>(p->loss.rows) * 2 * sizeof(float);
        slope = loss + static_cast<size_t>(p->pairs) * sizeof(float);
        bytes = slope + static_cast<size_t>(2 * p->pairs) * sizeof(float) + 256;
    }
};

int check_workspace(const isa_train_preference* p, const void* workspace, size_t bytes) {
    if (bytes < PreferenceSpace(p).bytes) return fail("workspace too small: %zu bytes", bytes);
    if (!workspace || !aligned(workspace, 256)) return fail("workspace must be 256-byte aligned");
    return 0;
}

// l of rows, sequences' sums, losses and slopes of pairs, and unless out is null their losses' sum or mean.
int run_pairs(const isa_train_preference* p, float* stats, float* losses, float* logp, float* slope, int mean, float* out,
              void* workspace, hipStream_t s) {
    LossArgs a = args_of(&p->loss);
    a.row_logp = static_cast<double*>(workspace);
    a.stats = stats;
    if (p->loss.rows) run_rows<Of::kStats>(p->loss.type, a, s);
    if (int rc = launched("loss_kernel")) return rc;
    const PairArgs b{a.row_logp, p->ref_logp, p->pairs, p->tokens, losses, logp, slope, p->beta};
    if (out && p->loss.rows <= kPairsHere && p->pairs <= kPairsHere) {
        preference_pairs_kernel<<<1, kMostThreads, 0, s>>>(b, mean, out);
        return launched("preference_pairs_kernel");
    }
    const int64_t blocks = std::min<int64_t>(p->pairs, 4096);
    if (blocks) preference_pair_kernel<<<dim3(static_cast<unsigned>(blocks)), dim3(kPairThreads), 0, s>>>(b);
    if (int rc = launched("preference_pair_kernel")) return rc;
    if (!out) return 0;
    preference_sum_kernel<<<1, kPairThreads, 0, s>>>(losses, p->pairs, mean, out);
    return launched("preference_sum_kernel");
}

// Few rows: l and statistics, then all the rest in one launch.
int run_few_pairs(const isa_train_preference* p, float scale, float* stats, float* logp, float* out, void* grad,
                  int64_t grad_stride, void* workspace, hipStream_t s) {
    LossArgs a = args_of(&p->loss);
    a.row_logp = static_cast<double*>(workspace);
    a.stats = stats;
    run_rows<Of::kStats>(p->loss.type, a, s);
    if (int rc = launched("loss_kernel")) return rc;
    a.grad = grad;
    a.grad_stride = grad_stride;
    a.scale = scale;
    const PairArgs b{a.row_logp, p->ref_logp, p->pairs, p->tokens, nullptr, logp, nullptr, p->beta};
    const dim3 grid(static_cast<unsigned>(a.rows + 1));
    if (p->loss.type == ISA_BLOCK_F32) preference_rows_kernel<float><<<grid, dim3(kPairThreads), 0, s>>>(a, b, out);
    else if (p->loss.type == ISA_BLOCK_BF16) preference_rows_kernel<bf16><<<grid, dim3(kPairThreads), 0, s>>>(a, b, out);
    else preference_rows_kernel<f16><<<grid, dim3(kPairThreads), 0, s>>>(a, b, out);
    return launched("preference_rows_kernel");
}

int run_pairs_backward(const isa_train_preference* p, const float* stats, const float* slope, const float* by, int step,
                       float scale, void* grad, int64_t grad_stride, hipStream_t s) {
    LossArgs a = args_of(&p->loss);
    a.stats = const_cast<float*>(stats);
    a.slope = slope;
    a.tokens = p->tokens;
    a.pairs = p->pairs;
    a.scale_by = by;
    a.scale_step = step;
    a.scale = scale;
    a.grad = grad;
    a.grad_stride = grad_stride;
    a.backwards = true;  // those that were read last are in the caches
    a.past = past_caches(p->loss);
    run_backward<true>(p->loss.type, a, s);
    return launched("loss_backward_kernel");
}

}  // namespace
}  // namespace isa_block

using namespace isa_block;

extern "C" int isa_train_policy_forward(const isa_train_policy* p, int reduction, float* out, float* logp, float* stats,
                                        float* slope, float* count, void* workspace, size_t workspace_bytes,
                                        void* stream) {
    if (int rc = check(p)) return rc;
    const isa_block_loss* l = &p->loss;
    if (reduction < ISA_BLOCK_MEAN || reduction > ISA_BLOCK_NONE) return fail("unknown reduction %d", reduction);
    if (reduction == ISA_BLOCK_NONE && l->rows == 0) return 0;
    if (!out || (l->rows && !logp)) return fail("out and logp must be set");
    if (l->rows && ((stats == nullptr) != (slope == nullptr) || (stats == nullptr) != (count == nullptr)))
        return fail("stats, slope and count go together");
    if (int rc = check_workspace(l, workspace, workspace_bytes)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(workspace);
    if (!count) count = ws;
    if (reduction == ISA_BLOCK_MEAN) {
        loss_count_kernel<<<1, kMostThreads, 0, s>>>(l->targets, l->rows, l->ignore_index, count);
        if (int rc = launched("loss_count_kernel")) return rc;
    }
    LossArgs a = args_of(p);
    a.row_loss = reduction == ISA_BLOCK_NONE ? out : ws + 64;
    a.logp = logp;
    a.stats = stats;
    a.row_slope = slope;
    if (l->rows) run_rows<Of::kPolicy>(l->type, a, s);
    if (int rc = launched("loss_kernel")) return rc;
    if (reduction == ISA_BLOCK_NONE) return 0;
    loss_sum_kernel<<<1, kMostThreads, 0, s>>>(ws + 64, l->rows, reduction == ISA_BLOCK_MEAN ? count : nullptr, out);
    return launched("loss_sum_kernel");
}

extern "C" int isa_train_policy_backward(const isa_block_loss* l, int reduction, const float* stats, const float* slope,
                                         const float* count, const float* grad_out, void* grad, int64_t grad_stride,
                                         void* stream) {
    if (int rc = check(l)) return rc;
    if (reduction < ISA_BLOCK_MEAN || reduction > ISA_BLOCK_NONE) return fail("unknown reduction %d", reduction);
    if (l->rows == 0) return 0;
    if (!stats || !slope || !grad_out || !grad || (reduction == ISA_BLOCK_MEAN && !count))
        return fail("stats, slope, grad_out, grad_logits and a mean's count must be set");
    if (!aligned(grad, type_bytes(l->type))) return fail("grad_logits is not aligned to its type");
    LossArgs a = args_of(l);
    a.stats = const_cast<float*>(stats);
    a.slope = slope;
    a.tokens = 1;
    a.pairs = l->rows;
    a.count = reduction == ISA_BLOCK_MEAN ? count : nullptr;
    a.scale_by = grad_out;
    a.scale_step = reduction == ISA_BLOCK_NONE;
    a.scale = 1.0f;
    a.past = past_caches(*l);
    a.grad = grad;
    a.grad_stride = grad_stride;
    run_backward<true>(l->type, a, static_cast<hipStream_t>(stream));
    return launched("loss_backward_kernel");
}

extern "C" int isa_train_policy_with_grad(const isa_train_policy* p, float grad_scale, float* out, float* logp,
                                          void* grad, int64_t grad_stride, void* workspace, size_t workspace_bytes,
                                          void* stream) {
    if (int rc = check(p)) return rc;
    const isa_block_loss* l = &p->loss;
    if (!out || (l->rows && (!grad || !logp))) return fail("out, logp and grad_logits must be set");
    if (l->rows && !aligned(grad, type_bytes(l->type))) return fail("grad_logits is not aligned to its type");
    if (int rc = check_workspace(l, workspace, workspace_bytes)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(workspace);
    LossArgs a = args_of(p);
    a.count_here = l->rows <= kCountHere;
    if (!a.count_here) {
        loss_count_kernel<<<1, kMostThreads, 0, s>>>(l->targets, l->rows, l->ignore_index, ws);
        if (int rc = launched("loss_count_kernel")) return rc;
        a.count = ws;
    }
    a.row_loss = ws + 64;
    a.logp = logp;
    a.past = past_caches(*l);
    a.scale = grad_scale;
    a.grad = grad;
    a.grad_stride = grad_stride;
    if (l->rows) run_rows<Of::kPolicy>(l->type, a, s);
    if (int rc = launched("loss_kernel")) return rc;
    if (a.count_here)
        loss_mean_kernel<<<1, kMostThreads, 0, s>>>(ws + 64, l->targets, l->rows, l->ignore_index, out);
    else
        loss_sum_kernel<<<1, kMostThreads, 0, s>>>(ws + 64, l->rows, ws, out);
    return launched("loss_sum_kernel");
}

extern "C" size_t isa_train_preference_workspace(const isa_train_preference* p) {
    return check(p) ? 0 : PreferenceSpace(p).bytes;
}

extern "C" int isa_train_preference_forward(const isa_train_preference* p, int reduction, float* out, float* logp,
                                            float* stats, float* slope, void* workspace, size_t workspace_bytes,
                                            void* stream) {
    if (int rc = check(p)) return rc;
    if (reduction < ISA_BLOCK_MEAN || reduction > ISA_BLOCK_NONE) return fail("unknown reduction %d", reduction);
    if (reduction == ISA_BLOCK_NONE && p->pairs == 0) return 0;
    if (!out || (p->pairs && !logp)) return fail("out and logp must be set");
    if (p->loss.rows && (stats == nullptr) != (slope == nullptr)) return fail("stats and slope go together");
    if (int rc = check_workspace(p, workspace, workspace_bytes)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    float* losses = reduction == ISA_BLOCK_NONE ? out : reinterpret_cast<float*>(ws + PreferenceSpace(p).loss);
    return run_pairs(p, stats, losses, logp, slope, reduction == ISA_BLOCK_MEAN,
                     reduction == ISA_BLOCK_NONE ? nullptr : out, ws, s);
}

extern "C" int isa_train_preference_backward(const isa_train_preference* p, int reduction, const float* stats,
                                             const float* slope, const float* grad_out, void* grad, int64_t grad_stride,
                                             void* stream) {
    if (int rc = check(p)) return rc;
    if (reduction < ISA_BLOCK_MEAN || reduction > ISA_BLOCK_NONE) return fail("unknown reduction %d", reduction);
    if (p->loss.rows == 0) return 0;
    if (!stats || !slope || !grad_out || !grad) return fail("stats, slope, grad_out and grad_logits must be set");
    if (!aligned(grad, type_bytes(p->loss.type))) return fail("grad_logits is not aligned to its type");
    return run_pairs_backward(p, stats, slope, grad_out, reduction == ISA_BLOCK_NONE,
                              reduction == ISA_BLOCK_MEAN ? 1.0f / static_cast<float>(p->pairs) : 1.0f, grad, grad_stride,
                              static_cast<hipStream_t>(stream));
}

extern "C" int isa_train_preference_with_grad(const isa_train_preference* p, float grad_scale, float* out, float* logp,
                                              void* grad, int64_t grad_stride, void* workspace, size_t workspace_bytes,
                                              void* stream) {
    if (int rc = check(p)) return rc;
    if (!out || (p->pairs && !logp) || (p->loss.rows && !grad)) return fail("out, logp and grad_logits must be set");
    if (p->loss.rows && !aligned(grad, type_bytes(p->loss.type))) return fail("grad_logits is not aligned to its type");
    if (int rc = check_workspace(p, workspace, workspace_bytes)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const PreferenceSpace at(p);
    char* ws = static_cast<char*>(workspace);
    float *stats = reinterpret_cast<float*>(ws + at.stats), *losses = reinterpret_cast<float*>(ws + at.loss),
          *slope = reinterpret_cast<float*>(ws + at.slope);
    const float scale = grad_scale / static_cast<float>(p->pairs);
    const int64_t row_bytes = p->loss.vocab * static_cast<int64_t>(type_bytes(p->loss.type));
    if (p->loss.rows && p->loss.rows <= kFewRows && p->pairs <= kFewPairs && row_bytes <= kFewBytes)
        return run_few_pairs(p, scale, stats, logp, out, grad, grad_stride, ws, s);
    if (int rc = run_pairs(p, stats, losses, logp, slope, 1, out, ws, s)) return rc;
    if (p->loss.rows == 0) return 0;
    return run_pairs_backward(p, stats, slope, nullptr, 0, scale, grad, grad_stride, s);
}
