// Attention with a sliding window and sinks, for gfx950: the forward pass.
//
//   s_ij = c q_i k_j  (c = scale log2 e),  p_ij = exp2(s_ij - lse_i) over the keys j that i sees
//   out = p v
//
// Products run on the matrix cores in 32 x 32 tiles with fp32 sums: 16-bit types as 32x32x16,
// fp32 as 32x32x2. Scores are taken as s^T = K Q^T, so a lane holds one query's scores and a
// row's maximum and sum are lane-local but for one exchange of the wave's halves; and those
// scores are, register for register, the second operand of the next product (out^T = V^T p^T),
// because the order in which a product sums its inner index is free: each half of the wave
// takes the keys that it holds. The first operand (V^T) follows that order and is read across the
// tile's rows.
//
// The rows of a product are the queries of all heads that share a key head, position by
// position, so K and V are read once for the group. A block walks the tiles of keys that any of
// its rows sees: the sinks' tiles, then the window's, while the next tile's copy to LDS runs.
// Masks are evaluated only in tiles that some row of a wave sees in part. A running sum is
// rescaled only where a score passes the last maximum by 8 powers of two: until then the weights
// are at most 256 times too large, which costs fp32 sums and both 16-bit types nothing.
//
// In 16-bit types p is rounded to the type for the product, as ds is in the backward: products of fp32 operands run
// at an eighth of the rate, and one more product for what the rounding leaves would be half as many again.
// It is taken only of sinks, which hold most of a row's weight. Against 64 bits rounded once, errors
// are 1.3 times as large for out and 1.4 to 1.5 for the gradients (300 tokens, window 64), with strong sinks 1.0
// for out and 1.1 for dq.
#include "block_attention.hpp"

namespace isa_block {
namespace {

constexpr int kCombineWaves = 4;

// A row's running softmax: base = c times a maximum, the weights' sum, and the product.
//
// `sum` is that of the weights as the product takes them, which out is divided by; `whole`, where lse is asked
// for, that of the weights as the backward makes them, from its own scores and unrounded:
//  * in 16-bit types not of the rounded ones. All of a row's p, dv and ds would be off by what its largest weight
//    was rounded by (bf16 rows with a weight of 0.97: dq 3.4e-3 off, with `whole` 2.6e-3, of which its own rounding
//    is 1.7e-3; the adding takes 4% of a training forward of 128-wide heads, nothing that shows of 64-wide ones);
//  * in fp32, where few rows' scores are four sums, of scores as one, which round as the backward's do (7 x 26 tokens
//    of 128-wide heads, weights near 1: dv 2.8e-6 off, with `whole` 1.2e-7).
template <int DB>
struct Running {
    float top = 0.0f, base = 0.0f, bound = -INFINITY, sum = 0.0f, whole = 0.0f;
    acc16 o[DB] = {};
};

constexpr float kSlack = 8.0f;

// Past it base's rounding, which all weights of a row have in them as a factor until they are divided by their
// sum, may be a power of two that passes the type's range.
constexpr float kFar = 0x1p24f;

// Weights of 32 NK keys join the running sums of their rows.
template <typename T, int D, int NK>
__device__ __forceinline__ void add_weighted(Running<D / 32>& r, const acc16 (&p)[NK], const T* vtile, int lane) {
    using L = Tile<T, D>;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int u = 0; u < L::kUses; ++u) {
            const typename Frag<T>::V f = operand<T>(p[n], u);
            r.sum = add_all(f, r.sum);
#pragma unroll
            for (int db = 0; db < D / 32; ++db) mma(r.o[db], L::column(vtile, 32 * n, u, db, lane), f);
        }
    constexpr int kProducts = NK * L::kUses * (D / 32);
    reads_ahead<kProducts * L::kColumnReads, kProducts * L::kMmas, 4 * L::kColumnReads>();
}

// What `whole` is made of.
enum Whole { kNone, kWeights, kOtherScores };

// Scores of 32 NK keys (lane: a query) join the running sums of their rows.
template <typename T, int D, int NK, Whole WHOLE>
__device__ __forceinline__ void attend(Running<D / 32>& r, acc16 (&s)[NK], const T* vtile, const AttnArgs& a, bool sinks,
                                       int lane, const acc16* others = nullptr) {
    float t = s[0][0];
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) t = fmaxf(t, s[n][i]);
    const float top = half_max(t);
    t = top * a.c;
    if (__any(t > r.bound)) {
        const bool moves = t > r.bound;
        // 1 in rows whose base stays, 0 in those that had none
        const float decay = !moves ? 1.0f : r.bound == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r.base - t);
        if (moves) {
            r.bound = t + kSlack;
            r.base = t;
            r.top = top;
        }
        r.sum *= decay;
        if constexpr (WHOLE != kNone) r.whole *= decay;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) r.o[db][i] *= decay;
    }
    float base = r.base, less = 0.0f;
    if (__any(fabsf(base) > kFar)) {  // there the scores' differences are taken first
        const bool far = fabsf(base) > kFar;
        base = far ? 0.0f : base;
        less = far ? r.top : 0.0f;
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] -= less;
    }
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = weight(s[n][i], a.c, base);
    if constexpr (WHOLE != kNone) {
        float part[4] = {};
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                part[i % 4] += WHOLE == kWeights ? s[n][i] : weight(others[n][i] - less, a.c, base);
        r.whole += (part[0] + part[1]) + (part[2] + part[3]);
    }
    add_weighted<T, D, NK>(r, s, vtile, lane);
    if (sizeof(T) == 2 && sinks) {
#pragma unroll
        for (int n = 0; n < NK; ++n) s[n] = remainder<T>(s[n]);
        add_weighted<T, D, NK>(r, s, vtile, lane);
    }
}

// Where a row's sums go: its result, or with several blocks to a tile of rows their partial sums
// [splits][rows of all heads][D + 4]: the product, base, sum, whole. A sum of 0 is that of a row that sees nothing; one
// of NaN goes on to the result.
template <typename T, int D, Whole WHOLE>
__device__ __forceinline__ void finish(Running<D / 32>& r, const AttnArgs& a, const RowAt& at, int b, int split,
                                       int lane) {
    const float sum = half_sum(r.sum), whole = WHOLE == kNone ? sum : half_sum(r.whole);
    const int64_t row = at.packed(a, b);
    if (a.splits > 1) {
        const int64_t rows = static_cast<int64_t>(a.batch) * a.queries * a.heads;
        float* p = a.partial + (split * rows + row / a.dim) * (D + 4);
        store_row<float, D / 32>(p, r.o, 1.0f, D, lane);
        if (lane < 32) {
            p[D] = sum == 0.0f ? -INFINITY : r.base;
            p[D + 1] = sum;
            p[D + 2] = whole;
        }
        return;
    }
    store_row<T, D / 32>(static_cast<T*>(a.result) + row, r.o, sum == 0.0f ? 0.0f : 1.0f / sum, a.dim, lane,
                         a.rest ? static_cast<T*>(a.rest) + row : nullptr);
    if (a.lse && lane < 32) {
        float* lse = a.lse + 2 * at.stat(a, b);
        lse[0] = sum == 0.0f ? -INFINITY : r.base;
        lse[1] = sum == 0.0f ? 0.0f : log2f(whole);
    }
}

// Waves to a SIMD that registers are to leave room for.
template <typename T, int D>
constexpr int kForwardWaves = sizeof(T) == 4 && D <= 64 ? 3 : 1;

template <typename T, int D, Whole WHOLE>
__global__ __launch_bounds__(kThreads<T>, (kForwardWaves<T, D>)) void attention_forward_kernel(AttnArgs a) {
    using L = Tile<T, D>;
    constexpr int BN = kKeyTile<T>, NK = BN / 32, kRows = isa_block::kRows<T>;
    constexpr int kSecond = kOneTile<T> ? 1 : BN * L::kPitch;
    __shared__ __attribute__((aligned(1024))) T k0[BN * L::kPitch], v0[BN * L::kPitch], k1[kSecond], v1[kSecond];
    const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), half = lane / 32;
    const int rows = a.queries * a.group, tiles = (rows + kRows - 1) / kRows;
    const Piece piece(blockIdx.x, gridDim.x, a.batch * a.kv_heads, tiles * a.splits);
    const int kv_head = piece.head % a.kv_heads, b = piece.head / a.kv_heads, split = piece.slot % a.splits;
    const int row0 = (tiles - 1 - piece.slot / a.splits) * kRows;  // rows that see the most keys first
    const int shift = length_of(a, b) - a.queries, last = min(row0 + kRows, rows) - 1;
    const Span<BN> span(a, shift + row0 / a.group, shift + last / a.group);
    const int begin = span.count * split / a.splits, end = span.count * (split + 1) / a.splits;

    const int mine = row0 + wave * kTile, row = mine + lane % 32;
    const int pmin = shift + min(mine, last) / a.group, pmax = shift + min(mine + kTile - 1, last) / a.group;
    const RowAt at(a, min(row, last), kv_head);
    const int p = shift + at.query;
    RowFrags<T, D> q;
    q.load(row <= last ? static_cast<const T*>(a.q) + at.in(a.qs, b) : nullptr, a.dim, lane);

    Running<D / 32> r;
    const Loader<T, D, BN, kThreads<T>> kload(static_cast<const T*>(a.k) + b * a.ks[0] + kv_head * a.ks[2], a.ks[1], a.dim,
                                           threadIdx.x);
    const Loader<T, D, BN, kThreads<T>> vload(static_cast<const T*>(a.v) + b * a.vs[0] + kv_head * a.vs[2], a.vs[1], a.dim,
                                           threadIdx.x);
    auto fetch_k = [&](int it, T* kt) { kload.load(kt, 0, span.first(it), span.end(it), wave); };
    auto fetch_v = [&](int it, T* vt) { vload.load(vt, 0, span.first(it), span.end(it), wave); };
    // false where no row of the wave sees a key of the tile
    auto scores = [&](int it, const T* kt, acc16(&s)[NK]) {
        const int j0 = span.first(it);
        const Sight<BN> sight(a, span, it, j0, pmin, pmax);
        if (sight.none) return false;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            s[n] = acc16{};
#pragma unroll
            for (int t = 0; t < L::kSteps; ++t) mma(s[n], L::row(kt, 32 * n, t, lane), q[t]);
        }
        reads_ahead<NK * L::kSteps, NK * L::kSteps * L::kMmas, 4>();
        if (!sight.all) {
            const Range seen(a, span.of_sinks(it), span.sink, p, j0, half);
#pragma unroll
            for (int n = 0; n < NK; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[n][i] = seen.has(32 * n + product_row(i, 0)) ? s[n][i] : -INFINITY;
        }
        return true;
    };
    if constexpr (kOneTile<T>) {  // V's copy runs beside the scores, the next K's beside V's product
        if (begin < end) fetch_k(begin, k0);
        for (int it = begin; it < end; ++it) {
            loads_arrived();
            __syncthreads();
            fetch_v(it, v0);
            acc16 s[NK];
            const bool any = scores(it, k0, s);
            loads_arrived();
            __syncthreads();
            if (it + 1 < end) fetch_k(it + 1, k0);
            if (any) attend<T, D, NK, WHOLE>(r, s, v0, a, span.of_sinks(it), lane);
        }
    } else {
        auto compute = [&](int it, const T* kt, const T* vt) {
            acc16 s[NK];
            if (scores(it, kt, s)) attend<T, D, NK, WHOLE>(r, s, vt, a, span.of_sinks(it), lane);
        };
        auto fetch = [&](int it, T* kt, T* vt) {
            fetch_k(it, kt);
            fetch_v(it, vt);
        };
        if (begin < end) fetch(begin, k0, v0);
        for (int it = begin; it < end; it += 2) {
            loads_arrived();
            __syncthreads();
            if (it + 1 < end) fetch(it + 1, k1, v1);
            compute(it, k0, v0);
            if (it + 1 >= end) break;
            loads_arrived();
            __syncthreads();
            if (it + 2 < end) fetch(it + 2, k0, v0);
            compute(it + 1, k1, v1);
        }
    }
    if (row <= last) finish<T, D, WHOLE>(r, a, at, b, split, lane);
}

// ---- few rows: tokens over a cache ---------------------------------------------------------------
// One tile holds all rows of a key head, so the work is the keys': each wave walks its own part of
// them through tiles of its own in LDS, without barriers, the next tile's copy in flight; the waves'
// sums are joined at the end, and those of several blocks by the kernel below. Bound by HBM: with
// 32 keys of 16-bit 128-wide heads a wave computes 512 cycles for 16 KB.

template <typename T, int D>
struct TokenShape {
    static constexpr int kTileBytes = kTile * Tile<T, D>::kPitch * static_cast<int>(sizeof(T));
    // two tiles each of K and V a wave, in 128 KB
    static constexpr int kWaveCount = std::min(8, (128 << 10) / (4 * kTileBytes));
    static constexpr int kThreadCount = kWaveCount * kWave;
};

template <int DB, Whole WHOLE>
__device__ __forceinline__ void put(float* to, const Running<DB>& r, int lane) {
    using F = vec<float, 4>;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            reinterpret_cast<F*>(to)[(db * 4 + i / 4) * kWave + lane] =
                F{r.o[db][i], r.o[db][i + 1], r.o[db][i + 2], r.o[db][i + 3]};
    to[DB * 16 * kWave + lane] = r.bound == -INFINITY ? -INFINITY : r.base;
    to[DB * 16 * kWave + kWave + lane] = r.sum;
    if constexpr (WHOLE != kNone) to[DB * 16 * kWave + 2 * kWave + lane] = r.whole;
}

// Joins the sums that another wave put. Where neither has a maximum they are 0, or NaN if all scores were.
template <int DB, Whole WHOLE>
__device__ __forceinline__ void join(Running<DB>& r, const float* from, int lane) {
    using F = vec<float, 4>;
    const float other = from[DB * 16 * kWave + lane], mine = r.bound == -INFINITY ? -INFINITY : r.base;
    const float top = fmaxf(mine, other);
    const float keep = mine == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mine - top);
    const float take = other == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(other - top);
    r.bound = top;
    r.base = top == -INFINITY ? 0.0f : top;
    r.sum = r.sum * keep + from[DB * 16 * kWave + kWave + lane] * take;
    if constexpr (WHOLE != kNone) r.whole = r.whole * keep + from[DB * 16 * kWave + 2 * kWave + lane] * take;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const F x = reinterpret_cast<const F*>(from)[(db * 4 + i / 4) * kWave + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[db][i + e] = r.o[db][i + e] * keep + x[e] * take;
        }
}

template <typename T, int D, Whole WHOLE>
__global__ __launch_bounds__((TokenShape<T, D>::kThreadCount)) void attention_token_kernel(AttnArgs a) {
    using L = Tile<T, D>;
    using S = TokenShape<T, D>;
    constexpr int DB = D / 32, kElements = kTile * L::kPitch, W = S::kWaveCount;
    __shared__ __attribute__((aligned(1024))) T k0[W * kElements], v0[W * kElements], k1[W * kElements], v1[W * kElements];
    const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), half = lane / 32;
    const int task = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const int kv_head = task % a.kv_heads, b = task / a.kv_heads;
    const int shift = length_of(a, b) - a.queries, last = a.queries * a.group - 1;
    const int pmin = shift, pmax = shift + a.queries - 1;
    const Span<kTile> span(a, pmin, pmax);
    const int part = split * W + wave, parts = a.splits * W;
    const int begin = static_cast<int>(static_cast<int64_t>(span.count) * part / parts);
    const int end = static_cast<int>(static_cast<int64_t>(span.count) * (part + 1) / parts);

    const int row = lane % 32;
    const RowAt at(a, min(row, last), kv_head);
    const int p = shift + at.query;
    RowFrags<T, D> q;
    q.load(row <= last ? static_cast<const T*>(a.q) + at.in(a.qs, b) : nullptr, a.dim, lane);

    Running<DB> r;
    const Loader<T, D, kTile, kWave> kload(static_cast<const T*>(a.k) + b * a.ks[0] + kv_head * a.ks[2], a.ks[1], a.dim,
                                           lane);
    const Loader<T, D, kTile, kWave> vload(static_cast<const T*>(a.v) + b * a.vs[0] + kv_head * a.vs[2], a.vs[1], a.dim,
                                           lane);
    auto fetch = [&](int it, T* kt, T* vt) {
        const int j0 = span.first(it), je = span.end(it);
        kload.load(kt, wave * S::kTileBytes, j0, je, 0);
        vload.load(vt, wave * S::kTileBytes, j0, je, 0);
    };
    auto compute = [&](int it, const T* kt, const T* vt) {
        const int j0 = span.first(it);
        const Sight<kTile> sight(a, span, it, j0, pmin, pmax);
        // fp32 scores as four sums: one chain of 64 products was most of the error of a token (12 heads of 64,
        // 516 keys: out 4.1e-7 to 7.0e-7 off, with four sums 2.1e-7 to 3.0e-7, the time is the same)
        constexpr int kSums = sizeof(T) == 4 ? 4 : 1;
        acc16 sums[kSums] = {}, s[1], chain[1] = {};
#pragma unroll
        for (int t = 0; t < L::kSteps; ++t) {
            const auto keys = L::row(kt + wave * kElements, 0, t, lane);
            mma(sums[t % kSums], keys, q[t]);
            if constexpr (WHOLE == kOtherScores) mma(chain[0], keys, q[t]);
        }
        s[0] = kSums == 4 ? (sums[0] + sums[1 % kSums]) + (sums[2 % kSums] + sums[3 % kSums]) : sums[0];
        if (!sight.all) {
            const Range seen(a, span.of_sinks(it), span.sink, p, j0, half);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool has = seen.has(product_row(i, 0));
                s[0][i] = has ? s[0][i] : -INFINITY;
                if constexpr (WHOLE == kOtherScores) chain[0][i] = has ? chain[0][i] : -INFINITY;
            }
        }
        attend<T, D, 1, WHOLE>(r, s, vt + wave * kElements, a, span.of_sinks(it), lane, chain);
    };
    if (begin < end) fetch(begin, k0, v0);
    for (int it = begin; it < end; it += 2) {
        loads_arrived();
        if (it + 1 < end) fetch(it + 1, k1, v1);
        compute(it, k0, v0);
        if (it + 1 >= end) break;
        loads_arrived();
        if (it + 2 < end) fetch(it + 2, k0, v0);
        compute(it + 1, k1, v1);
    }
    // joined by halves through the tiles' memory, a wave's sums in each of the four
    static_assert((DB * 16 + 3) * kWave * sizeof(float) <= sizeof(k0) && W <= 8);
    auto place = [&](int n) { return reinterpret_cast<float*>(n == 0 ? k0 : n == 1 ? v0 : n == 2 ? k1 : v1); };
    __syncthreads();
#pragma unroll
    for (int n = W / 2; n >= 1; n /= 2) {
        if (wave >= n && wave < 2 * n) put<DB, WHOLE>(place(wave - n), r, lane);
        __syncthreads();
        if (wave < n) join<DB, WHOLE>(r, place(wave), lane);
        __syncthreads();
    }
    if (wave == 0 && row <= last) finish<T, D, WHOLE>(r, a, at, b, split, lane);
}

// Rows from the partial sums of `splits` blocks (at most 64): a wave each, a lane for a block's sum.
template <typename T, int D>
__global__ __launch_bounds__(kCombineWaves * kWave) void attention_combine_kernel(AttnArgs a) {
    const int lane = threadIdx.x % kWave;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.queries * a.heads;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kCombineWaves + threadIdx.x / kWave;
    if (row >= rows) return;
    const float* p = a.partial + row * (D + 4);
    const int64_t step = rows * (D + 4);
    const bool have = lane < a.splits;
    const float base = have ? p[lane * step + D] : -INFINITY, part = have ? p[lane * step + D + 1] : 0.0f;
    const float top = wave_max(base);
    const float mine = base == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(base - top);
    const float sum = wave_sum(part * mine);
    constexpr int E = (D + 63) / 64;
    float o[E] = {};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), s));
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e * 64 + lane < a.dim) o[e] = fmaf(p[s * step + e * 64 + lane], f, o[e]);
    }
    const float factor = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e * 64 + lane < a.dim) {
            const float x = o[e] * factor;
            const T y = static_cast<T>(x);
            static_cast<T*>(a.result)[row * a.dim + e * 64 + lane] = y;
            if (a.rest) static_cast<T*>(a.rest)[row * a.dim + e * 64 + lane] = static_cast<T>(x - static_cast<float>(y));
        }
    const float whole = a.lse ? wave_sum(have ? p[lane * step + D + 2] * mine : 0.0f) : 0.0f;
    if (a.lse && lane == 0) {
        const int64_t token = row / a.heads;
        float* lse = a.lse + 2 * ((token / a.queries * a.heads + row % a.heads) * a.queries + token % a.queries);
        lse[0] = top;
        lse[1] = sum == 0.0f ? 0.0f : log2f(whole);
    }
}

// ---- host -----------------------------------------------------------------------------------------

constexpr int kComputeUnits = 256;

// One tile holds all rows of a key head.
bool few_rows(const isa_block_attention* t) { return t->queries * (t->heads / t->kv_heads) <= kTile; }

// Blocks that share a tile of rows: where the tiles alone leave compute units idle, as many as fill
// them (twice, of the kernel of which two share a unit), each wave or block with a tile of keys or two.
int splits_of(const isa_block_attention* t) {
    const bool few = few_rows(t);
    const int64_t group = t->heads / t->kv_heads, tile_rows = few ? kTile : t->type == ISA_BLOCK_F32 ? kRows<float> : kRows<bf16>;
    const int64_t tasks = ceil_div(t->queries * group, tile_rows) * t->batch * t->kv_heads;
    if (tasks == 0 || tasks >= kComputeUnits) return 1;
    const int64_t rows = std::min<int64_t>(t->queries, ceil_div(tile_rows, group) + 1);
    const int64_t seen = t->window ? std::min(t->keys, t->window + rows + t->sinks) : t->keys;
    int64_t least = 2 * (t->type == ISA_BLOCK_F32 ? 32 : 64), want = 2 * kComputeUnits / tasks;
    if (few) {
        int waves = 0;
        for_type(t->type, static_cast<int>(t->head_dim), [&](auto type, auto dim) {
            waves = TokenShape<decltype(type), decltype(dim)::value>::kWaveCount;
        });
        least = kTile * waves;
        want = ceil_div(kComputeUnits, tasks);
    }
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, seen / least, 64})));
}

int padded_dim(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }

}  // namespace

bool strided(const void* p, const int64_t (&s)[3], int64_t tokens, int64_t dim, size_t bytes) {
    // a tile's rows are told apart, and its last one's end from memory, by 32-bit offsets
    if (tokens > 1 && (s[1] < dim || s[1] * static_cast<int64_t>(bytes) > (INT_MAX >> 7))) return false;
    return aligned(p, 16) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
}

int check_attention(const isa_block_attention* t) {
    if (!t) return fail("attention is null");
    if (!known_type(t->type)) return fail("unknown element type %d", t->type);
    for (int64_t n : {t->batch, t->queries, t->keys, t->heads, t->kv_heads, t->window, t->sinks})
        if (n < 0 || n > kMaxLength)
            return fail("sizes must be 0 to %d, got %lld", kMaxLength, static_cast<long long>(n));
    if (t->kv_heads < 1 || t->heads < 1 || t->heads % t->kv_heads)
        return fail("heads (%lld) must be a multiple of kv_heads (%lld)", static_cast<long long>(t->heads),
                    static_cast<long long>(t->kv_heads));
    if (t->head_dim < 8 || t->head_dim > ISA_BLOCK_ATTENTION_MAX_DIM || t->head_dim % 8)
        return fail("head_dim must be a multiple of 8 up to %d, got %lld", ISA_BLOCK_ATTENTION_MAX_DIM,
                    static_cast<long long>(t->head_dim));
    if (!(t->scale > 0.0f) || t->scale > 1e30f) return fail("scale must be positive and finite");
    // a block of a launch takes at least 16 rows or keys of a head
    const int64_t most = std::max(t->queries, t->keys) / 16 + 1;
    if (t->batch * t->heads > kMaxLength || t->batch * t->heads * most > INT_MAX ||
        t->queries * (t->heads / t->kv_heads) > kMaxLength)
        return fail("too many rows for one launch");
    if (t->batch && t->queries && !t->q) return fail("q is null");
    if (t->batch && t->keys && (!t->k || !t->v)) return fail("k and v must be set");
    const size_t bytes = type_bytes(t->type);
    if (!strided(t->q, t->q_strides, t->queries, t->head_dim, bytes) ||
        !strided(t->k, t->k_strides, t->keys, t->head_dim, bytes) ||
        !strided(t->v, t->v_strides, t->keys, t->head_dim, bytes))
        return fail("q, k and v must be 16-byte aligned, their strides multiples of 8 elements, those of tokens at "
                    "least head_dim and under 16 MiB");
    return 0;
}

AttnArgs attention_args(const isa_block_attention* t) {
    AttnArgs a{};
    a.q = t->q;
    a.k = t->k;
    a.v = t->v;
    a.lengths = t->key_lengths;
    std::copy(t->q_strides, t->q_strides + 3, a.qs);
    std::copy(t->k_strides, t->k_strides + 3, a.ks);
    std::copy(t->v_strides, t->v_strides + 3, a.vs);
    a.batch = static_cast<int>(t->batch);
    a.queries = static_cast<int>(t->queries);
    a.keys = static_cast<int>(t->keys);
    a.heads = static_cast<int>(t->heads);
    a.kv_heads = static_cast<int>(t->kv_heads);
    a.group = a.heads / a.kv_heads;
    a.dim = static_cast<int>(t->head_dim);
    a.window = t->window ? static_cast<int>(t->window) : kMaxLength;
    a.sinks = t->window ? static_cast<int>(t->sinks) : 0;  // all keys are in the window
    a.scale = t->scale;
    a.c = static_cast<float>(static_cast<double>(t->scale) * 1.44269504088896340736);
    a.splits = 1;
    // a single token's stride says nothing
    if (t->keys <= 1) a.ks[1] = a.vs[1] = t->head_dim;
    if (t->queries <= 1) a.qs[1] = t->head_dim;
    return a;
}

}  // namespace isa_block

using namespace isa_block;

extern "C" size_t isa_block_attention_forward_workspace(const isa_block_attention* t) {
    if (!t || check_attention(t)) return 0;
    const int splits = splits_of(t);
    if (splits == 1) return 0;
    return static_cast<size_t>(splits) * t->batch * t->queries * t->heads * (padded_dim(t->head_dim) + 4) *
           sizeof(float);
}

extern "C" int isa_block_attention_forward(const isa_block_attention* t, void* out, void* rest, float* lse,
                                           void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_attention(t)) return rc;
    if (t->batch == 0 || t->queries == 0) return 0;
    if (!out || !aligned(out, 16) || !aligned(rest, 16)) return fail("out must be set, it and rest 16-byte aligned");
    const size_t need = isa_block_attention_forward_workspace(t);
    if (workspace_bytes < need) return fail("workspace too small: %zu bytes", workspace_bytes);
    if (need && (!workspace || !aligned(workspace, 256))) return fail("workspace must be 256-byte aligned");
    AttnArgs a = attention_args(t);
    a.result = out;
    a.rest = rest;
    a.lse = lse;
    a.partial = static_cast<float*>(workspace);
    a.splits = splits_of(t);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    for_type(t->type, a.dim, [&](auto type, auto dim) {
        using T = decltype(type);
        constexpr int D = decltype(dim)::value;
        const int64_t tiles = few_rows(t) ? 1 : ceil_div(static_cast<int64_t>(a.queries) * a.group, kRows<T>);
        const dim3 blocks(static_cast<unsigned>(tiles * a.batch * a.kv_heads * a.splits));
        const auto launch = [&](auto kernel, int threads) { kernel<<<blocks, threads, 0, s>>>(a); };
        constexpr Whole kTokens = sizeof(T) == 4 ? kOtherScores : kWeights, kRowsOf = sizeof(T) == 4 ? kNone : kWeights;
        if (few_rows(t))
            launch(a.lse ? attention_token_kernel<T, D, kTokens> : attention_token_kernel<T, D, kNone>,
                   TokenShape<T, D>::kThreadCount);
        else
            launch(a.lse ? attention_forward_kernel<T, D, kRowsOf> : attention_forward_kernel<T, D, kNone>, kThreads<T>);
        if (a.splits > 1) {
            const int64_t rows = static_cast<int64_t>(a.batch) * a.queries * a.heads;
            attention_combine_kernel<T, D>
                <<<dim3(static_cast<unsigned>(ceil_div(rows, kCombineWaves))), kCombineWaves * kWave, 0, s>>>(a);
        }
    });
    return launched("the attention's forward");
}
