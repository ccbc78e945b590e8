// Attention with a sliding window and sinks, for gfx950: the backward pass (block_attention.hip has
// the forward's layout of products, which is used here too).
//
//   delta_i = do_i out_i,  p = exp2(c q k - lse),  dp = do v^T,  ds = p (dp - delta)
//   dv = p^T do,  dk = scale ds^T q,  dq = scale ds k
//
// Two walks, each of which recomputes p and dp from what it needs anyway, so that no sum crosses
// blocks in an order that changes: dq's over the keys that a tile of rows sees, dk's and dv's over
// the queries that see a tile of keys, head by head of those that share the key head.
// 7 products instead of the 5 that one walk with atomic sums of dq would take.
#include "block_attention.hpp"

namespace isa_block {
namespace {

constexpr int kRowThreads = 256;

// What both walks read of a row beside q and do, in planes of the workspace: delta, and lse as one
// float (16-bit types) or as two (fp32, where its rounding alone would be an error of the size of
// all others together).
enum Plane { kDelta = 0, kLse = 1, kLseRest = 2, kPlanes = 3 };

__device__ __forceinline__ int64_t plane_rows(const AttnArgs& a) {
    return (static_cast<int64_t>(a.batch) * a.heads * a.queries + 63) / 64 * 64;
}

template <typename T>
__device__ __forceinline__ void put_planes(const AttnArgs& a, int64_t at, float delta, float base, float log_sum) {
    const int64_t plane = plane_rows(a);
    a.delta[kDelta * plane + at] = delta;
    a.delta[kLse * plane + at] = sizeof(T) == 4 ? base : base + log_sum;
    if (sizeof(T) == 4) a.delta[kLseRest * plane + at] = log_sum;
}

// delta = rows' do . out, 16 threads a row, where no dq is asked for, whose kernel does it on its way.
// Where one weight is close to 1, its key's dp is close to delta and ds is their difference: out's own
// rounding would be most of it, so a 16-bit out comes with what that left.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void attention_rows_kernel(AttnArgs a) {
    const int64_t r = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) / 16;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.queries * a.heads;
    const int c = threadIdx.x % 16 * 8;
    float s = 0.0f;
    const int head = static_cast<int>(r % a.heads);
    const int64_t token = r / a.heads, b = token / a.queries, i = token % a.queries;
    if (r < rows && c < a.dim) {
        const Pack<T, 8> x = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.out) + r * a.dim + c);
        const Pack<T, 8> y = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.dout) + b * a.gs[0] +
                                                                  i * a.gs[1] + head * a.gs[2] + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(static_cast<float>(x.v[e]), static_cast<float>(y.v[e]), s);
        if (a.rest) {
            const Pack<T, 8> z = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.rest) + r * a.dim + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(static_cast<float>(z.v[e]), static_cast<float>(y.v[e]), s);
        }
    }
    s += dpp<0xB1>(s);
    s += dpp<0x4E>(s);
    s += dpp<0x141>(s);
    s += dpp<0x140>(s);
    if (r >= rows || threadIdx.x % 16 != 0) return;
    const int64_t at = (b * a.heads + head) * a.queries + i;
    put_planes<T>(a, at, s, a.lse[2 * at], a.lse[2 * at + 1]);
}

template <typename T, int D>
__device__ __forceinline__ float dot(const RowFrags<T, D>& x, const RowFrags<T, D>& y, float sum) {
#pragma unroll
    for (int t = 0; t < Tile<T, D>::kSteps; ++t)
#pragma unroll
        for (int e = 0; e < Frag<T>::N; ++e)
            sum = fmaf(static_cast<float>(x[t][e]), static_cast<float>(y[t][e]), sum);
    return sum;
}

// fp16 has 5 bits of exponent: gradients of a mean loss, some 1e-5, would leave ds a few bits, and values of some
// 1000 could take it past the range. A lane's ds belong to one row (dq) or one key (dk), and so do its sums of
// them times the other operand: both are held times a power of two that brings the largest ds so far
// to between 1 and kMostDs, so that rows' and keys' sizes do not meet. (2 x 4096 tokens, 16 heads on 4 of 128,
// window 1024: dq 128 us, dk and dv 165, as bf16 without a scale takes.)
template <typename T>
constexpr bool kScaled = std::is_same_v<T, f16>;
constexpr float kFirstFactor = 0x1p126f;  // of a lane that has seen no ds (past 2^-113)
constexpr float kMostDs = 0x1p13f;

__device__ __forceinline__ float to_one(float peak) {
    const int e = static_cast<int>(__float_as_uint(peak) >> 23);  // (peak is not negative)
    return e < 1 || e > 253 ? 1.0f : __uint_as_float(static_cast<unsigned>(254 - e) << 23);
}

template <int DB>
__device__ __forceinline__ void scale_to_one(acc16& ds, float& factor, acc16 (&sums)[DB]) {
    float peak = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) peak = fmaxf(peak, fabsf(ds[i]));
    peak = half_max(peak);
    if (__any(peak * factor > kMostDs)) {
        const float next = peak * factor > kMostDs ? to_one(peak) : factor, change = next / factor;
        factor = next;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[db][i] *= change;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) ds[i] *= factor;
}

template <typename T>
__device__ __forceinline__ float probability(float s, const AttnArgs& a, float lse, float lse_rest) {
    const float x = fmaf(s, a.c, -lse);
    return __builtin_amdgcn_exp2f(sizeof(T) == 4 ? x - lse_rest : x);
}

// Two waves to a SIMD, so that one's products run beside the other's softmax, where 256 registers hold
// a wave's operands and sums; three where 168 do (dk and dv of fp16 heads of 64, 8 x 1024 tokens without a
// window: 47 us against 54).
template <typename T, int D>
constexpr int kDqWaves = sizeof(T) == 2 || D <= 64 ? 2 : 1;
template <typename T, int D>
constexpr int kDkvWaves = sizeof(T) == 2 ? (D <= 64 ? 3 : 2) : D <= 64 ? 2 : 1;

template <typename T, int D>
__global__ __launch_bounds__(kThreads<T>, (kDqWaves<T, D>)) void attention_dq_kernel(AttnArgs a) {
    using L = Tile<T, D>;
    constexpr int BN = kKeyTile<T>, DB = D / 32, kRows = isa_block::kRows<T>;
    __shared__ __attribute__((aligned(1024))) T k0[BN * L::kPitch], v0[BN * L::kPitch], k1[BN * L::kPitch],
        v1[BN * L::kPitch];
    const int lane = threadIdx.x % kWave, wave = uniform(threadIdx.x / kWave), half = lane / 32;
    const int rows = a.queries * a.group, tiles = (rows + kRows - 1) / kRows;
    const Piece piece(blockIdx.x, gridDim.x, a.batch * a.kv_heads, tiles);
    const int kv_head = piece.head % a.kv_heads, b = piece.head / a.kv_heads;
    const int row0 = (tiles - 1 - piece.slot) * kRows;
    const int shift = length_of(a, b) - a.queries, last = min(row0 + kRows, rows) - 1;
    const Span<BN> span(a, shift + row0 / a.group, shift + last / a.group);

    const int mine = row0 + wave * kTile, row = mine + lane % 32;
    const int pmin = shift + min(mine, last) / a.group, pmax = shift + min(mine + kTile - 1, last) / a.group;
    const RowAt at(a, min(row, last), kv_head);
    const int p = shift + at.query;
    RowFrags<T, D> q, g;
    q.load(row <= last ? static_cast<const T*>(a.q) + at.in(a.qs, b) : nullptr, a.dim, lane);
    g.load(row <= last ? static_cast<const T*>(a.dout) + at.in(a.gs, b) : nullptr, a.dim, lane);
    float delta = 0.0f;
    {
        RowFrags<T, D> o;
        o.load(row <= last ? static_cast<const T*>(a.out) + at.packed(a, b) : nullptr, a.dim, lane);
        delta = dot<T, D>(o, g, delta);
        if (a.rest) {
            o.load(row <= last ? static_cast<const T*>(a.rest) + at.packed(a, b) : nullptr, a.dim, lane);
            delta = dot<T, D>(o, g, delta);
        }
        delta = half_sum(delta);
    }
    const int64_t stat = at.stat(a, b);
    const float base = a.lse[2 * stat], log_sum = a.lse[2 * stat + 1];
    const float lse = sizeof(T) == 4 ? base : base + log_sum, lse_rest = log_sum;
    if (row <= last && lane < 32) put_planes<T>(a, stat, delta, base, log_sum);
    float factor = kScaled<T> ? kFirstFactor : 1.0f;
    acc16 dq[DB] = {};
    const Loader<T, D, BN, kThreads<T>> kload(static_cast<const T*>(a.k) + b * a.ks[0] + kv_head * a.ks[2], a.ks[1], a.dim,
                                           threadIdx.x);
    const Loader<T, D, BN, kThreads<T>> vload(static_cast<const T*>(a.v) + b * a.vs[0] + kv_head * a.vs[2], a.vs[1], a.dim,
                                           threadIdx.x);
    auto fetch = [&](int it, T* kt, T* vt) {
        const int j0 = span.first(it), je = span.end(it);
        kload.load(kt, 0, j0, je, wave);
        vload.load(vt, 0, j0, je, wave);
    };
    auto compute = [&](int it, const T* kt, const T* vt) {
        const int j0 = span.first(it);
        const Sight<BN> sight(a, span, it, j0, pmin, pmax);
        if (sight.none) return;
#pragma unroll
        for (int n = 0; n < BN / 32; ++n) {
            acc16 s = {}, d = {};
#pragma unroll
            for (int t = 0; t < L::kSteps; ++t) {
                mma(s, L::row(kt, 32 * n, t, lane), q[t]);
                mma(d, L::row(vt, 32 * n, t, lane), g[t]);
            }
            reads_ahead<2 * L::kSteps, 2 * L::kSteps * L::kMmas, 4>();
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = probability<T>(s[i], a, lse, lse_rest) * (d[i] - delta);
            if (!sight.all) {
                const Range seen(a, span.of_sinks(it), span.sink, p, j0, half);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = seen.has(32 * n + product_row(i, 0)) ? s[i] : 0.0f;
            }
            if constexpr (kScaled<T>) scale_to_one(s, factor, dq);
#pragma unroll
            for (int u = 0; u < L::kUses; ++u) {
                const typename Frag<T>::V f = operand<T>(s, u);
#pragma unroll
                for (int db = 0; db < DB; ++db) mma(dq[db], L::column(kt, 32 * n, u, db, lane), f);
            }
            reads_ahead<L::kUses * DB * L::kColumnReads, L::kUses * DB * L::kMmas, 4 * L::kColumnReads>();
            if (sizeof(T) == 2 && span.of_sinks(it)) {
                s = remainder<T>(s);
#pragma unroll
                for (int u = 0; u < L::kUses; ++u) {
                    const typename Frag<T>::V f = operand<T>(s, u);
#pragma unroll
                    for (int db = 0; db < DB; ++db) mma(dq[db], L::column(kt, 32 * n, u, db, lane), f);
                }
            }
        }
    };
    if (span.count) fetch(0, k0, v0);
    for (int it = 0; it < span.count; it += 2) {
        loads_arrived();
        __syncthreads();
        if (it + 1 < span.count) fetch(it + 1, k1, v1);
        compute(it, k0, v0);
        if (it + 1 >= span.count) break;
        loads_arrived();
        __syncthreads();
        if (it + 2 < span.count) fetch(it + 2, k0, v0);
        compute(it + 1, k1, v1);
    }
    if (row <= last) store_row<T, DB>(static_cast<T*>(a.result) + at.packed(a, b), dq, a.scale / factor, a.dim, lane);
}

// ---- dk and dv ------------------------------------------------------------------------------
// A block takes kKeys keys of a key head, a wave 32 of them, and walks the tiles of BR queries of
// each head that see one of the keys. The blocks of one tile of keys, if several, take equal parts
// of that walk and leave partial sums.

template <typename T, int D>
struct DkvShape {
    static constexpr int kWaveCount = sizeof(T) == 4 ? 1 : 4;
    static constexpr int kKeys = kWaveCount * 32, kThreadCount = kWaveCount * kWave;
    // 16-bit rows of 128: V waits in LDS instead of in registers, and tiles of 32 queries leave room for
    // it, so that two blocks still share a compute unit
    static constexpr bool kHoldV = !(sizeof(T) == 2 && D == 128);
    static constexpr int BR = kHoldV ? kKeyTile<T> : 32;
};

// Pieces of a key head's tiles that are cut, of which `plain` hold no sinks: those first.
__device__ __forceinline__ int pieces_per_head(const AttnArgs& a, int plain) {
    return (a.near > 1 ? plain * a.near : 0) + (a.far > 1 ? a.far_tiles * a.far : 0);
}

// The queries first .. end - 1 that see one of the keys j0 .. j1 - 1.
struct Seen {
    int first, end;
    __device__ __forceinline__ Seen(const AttnArgs& a, int length, int j0, int j1) {
        const int shift = length - a.queries;
        const int64_t reach = static_cast<int64_t>(min(j1, length)) - 1 + a.window - 1;
        const int plast = j0 < a.sinks || reach > length - 1 ? length - 1 : static_cast<int>(reach);
        first = max(0, j0 - shift);
        end = j0 < length ? max(first, plast - shift + 1) : first;
    }
};

template <typename T, int D>
__global__ __launch_bounds__((DkvShape<T, D>::kThreadCount), (kDkvWaves<T, D>)) void attention_dkv_kernel(AttnArgs a) {
    using L = Tile<T, D>;
    using S = DkvShape<T, D>;
    constexpr int BR = S::BR, DB = D / 32;
    constexpr int kSecond = kOneTile<T> ? 1 : BR * L::kPitch;
    __shared__ __attribute__((aligned(1024))) T q0[BR * L::kPitch], g0[BR * L::kPitch], q1[kSecond], g1[kSecond];
    __shared__ __attribute__((aligned(1024))) float stat0[kPlanes * 64], stat1[kOneTile<T> ? 1 : kPlanes * 64];
    const int outer = threadIdx.x % kWave, lane = outer, wave = uniform(threadIdx.x / kWave);
    const int tiles = (a.keys + S::kKeys - 1) / S::kKeys;
    // a key head's blocks: those of the tiles without sinks, then those of the tiles with
    const int plain = tiles - a.far_tiles, per_head = plain * a.near + a.far_tiles * a.far;
    const Piece piece(blockIdx.x, gridDim.x, a.batch * a.kv_heads, per_head);
    const int kv_head = piece.head % a.kv_heads, b = piece.head / a.kv_heads, slot = piece.slot;
    const bool far = slot >= plain * a.near;
    const int splits = far ? a.far : a.near, in = far ? slot - plain * a.near : slot;
    const int tile = (far ? 0 : a.far_tiles) + in / splits, split = in % splits;
    const int j0 = tile * S::kKeys, length = length_of(a, b), shift = length - a.queries;

    const int mine = j0 + wave * 32;
    __shared__ __attribute__((aligned(1024))) T held[S::kHoldV ? 1 : S::kKeys * L::kPitch];
    if constexpr (!S::kHoldV) {
        const Loader<T, D, S::kKeys, S::kThreadCount> vload(
            static_cast<const T*>(a.v) + b * a.vs[0] + kv_head * a.vs[2], a.vs[1], a.dim, threadIdx.x);
        vload.load(held, 0, j0, length, wave);
    }
    RowFrags<T, D> k, v;
    const int key = mine + lane % 32;
    k.load(key < length ? static_cast<const T*>(a.k) + b * a.ks[0] + kv_head * a.ks[2] + key * a.ks[1] : nullptr, a.dim, lane);
    if constexpr (S::kHoldV)
        v.load(key < length ? static_cast<const T*>(a.v) + b * a.vs[0] + kv_head * a.vs[2] + key * a.vs[1] : nullptr, a.dim,
               lane);
    float factor = kScaled<T> ? kFirstFactor : 1.0f;
    const Seen seen(a, length, j0, j0 + S::kKeys);
    const int turns = (seen.end - seen.first + BR - 1) / BR, all_turns = turns * a.group;
    const int begin = static_cast<int>(static_cast<int64_t>(all_turns) * split / splits);
    const int end = static_cast<int>(static_cast<int64_t>(all_turns) * (split + 1) / splits);

    acc16 dk[DB] = {}, dv[DB] = {};
    const int64_t plane = plane_rows(a);
    const Loader<T, D, BR, S::kThreadCount> qload(
        static_cast<const T*>(a.q) + b * a.qs[0] + static_cast<int64_t>(kv_head) * a.group * a.qs[2], a.qs[1], a.dim,
        threadIdx.x);
    const Loader<T, D, BR, S::kThreadCount> gload(
        static_cast<const T*>(a.dout) + b * a.gs[0] + static_cast<int64_t>(kv_head) * a.group * a.gs[2], a.gs[1], a.dim,
        threadIdx.x);
    const float* stats = a.delta + (static_cast<int64_t>(b) * a.heads + kv_head * a.group) * a.queries;
    auto fetch_q = [&](int it, T* qt, float* stat) {
        const int head = it / turns, i0 = seen.first + (it - head * turns) * BR;
        const int64_t from = (head * a.qs[2] + i0 * a.qs[1]) * static_cast<int64_t>(sizeof(T));
        qload.load_from(qt, 0, qload.base + from, seen.end - i0, wave);
        const int64_t at = static_cast<int64_t>(head) * a.queries + i0;
#pragma unroll
        for (int n = 0; n < (sizeof(T) == 4 ? 3 : 2); ++n)
            if (n % S::kWaveCount == wave) load_floats(stat, 64 * n, stats + n * plane, at, seen.end - i0, lane);
    };
    auto fetch_g = [&](int it, T* gt) {
        const int head = it / turns, i0 = seen.first + (it - head * turns) * BR;
        const int64_t from = (head * a.gs[2] + i0 * a.gs[1]) * static_cast<int64_t>(sizeof(T));
        gload.load_from(gt, 0, gload.base + from, seen.end - i0, wave);
    };
    // s = p and d = ds of 32 queries and 32 keys; false where none of them sees any
    auto gradients = [&](int it, int r, const T* qt, const T* gt, const float* stat, acc16& s, acc16& d, int lane) {
        const int half = lane / 32, i0 = seen.first + it % turns * BR;
        const int pmin = shift + i0, pmax = shift + min(i0 + BR, seen.end) - 1;
        const int key = mine + lane % 32, plo = pmin + 32 * r, phi = min(plo + 31, pmax);
        if (mine > phi || (mine + 31 <= plo - a.window && mine >= a.sinks)) return false;
        const bool all = mine + 31 <= plo && (mine + 32 <= a.sinks || mine > phi - a.window);
        s = acc16{};
        d = acc16{};
#pragma unroll
        for (int t = 0; t < L::kSteps; ++t) {
            mma(s, L::row(qt, 32 * r, t, lane), k[t]);
            mma(d, L::row(gt, 32 * r, t, lane), S::kHoldV ? v[t] : L::row(held, wave * 32, t, lane));
        }
        reads_ahead<(S::kHoldV ? 2 : 3) * L::kSteps, 2 * L::kSteps * L::kMmas, 4>();
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int at = 32 * r + product_row(i, half);
            using F = vec<float, 4>;
            const F delta = *reinterpret_cast<const F*>(stat + 64 * kDelta + at);
            const F lse = *reinterpret_cast<const F*>(stat + 64 * kLse + at);
            F rest{};
            if constexpr (sizeof(T) == 4) rest = *reinterpret_cast<const F*>(stat + 64 * kLseRest + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i + e] = probability<T>(s[i + e], a, lse[e], rest[e]);
                d[i + e] = s[i + e] * (d[i + e] - delta[e]);
            }
        }
        if (!all) {
            // queries at key .. key + window - 1 see it, of a sink all from it on
            const int from = key - pmin - 32 * r - 4 * half;
            const unsigned count = key < a.sinks ? INT_MAX : a.window;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool seen = static_cast<unsigned>(product_row(i, 0) - from) < count;
                s[i] = seen ? s[i] : 0.0f;
                d[i] = seen ? d[i] : 0.0f;
            }
        }
        if constexpr (kScaled<T>) scale_to_one(d, factor, dk);
        return true;
    };
    if constexpr (kOneTile<T>) {  // Q's tile is free after dk, dO's after dv
        static_assert(BR == kTile);
        auto add = [&](acc16(&sum)[DB], const T* tile, const acc16& x, int lane) {
#pragma unroll
            for (int u = 0; u < L::kUses; ++u) {
                const typename Frag<T>::V f = operand<T>(x, u);
#pragma unroll
                for (int db = 0; db < DB; ++db) mma(sum[db], L::column(tile, 0, u, db, lane), f);
            }
            reads_ahead<L::kUses * DB * L::kColumnReads, L::kUses * DB * L::kMmas, 4 * L::kColumnReads>();
        };
        if (begin < end) {
            fetch_q(begin, q0, stat0);
            fetch_g(begin, g0);
        }
        for (int it = begin; it < end; ++it) {
            loads_arrived();
            __syncthreads();
            const int lane = opaque(outer);
            acc16 s, d;
            const bool any = gradients(it, 0, q0, g0, stat0, s, d, lane);
            if (any) add(dk, q0, d, lane);
            __syncthreads();
            if (it + 1 < end) fetch_q(it + 1, q0, stat0);
            if (any) add(dv, g0, s, lane);
            __syncthreads();
            if (it + 1 < end) fetch_g(it + 1, g0);
        }
    } else {
        auto fetch = [&](int it, T* qt, T* gt, float* stat) {
            fetch_q(it, qt, stat);
            fetch_g(it, gt);
        };
        auto compute = [&](int it, const T* qt, const T* gt, const float* stat) {
            const int lane = opaque(outer);
#pragma unroll
            for (int r = 0; r < BR / 32; ++r) {
                acc16 s, d;
                if (!gradients(it, r, qt, gt, stat, s, d, lane)) continue;
#pragma unroll
                for (int u = 0; u < L::kUses; ++u) {
                    const typename Frag<T>::V f = operand<T>(s, u), h = operand<T>(d, u);
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        mma(dv[db], L::column(gt, 32 * r, u, db, lane), f);
                        mma(dk[db], L::column(qt, 32 * r, u, db, lane), h);
                    }
                }
                reads_ahead<2 * L::kUses * DB * L::kColumnReads, 2 * L::kUses * DB * L::kMmas, 4 * L::kColumnReads>();
            }
        };
        if (begin < end) fetch(begin, q0, g0, stat0);
        for (int it = begin; it < end; it += 2) {
            loads_arrived();
            __syncthreads();
            if (it + 1 < end) fetch(it + 1, q1, g1, stat1);
            compute(it, q0, g0, stat0);
            if (it + 1 >= end) break;
            loads_arrived();
            __syncthreads();
            if (it + 2 < end) fetch(it + 2, q0, g0, stat0);
            compute(it + 1, q1, g1, stat1);
        }
    }
    if (splits > 1) {  // [piece of a cut tile][dk, dv][dims' quarter of 32][thread]
        const int64_t mine_at = (static_cast<int64_t>(b) * a.kv_heads + kv_head) * pieces_per_head(a, plain) +
                                (far && a.near > 1 ? plain * a.near : 0) + in;
        float* p = a.partial + mine_at * (2 * S::kKeys * D) + threadIdx.x * 4;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int at = (db * 4 + i / 4) * S::kThreadCount * 4;
                using F = vec<float, 4>;
                *reinterpret_cast<F*>(p + at) = F{dk[db][i], dk[db][i + 1], dk[db][i + 2], dk[db][i + 3]} * (1.0f / factor);
                *reinterpret_cast<F*>(p + S::kKeys * D + at) = F{dv[db][i], dv[db][i + 1], dv[db][i + 2], dv[db][i + 3]};
            }
        return;
    }
    if (key >= a.keys) return;
    const int64_t out = ((static_cast<int64_t>(b) * a.keys + key) * a.kv_heads + kv_head) * a.dim;
    store_row<T, DB>(static_cast<T*>(a.dk) + out, dk, a.scale / factor, a.dim, lane);
    store_row<T, DB>(static_cast<T*>(a.dv) + out, dv, 1.0f, a.dim, lane);
}

// The partial sums of a tile's blocks, added in their order: a block takes 4 dims of each key.
template <typename T, int D>
__global__ __launch_bounds__((DkvShape<T, D>::kThreadCount)) void attention_dkv_sum_kernel(AttnArgs a) {
    using S = DkvShape<T, D>;
    using F = vec<float, 4>;
    constexpr int kQuads = D / 8;
    const int tiles = (a.keys + S::kKeys - 1) / S::kKeys, plain = tiles - a.far_tiles;
    const int quad = blockIdx.x % kQuads, which = blockIdx.x / kQuads % 2, task = blockIdx.x / kQuads / 2;
    const int summed = (a.near > 1 ? plain : 0) + (a.far > 1 ? a.far_tiles : 0);
    const int t = task % summed, head = task / summed;  // head: of all batches
    const bool far = a.near == 1 || t >= plain;
    const int in = far && a.near > 1 ? t - plain : t, splits = far ? a.far : a.near;
    const int tile = (far ? 0 : a.far_tiles) + in;
    const int64_t slot = static_cast<int64_t>(head) * pieces_per_head(a, plain) +
                         (far && a.near > 1 ? plain * a.near : 0) + in * splits;
    const F* p = reinterpret_cast<const F*>(a.partial + slot * (2 * S::kKeys * D) + which * S::kKeys * D) +
                 quad * S::kThreadCount + threadIdx.x;
    F x{};
#pragma unroll 8
    for (int s = 0; s < splits; ++s) x += p[static_cast<int64_t>(s) * (S::kKeys * D / 2)];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int dims = quad * 8 + lane / 32 * 4, key = tile * S::kKeys + wave * 32 + lane % 32;
    if (key >= a.keys || dims >= a.dim) return;
    const int64_t out = ((static_cast<int64_t>(head / a.kv_heads) * a.keys + key) * a.kv_heads + head % a.kv_heads) * a.dim;
    Pack<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.v[e] = static_cast<T>(x[e] * (which ? 1.0f : a.scale));
    *reinterpret_cast<Pack<T, 4>*>(static_cast<T*>(which ? a.dv : a.dk) + out + dims) = y;
}

// ---- host -----------------------------------------------------------------------------------------

constexpr int kComputeUnits = 256;

// How the walks over queries are cut. A tile of keys without sinks is seen by the queries of a
// window, one with sinks by all that follow, which may be many times more: those are cut to a quarter
// of the others' length, so that they fill what those leave. Others are cut where they are fewer than
// one and a half to a compute unit, which two share (248 blocks of 128-wide bf16 heads, 2 x 4096
// tokens: 235 us whole, 189 in halves and 27 to add those). Without a window their lengths range from
// all to nothing, and they are cut where they are fewer than three to a compute unit (bf16, 1 x 4096
// tokens, 12 heads of 64, 384 tiles: 119 us whole, 72 + 17 cut; 8 x 1024 tokens, 768: 40 whole, 45 + 31).
struct Cuts {
    int tiles, far_tiles, near, far;
    int64_t heads, slots, pieces;  // blocks of all heads, and those of tiles that are cut
    Cuts(const isa_block_attention* t, int keys_per_tile) {
        heads = t->batch * t->kv_heads;
        tiles = static_cast<int>(ceil_div(t->keys, keys_per_tile));
        const int64_t turn = t->type == ISA_BLOCK_F32 ? 32 : 64, group = t->heads / t->kv_heads;
        const int64_t longest = std::min(t->queries, t->window ? t->window + keys_per_tile - 1 : t->queries);
        const bool limited = longest < t->queries;
        far_tiles = limited ? static_cast<int>(std::min<int64_t>(ceil_div(t->sinks, keys_per_tile), tiles)) : 0;
        const int64_t plain = (tiles - far_tiles) * heads, turns = std::max<int64_t>(1, ceil_div(longest, turn) * group);
        const int64_t most = std::min<int64_t>(64, ceil_div(turns, 4));
        const int64_t enough = limited ? kComputeUnits * 3 / 2 : 3 * kComputeUnits;
        near = plain && plain < enough ? static_cast<int>(std::min(ceil_div(enough, plain), most)) : 1;
        const int64_t piece = std::max<int64_t>(4, turns / near / 4);
        // (where tiles with sinks are many, they fill the chip uncut, and their sums would fill its memory)
        const int64_t most_pieces = ceil_div(ceil_div(t->queries, turn) * group, piece);
        far = far_tiles ? static_cast<int>(std::max<int64_t>(1, std::min(most_pieces, 4 * kComputeUnits / (far_tiles * heads)))) : 1;
        slots = heads * (static_cast<int64_t>(tiles - far_tiles) * near + static_cast<int64_t>(far_tiles) * far);
        pieces = heads * ((near > 1 ? static_cast<int64_t>(tiles - far_tiles) * near : 0) +
                          (far > 1 ? static_cast<int64_t>(far_tiles) * far : 0));
    }
    int64_t summed() const { return heads * ((near > 1 ? tiles - far_tiles : 0) + (far > 1 ? far_tiles : 0)); }
};

size_t plane_bytes(const isa_block_attention* t) {
    return ceil_div(t->batch * t->heads * t->queries, 64) * 64 * kPlanes * sizeof(float);
}

template <typename T, int D>
void launch(AttnArgs a, const isa_block_attention* t, hipStream_t s) {
    using S = DkvShape<T, D>;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.queries * a.heads;
    if (rows) {
        const int64_t tiles = ceil_div(static_cast<int64_t>(a.queries) * a.group, kRows<T>);
        if (a.result)
            attention_dq_kernel<T, D><<<dim3(static_cast<unsigned>(tiles * a.batch * a.kv_heads)), kThreads<T>, 0, s>>>(a);
        else
            attention_rows_kernel<T><<<dim3(static_cast<unsigned>(ceil_div(rows * 16, kRowThreads))), kRowThreads, 0, s>>>(a);
    }
    if (!a.dk || !a.keys) return;
    const Cuts cuts(t, S::kKeys);
    a.near = cuts.near;
    a.far = cuts.far;
    a.far_tiles = cuts.far_tiles;
    attention_dkv_kernel<T, D><<<dim3(static_cast<unsigned>(cuts.slots)), S::kThreadCount, 0, s>>>(a);
    if (cuts.summed())
        attention_dkv_sum_kernel<T, D>
            <<<dim3(static_cast<unsigned>(cuts.summed() * 2 * (D / 8))), S::kThreadCount, 0, s>>>(a);
}

template <typename F>
void for_shape(const isa_block_attention* t, F f) {
    for_type(t->type, static_cast<int>(t->head_dim), [&](auto type, auto dim) {
        using T = decltype(type);
        constexpr int D = decltype(dim)::value;
        f(type, dim, DkvShape<T, D>{});
    });
}

}  // namespace
}  // namespace isa_block

using namespace isa_block;

extern "C" size_t isa_block_attention_backward_workspace(const isa_block_attention* t) {
    if (!t || check_attention(t)) return 0;
    size_t bytes = plane_bytes(t);
    for_shape(t, [&](auto, auto dim, auto shape) {
        using S = decltype(shape);
        const Cuts cuts(t, S::kKeys);
        bytes += cuts.pieces * 2 * S::kKeys * decltype(dim)::value * sizeof(float);
    });
    return bytes;
}

extern "C" int isa_block_attention_backward(const isa_block_attention* t, const void* out, const void* rest,
                                            const float* lse, const void* dout, const int64_t dout_strides[3],
                                            void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                            void* stream) {
    if (int rc = check_attention(t)) return rc;
    if (t->batch == 0 || (t->queries == 0 && t->keys == 0)) return 0;
    if (t->queries && (!out || !lse || !dout || !dout_strides)) return fail("out, lse and grad_out must be set");
    if ((dk == nullptr) != (dv == nullptr)) return fail("grad_k and grad_v go together");
    AttnArgs a = attention_args(t);
    if (t->queries) {
        std::copy(dout_strides, dout_strides + 3, a.gs);
        if (t->queries == 1) a.gs[1] = t->head_dim;
        if (!strided(dout, a.gs, t->queries, t->head_dim, type_bytes(t->type)))
            return fail("grad_out must be 16-byte aligned, its strides multiples of 8 elements, that of tokens at "
                        "least head_dim and under 16 MiB");
    }
    if (workspace_bytes < isa_block_attention_backward_workspace(t))
        return fail("workspace too small: %zu bytes", workspace_bytes);
    if (workspace_bytes && (!workspace || !aligned(workspace, 256))) return fail("workspace must be 256-byte aligned");
    for (const void* p : {out, rest, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
        if (!aligned(p, 16)) return fail("out and the gradients must be 16-byte aligned");
    a.out = out;
    a.rest = const_cast<void*>(rest);
    a.dout = dout;
    a.lse = const_cast<float*>(lse);
    a.delta = static_cast<float*>(workspace);
    a.partial = a.delta + plane_bytes(t) / sizeof(float);
    a.result = dq;
    a.dk = dk;
    a.dv = dv;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    for_type(t->type, a.dim, [&](auto type, auto dim) { launch<decltype(type), decltype(dim)::value>(a, t, s); });
    return launched("the attention's backward");
}
