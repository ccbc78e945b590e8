// Attention with a sliding window and sinks, forward and backward, for gfx950.
//
//   s_ij = c q_i k_j  (c = scale log2 e),  p_ij = exp2(s_ij - lse_i) over the keys j that i sees
//   out = p v;  dv = p^T do,  dp = do v^T,  ds = p (dp - delta),  delta_i = do_i out_i,
//   dq = scale ds k,  dk = scale ds^T q
//
// Products run on the matrix cores in 32 x 32 tiles with fp32 sums: 16-bit types as 32x32x16,
// fp32 as 32x32x2. Scores are taken as s^T = K Q^T, so a lane holds one query's scores and a
// row's maximum and sum are lane-local but for one exchange of the wave's halves; and those
// scores are, register for register, the second operand of the next product (out^T = V^T p^T),
// because the order in which a product sums its inner index is free: each half of the wave
// takes the keys that it holds. The first operand (V^T, K^T, Q^T, dO^T) follows that order and is
// read across the tile's rows.
//
// The rows of a product are the queries of all heads that share a key head, position by
// position, so K and V are read once for the group. A block walks the tiles of keys that any of
// its rows sees: the sinks' tiles, then the window's. Masks are evaluated only in tiles that some
// row sees in part.
#include "block_common.hpp"

#include <algorithm>
#include <climits>

namespace isa_block {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kTile = 32;               // of the matrix instruction, both ways
constexpr int kBlockRows = kWaves * kTile;
constexpr float kLog2E = 1.44269504088896340736f;
constexpr int kMaxLength = 1 << 30;

using acc16 = vec<float, 16>;

struct AttnArgs {
    const void *q, *k, *v, *out, *dout;
    void *result, *rest, *dk, *dv;  // result: out, or dq
    float *lse, *delta;
    const int32_t* lengths;
    int64_t qs[3], ks[3], vs[3], gs[3];
    int batch, queries, keys, heads, kv_heads, group, dim, window, sinks;
    float c, scale;
};

// ---- fragments: 16 bytes a lane, of an operand's row (lane % 32) the chunk of its half --------

template <typename T>
struct Frag {
    static constexpr int N = 16 / sizeof(T);  // elements
    using V = vec<T, N>;
};

__device__ __forceinline__ void mma(acc16& acc, vec<bf16, 8> a, vec<bf16, 8> b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(acc16& acc, vec<f16, 8> a, vec<f16, 8> b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(acc16& acc, vec<float, 4> a, vec<float, 4> b) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
}

// Values u N .. u N + N - 1 of a lane's column of a product, as an operand of the next one.
template <typename T>
__device__ __forceinline__ typename Frag<T>::V operand(const acc16& x, int u) {
    typename Frag<T>::V f;
#pragma unroll
    for (int e = 0; e < Frag<T>::N; ++e) f[e] = static_cast<T>(x[u * Frag<T>::N + e]);
    return f;
}

// sum plus an operand's values as they were rounded: a row's weights, whose sum is what they are
// divided by, then add up to 1 as the product sees them.
__device__ __forceinline__ float add_all(vec<bf16, 8> x, float sum) {
    const vec<bf16, 2> one = {static_cast<bf16>(1.0f), static_cast<bf16>(1.0f)};
#pragma unroll
    for (int e = 0; e < 8; e += 2)
        sum = __builtin_amdgcn_fdot2_f32_bf16(vec<bf16, 2>{x[e], x[e + 1]}, one, sum, false);
    return sum;
}
__device__ __forceinline__ float add_all(vec<f16, 8> x, float sum) {
    const vec<f16, 2> one = {static_cast<f16>(1.0f), static_cast<f16>(1.0f)};
#pragma unroll
    for (int e = 0; e < 8; e += 2)
        sum = __builtin_amdgcn_fdot2(vec<f16, 2>{x[e], x[e + 1]}, one, sum, false);
    return sum;
}
__device__ __forceinline__ float add_all(vec<float, 4> x, float sum) { return sum + ((x[0] + x[1]) + (x[2] + x[3])); }

// The row of a 32-row product that register i of a lane in `half` holds.
__device__ __forceinline__ constexpr int product_row(int i, int half) { return 8 * (i / 4) + 4 * half + i % 4; }

// ---- tiles in LDS: rows of D elements, 16 bytes apart from the next, so that 16-byte reads of one
// chunk down the rows use all banks ----------------------------------------------------------

template <typename T, int D>
struct Tile {
    static constexpr int N = Frag<T>::N;
    static constexpr int kChunks = D / N;
    static constexpr int kPitch = D + N;  // elements
    static constexpr int kSteps = kChunks / 2;
    static constexpr int kUses = kTile / (2 * N);  // operand()s of 32 rows

    // of row (r0 + lane % 32), dims of step t
    static __device__ __forceinline__ typename Frag<T>::V row(const T* tile, int r0, int t, int lane) {
        return *reinterpret_cast<const typename Frag<T>::V*>(tile + (r0 + lane % 32) * kPitch +
                                                             (2 * t + lane / 32) * N);
    }

    // of column (32 db + lane % 32), the rows r0 .. r0 + 31 that operand(x, u) holds in this half
    static __device__ __forceinline__ typename Frag<T>::V column(const T* tile, int r0, int u, int db, int lane) {
        if constexpr (sizeof(T) == 4) {
            typename Frag<T>::V f;
            const T* p = tile + (r0 + 8 * u + 4 * (lane / 32)) * kPitch + 32 * db + lane % 32;
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = p[e * kPitch];
            return f;
        } else {
            // the transposing read: 16 lanes give the addresses of 4 rows x 16 columns, 4 columns each,
            // and get a column's 4 rows each
            using s4 = vec<short, 4>;
            using lds = __attribute__((address_space(3))) s4;
            const int at = (r0 + 16 * u + 4 * (lane / 32) + lane % 16 / 4) * kPitch + 32 * db + lane / 16 % 2 * 16 +
                           lane % 4 * 4;
            union {
                s4 part[2];
                typename Frag<T>::V f;
            } x;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                x.part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)(tile + at + 8 * j * kPitch));
            return x.f;
        }
    }
};

// A tile's chunks on their way from global memory to LDS: held in registers while the last tile
// is computed on.
template <typename T, int D, int ROWS>
struct Staged {
    using L = Tile<T, D>;
    using V = typename Frag<T>::V;
    static constexpr int kEach = ROWS * L::kChunks / kThreads;
    static_assert(ROWS * L::kChunks % kThreads == 0);
    V v[kEach];

    // row_of(row): the row's elements in global memory, or null for a row of zeros
    template <typename F>
    __device__ __forceinline__ void load(int dim, F row_of) {
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int at = threadIdx.x + n * kThreads, c = at % L::kChunks;
            const T* p = row_of(at / L::kChunks);
            v[n] = V{};
            if (p && c * L::N < dim) v[n] = *reinterpret_cast<const V*>(p + c * L::N);
        }
    }
    __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int at = threadIdx.x + n * kThreads;
            *reinterpret_cast<V*>(tile + at / L::kChunks * L::kPitch + at % L::kChunks * L::N) = v[n];
        }
    }
};

// Dispatch gives block i to XCD i % 8; this gives each XCD a run of adjacent work, whose keys its
// L2 then holds once.
__device__ __forceinline__ int xcd_order(int id, int n) {
    const int per = n / 8, rest = n % 8, x = id % 8;
    return x * per + min(x, rest) + id / 8;
}

// ---- which keys a block of rows sees --------------------------------------------------------

__device__ __forceinline__ int length_of(const AttnArgs& a, int b) {
    return a.lengths ? min(max(a.lengths[b], 0), a.keys) : a.keys;
}

__device__ __forceinline__ bool sees(const AttnArgs& a, int p, int j) {
    return j <= p && (j < a.sinks || j > p - a.window);
}

struct Span {
    int lo, hi, sink_tiles, first, count;
    int pmin, pmax;

    // Tiles of BN keys that some query at pmin .. pmax sees: the sinks' tiles that lie before the
    // window's, then the window's.
    template <int BN>
    static __device__ __forceinline__ Span of(const AttnArgs& a, int pmin, int pmax) {
        Span s;
        s.pmin = pmin;
        s.pmax = pmax;
        s.hi = pmax + 1;
        s.lo = max(0, pmin - a.window + 1);
        s.first = s.lo / BN;
        s.sink_tiles = min((min(a.sinks, s.lo) + BN - 1) / BN, s.first);
        s.count = s.hi <= 0 ? 0 : s.sink_tiles + (s.hi + BN - 1) / BN - s.first;
        return s;
    }
    __device__ __forceinline__ int tile(int it) const { return it < sink_tiles ? it : first + it - sink_tiles; }
    // whether some row sees key j: others are not read
    __device__ __forceinline__ bool read(const AttnArgs& a, int j) const { return j < hi && (j >= lo || j < a.sinks); }
    // whether every row sees all of j0 .. j1 - 1
    __device__ __forceinline__ bool all(const AttnArgs& a, int j0, int j1) const {
        return j1 - 1 <= pmin && (j1 <= a.sinks || j0 > pmax - a.window);
    }
};

// A row of a block: its query's place in the sequence and its pointers' offsets.
struct RowAt {
    int query, head;
    __device__ __forceinline__ RowAt(const AttnArgs& a, int row, int kv_head)
        : query(row / a.group), head(kv_head * a.group + row % a.group) {}
    __device__ __forceinline__ int64_t in(const int64_t (&s)[3], int b) const {
        return b * s[0] + query * s[1] + head * s[2];
    }
    __device__ __forceinline__ int64_t stat(const AttnArgs& a, int b) const {
        return (static_cast<int64_t>(b) * a.heads + head) * a.queries + query;
    }
    __device__ __forceinline__ int64_t packed(const AttnArgs& a, int b) const {
        return ((static_cast<int64_t>(b) * a.queries + query) * a.heads + head) * a.dim;
    }
};

template <typename T, int D>
struct RowFrags {
    typename Frag<T>::V v[Tile<T, D>::kSteps];
    __device__ __forceinline__ const typename Frag<T>::V& operator[](int t) const { return v[t]; }
};

// A row's elements, or zeros.
template <typename T, int D>
__device__ __forceinline__ void load_row_frags(RowFrags<T, D>& f, const T* row, int dim, int lane) {
    using V = typename Frag<T>::V;
#pragma unroll
    for (int t = 0; t < Tile<T, D>::kSteps; ++t) {
        const int at = (2 * t + lane / 32) * Frag<T>::N;
        f.v[t] = V{};
        if (row && at < dim) f.v[t] = *reinterpret_cast<const V*>(row + at);
    }
}

// Rows of a transposed product (lane: a row, registers: its dims), each times `factor`; what their
// rounding leaves goes to `rest` if that is set.
template <typename T, int DB>
__device__ __forceinline__ void store_rows(T* row, const acc16 (&x)[DB], float factor, int dim, int lane,
                                           T* rest = nullptr) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int at = 32 * db + product_row(i, lane / 32);
            Pack<T, 4> p;
#pragma unroll
            for (int e = 0; e < 4; ++e) p.v[e] = static_cast<T>(x[db][i + e] * factor);
            if (at < dim) *reinterpret_cast<Pack<T, 4>*>(row + at) = p;
            if (!rest) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) p.v[e] = static_cast<T>(x[db][i + e] * factor - static_cast<float>(p.v[e]));
            if (at < dim) *reinterpret_cast<Pack<T, 4>*>(rest + at) = p;
        }
}

template <typename T>
constexpr int kKeyTile = sizeof(T) == 4 ? 32 : 64;

// ---- forward ----------------------------------------------------------------------------------

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attention_forward_kernel(AttnArgs a) {
    using L = Tile<T, D>;
    constexpr int BN = kKeyTile<T>, DB = D / 32;
    __shared__ __attribute__((aligned(16))) T ktile[BN * L::kPitch], vtile[BN * L::kPitch];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, half = lane / 32;
    const int rows = a.queries * a.group, tiles = (rows + kBlockRows - 1) / kBlockRows;
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int kv_head = id / tiles % a.kv_heads, b = id / tiles / a.kv_heads;
    const int row0 = (tiles - 1 - id % tiles) * kBlockRows;  // rows that see the most keys first
    const int length = length_of(a, b), shift = length - a.queries;
    const int last = min(row0 + kBlockRows, rows) - 1;
    const Span span = Span::of<BN>(a, shift + row0 / a.group, shift + last / a.group);

    const int row = row0 + wave * kTile + lane % 32;
    const RowAt at(a, min(row, last), kv_head);
    const int p = shift + at.query;
    RowFrags<T, D> q;
    load_row_frags<T, D>(q, row <= last ? static_cast<const T*>(a.q) + at.in(a.qs, b) : nullptr, a.dim, lane);

    acc16 o[DB] = {};
    float top = -INFINITY, sum = 0.0f;
    Staged<T, D, BN> ks, vs;
    const T* kbase = static_cast<const T*>(a.k) + b * a.ks[0] + kv_head * a.ks[2];
    const T* vbase = static_cast<const T*>(a.v) + b * a.vs[0] + kv_head * a.vs[2];
    auto fetch = [&](int it) {
        const int j0 = span.tile(it) * BN;
        ks.load(a.dim, [&](int r) { return span.read(a, j0 + r) ? kbase + (j0 + r) * a.ks[1] : nullptr; });
        vs.load(a.dim, [&](int r) { return span.read(a, j0 + r) ? vbase + (j0 + r) * a.vs[1] : nullptr; });
    };
    if (span.count) fetch(0);
    for (int it = 0; it < span.count; ++it) {
        ks.store(ktile);
        vs.store(vtile);
        __syncthreads();
        if (it + 1 < span.count) fetch(it + 1);
        const int j0 = span.tile(it) * BN;
        acc16 s[BN / 32];
#pragma unroll
        for (int n = 0; n < BN / 32; ++n) {
            s[n] = acc16{};
#pragma unroll
            for (int t = 0; t < L::kSteps; ++t) mma(s[n], L::row(ktile, 32 * n, t, lane), q[t]);
        }
        if (!span.all(a, j0, j0 + BN)) {
#pragma unroll
            for (int n = 0; n < BN / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!sees(a, p, j0 + 32 * n + product_row(i, half))) s[n][i] = -INFINITY;
        }
        float t = top;
#pragma unroll
        for (int n = 0; n < BN / 32; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) t = fmaxf(t, s[n][i]);
        t = half_max(t);
        const float base = t == -INFINITY ? 0.0f : t * a.c;  // a row that has seen nothing yet
        const float decay = __builtin_amdgcn_exp2f(top * a.c - base);
        top = t;
        sum *= decay;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] *= decay;
#pragma unroll
        for (int n = 0; n < BN / 32; ++n) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = __builtin_amdgcn_exp2f(fmaf(s[n][i], a.c, -base));
#pragma unroll
            for (int u = 0; u < L::kUses; ++u) {
                const typename Frag<T>::V f = operand<T>(s[n], u);
                sum = add_all(f, sum);
#pragma unroll
                for (int db = 0; db < DB; ++db) mma(o[db], L::column(vtile, 32 * n, u, db, lane), f);
            }
        }
        __syncthreads();
    }
    sum = half_sum(sum);
    if (row > last) return;
    const int64_t to = at.packed(a, b);
    store_rows<T, DB>(static_cast<T*>(a.result) + to, o, sum > 0.0f ? 1.0f / sum : 0.0f, a.dim, lane,
                      a.rest ? static_cast<T*>(a.rest) + to : nullptr);
    if (a.lse && half == 0)
        a.lse[at.stat(a, b)] = sum > 0.0f ? fmaf(top, a.c, log2f(sum)) : -INFINITY;
}

// ---- backward -----------------------------------------------------------------------------------

// delta = rows' do . out, 16 threads a row. Where one weight is close to 1, its key's dp is close to
// delta and ds is their difference: out's own rounding would be most of it, so a 16-bit out comes
// with what that left.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_delta_kernel(AttnArgs a) {
    const int64_t r = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / 16;
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
    if (r < rows && threadIdx.x % 16 == 0) a.delta[(b * a.heads + head) * a.queries + i] = s;
}

// dq: the forward's walk, with p from the saved sums.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attention_dq_kernel(AttnArgs a) {
    using L = Tile<T, D>;
    constexpr int BN = kKeyTile<T>, DB = D / 32;
    __shared__ __attribute__((aligned(16))) T ktile[BN * L::kPitch], vtile[BN * L::kPitch];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, half = lane / 32;
    const int rows = a.queries * a.group, tiles = (rows + kBlockRows - 1) / kBlockRows;
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int kv_head = id / tiles % a.kv_heads, b = id / tiles / a.kv_heads;
    const int row0 = (tiles - 1 - id % tiles) * kBlockRows;
    const int length = length_of(a, b), shift = length - a.queries;
    const int last = min(row0 + kBlockRows, rows) - 1;
    const Span span = Span::of<BN>(a, shift + row0 / a.group, shift + last / a.group);

    const int row = row0 + wave * kTile + lane % 32;
    const RowAt at(a, min(row, last), kv_head);
    const int p = shift + at.query;
    RowFrags<T, D> q, g;
    load_row_frags<T, D>(q, row <= last ? static_cast<const T*>(a.q) + at.in(a.qs, b) : nullptr, a.dim, lane);
    load_row_frags<T, D>(g, row <= last ? static_cast<const T*>(a.dout) + at.in(a.gs, b) : nullptr, a.dim, lane);
    const float lse = row <= last ? a.lse[at.stat(a, b)] : 0.0f, delta = row <= last ? a.delta[at.stat(a, b)] : 0.0f;

    acc16 dq[DB] = {};
    Staged<T, D, BN> ks, vs;
    const T* kbase = static_cast<const T*>(a.k) + b * a.ks[0] + kv_head * a.ks[2];
    const T* vbase = static_cast<const T*>(a.v) + b * a.vs[0] + kv_head * a.vs[2];
    auto fetch = [&](int it) {
        const int j0 = span.tile(it) * BN;
        ks.load(a.dim, [&](int r) { return span.read(a, j0 + r) ? kbase + (j0 + r) * a.ks[1] : nullptr; });
        vs.load(a.dim, [&](int r) { return span.read(a, j0 + r) ? vbase + (j0 + r) * a.vs[1] : nullptr; });
    };
    if (span.count) fetch(0);
    for (int it = 0; it < span.count; ++it) {
        ks.store(ktile);
        vs.store(vtile);
        __syncthreads();
        if (it + 1 < span.count) fetch(it + 1);
        const int j0 = span.tile(it) * BN;
        const bool all = span.all(a, j0, j0 + BN);
#pragma unroll
        for (int n = 0; n < BN / 32; ++n) {
            acc16 s = {}, d = {};
#pragma unroll
            for (int t = 0; t < L::kSteps; ++t) {
                mma(s, L::row(ktile, 32 * n, t, lane), q[t]);
                mma(d, L::row(vtile, 32 * n, t, lane), g[t]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.c, -lse)) * (d[i] - delta);
            if (!all) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!sees(a, p, j0 + 32 * n + product_row(i, half))) s[i] = 0.0f;
            }
#pragma unroll
            for (int u = 0; u < L::kUses; ++u) {
                const typename Frag<T>::V f = operand<T>(s, u);
#pragma unroll
                for (int db = 0; db < DB; ++db) mma(dq[db], L::column(ktile, 32 * n, u, db, lane), f);
            }
        }
        __syncthreads();
    }
    if (row <= last) store_rows<T, DB>(static_cast<T*>(a.result) + at.packed(a, b), dq, a.scale, a.dim, lane);
}

// dk and dv: a block takes 128 keys, a wave 32 of them, and walks the rows that see them.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attention_dkv_kernel(AttnArgs a) {
    using L = Tile<T, D>;
    constexpr int BR = kKeyTile<T>, DB = D / 32;
    __shared__ __attribute__((aligned(16))) T qtile[BR * L::kPitch], gtile[BR * L::kPitch];
    __shared__ __attribute__((aligned(16))) float lses[BR], deltas[BR];
    __shared__ __attribute__((aligned(16))) int places[BR];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, half = lane / 32;
    const int tiles = (a.keys + kBlockRows - 1) / kBlockRows;
    const int id = xcd_order(blockIdx.x, gridDim.x);
    const int kv_head = id / tiles % a.kv_heads, b = id / tiles / a.kv_heads;
    const int j0 = id % tiles * kBlockRows;
    const int length = length_of(a, b), shift = length - a.queries;

    const int mine = j0 + wave * kTile, key = mine + lane % 32;
    RowFrags<T, D> k, v;
    load_row_frags<T, D>(k, key < length ? static_cast<const T*>(a.k) + b * a.ks[0] + kv_head * a.ks[2] + key * a.ks[1]
                                         : nullptr, a.dim, lane);
    load_row_frags<T, D>(v, key < length ? static_cast<const T*>(a.v) + b * a.vs[0] + kv_head * a.vs[2] + key * a.vs[1]
                                         : nullptr, a.dim, lane);
    // the queries at p = j0 .. that see one of the keys
    const int64_t reach = static_cast<int64_t>(min(j0 + kBlockRows, length)) - 1 + a.window - 1;
    const int plast = j0 < a.sinks || reach > length - 1 ? length - 1 : static_cast<int>(reach);
    const int first = max(0, j0 - shift) * a.group;
    const int end = j0 < length ? (plast - shift + 1) * a.group : 0;

    acc16 dk[DB] = {}, dv[DB] = {};
    Staged<T, D, BR> qs, gs;
    float lse = 0.0f, delta = 0.0f;
    const T *qbase = static_cast<const T*>(a.q), *gbase = static_cast<const T*>(a.dout);
    auto fetch = [&](int r0) {
        qs.load(a.dim, [&](int r) { return r0 + r < end ? qbase + RowAt(a, r0 + r, kv_head).in(a.qs, b) : nullptr; });
        gs.load(a.dim, [&](int r) { return r0 + r < end ? gbase + RowAt(a, r0 + r, kv_head).in(a.gs, b) : nullptr; });
        if (threadIdx.x < BR) {
            const int r = r0 + threadIdx.x;
            const int64_t at = RowAt(a, min(r, end - 1), kv_head).stat(a, b);
            lse = r < end ? a.lse[at] : 0.0f;
            delta = r < end ? a.delta[at] : 0.0f;
        }
    };
    if (first < end) fetch(first);
    for (int r0 = first; r0 < end; r0 += BR) {
        qs.store(qtile);
        gs.store(gtile);
        if (threadIdx.x < BR) {
            lses[threadIdx.x] = lse;
            deltas[threadIdx.x] = delta;
            places[threadIdx.x] = shift + (r0 + static_cast<int>(threadIdx.x)) / a.group;
        }
        __syncthreads();
        if (r0 + BR < end) fetch(r0 + BR);
        const int pmin = shift + r0 / a.group, pmax = shift + (min(r0 + BR, end) - 1) / a.group;
        const bool all = mine + kTile - 1 <= pmin && (mine + kTile <= a.sinks || mine > pmax - a.window);
#pragma unroll
        for (int n = 0; n < BR / 32; ++n) {
            acc16 s = {}, d = {};
#pragma unroll
            for (int t = 0; t < L::kSteps; ++t) {
                mma(s, L::row(qtile, 32 * n, t, lane), k[t]);
                mma(d, L::row(gtile, 32 * n, t, lane), v[t]);
            }
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int r = 32 * n + product_row(i, half);
                const vec<float, 4> l = *reinterpret_cast<const vec<float, 4>*>(lses + r);
                const vec<float, 4> m = *reinterpret_cast<const vec<float, 4>*>(deltas + r);
                const vec<int, 4> at = *reinterpret_cast<const vec<int, 4>*>(places + r);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = __builtin_amdgcn_exp2f(fmaf(s[i + e], a.c, -l[e])), y = x * (d[i + e] - m[e]);
                    if (!all && !sees(a, at[e], key)) x = y = 0.0f;
                    s[i + e] = x;
                    d[i + e] = y;
                }
            }
#pragma unroll
            for (int u = 0; u < L::kUses; ++u) {
                const typename Frag<T>::V f = operand<T>(s, u), h = operand<T>(d, u);
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    mma(dv[db], L::column(gtile, 32 * n, u, db, lane), f);
                    mma(dk[db], L::column(qtile, 32 * n, u, db, lane), h);
                }
            }
        }
        __syncthreads();
    }
    if (key >= a.keys) return;
    const int64_t out = ((static_cast<int64_t>(b) * a.keys + key) * a.kv_heads + kv_head) * a.dim;
    store_rows<T, DB>(static_cast<T*>(a.dk) + out, dk, a.scale, a.dim, lane);
    store_rows<T, DB>(static_cast<T*>(a.dv) + out, dv, 1.0f, a.dim, lane);
}

// ---- host -----------------------------------------------------------------------------------------

constexpr int64_t kMaxBlocks = INT_MAX;

template <typename T, int D>
void launch_forward(const AttnArgs& a, hipStream_t s) {
    const int64_t tiles = ceil_div(static_cast<int64_t>(a.queries) * a.group, kBlockRows);
    attention_forward_kernel<T, D><<<dim3(static_cast<unsigned>(tiles * a.batch * a.kv_heads)), kThreads, 0, s>>>(a);
}

template <typename T, int D>
void launch_backward(const AttnArgs& a, hipStream_t s) {
    const int64_t rows = static_cast<int64_t>(a.batch) * a.queries * a.heads;
    if (rows) {
        attention_delta_kernel<T><<<dim3(static_cast<unsigned>(ceil_div(rows * 16, kThreads))), kThreads, 0, s>>>(a);
        const int64_t tiles = ceil_div(static_cast<int64_t>(a.queries) * a.group, kBlockRows);
        if (a.result)
            attention_dq_kernel<T, D><<<dim3(static_cast<unsigned>(tiles * a.batch * a.kv_heads)), kThreads, 0, s>>>(a);
    }
    const int64_t tiles = ceil_div(a.keys, kBlockRows);
    if (tiles && a.dk)
        attention_dkv_kernel<T, D><<<dim3(static_cast<unsigned>(tiles * a.batch * a.kv_heads)), kThreads, 0, s>>>(a);
}

template <typename T>
void launch(const AttnArgs& a, bool backward, hipStream_t s) {
    if (a.dim <= 32) return backward ? launch_backward<T, 32>(a, s) : launch_forward<T, 32>(a, s);
    if (a.dim <= 64) return backward ? launch_backward<T, 64>(a, s) : launch_forward<T, 64>(a, s);
    if (a.dim <= 96) return backward ? launch_backward<T, 96>(a, s) : launch_forward<T, 96>(a, s);
    return backward ? launch_backward<T, 128>(a, s) : launch_forward<T, 128>(a, s);
}

void run(int type, const AttnArgs& a, bool backward, hipStream_t s) {
    if (type == ISA_BLOCK_F32) launch<float>(a, backward, s);
    else if (type == ISA_BLOCK_BF16) launch<bf16>(a, backward, s);
    else launch<f16>(a, backward, s);
}

bool strided(const void* p, const int64_t (&s)[3]) {
    return aligned(p, 16) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
}

int check(const isa_block_attention* t) {
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
    if (t->queries * (t->heads / t->kv_heads) > kMaxLength)
        return fail("more than 2^30 queries times heads of a key head");
    // blocks of 128 rows or keys, and of 16 rows in the backward's first pass
    if (t->batch * t->kv_heads > kMaxLength || t->batch * t->heads * std::max<int64_t>(t->queries, t->keys) / 16 > kMaxBlocks ||
        t->batch * t->kv_heads * (std::max<int64_t>(t->queries * (t->heads / t->kv_heads), t->keys) / kBlockRows + 1) > kMaxBlocks)
        return fail("too many rows for one launch");
    if (t->batch && t->queries && !t->q) return fail("q is null");
    if (t->batch && t->keys && (!t->k || !t->v)) return fail("k and v must be set");
    if (!strided(t->q, t->q_strides) || !strided(t->k, t->k_strides) || !strided(t->v, t->v_strides))
        return fail("q, k and v must be 16-byte aligned, their strides multiples of 8 elements");
    return 0;
}

AttnArgs args_of(const isa_block_attention* t) {
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
    a.sinks = static_cast<int>(t->sinks);
    a.scale = t->scale;
    a.c = t->scale * kLog2E;
    return a;
}

size_t delta_bytes(const isa_block_attention* t) {
    return ceil_div(t->batch * t->heads * t->queries * static_cast<int64_t>(sizeof(float)), 256) * 256;
}

}  // namespace
}  // namespace isa_block

using namespace isa_block;

extern "C" size_t isa_block_attention_forward_workspace(const isa_block_attention* t) {
    (void)t;
    return 0;
}

extern "C" int isa_block_attention_forward(const isa_block_attention* t, void* out, void* rest, float* lse,
                                           void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(t)) return rc;
    if (t->batch == 0 || t->queries == 0) return 0;
    if (!out || !aligned(out, 16) || !aligned(rest, 16)) return fail("out must be set, it and rest 16-byte aligned");
    AttnArgs a = args_of(t);
    a.result = out;
    a.rest = rest;
    a.lse = lse;
    run(t->type, a, false, static_cast<hipStream_t>(stream));
    return launched("attention_forward_kernel");
}

extern "C" size_t isa_block_attention_backward_workspace(const isa_block_attention* t) {
    if (!t || check(t)) return 0;
    return delta_bytes(t);
}

extern "C" int isa_block_attention_backward(const isa_block_attention* t, const void* out, const void* rest,
                                            const float* lse, const void* dout, const int64_t dout_strides[3], void* dq, void* dk,
                                            void* dv, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(t)) return rc;
    if (t->batch == 0 || (t->queries == 0 && t->keys == 0)) return 0;
    if (t->queries && (!out || !lse || !dout || !dout_strides)) return fail("out, lse and grad_out must be set");
    if ((dk == nullptr) != (dv == nullptr)) return fail("grad_k and grad_v go together");
    AttnArgs a = args_of(t);
    if (t->queries) {
        std::copy(dout_strides, dout_strides + 3, a.gs);
        if (!strided(dout, a.gs)) return fail("grad_out must be 16-byte aligned, its strides multiples of 8 elements");
        if (workspace_bytes < isa_block_attention_backward_workspace(t))
            return fail("workspace too small: %zu bytes", workspace_bytes);
        if (!workspace || !aligned(workspace, 256)) return fail("workspace must be 256-byte aligned");
    }
    for (const void* p : {out, rest, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
        if (!aligned(p, 16)) return fail("out and the gradients must be 16-byte aligned");
    a.out = out;
    a.rest = const_cast<void*>(rest);
    a.dout = dout;
    a.lse = const_cast<float*>(lse);
    a.delta = static_cast<float*>(workspace);
    a.result = dq;
    a.dk = dk;
    a.dv = dv;
    run(t->type, a, true, static_cast<hipStream_t>(stream));
    return launched("the attention's backward");
}
