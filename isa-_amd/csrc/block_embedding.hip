// Embedding lookup of tokens and places, and the tables' gradients, for gfx950.
//
//   y_t = round(scale W[id_t] + P[place_t]),   dW_v = scale sum_{t: id_t = v} dy_t
//
// Both are bound by HBM: the lookup reads and writes rows, the gradient reads dy and writes all of dW, most of
// whose rows are zeros. The gradient's sums use no atomics: tokens are sorted by their row, in order within
// one, and a row's sum is taken in that order.
//
// The sort is one launch without any exchange between its blocks: a block owns a range of rows, reads all
// keys, counts those below its range (where its part of the list starts) and places those inside.
// A row with many tokens would be one wave's long walk: lists longer than a tile are summed by tiles of
// the sorted list, whose sums of a row are added up in a third launch.
#include "block_common.hpp"

#include <algorithm>

#include "isa_train.h"

namespace isa_block {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 8192;

// ---- lookup -------------------------------------------------------------------------------

struct LookupArgs {
    const int64_t *ids, *place_ids;
    const void *weight, *place_weight;
    void* y;
    int64_t tokens, vocab, weight_stride, places, places_stride, period;
    int dim;
    float scale;
};

// A row of y is taken by `lanes` threads of a block, 16 bytes at a time.
template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_kernel(LookupArgs a, int lanes) {
    constexpr int N = 16 / sizeof(T);
    const int per_block = kThreads / lanes, lane = threadIdx.x % lanes;
    const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / lanes; t < a.tokens; t += step) {
        const int64_t id = a.ids[t];
        const int64_t place = !a.places ? 0 : a.place_ids ? a.place_ids[t] : t % a.period;
        const bool inside = id >= 0 && id < a.vocab && (!a.places || (place >= 0 && place < a.places));
        const T* w = static_cast<const T*>(a.weight) + (inside ? id : 0) * a.weight_stride;
        const T* p = static_cast<const T*>(a.place_weight) + (inside ? place : 0) * a.places_stride;
        T* y = static_cast<T*>(a.y) + t * a.dim;
        for (int at = lane * N; at < a.dim; at += lanes * N) {
            Pack<T, N> r, q;
            if (inside) {
                load_loose(r, w + at, a.dim - at);
                if (a.places) load_loose(q, p + at, a.dim - at);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float x = a.scale * static_cast<float>(r.v[e]);
                if (a.places) x = fmaf(a.scale, static_cast<float>(r.v[e]), static_cast<float>(q.v[e]));
                r.v[e] = static_cast<T>(inside ? x : NAN);
            }
            store_loose(y + at, r, a.dim - at);
        }
    }
}

// ---- the tokens of each row ---------------------------------------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortRange = 512;  // rows of a block: 32 KiB of counters, so that blocks share a compute unit
constexpr int kSortBlocks = 256;

struct SortArgs {
    const int64_t* keys;
    int64_t tokens, rows, skip;
    int range;
    int* order;   // [tokens]: tokens by row, then by their own place
    int* starts;  // [rows + 1]: where a row's begin in `order`
};

__global__ __launch_bounds__(kSortThreads) void sort_kernel(SortArgs a) {
    __shared__ int counts[kSortWaves][kSortRange];
    __shared__ int sums[kSortWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int64_t low = static_cast<int64_t>(blockIdx.x) * a.range;
    const int range = static_cast<int>(std::min<int64_t>(a.range, a.rows - low));
    for (int i = threadIdx.x; i < kSortWaves * kSortRange; i += kSortThreads) counts[i / kSortRange][i % kSortRange] = 0;
    __syncthreads();
    // a wave's tokens are adjacent ones
    const int64_t each = ceil_div(ceil_div(a.tokens, kSortWaves), kWave) * kWave;
    const int64_t from = wave * each, to = std::min<int64_t>(from + each, a.tokens);
    int below = 0;
    for (int64_t i = from + lane; i < to; i += kWave) {
        const int64_t key = a.keys[i];
        if (key < 0 || key >= a.rows || key == a.skip) continue;
        if (key < low) ++below;
        else if (key < low + range) atomicAdd(&counts[wave][key - low], 1);  // counts have one value in any order
    }
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) below += __shfl_xor(below, by);
    if (lane == 0) sums[wave] = below;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k) before += sums[k];
    __syncthreads();
    // where each row's tokens start, and in them each wave's
    int mine = 0;
    const int row = threadIdx.x;
    if (row < range)
#pragma unroll
        for (int k = 0; k < kSortWaves; ++k) mine += counts[k][row];
    int scan = mine;
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) {
        const int other = __shfl_up(scan, by);
        if (lane >= by) scan += other;
    }
    if (lane == kWave - 1) sums[wave] = scan;
    __syncthreads();
    int at = before + scan - mine;
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k)
        if (k < wave) at += sums[k];
    if (row < range) {
        a.starts[low + row] = at;
        if (low + row == a.rows - 1) a.starts[a.rows] = at + mine;
#pragma unroll
        for (int k = 0; k < kSortWaves; ++k) {
            const int n = counts[k][row];
            counts[k][row] = at;
            at += n;
        }
    }
    __syncthreads();
    for (int64_t first = from; first < to; first += kWave) {
        const int64_t i = first + lane;
        const int64_t key = i < to ? a.keys[i] : -1;
        const bool inside = key >= low && key < low + range && key != a.skip && key >= 0;
        const int local = inside ? static_cast<int>(key - low) : -1;
        uint64_t left = __ballot(inside);
        while (left) {  // once for each row that some lane's token has
            const int leader = __builtin_ctzll(left);
            const int which = __shfl(local, leader);
            const uint64_t same = __ballot(local == which);
            int place = 0;
            if (lane == leader) place = atomicAdd(&counts[wave][which], static_cast<int>(__popcll(same)));
            place = __shfl(place, leader);
            if (local == which) a.order[place + __popcll(same & ((uint64_t{1} << lane) - 1))] = static_cast<int>(i);
            left &= ~same;
        }
    }
}

// ---- sums -----------------------------------------------------------------------------------

struct SumArgs {
    const int64_t* keys;        // null: key_t = t mod period
    const int *order, *starts;  // null without keys
    const void* dy;
    void* grad;
    float* partial;  // [tiles][2][dim]
    int64_t tokens, rows, period, tiles;
    int dim, tile;
    float scale;
};

// The list of tokens sorted by row: as sorted, or known where keys count 0 .. period - 1 again and again.
__device__ __forceinline__ int64_t start_of(const SumArgs& a, int64_t row) {
    return a.starts ? a.starts[row] : std::min(row, a.period) * (a.tokens / a.period);
}
__device__ __forceinline__ int64_t token_at(const SumArgs& a, int64_t place) {
    if (a.order) return a.order[place];
    const int64_t times = a.tokens / a.period;
    return place % times * a.period + place / times;
}
__device__ __forceinline__ int64_t row_at(const SumArgs& a, int64_t place) {
    return a.order ? a.keys[a.order[place]] : place / (a.tokens / a.period);
}

template <typename T, int N>
__device__ __forceinline__ void add_rows(const SumArgs& a, int64_t from, int64_t to, int at, float (&sum)[N]) {
    const T* dy = static_cast<const T*>(a.dy) + at;
    const int left = a.dim - at;
#pragma unroll 4
    for (int64_t i = from; i < to; ++i) {
        Pack<T, N> p;
        load_loose(p, dy + token_at(a, i) * a.dim, left);
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += static_cast<float>(p.v[e]);
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_sum(const SumArgs& a, int64_t row, int at, const float (&sum)[N]) {
    Pack<T, N> p;
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = static_cast<T>(a.scale * sum[e]);
    store_loose(static_cast<T*>(a.grad) + row * a.dim + at, p, a.dim - at);
}

// Rows of at most a tile's tokens: `lanes` threads a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void row_sum_kernel(SumArgs a, int lanes) {
    constexpr int N = 16 / sizeof(T);
    const int per_block = kThreads / lanes, lane = threadIdx.x % lanes;
    const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / lanes; v < a.rows; v += step) {
        const int64_t from = start_of(a, v), to = start_of(a, v + 1);
        if (to - from > a.tile) continue;
        for (int at = lane * N; at < a.dim; at += lanes * N) {
            float sum[N] = {};
            add_rows<T>(a, from, to, at, sum);
            store_sum<T>(a, v, at, sum);
        }
    }
}

// A tile of the sorted list: its parts of rows longer than a tile, of which it meets two at most (one that ends
// in it and one that starts in it).
template <typename T>
__global__ __launch_bounds__(kThreads) void tile_sum_kernel(SumArgs a) {
    constexpr int N = 16 / sizeof(T);
    const int64_t total = start_of(a, a.rows), k = blockIdx.x;
    const int64_t from = k * a.tile, to = std::min<int64_t>(from + a.tile, total);
    if (from >= to) return;
    const int64_t first = row_at(a, from), last = row_at(a, to - 1);
    for (int part = 0; part < 2; ++part) {
        const int64_t row = part ? last : first;
        if (part && last == first) return;
        const int64_t s = start_of(a, row), e = start_of(a, row + 1);
        if (e - s <= a.tile) continue;
        float* out = a.partial + (2 * k + part) * a.dim;
        for (int at = (blockIdx.y * kThreads + threadIdx.x) * N; at < a.dim; at += gridDim.y * kThreads * N) {
            float sum[N] = {};
            add_rows<T>(a, std::max(s, from), std::min(e, to), at, sum);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < a.dim) out[at + i] = sum[i];
        }
    }
}

// The row longer than a tile that starts in tile k, if there is one: the sum of its tiles' sums. A block takes 64
// columns, its waves every 16th tile.
template <typename T>
__global__ __launch_bounds__(kSortThreads) void tile_join_kernel(SumArgs a) {
    __shared__ float sums[kSortWaves][kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int64_t total = start_of(a, a.rows), k = blockIdx.x;
    const int64_t from = k * a.tile, to = std::min<int64_t>(from + a.tile, total);
    if (from >= to) return;
    const int64_t row = row_at(a, to - 1), s = start_of(a, row), e = start_of(a, row + 1);
    if (e - s <= a.tile || s < from) return;
    const int64_t last = (e - 1) / a.tile;
    for (int first = blockIdx.y * kWave; first < a.dim; first += gridDim.y * kWave) {
        const int at = first + lane;
        float sum = 0.0f;
        if (at < a.dim)
            for (int64_t t = k + wave; t <= last; t += kSortWaves)
                sum += a.partial[(2 * t + (t == k && s > from ? 1 : 0)) * a.dim + at];
        sums[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && at < a.dim) {
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) sum += sums[w][lane];
            static_cast<T*>(a.grad)[row * a.dim + at] = static_cast<T>(a.scale * sum);
        }
        __syncthreads();
    }
}

// ---- host -----------------------------------------------------------------------------------

// Threads of a row of `chunks` 16-byte pieces: a power of two, the whole block at most.
int lanes_of(int64_t chunks) {
    int lanes = 8;
    while (lanes < kThreads && lanes < chunks) lanes *= 2;
    return lanes;
}

// A tile's tokens: 64, and more where that would make more than 2048 tiles, whose sums are added up.
int tile_of(int64_t tokens) { return static_cast<int>(std::max<int64_t>(64, ceil_div(tokens, 2048))); }
// No row is longer than a tile where there are no more tokens.
int64_t tiles_of(int64_t tokens) { return tokens > tile_of(tokens) ? ceil_div(tokens, tile_of(tokens)) : 0; }

constexpr int64_t kMaxTokens = int64_t{1} << 30, kMaxDim = int64_t{1} << 24;

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

struct Space {
    size_t starts, partial, bytes;
    Space(int64_t tokens, int64_t rows, int64_t dim, bool has_keys) {
        starts = has_keys ? rounded(tokens * sizeof(int)) : 0;
        partial = starts + (has_keys ? rounded((rows + 1) * sizeof(int)) : 0);
        bytes = partial + static_cast<size_t>(tiles_of(tokens)) * 2 * dim * sizeof(float);
    }
};

bool sizes_fit(int64_t tokens, int64_t rows, int64_t dim) {
    return tokens >= 0 && tokens <= kMaxTokens && rows >= 0 && rows <= ISA_TRAIN_EMBEDDING_MAX_ROWS && dim >= 1 &&
           dim <= kMaxDim;
}

template <typename T>
int sums(const SumArgs& a, hipStream_t s) {
    const int lanes = lanes_of(ceil_div(a.dim, 16 / sizeof(T)));
    const int64_t blocks = std::min<int64_t>(ceil_div(a.rows, kThreads / lanes), kMaxBlocks);
    row_sum_kernel<T><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s>>>(a, lanes);
    if (int rc = launched("row_sum_kernel")) return rc;
    if (!a.tiles) return 0;
    const auto across = [&](int64_t each) { return static_cast<unsigned>(std::min<int64_t>(ceil_div(a.dim, each), 1024)); };
    const unsigned tiles = static_cast<unsigned>(a.tiles);
    tile_sum_kernel<T><<<dim3(tiles, across(kThreads * 16 / sizeof(T))), dim3(kThreads), 0, s>>>(a);
    if (int rc = launched("tile_sum_kernel")) return rc;
    tile_join_kernel<T><<<dim3(tiles, across(kWave)), dim3(kSortThreads), 0, s>>>(a);
    return launched("tile_join_kernel");
}

}  // namespace
}  // namespace isa_block

using namespace isa_block;

extern "C" int isa_train_abi_version(void) { return ISA_TRAIN_ABI_VERSION; }

extern "C" int isa_train_embedding_forward(const isa_train_embedding* e, void* y, void* stream) {
    if (!e) return fail("embedding is null");
    if (!known_type(e->type)) return fail("unknown element type %d", e->type);
    if (!sizes_fit(e->tokens, e->vocab, e->dim) || e->places < 0 || e->places > ISA_TRAIN_EMBEDDING_MAX_ROWS)
        return fail("sizes out of range: tokens %lld, tables of %lld and %lld rows, dim %lld",
                    static_cast<long long>(e->tokens), static_cast<long long>(e->vocab),
                    static_cast<long long>(e->places), static_cast<long long>(e->dim));
    if (e->tokens == 0) return 0;
    if (!e->ids || !y || (e->vocab && !e->weight)) return fail("ids, weight and y must be set");
    if (e->places && !e->place_weight) return fail("place_weight must be set");
    if (e->places && !e->place_ids && (e->period < 1 || e->tokens % e->period))
        return fail("period must divide the tokens, got %lld", static_cast<long long>(e->period));
    const size_t b = type_bytes(e->type);
    if (!aligned(y, b) || !aligned(e->weight, b) || (e->places && !aligned(e->place_weight, b)))
        return fail("y or a table is not aligned to its type");
    const LookupArgs a{e->ids,           e->place_ids, e->weight, e->place_weight, y, e->tokens, e->vocab, e->weight_stride, e->places,
                       e->places_stride, e->period,    static_cast<int>(e->dim), e->scale};
    const int lanes = lanes_of(ceil_div(e->dim, static_cast<int64_t>(16 / b)));
    const int64_t blocks = std::min<int64_t>(ceil_div(e->tokens, kThreads / lanes), kMaxBlocks);
    const dim3 grid(static_cast<unsigned>(blocks));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (e->type == ISA_BLOCK_F32) lookup_kernel<float><<<grid, dim3(kThreads), 0, s>>>(a, lanes);
    else if (e->type == ISA_BLOCK_BF16) lookup_kernel<bf16><<<grid, dim3(kThreads), 0, s>>>(a, lanes);
    else lookup_kernel<f16><<<grid, dim3(kThreads), 0, s>>>(a, lanes);
    return launched("lookup_kernel");
}

extern "C" size_t isa_train_embedding_backward_workspace(int64_t tokens, int64_t rows, int64_t dim, int has_keys) {
    return sizes_fit(tokens, rows, dim) ? Space(tokens, rows, dim, has_keys != 0).bytes : 0;
}

extern "C" int isa_train_embedding_backward(int type, int64_t tokens, int64_t rows, int64_t dim, const int64_t* keys,
                                            int64_t period, int64_t skip, float scale, const void* dy, void* grad,
                                            void* workspace, size_t workspace_bytes, void* stream) {
    if (!known_type(type)) return fail("unknown element type %d", type);
    if (!sizes_fit(tokens, rows, dim))
        return fail("sizes out of range: tokens %lld, rows %lld, dim %lld", static_cast<long long>(tokens),
                    static_cast<long long>(rows), static_cast<long long>(dim));
    if (rows == 0) return 0;
    if (!grad || (tokens && !dy)) return fail("grad_y and grad must be set");
    if (!aligned(grad, type_bytes(type)) || !aligned(dy, type_bytes(type)))
        return fail("grad_y or grad is not aligned to its type");
    if (tokens && !keys && (period < 1 || tokens % period))
        return fail("period must divide the tokens, got %lld", static_cast<long long>(period));
    const bool has_keys = keys && tokens;
    const Space at(tokens, rows, dim, has_keys);
    if (workspace_bytes < at.bytes) return fail("workspace too small: %zu bytes", workspace_bytes);
    if (at.bytes && (!workspace || !aligned(workspace, 256))) return fail("workspace must be 256-byte aligned");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    SumArgs a{};
    if (has_keys) {
        SortArgs b{keys, tokens, rows, skip, 0, reinterpret_cast<int*>(ws), reinterpret_cast<int*>(ws + at.starts)};
        b.range = static_cast<int>(std::min<int64_t>(ceil_div(rows, kSortBlocks), kSortRange));
        sort_kernel<<<dim3(static_cast<unsigned>(ceil_div(rows, b.range))), dim3(kSortThreads), 0, s>>>(b);
        if (int rc = launched("sort_kernel")) return rc;
        a.keys = keys;
        a.order = b.order;
        a.starts = b.starts;
    }
    a.dy = dy;
    a.grad = grad;
    a.partial = reinterpret_cast<float*>(ws + at.partial);
    a.tokens = tokens;
    a.rows = rows;
    a.period = has_keys || !tokens ? 1 : period;
    a.tiles = tiles_of(tokens);
    a.dim = static_cast<int>(dim);
    a.tile = tile_of(tokens);
    a.scale = scale;
    if (type == ISA_BLOCK_F32) return sums<float>(a, s);
    if (type == ISA_BLOCK_BF16) return sums<bf16>(a, s);
    return sums<f16>(a, s);
}
