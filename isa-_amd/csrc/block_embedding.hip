// Embedding lookup of tokens and places, and the tables' gradients, for gfx950.
//
//   y_t = round(scale W[id_t] + P[place_t]),   dW_v = scale sum_{t: id_t = v} dy_t
//
// Both are bound by HBM: the lookup reads and writes rows, the gradient reads dy and writes all of dW, most of
// whose rows are zeros. The gradient's sums use no atomics: tokens are sorted by their row, in order within
// one, and a row's sum is taken in that order.
//
// The sort needs no exchange between its blocks: a block owns a range of rows, reads all keys, counts those
// below its range (where its part of the list starts) and places those inside. It runs in the lookup's launch.
// A row with many tokens would be one wave's long walk: lists longer than a tile are summed by tiles of
// the sorted list, in the rows' launch, and a third launch adds up their sums. Both tables share the launches.
//
// 65536 tokens of a 50304 x 1024 bf16 table: lookup with its sort 31 us (162 MB), rows and tiles 37 (237 MB, 6.4 TB/s),
// join 7; 8192 tokens of 50304 x 768 and 1024 x 768 in fp32: 13, 34 (207 MB) and 4.
#include "block_common.hpp"

#include <algorithm>

#include "isa_train.h"

namespace isa_block {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 8192;

// ---- columns ------------------------------------------------------------------------------

// 16 bytes of a row of `dim` elements from column `at` on, which ends with the row: a row's last piece starts
// earlier where its width is no multiple, and two lanes then have the same elements with the same values. So all loads
// and stores are whole vectors, at any element's address. SHORT: rows of less than 16 bytes, element by element.
template <typename T>
constexpr int kPiece = 16 / sizeof(T);

template <typename T, bool SHORT>
__device__ __forceinline__ int piece_at(int column, int dim) {
    return SHORT ? 0 : std::min(column, dim - kPiece<T>);
}

template <typename T, bool SHORT>
__device__ __forceinline__ void load_piece(vec<T, kPiece<T>>& p, const T* from, int dim) {
    if constexpr (SHORT) {
#pragma unroll
        for (int e = 0; e < kPiece<T>; ++e) p[e] = e < dim ? from[e] : static_cast<T>(0.0f);
    } else {
        p = *reinterpret_cast<const typename Loose<T, kPiece<T>>::type*>(from);
    }
}

// `past`: the caches, for results too large to be found there by their reader.
template <typename T, bool SHORT>
__device__ __forceinline__ void store_piece(T* to, const vec<T, kPiece<T>>& p, int dim, bool past) {
    using V = typename Loose<T, kPiece<T>>::type;
    if constexpr (SHORT) {
#pragma unroll
        for (int e = 0; e < kPiece<T>; ++e)
            if (e < dim) to[e] = p[e];
    } else if (past) {
        asm volatile("");  // two stores of one value to one place become one, of the ordinary kind: not with these between
        __builtin_nontemporal_store(static_cast<V>(p), reinterpret_cast<V*>(to));
        asm volatile("");
    } else {
        *reinterpret_cast<V*>(to) = p;
    }
}

// ---- lookup -------------------------------------------------------------------------------

struct LookupArgs {
    const int64_t *ids, *place_ids;
    const void *weight, *place_weight;
    void* y;
    int64_t tokens, vocab, weight_stride, places, places_stride, period;
    int dim;
    float scale;
    bool past;  // the caches, for y
};

// `lanes` threads of a block take K adjacent tokens at a time, whose ids and then whose rows are in flight together.
template <typename T, bool PLACES, bool SHORT, int K, int THREADS>
__device__ __forceinline__ void look_up(const LookupArgs& a, int lanes, int block, int blocks) {
    constexpr int N = kPiece<T>;
    const int per_block = THREADS / lanes, group = threadIdx.x / lanes, lane = threadIdx.x - group * lanes;
    if (group >= per_block) return;
    const int64_t step = static_cast<int64_t>(blocks) * per_block * K;
    for (int64_t t = (static_cast<int64_t>(block) * per_block + group) * K; t < a.tokens; t += step) {
        int64_t id[K], place[K];
#pragma unroll
        for (int k = 0; k < K; ++k) id[k] = a.ids[std::min(t + k, a.tokens - 1)];
        if constexpr (PLACES) {
            if (a.place_ids)
#pragma unroll
                for (int k = 0; k < K; ++k) place[k] = a.place_ids[std::min(t + k, a.tokens - 1)];
            else
#pragma unroll
                for (int k = 0; k < K; ++k)
                    place[k] = static_cast<uint32_t>(std::min(t + k, a.tokens - 1)) % static_cast<uint32_t>(a.period);
        }
        __builtin_amdgcn_sched_barrier(0);  // all of them before the first is waited for
        const T *w[K], *p[K];
        bool inside[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            inside[k] = static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(a.vocab);
            if constexpr (PLACES) {
                inside[k] = inside[k] & (static_cast<uint64_t>(place[k]) < static_cast<uint64_t>(a.places));
                p[k] = static_cast<const T*>(a.place_weight) + (inside[k] ? place[k] : 0) * a.places_stride;
            }
            w[k] = static_cast<const T*>(a.weight) + (inside[k] ? id[k] : 0) * a.weight_stride;
        }
        for (int column = lane * N; column < a.dim; column += lanes * N) {
            const int at = piece_at<T, SHORT>(column, a.dim);
            vec<T, N> r[K], q[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                load_piece<T, SHORT>(r[k], w[k] + at, a.dim);
                if constexpr (PLACES) load_piece<T, SHORT>(q[k], p[k] + at, a.dim);
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (t + k >= a.tokens) break;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float x = static_cast<float>(r[k][e]);
                    const float y = PLACES ? fmaf(a.scale, x, static_cast<float>(q[k][e])) : a.scale * x;
                    r[k][e] = static_cast<T>(inside[k] ? y : NAN);
                }
                store_piece<T, SHORT>(static_cast<T*>(a.y) + (t + k) * a.dim + at, r[k], a.dim, a.past);
            }
        }
    }
}

// ---- the tokens of each row ---------------------------------------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortRange = 512;  // rows of a block: 32 KiB of counters, so that blocks share a compute unit
constexpr int kSortBlocks = 128;  // 13.3 us with the lookup of 8192 x 768 in fp32; 256, which leave it less room, 17.6
constexpr int kSortBatch = 8;  // keys of a lane in flight
constexpr int kSortFound = 448;  // tokens of its range that a wave keeps: 28 KiB
// Up to so many of a step's tokens inside find their row's others in a turn a row, more by the bits of their rows. Steps of
// 131072 tokens of 50304 x 256 in bf16, ids numbered by frequency (the first block's are half of all) and in any order:
// 165 and 102 us; up to 6 165 and 110, by bits alone 162 and 145, by turns alone, each with its counter, 838 and 112.
constexpr int kSortTurns = 12;
constexpr int kSortListed = (1 << 30) / kSortRange * 4;  // tokens of a wave that 32 bits number beside their rows

struct SortArgs {
    const int64_t* keys;
    uint32_t skip;
    int tokens, rows, range, blocks;
    int* order;   // [tokens]: tokens by row, then by their own place
    int* starts;  // [rows + 1]: where a row's begin in `order`
};

// A key as a row, or one that no block has.
__device__ __forceinline__ uint32_t row_of(int64_t key, const SortArgs& a) {
    const uint32_t low = static_cast<uint32_t>(key), high = static_cast<uint32_t>(static_cast<uint64_t>(key) >> 32);
    return high != 0 || low >= static_cast<uint32_t>(a.rows) || low == a.skip ? ~0u : low;
}

// The tokens of one step of a wave into their rows' lists: `local` is a token's row in the range, if inside. A lane finds
// the others of its row, and the first of them moves the wave's own counter.
__device__ __forceinline__ void place_tokens(const SortArgs& a, int* next, uint32_t local, bool inside, int token, int lane) {
    uint64_t left = __ballot(inside), same = left;
    if (!left) return;
    if (__popcll(left) <= kSortTurns) {
        while (left) {  // once for each row that some lane's token has
            const uint32_t which = __builtin_amdgcn_readlane(local, __builtin_ctzll(left));
            const uint64_t its = __ballot(inside && local == which);
            if (local == which) same = its;
            left &= ~its;
        }
    } else {
        for (uint32_t bit = 1; bit < static_cast<uint32_t>(a.range); bit *= 2) {  // those that agree in every bit
            const uint64_t set = __ballot(local & bit);
            same &= local & bit ? set : ~set;
        }
    }
    if (!inside) return;
    const uint64_t before = same & ((uint64_t{1} << lane) - 1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the counter as the last step left it,
    const int place = next[local];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // read by all lanes before one moves it
    if (!before) next[local] = place + static_cast<int>(__popcll(same));
    a.order[place + __popcll(before)] = token;
}

__device__ void sort_range(const SortArgs& a, int block) {
    __shared__ int counts[kSortWaves * kSortRange];
    __shared__ uint32_t found[kSortWaves][kSortFound];
    __shared__ int sums[kSortWaves];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t low = static_cast<uint32_t>(block) * a.range;
    const uint32_t range = std::min<uint32_t>(a.range, a.rows - low);
    for (uint32_t i = threadIdx.x; i < kSortWaves * range; i += kSortThreads) counts[i] = 0;
    __syncthreads();
    int* mine = counts + wave * range;
    // a wave's tokens are adjacent ones
    const int each = static_cast<int>(ceil_div(ceil_div(a.tokens, kSortWaves), kWave) * kWave);
    const int64_t from = static_cast<int64_t>(wave) * each;
    const int n = static_cast<int>(std::max<int64_t>(0, std::min<int64_t>(each, a.tokens - from)));
    const int64_t* keys = a.keys + from;
    const uint64_t before_me = (uint64_t{1} << lane) - 1;
    int below = 0, listed = 0;
    for (int first = 0; first < n; first += kSortBatch * kWave) {
        int64_t key[kSortBatch];
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k) {
            const int i = first + k * kWave + lane;
            key[k] = i < n ? keys[i] : -1;
        }
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k) {
            const uint32_t row = row_of(key[k], a), local = row - low;
            const bool inside = local < range;
            if (row < low) ++below;
            if (const uint64_t mask = __ballot(inside)) {
                const int at = listed + static_cast<int>(__popcll(mask & before_me));
                if (inside) {
                    atomicAdd(&mine[local], 1);  // counts have one value in any order
                    if (at < kSortFound) found[wave][at] = static_cast<uint32_t>(first + k * kWave + lane) * kSortRange + local;
                }
                listed += static_cast<int>(__popcll(mask));
            }
        }
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
    const uint32_t row = threadIdx.x;
    int count = 0;
    if (row < range)
#pragma unroll
        for (int k = 0; k < kSortWaves; ++k) count += counts[k * range + row];
    int scan = count;
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) {
        const int other = __shfl_up(scan, by);
        if (lane >= by) scan += other;
    }
    if (lane == kWave - 1) sums[wave] = scan;
    __syncthreads();
    int at = before + scan - count;
#pragma unroll
    for (int k = 0; k < kSortWaves; ++k)
        if (k < wave) at += sums[k];
    if (row < range) {
        a.starts[low + row] = at;
        if (low + row == static_cast<uint32_t>(a.rows) - 1) a.starts[a.rows] = at + count;
#pragma unroll
        for (int k = 0; k < kSortWaves; ++k) {
            const int c = counts[k * range + row];
            counts[k * range + row] = at;
            at += c;
        }
    }
    __syncthreads();
    // the tokens that were found, in their order, or all keys again where those did not fit
    if (listed <= kSortFound && n <= kSortListed) {
        for (int i = lane; i - lane < listed; i += kWave) {
            const bool inside = i < listed;
            const uint32_t f = inside ? found[wave][i] : 0;
            place_tokens(a, mine, f % kSortRange, inside, static_cast<int>(from) + static_cast<int>(f / kSortRange), lane);
        }
        return;
    }
    for (int first = 0; first < n; first += kSortBatch * kWave) {
        int64_t key[kSortBatch];
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k) {
            const int i = first + k * kWave + lane;
            key[k] = i < n ? keys[i] : -1;
        }
#pragma unroll
        for (int k = 0; k < kSortBatch; ++k) {
            const uint32_t local = row_of(key[k], a) - low;
            place_tokens(a, mine, local, local < range, static_cast<int>(from) + first + k * kWave + lane, lane);
        }
    }
}

// The lookup and, for a backward pass, both tables' sorts: they need the ids alone, and their few blocks, whose time
// is latency, run beside the lookup's: two blocks of 1024 threads share a compute unit, hence at most 64 registers.
// THREADS 256: a lookup without sorts.
template <typename T, bool PLACES, bool SHORT, int K, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS == kSortThreads ? 8 : 1) void lookup_kernel(LookupArgs a, int lanes, SortArgs first, SortArgs second) {
    int block = static_cast<int>(blockIdx.x), blocks = static_cast<int>(gridDim.x);
    if constexpr (THREADS == kSortThreads) {
        if (block < first.blocks) return sort_range(first, block);
        block -= first.blocks;
        if (block < second.blocks) return sort_range(second, block);
        block -= second.blocks;
        blocks -= first.blocks + second.blocks;
    }
    look_up<T, PLACES, SHORT, K, THREADS>(a, lanes, block, blocks);
}

// ---- sums -----------------------------------------------------------------------------------

constexpr int kJoinThreads = 512, kJoinTiles = 4, kFewThreads = 1024;

struct SumArgs {
    const int64_t* keys;        // null: key_t = t mod period
    const int *order, *starts;  // null without keys
    const void* dy;
    void* grad;
    float* partial;  // [tiles][2][dim]
    int* joins;      // [tiles]: the row longer than a tile that starts in a tile, or -1
    int rows, period, times;  // without keys: tokens / period
    int dim, tile, tiles;
    int each;                // rows of a group of lanes
    int tile_blocks, blocks;  // of the tiles, in all
    float scale;
    bool past;  // the caches, for grad
};

// The list of tokens sorted by row: as sorted, or known where keys count 0 .. period - 1 again and again.
__device__ __forceinline__ int start_of(const SumArgs& a, int row) {
    return a.starts ? a.starts[row] : std::min(row, a.period) * a.times;
}
__device__ __forceinline__ int token_at(const SumArgs& a, int place) {
    if (a.order) return a.order[place];
    return place % a.times * a.period + place / a.times;
}
// (Held to the table: keys that were overwritten since they were sorted give wrong sums, not other memory.)
__device__ __forceinline__ int row_at(const SumArgs& a, int place) {
    if (!a.order) return place / a.times;
    return static_cast<int>(std::min<uint64_t>(static_cast<uint64_t>(a.keys[a.order[place]]), static_cast<uint64_t>(a.rows - 1)));
}

// `from`'s value in a group of LANES lanes: uniform in a wave where that is the group.
template <int LANES>
__device__ __forceinline__ int lane_value(int x, int from) {
    if constexpr (LANES == kWave) return __builtin_amdgcn_readlane(x, from);
    return __shfl(x, from, LANES);
}

// A group of LANES lanes, whose lanes hold C pieces of a row each, LANES apart. (Lanes past a row's end read its
// last piece, too, and write nothing.)
template <typename T, int LANES, int C, bool SHORT>
struct Group {
    static constexpr int N = kPiece<T>;
    static constexpr int kBatch = C <= 2 ? 8 : 4;  // rows in flight
    const SumArgs& a;
    int lane, first;  // lane of the group, column of its first piece
    int at[C];        // where its pieces start
    int end;          // of the places that it may add
    int base, token;  // the tokens of places base .. base + LANES - 1 up to the end, one a lane
    float sum[C][N];

    __device__ Group(const SumArgs& args, int columns, int places_end)
        : a(args), lane(threadIdx.x % LANES), end(places_end), base(-LANES - 1), token(0) {
        first = columns + lane * N;
#pragma unroll
        for (int c = 0; c < C; ++c) at[c] = piece_at<T, SHORT>(first + c * LANES * N, a.dim);
    }
    __device__ void clear() {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < N; ++e) sum[c][e] = 0.0f;
    }
    // rows [place, place + K) of the list, of which the group's lanes know the tokens
    template <int K>
    __device__ __forceinline__ void add_batch(int place) {
        vec<T, N> p[K][C];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t t = lane_value<LANES>(token, place - base + k);
            const T* row = static_cast<const T*>(a.dy) + t * a.dim;
#pragma unroll
            for (int c = 0; c < C; ++c) load_piece<T, SHORT>(p[k][c], row + at[c], a.dim);
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[c][e] += static_cast<float>(p[k][c][e]);
    }
    __device__ __forceinline__ void add(int from, int to) {
        for (int i = from; i < to; i += kBatch) {
            const int n = std::min(kBatch, to - i);
            if (i < base || i + n > base + LANES) {
                base = i;
                token = i + lane < end ? token_at(a, i + lane) : 0;
            }
            if (n == kBatch) {
                add_batch<kBatch>(i);
                continue;
            }
            int done = 0;
            if (kBatch > 4 && n & 4) add_batch<4>(i), done = 4;
            if (n & 2) add_batch<2>(i + done), done += 2;
            if (n & 1) add_batch<1>(i + done);
        }
    }
    __device__ void store(int row) const {
        T* out = static_cast<T*>(a.grad) + static_cast<int64_t>(row) * a.dim;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (first + c * LANES * N >= a.dim) break;
            vec<T, N> p;
#pragma unroll
            for (int e = 0; e < N; ++e) p[e] = static_cast<T>(a.scale * sum[c][e]);
            store_piece<T, SHORT>(out + at[c], p, a.dim, a.past);
        }
    }
    __device__ void store_partial(int64_t slot) const {
        float* out = a.partial + slot * a.dim;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (first + c * LANES * N >= a.dim) break;
#pragma unroll
            for (int h = 0; h < N; h += 4) {
                vec<float, 4> p;
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = sum[c][h + e];
                if constexpr (SHORT) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (h + e < a.dim) out[h + e] = p[e];
                } else {
                    *reinterpret_cast<Loose<float, 4>::type*>(out + at[c] + h) = p;
                }
            }
        }
    }
};

// A tile of the sorted list: its parts of rows longer than a tile, of which it meets two at most (one that ends
// in it and one that starts in it).
template <typename T, int LANES, int C, bool SHORT>
__device__ __forceinline__ void sum_tile(const SumArgs& a, int k, int columns) {
    const int from = k * a.tile, to = std::min(from + a.tile, start_of(a, a.rows));
    Group<T, LANES, C, SHORT> g(a, columns, to);
    int join = -1;
    if (from < to) {
        const int ends[2] = {row_at(a, from), row_at(a, to - 1)};
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const int row = ends[part];
            if (part && row == ends[0]) break;
            const int s = start_of(a, row), e = start_of(a, row + 1);
            if (e - s <= a.tile) continue;
            if (s >= from) join = row;
            g.clear();
            g.add(std::max(s, from), std::min(e, to));
            g.store_partial(2 * static_cast<int64_t>(k) + part);
        }
    }
    if (g.lane == 0 && columns == 0) a.joins[k] = join;
}

// Rows of at most a tile's tokens, `each` adjacent ones: where they start is one load, and so are their tokens. Returns
// which of them were longer.
template <typename T, int LANES, int C, bool SHORT>
__device__ __forceinline__ uint64_t sum_rows(const SumArgs& a, int64_t row, int columns) {
    const int n = static_cast<int>(std::min<int64_t>(a.each, a.rows - row));
    if (n <= 0) return 0;
    const int start = start_of(a, static_cast<int>(row) + std::min<int>(threadIdx.x % LANES, n));
    Group<T, LANES, C, SHORT> g(a, columns, lane_value<LANES>(start, n));
    uint64_t longer = 0;
    for (int r = 0; r < n; ++r) {
        const int s = lane_value<LANES>(start, r), e = lane_value<LANES>(start, r + 1);
        if (e - s > a.tile) {
            longer |= uint64_t{1} << r;
            continue;
        }
        g.clear();
        g.add(s, e);
        g.store(static_cast<int>(row) + r);
    }
    return longer;
}

// The longer rows of a block's groups, by all of its groups: each a part of a row's tokens, added up in LDS.
template <typename T, int LANES, int C, bool SHORT>
__device__ __forceinline__ void sum_longer(const SumArgs& a, int64_t first_row, uint64_t longer, int columns) {
    constexpr int kGroups = kFewThreads / LANES, N = kPiece<T>;
    __shared__ uint64_t masks[kGroups];
    __shared__ float sums[kGroups][C * N][LANES];
    const int group = threadIdx.x / LANES;
    Group<T, LANES, C, SHORT> g(a, columns, start_of(a, a.rows));
    if (g.lane == 0) masks[group] = longer;
    __syncthreads();
    for (int k = 0; k < kGroups; ++k) {
        for (uint64_t left = masks[k]; left; left &= left - 1) {
            const int row = static_cast<int>(first_row) + k * a.each + __builtin_ctzll(left);
            const int s = start_of(a, row), e = start_of(a, row + 1), part = static_cast<int>(ceil_div(e - s, kGroups));
            const int from = s + group * part;
            g.clear();
            g.add(from, std::min(from + part, e));
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < N; ++i) sums[group][c * N + i][g.lane] = g.sum[c][i];
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        float all = 0.0f;
                        for (int w = 0; w < kGroups; ++w) all += sums[w][c * N + i][g.lane];
                        g.sum[c][i] = all;
                    }
                g.store(row);
            }
            __syncthreads();
        }
    }
}

// FEW tokens: rows alone, the longer ones by a whole block, and nothing is left to join. Else the first blocks take
// tiles, which have the longest walks, the others rows.
template <typename T, int LANES, int C, bool SHORT, bool FEW>
__global__ __launch_bounds__(FEW ? kFewThreads : kThreads, FEW ? 4 : 1) void sum_kernel(SumArgs first, SumArgs second) {
    constexpr int kGroups = (FEW ? kFewThreads : kThreads) / LANES;
    int block = static_cast<int>(blockIdx.x);
    const bool other = block >= first.blocks;
    if (other) block -= first.blocks;
    const SumArgs& a = other ? second : first;
    const int columns = static_cast<int>(blockIdx.y) * LANES * C * kPiece<T>;
    int group = threadIdx.x / LANES;
    if constexpr (LANES == kWave) group = __builtin_amdgcn_readfirstlane(group);
    if (!FEW && block < a.tile_blocks) {
        const int k = block * kGroups + group;
        if (k < a.tiles) sum_tile<T, LANES, C, SHORT>(a, k, columns);
        return;
    }
    const int64_t row = static_cast<int64_t>(block - a.tile_blocks) * kGroups * a.each;
    const uint64_t longer = sum_rows<T, LANES, C, SHORT>(a, row + group * a.each, columns);
    if constexpr (FEW) sum_longer<T, LANES, C, SHORT>(a, row, longer, columns);
}

// Rows longer than a tile, those that start in a block's tiles: the sum of their tiles' sums. A block takes 256
// columns, its waves every eighth tile.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(SumArgs first, SumArgs second, int first_blocks) {
    constexpr int kWaves = kJoinThreads / kWave, N = 4;
    __shared__ float sums[kWaves][kWave * N];
    int block = static_cast<int>(blockIdx.x);
    const bool other = block >= first_blocks;
    if (other) block -= first_blocks;
    const SumArgs& a = other ? second : first;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int mine = block * kJoinTiles + lane < a.tiles && lane < kJoinTiles ? a.joins[block * kJoinTiles + lane] : -1;
    for (uint64_t left = __ballot(mine >= 0); left; left &= left - 1) {
        const int at = __builtin_ctzll(left), k = block * kJoinTiles + at;
        const int row = __builtin_amdgcn_readlane(mine, at);
        const int s = start_of(a, row), last = (start_of(a, row + 1) - 1) / a.tile;
        for (int columns = static_cast<int>(blockIdx.y) * kWave * N; columns < a.dim;
             columns += static_cast<int>(gridDim.y) * kWave * N) {
            const int c = columns + lane * N;
            float sum[N] = {};
#pragma unroll 4
            for (int t = k + wave; t <= last; t += kWaves) {
                // (the row's first tile holds it second where another row ends in it)
                const int64_t slot = 2 * static_cast<int64_t>(t) + (t == k && s > k * a.tile ? 1 : 0);
                Pack<float, N> p;
                load_loose(p, a.partial + slot * a.dim + c, a.dim - c);
#pragma unroll
                for (int e = 0; e < N; ++e) sum[e] += p.v[e];
            }
#pragma unroll
            for (int e = 0; e < N; ++e) sums[wave][e * kWave + lane] = sum[e];
            __syncthreads();
            if (wave == 0) {
                Pack<T, N> p;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    float all = 0.0f;
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) all += sums[w][e * kWave + lane];
                    p.v[e] = static_cast<T>(a.scale * all);
                }
                store_loose(static_cast<T*>(a.grad) + static_cast<int64_t>(row) * a.dim + c, p, a.dim - c);
            }
            __syncthreads();
        }
    }
}

// ---- host -----------------------------------------------------------------------------------

// A tile's tokens: 16, and more where that would make more than 2048 tiles, whose sums are added up (65536 tokens by 32:
// rows and tiles 62 us and the join 7; by 64 65 and 7, by 16 63 and 12).
int tile_of(int64_t tokens) { return static_cast<int>(std::max<int64_t>(16, ceil_div(tokens, 2048))); }

// So many need no tiles in tables of so many bytes: a row of all of them is a walk of 128 tokens for each wave of a block, and
// a launch less (a step of 999 tokens of a 5003 x 390 bf16 table 49 us, by tiles 54). Larger tables' rows are written by
// waves that take more of a row: the gradient of 131072 x 1024 in bf16 51 us by tiles, else 66.
constexpr int64_t kFewTokens = 2048, kFewBytes = int64_t{32} << 20;

// Results that are written past the caches: y from half the last cache's size on, which the next operator reads, a
// gradient from a quarter on, which waits for the optimizer. A step of 65536 tokens of a 50304 x 1024 bf16 table: 110
// us on inputs that change, 119 through the caches (y alone 114, the gradient alone 117); of 8192 tokens of 50304 x 768 in
// fp32 59 and 61.5. With one set of inputs that the cache holds the latter's gradient takes 34 us past it, 30 in it.
// Rows of whole lines alone: parts of one line, of two waves, would each be a write of its own there.
constexpr size_t kResultPast = size_t{128} << 20, kGradientPast = size_t{64} << 20, kLine = 128;

constexpr int64_t kMaxTokens = int64_t{1} << 30;

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

// One table's parts of the lists that a lookup leaves and of a backward call's workspace.
struct Space {
    int64_t tiles = 0;
    size_t starts = 0, lists = 0;       // bytes before the lists' starts, in all
    size_t partial = 0, workspace = 0;  // bytes before the partial sums, in all
    Space() = default;                  // of a table that is not there
    Space(int64_t tokens, int64_t rows, int64_t dim, bool few, bool keys, int64_t period) {
        const int tile = tile_of(tokens);
        // of few tokens a row's block takes longer ones; without keys all rows have one length
        tiles = !few && tokens > tile && (keys || tokens / period > tile) ? ceil_div(tokens, tile) : 0;
        starts = keys ? rounded(tokens * sizeof(int)) : 0;
        lists = starts + (keys ? rounded((rows + 1) * sizeof(int)) : 0);
        partial = rounded(tiles * sizeof(int));
        workspace = partial + rounded(static_cast<size_t>(tiles) * 2 * dim * sizeof(float));
    }
};

int check(const isa_train_embedding* e) {
    if (!e) return fail("embedding is null");
    if (!known_type(e->type)) return fail("unknown element type %d", e->type);
    if (e->tokens < 0 || e->tokens > kMaxTokens || e->vocab < 0 || e->vocab > ISA_TRAIN_EMBEDDING_MAX_ROWS ||
        e->places < 0 || e->places > ISA_TRAIN_EMBEDDING_MAX_ROWS || e->dim < 1 ||
        e->dim > ISA_TRAIN_EMBEDDING_MAX_DIM)
        return fail("sizes out of range: tokens %lld, tables of %lld and %lld rows, dim %lld",
                    static_cast<long long>(e->tokens), static_cast<long long>(e->vocab),
                    static_cast<long long>(e->places), static_cast<long long>(e->dim));
    if (e->tokens && !e->ids) return fail("ids must be set");
    if (e->tokens && e->places && !e->place_ids && (e->period < 1 || e->tokens % e->period))
        return fail("period must divide the tokens, got %lld", static_cast<long long>(e->period));
    return 0;
}

// Whether no tiles are made: of few tokens, for tables that are not large.
bool few_of(const isa_train_embedding* e) {
    return e->tokens <= kFewTokens &&
           std::max(e->vocab, e->places) * e->dim * static_cast<int64_t>(type_bytes(e->type)) <= kFewBytes;
}

Space space_of(const isa_train_embedding* e, bool places) {
    if (!places) return Space(e->tokens, e->vocab, e->dim, few_of(e), true, 1);
    if (e->places == 0) return Space();  // whose period may be anything
    return Space(e->tokens, e->places, e->dim, few_of(e), e->place_ids != nullptr, e->tokens ? e->period : 1);
}

// Rows of a group: so many that some 8192 groups of 64 lanes take them all, at most the lanes that know where they
// start.
int rows_each(int64_t rows, int lanes, int64_t across) {
    return static_cast<int>(std::min<int64_t>(lanes - 1, std::max<int64_t>(1, ceil_div(rows * across * lanes, 8192 * kWave))));
}

struct Jobs {
    SumArgs sum[2];
};

template <typename T, int LANES, int C, bool FEW, bool SHORT = false>
int launch_sums(Jobs& j, hipStream_t s) {
    constexpr int N = kPiece<T>, kBlock = FEW ? kFewThreads : kThreads, kGroups = kBlock / LANES;
    const int64_t dim = std::max(j.sum[0].dim, j.sum[1].dim), across = ceil_div(dim, LANES * C * N);
    for (SumArgs& a : j.sum) {
        if (a.rows == 0) continue;
        a.each = rows_each(a.rows, LANES, across);
        a.tile_blocks = static_cast<int>(ceil_div(a.tiles, kGroups));
        a.blocks = a.tile_blocks + static_cast<int>(ceil_div(ceil_div(a.rows, a.each), kGroups));
    }
    // a grid's second dimension ends at 65535: 2^20 columns of fp32 are 4096 times 64 lanes of 4
    const dim3 grid(static_cast<unsigned>(j.sum[0].blocks + j.sum[1].blocks), static_cast<unsigned>(across));
    sum_kernel<T, LANES, C, SHORT, FEW><<<grid, dim3(kBlock), 0, s>>>(j.sum[0], j.sum[1]);
    if (int rc = launched("sum_kernel")) return rc;
    const int64_t blocks[2] = {ceil_div(j.sum[0].tiles, kJoinTiles), ceil_div(j.sum[1].tiles, kJoinTiles)};
    if (blocks[0] + blocks[1] == 0) return 0;
    const dim3 joins(static_cast<unsigned>(blocks[0] + blocks[1]),
                     static_cast<unsigned>(std::min<int64_t>(ceil_div(dim, kWave * 4), 1024)));
    join_kernel<T><<<joins, dim3(kJoinThreads), 0, s>>>(j.sum[0], j.sum[1], static_cast<int>(blocks[0]));
    return launched("join_kernel");
}

// Lanes of a group and pieces of a lane: a row's columns, at most 256 pieces at a time. Few tokens: one piece a lane, so
// that a long row's walk is shared by the blocks of its columns, too.
template <typename T>
int sums(Jobs& j, int64_t dim, bool few, hipStream_t s) {
    const int64_t pieces = ceil_div(dim, static_cast<int64_t>(kPiece<T>));
    if (few) {
        if (dim < kPiece<T>) return launch_sums<T, 8, 1, true, true>(j, s);
        if (pieces <= 8) return launch_sums<T, 8, 1, true>(j, s);
        if (pieces <= 16) return launch_sums<T, 16, 1, true>(j, s);
        if (pieces <= 32) return launch_sums<T, 32, 1, true>(j, s);
        return launch_sums<T, 64, 1, true>(j, s);
    }
    if (dim < kPiece<T>) return launch_sums<T, 8, 1, false, true>(j, s);
    if (pieces <= 8) return launch_sums<T, 8, 1, false>(j, s);
    if (pieces <= 16) return launch_sums<T, 16, 1, false>(j, s);
    if (pieces <= 32) return launch_sums<T, 32, 1, false>(j, s);
    if (pieces <= 64) return launch_sums<T, 64, 1, false>(j, s);
    if (pieces <= 128) return launch_sums<T, 64, 2, false>(j, s);
    if (pieces <= 192) return launch_sums<T, 64, 3, false>(j, s);
    return launch_sums<T, 64, 4, false>(j, s);
}

// The sorts of a table's tokens into its part of the lists.
SortArgs sort_of(const isa_train_embedding* e, bool places, int64_t skip, char* lists) {
    SortArgs o{};
    const int64_t rows = places ? e->places : e->vocab;
    o.keys = places ? e->place_ids : e->ids;
    o.skip = places || skip < 0 || skip >= rows ? ~0u : static_cast<uint32_t>(skip);
    o.tokens = static_cast<int>(e->tokens);
    o.rows = static_cast<int>(rows);
    o.range = static_cast<int>(std::min<int64_t>(ceil_div(rows, kSortBlocks), kSortRange));
    o.blocks = rows ? static_cast<int>(ceil_div(rows, o.range)) : 0;
    o.order = reinterpret_cast<int*>(lists);
    o.starts = reinterpret_cast<int*>(lists + space_of(e, places).starts);
    return o;
}

template <typename T, bool PLACES, bool SHORT, int K>
void launch_lookup(const LookupArgs& a, const SortArgs (&sorts)[2], int lanes, hipStream_t s) {
    const int others = sorts[0].blocks + sorts[1].blocks, threads = others ? kSortThreads : kThreads;
    const int64_t blocks = std::min<int64_t>(ceil_div(ceil_div(a.tokens, K), threads / lanes), kMaxBlocks) + others;
    const dim3 grid(static_cast<unsigned>(blocks)), block(threads);
    if (others) lookup_kernel<T, PLACES, SHORT, K, kSortThreads><<<grid, block, 0, s>>>(a, lanes, sorts[0], sorts[1]);
    else lookup_kernel<T, PLACES, SHORT, K, kThreads><<<grid, block, 0, s>>>(a, lanes, sorts[0], sorts[1]);
}

// Four tokens at a time (two with places, within 64 registers) where that leaves work for every compute unit: 37 us for
// 65536 x 1024 in bf16 without a sort, one by one 49.
template <typename T, bool PLACES>
void launch_lookup(const LookupArgs& a, const SortArgs (&sorts)[2], hipStream_t s) {
    const int64_t pieces = ceil_div(a.dim, static_cast<int64_t>(kPiece<T>));
    // a lane has one piece of a row, or as many as the others where a block of 256 has fewer lanes
    const int lanes = static_cast<int>(ceil_div(pieces, ceil_div(pieces, kThreads)));
    if (a.dim < kPiece<T>) return launch_lookup<T, PLACES, true, 1>(a, sorts, lanes, s);
    if (a.tokens * lanes >= 4 * 1024 * kThreads) return launch_lookup<T, PLACES, false, PLACES ? 2 : 4>(a, sorts, lanes, s);
    launch_lookup<T, PLACES, false, 1>(a, sorts, lanes, s);
}

template <typename T>
void launch_lookup(const LookupArgs& a, const SortArgs (&sorts)[2], hipStream_t s) {
    if (a.places) launch_lookup<T, true>(a, sorts, s);
    else launch_lookup<T, false>(a, sorts, s);
}

int check_lists(const void* lists, size_t bytes, size_t has) {
    if (has < bytes) return fail("lists too small: %zu bytes", has);
    if (bytes && (!lists || !aligned(lists, 256))) return fail("lists must be 256-byte aligned");
    return 0;
}

}  // namespace
}  // namespace isa_block

using namespace isa_block;

extern "C" int isa_train_abi_version(void) { return ISA_TRAIN_ABI_VERSION; }

extern "C" size_t isa_train_embedding_lists(const isa_train_embedding* e, int weight, int places) {
    if (check(e)) return 0;
    return (weight ? space_of(e, false).lists : 0) + (places ? space_of(e, true).lists : 0);
}

extern "C" int isa_train_embedding_forward(const isa_train_embedding* e, void* y, int weight, int places, int64_t skip,
                                           void* lists, size_t lists_bytes, void* stream) {
    if (int rc = check(e)) return rc;
    if (e->tokens && (!y || (e->vocab && !e->weight))) return fail("weight and y must be set");
    if (e->tokens && e->places && !e->place_weight) return fail("place_weight must be set");
    const size_t b = type_bytes(e->type);
    if (!aligned(y, b) || !aligned(e->weight, b) || (e->places && !aligned(e->place_weight, b)))
        return fail("y or a table is not aligned to its type");
    if (int rc = check_lists(lists, isa_train_embedding_lists(e, weight, places), lists_bytes)) return rc;
    SortArgs sorts[2] = {};
    char* list = static_cast<char*>(lists);
    if (weight) {
        sorts[0] = sort_of(e, false, skip, list);
        list += space_of(e, false).lists;
    }
    if (places && e->place_ids) sorts[1] = sort_of(e, true, -1, list);
    if (e->tokens == 0 && sorts[0].blocks + sorts[1].blocks == 0) return 0;
    // a table without rows has nothing to read: some memory stands for the row that no id is found in
    const LookupArgs a{e->ids,
                       e->place_ids,
                       e->vocab ? e->weight : y,
                       e->place_weight,
                       y,
                       e->tokens,
                       e->vocab,
                       e->vocab ? e->weight_stride : 0,
                       e->places,
                       e->places_stride,
                       e->period,
                       static_cast<int>(e->dim),
                       e->scale,
                       static_cast<size_t>(e->tokens) * e->dim * b >= kResultPast && e->dim * b % kLine == 0};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (e->type == ISA_BLOCK_F32) launch_lookup<float>(a, sorts, s);
    else if (e->type == ISA_BLOCK_BF16) launch_lookup<bf16>(a, sorts, s);
    else launch_lookup<f16>(a, sorts, s);
    return launched("lookup_kernel");
}

extern "C" size_t isa_train_embedding_backward_workspace(const isa_train_embedding* e, int weight, int places) {
    if (check(e)) return 0;
    return (weight ? space_of(e, false).workspace : 0) + (places ? space_of(e, true).workspace : 0);
}

extern "C" int isa_train_embedding_backward(const isa_train_embedding* e, const void* lists, size_t lists_bytes,
                                            const void* dy, void* dweight, void* dplaces, int listed_weight,
                                            int listed_places, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(e)) return rc;
    if ((dweight && !listed_weight) || (dplaces && !listed_places)) return fail("a gradient's table has no lists");
    if (int rc = check_lists(lists, isa_train_embedding_lists(e, listed_weight, listed_places), lists_bytes)) return rc;
    if (e->tokens && (dweight || dplaces) && !dy) return fail("grad_y must be set");
    const size_t b = type_bytes(e->type);
    if (!aligned(dy, b) || !aligned(dweight, b) || !aligned(dplaces, b)) return fail("a gradient is not aligned to its type");
    const size_t bytes = isa_train_embedding_backward_workspace(e, dweight != nullptr, dplaces != nullptr);
    if (workspace_bytes < bytes) return fail("workspace too small: %zu bytes", workspace_bytes);
    if (bytes && (!workspace || !aligned(workspace, 256))) return fail("workspace must be 256-byte aligned");
    if (e->vocab == 0) dweight = nullptr;
    if (e->places == 0) dplaces = nullptr;
    if (!dweight && !dplaces) return 0;
    Jobs j{};
    const char* list = static_cast<const char*>(lists);
    char* ws = static_cast<char*>(workspace);
    for (int k = 0; k < 2; ++k) {
        void* grad = k ? dplaces : dweight;
        const Space at = space_of(e, k == 1);
        if (grad) {
            SumArgs& a = j.sum[k];
            const int64_t* keys = k ? e->place_ids : e->ids;
            a.rows = static_cast<int>(k ? e->places : e->vocab);
            if (at.lists) {
                a.keys = keys;
                a.order = reinterpret_cast<const int*>(list);
                a.starts = reinterpret_cast<const int*>(list + at.starts);
            } else {
                a.period = static_cast<int>(e->tokens ? e->period : 1);
                a.times = static_cast<int>(e->tokens / a.period);
            }
            a.dy = dy;
            a.grad = grad;
            a.joins = reinterpret_cast<int*>(ws);
            a.partial = reinterpret_cast<float*>(ws + at.partial);
            a.tiles = static_cast<int>(at.tiles);
            a.dim = static_cast<int>(e->dim);
            a.tile = tile_of(e->tokens);
            a.scale = k ? 1.0f : e->scale;
            a.past = static_cast<size_t>(a.rows) * a.dim * b >= kGradientPast && a.dim * b % kLine == 0;
            ws += at.workspace;
        }
        if (k ? listed_places : listed_weight) list += at.lists;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool few = few_of(e);
    if (e->type == ISA_BLOCK_F32) return sums<float>(j, e->dim, few, s);
    if (e->type == ISA_BLOCK_BF16) return sums<bf16>(j, e->dim, few, s);
    return sums<f16>(j, e->dim, few, s);
}
