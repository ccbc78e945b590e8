// What the attention's forward and backward share: operands of the matrix cores, tiles in LDS, spans
// of keys. block_attention.hip describes the whole.
#pragma once

#include <algorithm>
#include <climits>

#include "block_common.hpp"

namespace isa_block {

constexpr int kTile = 32;  // of the matrix instruction, both ways
constexpr float kLog2E = 1.44269504088896340736f;
constexpr int kMaxLength = 1 << 30;

using acc16 = vec<float, 16>;

struct AttnArgs {
    const void *q, *k, *v, *out, *dout;
    void *result, *rest, *dk, *dv;  // result: out, or dq
    float *lse, *delta, *partial;
    const int32_t* lengths;
    int64_t qs[3], ks[3], vs[3], gs[3];
    int batch, queries, keys, heads, kv_heads, group, dim, window, sinks;
    int splits;         // forward: blocks that share a tile of rows
    int near, far;      // dk, dv: blocks that share a tile of keys, and one that holds sinks
    int far_tiles;      // tiles of keys that hold sinks
    float c, scale;  // c = scale log2 e
};

// ---- fragments: 16 bytes a lane: of an operand's row lane % 32, one of the two chunks of a step -----

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

// What rounding the values of a column to T leaves. A product is taken with it too where the keys are sinks:
// they draw most of many rows' weight, so their roundings would be most of out's and dq's error (dq of
// bf16 rows that give sinks 0.8 of their weight: 2.8e-3 off without, 2.0e-3 with, of which the result's
// own rounding is 1.7e-3).
template <typename T>
__device__ __forceinline__ acc16 remainder(acc16 x) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] -= static_cast<float>(static_cast<T>(x[i]));
    return x;
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

// c is one float in all types: its rounding scales all of a row's scores alike, and with c as two floats fp32's
// errors were the same to 3%.
__device__ __forceinline__ float weight(float s, float c, float base) {
    return __builtin_amdgcn_exp2f(fmaf(s, c, -base));
}

// ---- tiles in LDS -----------------------------------------------------------------------------
// A row's 16-byte chunks lie in a power of two of slots, chunk c in slot c ^ key(row), so that both
// kinds of reads use all banks: 16 rows' of one chunk, and 4 rows' of 4 adjacent chunks (the
// transposing read: with keys that leave those 4 chunks in their 64 bytes it takes twice the time).
// Tiles are loaded straight to LDS, 64 slots an instruction; a buffer descriptor that ends with the last
// row makes what is behind it zeros.

constexpr int slots_for(int chunks) { return chunks <= 4 ? 4 : chunks <= 8 ? 8 : chunks <= 16 ? 16 : 32; }

template <typename T, int D>
struct Tile {
    static constexpr int N = Frag<T>::N;
    static constexpr int kChunks = D / N;
    static constexpr int kSlots = slots_for(kChunks);
    static constexpr int kPitch = kSlots * N;              // elements
    static constexpr int kSteps = kChunks / 2;             // of a product over D
    static constexpr int kUses = kTile / (2 * N);          // operand()s of 32 rows
    static constexpr int kMmas = sizeof(T) == 4 ? 4 : 1;   // matrix instructions of a mma()
    static constexpr int kColumnReads = sizeof(T) == 4 ? 4 : 2;
    using V = typename Frag<T>::V;

    // 256 bytes of banks: 4, 2, 1 or half a row
    static __device__ __forceinline__ constexpr unsigned key(unsigned row) {
        const unsigned by_four = row / 4 % 4;
        return kSlots == 4 ? by_four : kSlots == 8 ? row / 2 % 2 * 4 + by_four : row % 4 * 4 + by_four;
    }

    // Below, what depends on the lane is one place, and a chunk's slot differs from it by an exclusive or
    // with a constant: the rest of an address goes into the instruction. In fp32 each other VALU
    // instruction is time that the products lose (they take the same units: 32x32x2 products of 3 waves
    // a SIMD alone 139 TF/s, with 4 instructions to each 116, with 8 102).

    // of row (r0 + lane % 32), the dims of step t
    static __device__ __forceinline__ V row(const T* tile, int r0, int t, int lane_) {
        const unsigned lane = lane_ % 64u, r = lane % 32;
        const unsigned place = r * kPitch + (lane / 32 ^ key(r)) * N;
        return *reinterpret_cast<const V*>(tile + r0 * kPitch + (place ^ 2 * t * N));
    }

    // of column (32 db + lane % 32), the rows r0 .. r0 + 31 that operand(x, u) holds in this half
    static __device__ __forceinline__ V column(const T* tile, int r0, int u, int db, int lane_) {
        const unsigned lane = lane_ % 64u, half = lane / 32;
        if constexpr (sizeof(T) == 4) {
            V f;
            const unsigned place = 4 * half * kPitch + (lane % 32 / 4 ^ half) * N + lane % 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int other = key(8 * u + e) ^ 8 * db;  // (that of row 4 is 1)
                f[e] = tile[(r0 + 8 * u + e) * kPitch + other / 8 * 8 * N + (place ^ other % 8 * N)];
            }
            return f;
        } else {
            // the transposing read: 16 lanes give the addresses of 4 rows x 16 columns, 4 columns each,
            // and get a column's 4 rows each
            using s4 = vec<short, 4>;
            using lds = __attribute__((address_space(3))) s4;
            union {
                s4 part[2];
                V f;
            } x;
            const unsigned r = 4 * half + lane % 16 / 4;
            const unsigned place = r * kPitch + (lane / 16 % 2 * 2 + lane % 4 / 2 ^ key(r)) * N + lane % 2 * 4;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // (8 rows further on the key differs by 2, 16 further it is the same)
                const T* p = tile + (r0 + 16 * u + 8 * j) * kPitch + (place ^ (4 * db ^ 2 * j) * N);
                x.part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds*)const_cast<T*>(p));
            }
            return x.f;
        }
    }
};

// x, of which the compiler knows nothing: what follows from it is computed again in each turn of a loop
// instead of being held in registers.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

using LdsPtr = __attribute__((address_space(3))) void*;
using LdsBytes = __attribute__((address_space(3))) char*;
constexpr int kBufferFlags = 0x00027000;  // raw buffer of 32-bit data
constexpr unsigned kOutside = 0x7fffffffu;

// COUNT times BYTES a lane to `lds` (an array: its address is known) + first, `step` bytes apart, from the
// buffer of `size` bytes at `base` (uniform); what lies outside is zeros.
// (The buffer's type exists for the device alone: the host's pass over the kernels does without.)
template <int BYTES, int COUNT>
__device__ __forceinline__ void load_to_lds(void* lds, int first, int step, const void* base, int size,
                                            const unsigned (&at)[COUNT]) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, uniform(size), kBufferFlags);
#pragma unroll
    for (int n = 0; n < COUNT; ++n)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (LdsPtr)((LdsBytes)lds + first + n * step), BYTES, at[n], 0, 0,
                                                 0);
#endif
}

// One block's (or wave's) copies of ROWS rows at a time from memory to a tile.
template <typename T, int D, int ROWS, int THREADS>
struct Loader {
    using L = Tile<T, D>;
    static constexpr int kEach = ROWS * L::kSlots / THREADS;
    static_assert(ROWS * L::kSlots % THREADS == 0);
    unsigned at[kEach];  // a lane's byte offsets from the tile's first row
    const char* base;    // of row 0 (uniform)
    int stride;          // bytes between rows, under 2^24

    // `thread`: of THREADS
    __device__ __forceinline__ Loader(const T* base_, int64_t row_stride, int dim, int thread)
        : base(reinterpret_cast<const char*>(base_)), stride(static_cast<int>(row_stride * sizeof(T))) {
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int slot = thread + n * THREADS, row = slot / L::kSlots;
            const int chunk = slot % L::kSlots ^ L::key(row);
            at[n] = chunk * L::N < dim ? static_cast<unsigned>(row * stride) + chunk * 16 : kOutside;
        }
    }

    // rows first .. first + ROWS - 1; those from `end` on become zeros
    // `place`: of the tile in `lds`, in bytes
    __device__ __forceinline__ void load(T* lds, int place, int first, int end, int wave) const {
        load_from(lds, place, base + static_cast<int64_t>(first) * stride, end - first, wave);
    }
    __device__ __forceinline__ void load_from(T* lds, int place, const char* from, int left, int wave) const {
        load_to_lds<16, kEach>(lds, place + wave * kWave * 16, THREADS * 16, from, min(max(left, 0), ROWS) * stride, at);
    }
};

// 64 floats to lds + place by one wave, zeros from `count` on.
__device__ __forceinline__ void load_floats(float* lds, int place, const float* base, int64_t first, int count, int lane) {
    const unsigned at[1] = {static_cast<unsigned>(lane) * 4};
    load_to_lds<4, 1>(lds, place * 4, 0, base + first, max(count, 0) * 4, at);
}

// All of this wave's loads to LDS have arrived.
__device__ __forceinline__ void loads_arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// Which of a key head's `slots` pieces of work, the longest first, block `id` of heads * slots takes.
// Dispatch gives block i to XCD i % 8 and there to compute unit i / 8 % 32. Heads are dealt to XCDs,
// whose L2 then holds their keys once, and taken in bundles of as many as fill an XCD (8 blocks a unit),
// the longest pieces of all heads of a bundle first; every other row of 32 blocks is turned round.
// So a unit gets long and short pieces; head by head, 16 pieces to a head would put all of one length in
// one unit (8 x 1024 tokens, 12 heads of 64 without a window: forward, dq, dk and dv in fp32 168 + 227 + 298 us
// against 224 + 369 + 437, in bf16 27 + 35 against 36 + 46; with a window the two are alike).
struct Piece {
    int head, slot;
    __device__ __forceinline__ Piece(int id, int total, int heads, int slots) {
        constexpr int kXcds = 8, kUnits = 32;
        const int x = id % kXcds, mine = (total - x + kXcds - 1) / kXcds;
        int at = id / kXcds;
        if (at / kUnits % 2) at = at / kUnits * kUnits + min(at / kUnits * kUnits + kUnits, mine) - 1 - at;
        id = at * kXcds + x;
        const int groups = min(heads & -heads, kXcds), each = heads / groups;  // a power of two that divides heads
        const int group = id % groups, rank = id / groups;
        const int bundle = min((kUnits * 8 + slots - 1) / slots, each), first = rank / (bundle * slots) * bundle;
        const int here = min(bundle, each - first), in = rank - first * slots;
        head = group * each + first + in % here;
        slot = in / here;
    }
};

// ---- which keys a block of rows sees --------------------------------------------------------

__device__ __forceinline__ int length_of(const AttnArgs& a, int b) {
    return a.lengths ? min(max(a.lengths[b], 0), a.keys) : a.keys;
}


// The tiles of BN keys that some query at pmin .. pmax sees: those of the sinks 0 .. sink - 1, then
// those of the window lo .. hi - 1 behind them.
template <int BN>
struct Span {
    int lo, hi, sink, sink_tiles, count;

    __device__ __forceinline__ Span(const AttnArgs& a, int pmin, int pmax) {
        hi = max(pmax + 1, 0);
        sink = min(a.sinks, hi);
        lo = max(sink, pmin - a.window + 1);
        sink_tiles = (sink + BN - 1) / BN;
        count = sink_tiles + (max(hi - lo, 0) + BN - 1) / BN;
    }
    __device__ __forceinline__ bool of_sinks(int it) const { return it < sink_tiles; }
    __device__ __forceinline__ int first(int it) const {
        return it < sink_tiles ? it * BN : lo + (it - sink_tiles) * BN;
    }
    __device__ __forceinline__ int end(int it) const { return it < sink_tiles ? sink : hi; }
};

// Rows of a wave against a tile's keys j0 .. j0 + BN - 1: whether all see all of them, or none any.
template <int BN>
struct Sight {
    bool all, none;
    __device__ __forceinline__ Sight(const AttnArgs& a, const Span<BN>& s, int it, int j0, int pmin, int pmax) {
        const bool sinks = s.of_sinks(it);
        all = j0 + BN - 1 <= pmin && (sinks ? j0 + BN <= s.sink : j0 > pmax - a.window);
        none = j0 > pmax || (!sinks && j0 + BN - 1 <= pmin - a.window);
    }
};

// What the query at p sees of a tile from j0 on, told for the registers of a product whose rows are
// the tile's keys: one range of them, so that a subtraction and a comparison decide.
struct Range {
    int from;
    unsigned count;
    __device__ __forceinline__ Range(const AttnArgs& a, bool of_sinks, int sink, int p, int j0, int half) {
        const int lo = of_sinks ? 0 : p - a.window + 1, hi = of_sinks ? min(p, sink - 1) : p;
        from = lo - j0 - 4 * half;
        count = max(hi - lo + 1, 0);
    }
    __device__ __forceinline__ bool has(int row) const { return static_cast<unsigned>(row - from) < count; }  // of half 0
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

// A row's elements as the fragments of a product over them, or zeros.
template <typename T, int D>
struct RowFrags {
    using V = typename Frag<T>::V;
    V v[Tile<T, D>::kSteps];
    __device__ __forceinline__ const V& operator[](int t) const { return v[t]; }
    __device__ __forceinline__ void load(const T* row, int dim, int lane) {
#pragma unroll
        for (int t = 0; t < Tile<T, D>::kSteps; ++t) {
            const int at = (2 * t + lane / 32) * Frag<T>::N;
            v[t] = V{};
            if (row && at < dim) v[t] = *reinterpret_cast<const V*>(row + at);
        }
    }
};

// 8 dims k 16 + 8 half .. of a 32-dim block of a row, rounded. Each half of the wave holds 4 of every 8
// dims of its lanes' rows; 16-bit types exchange them, so that a lane stores 16 bytes (stores of 8
// take a fifth of the forward's time at 2 x 4096 tokens of 128-wide heads).
template <typename T>
__device__ __forceinline__ Pack<T, 8> eight(const float (&x)[16], int k) {
    union {
        Pack<T, 4> v[2];
        unsigned u[2][2];
    } a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a.v[0].v[e] = static_cast<T>(x[8 * k + e]);
        a.v[1].v[e] = static_cast<T>(x[8 * k + 4 + e]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const auto r = __builtin_amdgcn_permlane32_swap(a.u[0][n], a.u[1][n], false, false);
        b.u[0][n] = r[0];
        b.u[1][n] = r[1];
    }
    Pack<T, 8> y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y.v[e] = b.v[e / 4].v[e % 4];
    return y;
}

// A row of a transposed product (lane: a row, registers: its dims) times `factor`; what its
// rounding leaves goes to `rest` if that is set. Both lanes of a row come here.
template <typename T, int DB>
__device__ __forceinline__ void store_row(T* row, const acc16 (&x)[DB], float factor, int dim, int lane,
                                          T* rest = nullptr) {
#pragma unroll
    for (int db = 0; db < DB; ++db) {
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = x[db][i] * factor;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int at = 32 * db + product_row(i, lane / 32);
                if (at < dim) *reinterpret_cast<vec<float, 4>*>(row + at) = vec<float, 4>{y[i], y[i + 1], y[i + 2], y[i + 3]};
            }
        } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int at = 32 * db + 16 * k + lane / 32 * 8;
                const Pack<T, 8> z = eight<T>(y, k);
                if (at < dim) *reinterpret_cast<Pack<T, 8>*>(row + at) = z;
            }
            if (!rest) continue;
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] -= static_cast<float>(static_cast<T>(y[i]));
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int at = 32 * db + 16 * k + lane / 32 * 8;
                const Pack<T, 8> z = eight<T>(y, k);
                if (at < dim) *reinterpret_cast<Pack<T, 8>*>(rest + at) = z;
            }
        }
    }
}

// Asks the scheduler for this block of code's READS reads of LDS to run AHEAD of the MMAS products that
// take them: left to itself it reads each operand right before its product, and the wave waits for
// LDS once a product.
template <int READS, int MMAS, int AHEAD>
__device__ __forceinline__ void reads_ahead() {
    constexpr int kFirst = AHEAD < READS ? AHEAD : READS, kEach = MMAS / READS > 0 ? MMAS / READS : 1;
    constexpr int kReads = MMAS / READS > 0 ? 1 : READS / MMAS;
    __builtin_amdgcn_sched_group_barrier(0x100, kFirst, 0);
#pragma unroll
    for (int i = kFirst; i < READS; i += kReads) {
        __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MMAS, 0);
}

template <typename T>
constexpr int kKeyTile = sizeof(T) == 4 ? 32 : 64;

// Waves, of 32 rows each, that share a block's tiles. At the edges of a window they wait for each other
// with nothing to compute; products in fp32 take 16 times as long as their operands' reads allow, so
// there fewer share (GPT-L's step in fp32, window 256, with two tiles of each operand: forward and dq
// 114 + 164 us by fours, 107 + 148 by twos, 121 + 169 alone; dk and dv 241, 205 and 188). 16-bit products
// need the sharing (2 x 4096 tokens of 128-wide heads, window 1024: 97 + 127 + 172 us by fours,
// 122 + 172 + 269 by twos).
template <typename T>
constexpr int kWaves = sizeof(T) == 4 ? 2 : 4;
template <typename T>
constexpr int kThreads = kWaves<T> * kWave;
template <typename T>
constexpr int kRows = kWaves<T> * kTile;

// One tile in LDS of each operand instead of two, in the forward and in dk's and dv's walk: the next one's copy
// starts when the products that read it are done, beside those of the other operand. In fp32 those take long
// enough for it to arrive, and LDS for two would be what limits the waves (8 x 1024 tokens of 64-wide heads,
// window 256: forward 90 us against 116; 2 x 4096 of 128-wide ones, window 1024: 597 against 627, dk and dv
// 1216 against 2201). dq, which reads K twice, gains nothing (924 against 890).
template <typename T>
constexpr bool kOneTile = sizeof(T) == 4;

int check_attention(const isa_block_attention* t);
AttnArgs attention_args(const isa_block_attention* t);
bool strided(const void* p, const int64_t (&s)[3], int64_t tokens, int64_t dim, size_t bytes);

// f(type, D) for the element type and the dims of a tile.
template <typename F>
void for_type(int type, int dim, F f) {
    auto dims = [&](auto t) {
        using T = decltype(t);
        if (dim <= 32) return f(T{}, std::integral_constant<int, 32>{});
        if (dim <= 64) return f(T{}, std::integral_constant<int, 64>{});
        if (dim <= 96) return f(T{}, std::integral_constant<int, 96>{});
        return f(T{}, std::integral_constant<int, 128>{});
    };
    if (type == ISA_BLOCK_F32) return dims(float{});
    if (type == ISA_BLOCK_BF16) return dims(bf16{});
    return dims(f16{});
}

}  // namespace isa_block
