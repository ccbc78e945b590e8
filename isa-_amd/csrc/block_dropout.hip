// Dropout from a counter-based generator, alone and in the norm's residual add, for gfx950.
//
//   y = keep ? x 65536 / (65536 - t) : 0,  keep iff the element's 16-bit number >= t
//
// No mask is stored: the backward makes the numbers again from the counter. Bound by HBM, one read and one write
// of each element; a thread takes eight adjacent elements, the numbers of one call of the generator. 65536 x 1024 in bf16
// 40 us (6.6 TB/s, a copy 37), 8192 x 768 in fp32 8.8 (5.7 TB/s, a copy 7.8), 65536 x 390 in bf16 20 (a copy 15).
#include "block_norm.hpp"

namespace isa_block {
namespace {

constexpr int kMaxDropoutBlocks = 4096;

struct DropoutArgs {
    Dropout drop;
    const void* x;
    void* y;
    int64_t x_stride, groups;  // of eight elements, in all rows
    uint32_t dim, per_row;
};

// How a group's elements are read. kFlat: rows lie one behind the other and groups fill them, so that a group's number
// says where. kCut: a row's last group may have fewer than eight, which are the end of the row's last eight. kShort: rows
// of less than eight.
enum Rows { kFlat, kCut, kShort };

// The elements from `by` on, in the first places: a register at a time, by 4, 2 and 1 elements.
template <typename T>
__device__ __forceinline__ Pack<T, 8> moved_down(const Pack<T, 8>& p, int by) {
    constexpr int W = 2 * sizeof(T), kStep = 4 / sizeof(T);  // registers, elements of one
    using Packed = Pack<T, 8>;
    struct Words {
        uint32_t w[W];
    };
    Words x = __builtin_bit_cast(Words, p);
#pragma unroll
    for (int n = 4; n >= kStep; n /= 2)
#pragma unroll
        for (int i = 0; i + n / kStep < W; ++i) x.w[i] = by & n ? x.w[i + n / kStep] : x.w[i];
    if constexpr (kStep == 2)
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const uint32_t half = __builtin_amdgcn_alignbit(i + 1 < W ? x.w[i + 1] : 0u, x.w[i], 16);
            x.w[i] = by & 1 ? half : x.w[i];
        }
    return __builtin_bit_cast(Packed, x);
}

template <typename T, Rows ROWS>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs a) {
    const DropoutKey key(a.drop);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < a.groups; i += step) {
        int64_t from = 8 * i, to = from;
        int left = 8;
        if constexpr (ROWS != kFlat) {
            // 64-bit quotients take several times the instructions
            const int64_t r = i <= UINT32_MAX ? static_cast<uint32_t>(i) / a.per_row : i / a.per_row;
            const int64_t at = 8 * (i - r * a.per_row);
            from = r * a.x_stride + at;
            to = r * a.dim + at;
            left = static_cast<int>(std::min<int64_t>(8, a.dim - at));
        }
        const T* x = static_cast<const T*>(a.x) + from;
        Pack<T, 8> p;
        if constexpr (ROWS == kShort) load_loose(p, x, left);
        else load_loose(p, x + (left - 8), 8);
        if constexpr (ROWS == kCut) p = moved_down(p, 8 - left);
        const DropoutNumbers n(key, static_cast<uint64_t>(i));
#pragma unroll
        for (int e = 0; e < 8; ++e) p.v[e] = static_cast<T>(dropped(static_cast<float>(p.v[e]), n.number(e), a.drop));
        store_loose(static_cast<T*>(a.y) + to, p, left);
    }
}

// fp32, flat: a group is two lanes' 16 bytes, so that a wave's loads are one piece of memory. A wave takes 64 groups as
// two loads; of a pair of lanes one makes the numbers of its group of the first load, the other of the second, and each
// sends the other half of them.
__global__ __launch_bounds__(kThreads) void dropout_pairs_kernel(DropoutArgs a) {
    const DropoutKey key(a.drop);
    const int lane = threadIdx.x % kWave;
    const bool odd = lane & 1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x - lane; base < a.groups; base += step) {
        const int64_t group[2] = {base + lane / 2, base + kWave / 2 + lane / 2};
        using V = typename Loose<float, 4>::type;
        V v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (group[k] < a.groups) v[k] = *reinterpret_cast<const V*>(static_cast<const float*>(a.x) + 8 * group[k] + 4 * odd);
        const DropoutNumbers n(key, static_cast<uint64_t>(group[odd]));
        uint32_t word[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t sent = odd ? n.word[h] : n.word[2 + h];
            const uint32_t got = __float_as_uint(dpp<0xB1>(__uint_as_float(sent)));  // lanes 1, 0, 3, 2
            word[0][h] = odd ? got : n.word[h];
            word[1][h] = odd ? n.word[2 + h] : got;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (group[k] >= a.groups) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = word[k][e >> 1];
                v[k][e] = dropped(v[k][e], e & 1 ? w >> 16 : w & 0xffffu, a.drop);
            }
            *reinterpret_cast<V*>(static_cast<float*>(a.y) + 8 * group[k] + 4 * odd) = v[k];
        }
    }
}

template <typename T>
void launch_dropout(const DropoutArgs& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(ceil_div(a.groups, kThreads), kMaxDropoutBlocks)));
    if (a.dim < 8) {
        dropout_kernel<T, kShort><<<grid, dim3(kThreads), 0, s>>>(a);
    } else if (a.dim % 8 || a.x_stride != a.dim) {
        dropout_kernel<T, kCut><<<grid, dim3(kThreads), 0, s>>>(a);
    } else {
        if constexpr (sizeof(T) == 4) dropout_pairs_kernel<<<grid, dim3(kThreads), 0, s>>>(a);
        else dropout_kernel<T, kFlat><<<grid, dim3(kThreads), 0, s>>>(a);
    }
}

}  // namespace
}  // namespace isa_block

using namespace isa_block;

extern "C" int isa_train_dropout_apply(const isa_train_dropout* drop, int type, int64_t rows, int64_t dim,
                                       const void* x, int64_t x_stride, void* y, void* stream) {
    if (int rc = check(drop)) return rc;
    if (!known_type(type)) return fail("unknown element type %d", type);
    if (rows < 0 || dim < 0 || dim > (int64_t{1} << 30) || rows > (int64_t{1} << 60) / std::max<int64_t>(dim, 1))
        return fail("rows must not be negative and dim be 0 to 2^30, got %lld and %lld", static_cast<long long>(rows),
                    static_cast<long long>(dim));
    if (rows == 0 || dim == 0) return 0;
    if (!x || !y) return fail("x and y must be set");
    if (!aligned(x, type_bytes(type)) || !aligned(y, type_bytes(type))) return fail("x or y is not aligned to its type");
    DropoutArgs a{};
    a.drop = dropout_of(*drop);
    a.x = x;
    a.y = y;
    a.x_stride = x_stride;
    a.dim = static_cast<uint32_t>(dim);
    a.per_row = static_cast<uint32_t>(ceil_div(dim, 8));
    a.groups = rows * a.per_row;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == ISA_BLOCK_F32) launch_dropout<float>(a, s);
    else if (type == ISA_BLOCK_BF16) launch_dropout<bf16>(a, s);
    else launch_dropout<f16>(a, s);
    return launched("dropout_kernel");
}

extern "C" int isa_train_dropout_norm_forward(const isa_block_norm* n, const isa_train_dropout* drop, const void* x,
                                              int64_t x_stride, const void* residual, int64_t residual_stride, void* y,
                                              void* h, float* mean, float* rstd, void* stream) {
    if (int rc = check(drop)) return rc;
    if (n && n->rows > 0 && !x) return fail("x must be set");
    return run_forward<Dropped>(n, dropout_of(*drop), x, x_stride, residual, residual_stride, y, h, mean, rstd, stream);
}

extern "C" int isa_train_dropout_norm_backward(const isa_block_norm* n, const isa_train_dropout* drop, const void* dy,
                                               const void* dh, const void* h, int64_t h_stride, const float* mean,
                                               const float* rstd, void* dx, void* dresidual, void* dweight,
                                               void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(drop)) return rc;
    if (n && n->rows > 0 && !dx) return fail("grad_x must be set");
    return run_backward<Dropped>(n, dropout_of(*drop), dy, dh, h, h_stride, mean, rstd, dx, dresidual, dweight, dbias,
                                 workspace, workspace_bytes, stream);
}
