// What the kernels of a transformer block share: element types, wave sums, errors.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "isa_block.h"

namespace isa_block {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T, int N>
using vec __attribute__((ext_vector_type(N))) = T;

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

constexpr int kWave = 64;

// N elements as one load or store at any element's address; `left` < N of them one by one.
template <typename T, int N>
struct Loose {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

template <typename T, int N>
__device__ __forceinline__ void load_loose(Pack<T, N>& p, const T* from, int left) {
    if (left >= N) {
        const typename Loose<T, N>::type x = *reinterpret_cast<const typename Loose<T, N>::type*>(from);
#pragma unroll
        for (int e = 0; e < N; ++e) p.v[e] = x[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) p.v[e] = e < left ? from[e] : static_cast<T>(0.0f);
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_loose(T* to, const Pack<T, N>& p, int left) {
    if (left >= N) {
        typename Loose<T, N>::type x;
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = p.v[e];
        *reinterpret_cast<typename Loose<T, N>::type*>(to) = x;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < left) to[e] = p.v[e];
    }
}

// v_permlane32_swap exchanges the upper half of one register with the lower half of another:
// given the same value twice, one result has the lower half's values in both halves, the
// other the upper half's.
__device__ __forceinline__ void both_halves(float x, float& lower, float& upper) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    lower = __uint_as_float(r[0]);
    upper = __uint_as_float(r[1]);
}

__device__ __forceinline__ float half_sum(float x) {
    float a, b;
    both_halves(x, a, b);
    return a + b;
}

__device__ __forceinline__ float half_max(float x) {
    float a, b;
    both_halves(x, a, b);
    return fmaxf(a, b);
}

template <int Ctrl>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), Ctrl, 0xf, 0xf, true));
}

__device__ __forceinline__ void both_rows(float x, float& a, float& b) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}

// Sum and maximum over the wave, in every lane: within 16 lanes by DPP (lane swaps by 1 and 2,
// then mirrors of 8 and 16), across them by lane-block swaps. Each step adds the same two values
// in both lanes, so all lanes hold the same bits.
__device__ __forceinline__ float wave_sum(float x) {
    x += dpp<0xB1>(x);   // quad_perm 1,0,3,2
    x += dpp<0x4E>(x);   // quad_perm 2,3,0,1
    x += dpp<0x141>(x);  // row_half_mirror
    x += dpp<0x140>(x);  // row_mirror
    float a, b;
    both_rows(x, a, b);
    return half_sum(a + b);
}

__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp<0xB1>(x));
    x = fmaxf(x, dpp<0x4E>(x));
    x = fmaxf(x, dpp<0x141>(x));
    x = fmaxf(x, dpp<0x140>(x));
    float a, b;
    both_rows(x, a, b);
    return half_max(fmaxf(a, b));
}

// ---- errors -----------------------------------------------------------------------------

char* error_buffer();
constexpr size_t kErrorBytes = 512;

__attribute__((format(printf, 1, 2))) inline int fail(const char* format, ...) {
    va_list args;
    va_start(args, format);
    std::vsnprintf(error_buffer(), kErrorBytes, format, args);
    va_end(args);
    return ISA_BLOCK_EINVAL;
}

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    std::snprintf(error_buffer(), kErrorBytes, "%s: %s", what, hipGetErrorString(e));
    return static_cast<int>(e);
}

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool known_type(int t) { return t == ISA_BLOCK_F32 || t == ISA_BLOCK_BF16 || t == ISA_BLOCK_F16; }
inline size_t type_bytes(int t) { return t == ISA_BLOCK_F32 ? 4 : 2; }
constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace isa_block
