// Dropout's numbers: Philox4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy
// as 1, 2, 3; 2011), eight 16-bit numbers of each call.
//
// 16 bits an element and not 32: a call is 20 products of 32 x 32 bits, which take four times an ordinary
// instruction's issue; at 32 bits an element a 16-bit dropout would be bound by them and not by HBM. The
// probability is then held to a multiple of 2^-16, and the factor of what is kept follows it exactly.
#pragma once

#include "block_common.hpp"

#include "isa_train.h"

namespace isa_block {

struct Dropout {
    const int64_t* seed;
    int64_t site;
    uint32_t threshold;
    float factor;  // of what is kept
};

// What a call's elements share: read once a thread.
struct DropoutKey {
    uint32_t key[2], offset[2];

    __device__ __forceinline__ explicit DropoutKey(const Dropout& d) {
        const uint64_t k = static_cast<uint64_t>(d.seed[0]);
        const uint64_t o = static_cast<uint64_t>(d.seed[1]) + static_cast<uint64_t>(d.site);
        key[0] = static_cast<uint32_t>(k);
        key[1] = static_cast<uint32_t>(k >> 32);
        offset[0] = static_cast<uint32_t>(o);
        offset[1] = static_cast<uint32_t>(o >> 32);
    }
};

// The numbers of eight adjacent elements of a row, the `group`-th eight of all rows.
struct DropoutNumbers {
    uint32_t word[4];

    __device__ __forceinline__ DropoutNumbers(const DropoutKey& k, uint64_t group) {
        uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32);
        uint32_t c2 = k.offset[0], c3 = k.offset[1], k0 = k.key[0], k1 = k.key[1];
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c0, b = static_cast<uint64_t>(0xCD9E8D57u) * c2;
            c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
            c1 = static_cast<uint32_t>(b);
            c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
            c3 = static_cast<uint32_t>(a);
            k0 += 0x9E3779B9u;
            k1 += 0xBB67AE85u;
        }
        word[0] = c0;
        word[1] = c1;
        word[2] = c2;
        word[3] = c3;
    }
    __device__ __forceinline__ uint32_t number(int e) const { return e & 1 ? word[e >> 1] >> 16 : word[e >> 1] & 0xffffu; }
};

// 0 of a dropped element by selection: a product would keep infinities and NaN.
__device__ __forceinline__ float dropped(float x, uint32_t number, const Dropout& d) {
    return number >= d.threshold ? x * d.factor : 0.0f;
}

inline Dropout dropout_of(const isa_train_dropout& d) {
    Dropout r{};
    r.seed = d.seed;
    r.site = d.site;
    r.threshold = static_cast<uint32_t>(d.threshold);
    r.factor = d.threshold < 65536 ? static_cast<float>(65536.0 / (65536 - d.threshold)) : 0.0f;
    return r;
}

inline int check(const isa_train_dropout* d) {
    if (!d) return fail("dropout is null");
    if (d->threshold < 0 || d->threshold > 65536) return fail("threshold must be 0 to 65536, got %d", d->threshold);
    if (!d->seed || !aligned(d->seed, 8)) return fail("seed must be set, two 64-bit numbers");
    return 0;
}

}  // namespace isa_block
