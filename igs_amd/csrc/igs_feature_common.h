// igs_feature_common.h -- element types, conversions and the counter-based generator shared by the
// feature operators (embedding lookup, layer norm, dropout).  Included by igs_feature.hip inside its
// anonymous namespace.
#pragma once

constexpr int kWave = 64;
constexpr int kBlock = 256;

typedef _Float16 f16;
typedef __bf16 bf16;

template <class T>
__device__ __forceinline__ float to_f32(T v) {
    return (float)v;
}
// one rounding, to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <class T>
__device__ __forceinline__ T from_f32(float v) {
    return (T)v;
}

// What a call's dropout needs: the keep rule, the factor of what stays, and the generator's state.
struct Dropout {
    uint32_t threshold;             // dropped iff u < threshold; 0: no dropout
    float factor;                   // 65536 / (65536 - threshold), 0 where everything is dropped
    uint64_t seed, offset;
    const uint64_t* seed_device;    // read by the kernel instead of `seed` when not NULL
};

struct PhiloxKey {
    uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ PhiloxKey philox_key(const Dropout& d) {
    const uint64_t s = d.seed_device ? *d.seed_device : d.seed;
    PhiloxKey k;
    k.k0 = (uint32_t)s;
    k.k1 = (uint32_t)(s >> 32);
    k.o0 = (uint32_t)d.offset;
    k.o1 = (uint32_t)(d.offset >> 32);
    return k;
}

// Philox4x32, seven rounds (Salmon, Moraes, Dror, Shaw 2011: the fewest that pass their test batteries;
// dropout asks no more of its numbers).  128 bits per block serve eight elements with 16 bits each,
// which keeps the integer products (quarter rate) below the time of the memory traffic.
__device__ __forceinline__ void philox(uint64_t block, const PhiloxKey& key, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = key.o0, c3 = key.o1;
    uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
}

// Number of element `j` (0..7) of a block.
__device__ __forceinline__ uint32_t philox_u16(const uint32_t (&w)[4], int j) {
    return (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
}
