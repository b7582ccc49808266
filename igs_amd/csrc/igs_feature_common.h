// igs_feature_common.h -- element types, wide loads, sums across lanes and the counter-based generator
// shared by the feature operators (embedding lookup, layer norm, dropout).  Included by igs_feature.hip and
// igs_norm.hip inside their anonymous namespaces.
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

// Elements of one 16-byte access.  A Pack has its element's alignment: global memory takes a 16-byte
// access at any address, so rows of odd lengths and misaligned views go the same way as others.
template <class T>
constexpr int kVec = 16 / (int)sizeof(T);
template <class T, int V>
struct Pack {
    T v[V];
};
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& q) {
    *reinterpret_cast<Pack<T, V>*>(p) = q;
}

// The same past the caches (non-temporal), for tensors that the last-level cache cannot hold anyway: what it does hold
// then stays.  `stream` is uniform; a call does so from kStreamBytes of reads (lookup and norm with a backward: writes)
// on.  us without / with, each call by itself: norm bf16 x 1024, 32768 rows forward 23 / 24, backward 39 / 39; 65536 rows
// 44 / 45, 77 / 69; 131072 rows 98 / 84, 148 / 129; lookup of 131072 tokens of 65536 x 1024 in bf16 83 / 57 (stores),
// its gradient 131 / 112.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p, bool stream) {
    if constexpr (sizeof(Pack<T, V>) == 16) {
        if (stream) {
            const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
            return __builtin_bit_cast(Pack<T, V>, v);
        }
    }
    return load_pack<T, V>(p);
}
// (a constant here: the compiler makes one store of the two of a branch, an ordinary one)
template <bool kStream, class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& q) {
    if constexpr (kStream && sizeof(Pack<T, V>) == 16) {
        const u32x4_any v = __builtin_bit_cast(u32x4, q);
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p));
    } else {
        store_pack<T, V>(p, q);
    }
}

// Sums over the TPR lanes of a row within a wave (TPR = 4, 8, 16, 32 or 64), the same bits in all of them.
// Every lane of the wave takes part.  Data-parallel moves inside 16 lanes; a whole wave's four sums
// of 16 are read as scalars.
template <int kCtrl>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xF, 0xF, true));
}
template <int TPR>
__device__ __forceinline__ float lanes_sum(float v) {
    static_assert(TPR == 4 || TPR == 8 || TPR == 16 || TPR == 32 || TPR == 64, "");
    v = dpp_add<0xB1>(v);   // lane ^ 1
    v = dpp_add<0x4E>(v);   // lane ^ 2
    if (TPR >= 8) v = dpp_add<0x141>(v);   // mirrored within 8
    if (TPR >= 16) v = dpp_add<0x140>(v);  // mirrored within 16
    if (TPR == 32) v += __shfl_xor(v, 16);
    if (TPR == 64) {
        const int i = __float_as_int(v);
        const float a = __int_as_float(__builtin_amdgcn_readlane(i, 0)), b = __int_as_float(__builtin_amdgcn_readlane(i, 16));
        const float c = __int_as_float(__builtin_amdgcn_readlane(i, 32)), d = __int_as_float(__builtin_amdgcn_readlane(i, 48));
        v = (a + b) + (c + d);
    }
    return v;
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

// a ^ b ^ c in one instruction
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
    return (uint32_t)__builtin_amdgcn_bitop3_b32((int)a, (int)b, (int)c, 0x96);
}

// Philox4x32, seven rounds (Salmon, Moraes, Dror, Shaw 2011: the fewest that pass their test batteries;
// dropout asks no more of its numbers).  128 bits per block serve eight elements with 16 bits each,
// which keeps the integer products (quarter rate) below the time of the memory traffic.  A pack of eight 16-bit elements
// takes one block; a pack of four fp32 ones takes one too and uses half of it, so that fp32 computes each block twice.
__device__ __forceinline__ void philox(uint64_t block, const PhiloxKey& key, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = key.o0, c3 = key.o1;
    uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = xor3((uint32_t)(b >> 32), c1, k0);
        c1 = (uint32_t)b;
        c2 = xor3((uint32_t)(a >> 32), c3, k1);
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
// Bit j: element j of the block stays.
__device__ __forceinline__ uint32_t keep_bits(uint64_t block, const Dropout& d, const PhiloxKey& key) {
    uint32_t w[4], bits = 0;
    philox(block, key, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) bits |= (philox_u16(w, j) >= d.threshold ? 1u : 0u) << j;
    return bits;
}

// v = dropped ? 0 : v * factor for V consecutive elements from linear index `first`.  `whole`
// (wave-uniform): every row length is a multiple of 8, so first is a multiple of V and the elements lie
// in one block; otherwise they may reach into the next one.
template <int V>
__device__ __forceinline__ void drop(float (&v)[V], uint64_t first, bool whole, const Dropout& d, const PhiloxKey& key) {
    if (V > 1 && whole) {
        uint32_t w[4];
        philox(first >> 3, key, w);
        if (V == 4 && (first & 4)) {
            w[0] = w[2];
            w[1] = w[3];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = philox_u16(w, j & 7) >= d.threshold ? v[j] * d.factor : 0.0f;
    } else {
        const uint32_t shift = (uint32_t)(first & 7);
        uint32_t bits = keep_bits(first >> 3, d, key);
        if (shift + V > 8) bits |= keep_bits((first >> 3) + 1, d, key) << 8;
        bits >>= shift;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (bits >> j) & 1 ? v[j] * d.factor : 0.0f;
    }
}
