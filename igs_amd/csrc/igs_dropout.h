// igs_dropout.h -- y = keep ? x * factor : 0 with a mask that is computed where it is used.
// Included by igs_feature.hip inside its anonymous namespace.
#pragma once

// A thread owns packs of 16 bytes (eight 16-bit elements, one generator block; four fp32 elements, half a
// block), kPacks of them in flight, 16 bytes times the workgroup's threads apart.
template <class T, int kPacks>
__global__ __launch_bounds__(kBlock) void k_dropout(const T* __restrict__ x, int64_t count, Dropout drop_,
                                                    T* __restrict__ y) {
    constexpr int V = kVec<T>;
    const PhiloxKey key = philox_key(drop_);
    const int64_t packs = count / V;
    const int64_t base = (int64_t)blockIdx.x * (kBlock * kPacks) + threadIdx.x;
    Pack<T, V> q[kPacks];
#pragma unroll
    for (int k = 0; k < kPacks; ++k)
        if (base + k * kBlock < packs) q[k] = load_pack<T, V>(x + (base + k * kBlock) * V);
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
        const int64_t p = base + k * kBlock;
        if (p < packs) {
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = to_f32(q[k].v[j]);
            drop<V>(v, (uint64_t)p * V, true, drop_, key);
#pragma unroll
            for (int j = 0; j < V; ++j) q[k].v[j] = from_f32<T>(v[j]);
            store_pack<T, V>(y + p * V, q[k]);
        }
    }
    if (blockIdx.x == 0 && threadIdx.x < count - packs * V) {  // the last count % V elements
        const int64_t i = packs * V + threadIdx.x;
        float v[1] = {to_f32(x[i])};
        drop<1>(v, (uint64_t)i, false, drop_, key);
        y[i] = from_f32<T>(v[0]);
    }
}
