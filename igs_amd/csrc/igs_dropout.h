// igs_dropout.h -- y = keep ? x * factor : 0 with a mask that is computed where it is used.
// Included by igs_feature.hip inside its anonymous namespace.
#pragma once

// A thread owns blocks of eight consecutive elements, one generator block each.
template <class T>
__global__ __launch_bounds__(kBlock) void k_dropout(const T* __restrict__ x, int64_t count, Dropout drop,
                                                    T* __restrict__ y) {
    const PhiloxKey key = philox_key(drop);
    const int64_t blocks = (count + 7) >> 3, step = (int64_t)gridDim.x * kBlock;
    for (int64_t b = (int64_t)blockIdx.x * kBlock + threadIdx.x; b < blocks; b += step) {
        uint32_t w[4];
        philox((uint64_t)b, key, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t i = 8 * b + j;
            if (i < count)
                y[i] = philox_u16(w, j) >= drop.threshold ? from_f32<T>(to_f32(x[i]) * drop.factor) : from_f32<T>(0.0f);
        }
    }
}
