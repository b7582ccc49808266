// igs_layer_norm.h -- layer norm over rows, forward and backward, with dropout of its result.
// Included by igs_feature.hip inside its anonymous namespace.
#pragma once

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int k = kWave / 2; k > 0; k >>= 1) v += __shfl_xor(v, k);
    __syncthreads();  // the previous sum has been read
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kBlock / kWave; ++w) s += red[w];
    return s;
}

__device__ __forceinline__ float drop_one(float v, int64_t i, const Dropout& drop, const PhiloxKey& key) {
    if (drop.threshold == 0) return v;
    uint32_t w[4];
    philox((uint64_t)(i >> 3), key, w);
    const uint32_t pair = (i & 4) ? ((i & 2) ? w[3] : w[2]) : ((i & 2) ? w[1] : w[0]);
    const uint32_t u = (i & 1) ? pair >> 16 : pair & 0xFFFFu;
    return u >= drop.threshold ? v * drop.factor : 0.0f;
}

// One workgroup per row: mean, then the sum of squared deviations, then the result.
template <class T, class W>
__global__ __launch_bounds__(kBlock) void k_norm_fwd(const T* __restrict__ x, int64_t stride,
                                                     const W* __restrict__ w, const W* __restrict__ b, int64_t rows,
                                                     int D, float eps, Dropout drop, T* __restrict__ y,
                                                     float* __restrict__ stats) {
    __shared__ float red[kBlock / kWave];
    const PhiloxKey key = philox_key(drop);
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * stride;
        float s = 0.0f;
        for (int d = threadIdx.x; d < D; d += kBlock) s += to_f32(xr[d]);
        const float mean = block_sum(s, red) / (float)D;
        s = 0.0f;
        for (int d = threadIdx.x; d < D; d += kBlock) {
            const float c = to_f32(xr[d]) - mean;
            s = fmaf(c, c, s);
        }
        const float rstd = 1.0f / sqrtf(block_sum(s, red) / (float)D + eps);
        for (int d = threadIdx.x; d < D; d += kBlock) {
            const float h = (to_f32(xr[d]) - mean) * rstd;
            const float v = fmaf(h, w ? to_f32(w[d]) : 1.0f, b ? to_f32(b[d]) : 0.0f);
            y[r * D + d] = from_f32<T>(drop_one(v, r * D + d, drop, key));
        }
        if (stats && threadIdx.x == 0) {
            stats[2 * r] = mean;
            stats[2 * r + 1] = rstd;
        }
    }
}

// d x, one workgroup per row.
template <class T, class W>
__global__ __launch_bounds__(kBlock) void k_norm_bwd_x(const T* __restrict__ gy, const T* __restrict__ x,
                                                       int64_t stride, const W* __restrict__ w,
                                                       const float* __restrict__ stats, int64_t rows, int D,
                                                       Dropout drop, T* __restrict__ gx) {
    __shared__ float red[kBlock / kWave];
    const PhiloxKey key = philox_key(drop);
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mean = stats[2 * r], rstd = stats[2 * r + 1];
        float s0 = 0.0f, s1 = 0.0f;
        for (int d = threadIdx.x; d < D; d += kBlock) {
            const float g = drop_one(to_f32(gy[r * D + d]), r * D + d, drop, key) * (w ? to_f32(w[d]) : 1.0f);
            s0 += g;
            s1 = fmaf(g, (to_f32(x[r * stride + d]) - mean) * rstd, s1);
        }
        s0 = block_sum(s0, red) / (float)D;
        s1 = block_sum(s1, red) / (float)D;
        for (int d = threadIdx.x; d < D; d += kBlock) {
            const float g = drop_one(to_f32(gy[r * D + d]), r * D + d, drop, key) * (w ? to_f32(w[d]) : 1.0f);
            const float h = (to_f32(x[r * stride + d]) - mean) * rstd;
            gx[r * D + d] = from_f32<T>(rstd * (g - s0 - h * s1));
        }
    }
}

// d weight, d bias: a workgroup owns 64 columns, its four waves every fourth row.
template <class T, class W>
__global__ __launch_bounds__(kBlock) void k_norm_bwd_w(const T* __restrict__ gy, const T* __restrict__ x,
                                                       int64_t stride, const float* __restrict__ stats, int64_t rows,
                                                       int D, Dropout drop, W* __restrict__ gw, W* __restrict__ gb) {
    __shared__ float red[2][kBlock];
    const PhiloxKey key = philox_key(drop);
    const int d = blockIdx.x * kWave + (threadIdx.x & (kWave - 1)), wave = threadIdx.x / kWave;
    float s0 = 0.0f, s1 = 0.0f;
    if (d < D)
        for (int64_t r = wave; r < rows; r += kBlock / kWave) {
            const float g = drop_one(to_f32(gy[r * D + d]), r * D + d, drop, key);
            s0 += g;
            s1 = fmaf(g, (to_f32(x[r * stride + d]) - stats[2 * r]) * stats[2 * r + 1], s1);
        }
    red[0][threadIdx.x] = s0;
    red[1][threadIdx.x] = s1;
    __syncthreads();
    if (threadIdx.x < kWave && d < D) {
        float t0 = 0.0f, t1 = 0.0f;
#pragma unroll
        for (int k = 0; k < kBlock / kWave; ++k) {
            t0 += red[0][k * kWave + threadIdx.x];
            t1 += red[1][k * kWave + threadIdx.x];
        }
        if (gb) gb[d] = from_f32<W>(t0);
        if (gw) gw[d] = from_f32<W>(t1);
    }
}
