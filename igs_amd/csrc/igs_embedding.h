// igs_embedding.h -- embedding lookup with scaling and its dense gradient.  Included by
// igs_feature.hip inside its anonymous namespace.
#pragma once

template <class I>
__device__ __forceinline__ bool token_ok(I t, int64_t vocab) {
    return (int64_t)t >= 0 && (int64_t)t < vocab;
}

// out[i,:] = scale * weight[tokens[i],:]; one element per thread.
template <class T, class I>
__global__ __launch_bounds__(kBlock) void k_embed_fwd(const T* __restrict__ weight, int64_t stride, int64_t vocab,
                                                      int D, const I* __restrict__ tokens, int64_t count,
                                                      float scale, T* __restrict__ out) {
    const int64_t total = count * D, step = (int64_t)gridDim.x * kBlock;
    for (int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x; e < total; e += step) {
        const int64_t i = e / D;
        const I t = tokens[i];
        out[e] = token_ok(t, vocab) ? from_f32<T>(to_f32(weight[(int64_t)t * stride + (e - i * D)]) * scale)
                                    : from_f32<T>(__builtin_nanf(""));
    }
}

// One workgroup per row of the table: it scans all tokens and adds the gradients of its own in
// increasing position.
template <class T, class I>
__global__ __launch_bounds__(kBlock) void k_embed_bwd(const T* __restrict__ grad, const I* __restrict__ tokens,
                                                      int64_t count, int64_t vocab, int D, float scale,
                                                      int64_t padding, T* __restrict__ out) {
    for (int64_t v = blockIdx.x; v < vocab; v += gridDim.x)
        for (int d = threadIdx.x; d < D; d += kBlock) {
            float s = 0.0f;
            if (v != padding)
                for (int64_t i = 0; i < count; ++i)
                    if ((int64_t)tokens[i] == v) s += to_f32(grad[i * D + d]);
            out[v * D + d] = from_f32<T>(s * scale);
        }
}
