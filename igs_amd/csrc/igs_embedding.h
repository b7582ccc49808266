// igs_embedding.h -- embedding lookup with scaling and its dense gradient.  Included by
// igs_feature.hip inside its anonymous namespace.
#pragma once

template <class I>
__device__ __forceinline__ bool token_ok(I t, int64_t vocab) {
    return (int64_t)t >= 0 && (int64_t)t < vocab;
}

// out[i,:] = scale * weight[tokens[i],:].  `lanes` threads (a power of two, at most a workgroup) share a
// token and walk its row in packs of V elements; the last pack of a row of another length is moved back
// to end with the row.  Rows of fewer elements than a pack go with V = 1.
template <class T, class I, int V>
__global__ __launch_bounds__(kBlock) void k_embed_fwd(const T* __restrict__ weight, int64_t stride, int64_t vocab,
                                                      int D, const I* __restrict__ tokens, int64_t count,
                                                      float scale, int lanes, T* __restrict__ out) {
    const int per = kBlock / lanes, slot = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
    for (int64_t i = (int64_t)blockIdx.x * per + slot; i < count; i += (int64_t)gridDim.x * per) {
        const I t = tokens[i];
        const bool ok = token_ok(t, vocab);
        const T* src = weight + (ok ? (int64_t)t : 0) * stride;
        T* dst = out + i * D;
        for (int d = lane * V; d < D; d += lanes * V) {
            const int at = d + V <= D ? d : D - V;
            Pack<T, V> q = load_pack<T, V>(src + at);
#pragma unroll
            for (int j = 0; j < V; ++j) q.v[j] = ok ? from_f32<T>(to_f32(q.v[j]) * scale) : from_f32<T>(__builtin_nanf(""));
            store_pack<T, V>(dst + at, q);
        }
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
