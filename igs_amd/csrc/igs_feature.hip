// igs_feature.hip -- operators in front of the module's head (the features that src/igs/gs2d.py:611-635
// of the reference takes as given): embedding lookup with its dense gradient, and dropout from a
// counter-based generator.  (Layer norm: igs_norm.hip.)  Kernels in the included headers, argument checks
// and launches here.
//
// Both are bound by memory traffic (a few operations per element); the sums of gradients of repeated tokens
// have a fixed order, so results are bit-reproducible run to run.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <atomic>
#include <utility>

#include "igs_hip.h"

namespace {
#include "igs_feature_common.h"
#include "igs_feature_host.h"

#include "igs_dropout.h"
#include "igs_embedding.h"

int embedding_shape(int64_t vocab, int D, int64_t count) {
    if (vocab < 1 || vocab > kMaxCount || D < 1 || D > kMaxRow || count < 0 || count > kMaxCount) return IGS_ERR_BAD_SHAPE;
    return IGS_OK;
}

// What the dense gradient of a lookup is made of, a function of its sizes alone.
struct EmbedPlan {
    bool small;              // k_embed_small does all of it
    int passes, bits;        // of the sort: digits and their width
    int tiles, tile;         // more than kSortOne tokens: tiles of so many keys
    SumShape sum;
    int64_t span;            // sorted places per group of k_embed_sum
    int64_t padded;          // elements of a key or position array
    size_t counts_at, partial_at, bytes;  // in the workspace, behind the arrays
};

constexpr int kSumWaves = 4096;        // of k_embed_sum on the device, about
constexpr int kFillBytes = 64 << 10;   // per filling workgroup

EmbedPlan make_embed_plan(int64_t vocab, int D, int dtype, int64_t n) {  // n >= 1
    EmbedPlan p;
    int total = 0;  // bits of the largest key, vocab itself
    while (vocab >> total) ++total;
    const bool one = n <= kSortOne;
    p.small = n <= kSmall;
    p.passes = (total + kSortBits - 1) / kSortBits;
    p.bits = (total + p.passes - 1) / p.passes;
    p.tiles = p.tile = 0;
    if (!one) {
        p.tiles = (int)at_most(kSortTiles, ceil_div(n, 2 * kSortThreads));
        p.tile = (int)(ceil_div(ceil_div(n, p.tiles), kSortThreads) * kSortThreads);
        p.tiles = (int)ceil_div(n, p.tile);
    }
    const int V = D < 16 / dtype_bytes(dtype) ? 1 : 16 / dtype_bytes(dtype);
    SumShape& s = p.sum;
    const int64_t packs = ceil_div(D, V);
    s.lanes = 8;
    while (s.lanes < packs && s.lanes < kWave) s.lanes *= 2;
    s.slices = (int)ceil_div(packs, s.lanes);
    // places per unit: short enough for so many waves on the device, eight (one group of loads) at least
    const int64_t waves = n * s.slices * s.lanes / kWave;
    const int64_t len = ceil_div(ceil_div(waves, kSumWaves), kUnroll) * kUnroll;
    s.len = (int)(len < kUnroll ? kUnroll : len);
    const int units = (p.small ? kSortThreads : kSumThreads) / s.lanes;
    p.span = (int64_t)units * s.len;
    s.groups = (int)ceil_div(n, p.span);
    s.stream = n * D * dtype_bytes(dtype) >= kStreamBytes;
    p.padded = ceil_div(n, 4) * 4;
    const size_t arrays = (size_t)p.padded * sizeof(int) * (one ? 2 : 4);
    p.counts_at = (arrays + 15) & ~(size_t)15;
    p.partial_at = (p.counts_at + ((size_t)p.tiles << p.bits) * sizeof(int) + 15) & ~(size_t)15;
    p.bytes = p.small ? 0 : p.partial_at + (s.groups > 1 ? (size_t)s.groups * 2 * D * sizeof(float) : 0);
    return p;
}

int embedding_plan(int64_t vocab, int D, int dtype, int64_t count, igs_embedding_plan_t* p) {
    if (!p) return IGS_ERR_NULL_POINTER;
    if (!dtype_ok(dtype)) return IGS_ERR_BAD_DTYPE;
    const int rc = embedding_shape(vocab, D, count);
    if (rc) return rc;
    p->vocab = vocab;
    p->count = count;
    p->D = D;
    p->reserved = 0;
    p->ws_bytes = count ? make_embed_plan(vocab, D, dtype, count).bytes : 0;
    return IGS_OK;
}

template <class T, class I>
int launch_embed_fwd(const void* weight, int64_t stride, int64_t vocab, int D, const void* tokens, int64_t count,
                     float scale, void* out, hipStream_t st) {
    constexpr int V = kVec<T>;
    const int packs = D < V ? D : (int)ceil_div(D, V);
    int lanes = 1;
    while (lanes < packs && lanes < kBlock) lanes *= 2;
    const int per = kBlock / lanes;
    // four tokens in flight per thread where that still leaves eight workgroups per compute unit
    const bool stream = count * D * (int64_t)sizeof(T) >= kStreamBytes;
    const bool four = (stream && D >= V) || ceil_div(count, 4 * per) >= 8 * (int64_t)device_cus();
    const dim3 grid(at_most(ceil_div(count, four ? 4 * per : per), 1 << 23));
#define IGS_EMBED_FWD(VV, U, S)                                                                                   \
    hipLaunchKernelGGL((k_embed_fwd<T, I, VV, U, S>), grid, dim3(kBlock), 0, st, (const T*)weight, stride, vocab, D, \
                       (const I*)tokens, count, scale, lanes, (T*)out)
    if (D < V) {
        if (four) IGS_EMBED_FWD(1, 4, false);
        else IGS_EMBED_FWD(1, 1, false);
    } else {
        if (stream) IGS_EMBED_FWD(V, 4, true);
        else if (four) IGS_EMBED_FWD(V, 4, false);
        else IGS_EMBED_FWD(V, 1, false);
    }
#undef IGS_EMBED_FWD
    return launch_status();
}

template <class T, int V>
void launch_embed_sum(const T* grad, const int* keys, const int* pos, int64_t n, int64_t vocab, int D, float scale,
                      const EmbedPlan& p, float* partial, T* out, hipStream_t st) {
    const SumShape& s = p.sum;
    const dim3 grid((int64_t)s.groups * s.slices);
    if (s.lanes == kWave)
        hipLaunchKernelGGL((k_embed_sum<T, V, true>), grid, dim3(kSumThreads), 0, st, grad, keys, pos, n, vocab, D, scale,
                           s, partial, out);
    else
        hipLaunchKernelGGL((k_embed_sum<T, V, false>), grid, dim3(kSumThreads), 0, st, grad, keys, pos, n, vocab, D, scale,
                           s, partial, out);
    if (s.groups > 1)
        hipLaunchKernelGGL((k_embed_join<T, V>), grid, dim3(kSumThreads), 0, st, keys, n, vocab, D, scale, s, p.span,
                           (const float*)partial, out);
}

template <class T, class I, int V>
void launch_embed_small(const T* grad, const I* tokens, int n, int64_t vocab, int64_t padding, int D, float scale,
                        const EmbedPlan& p, T* out, hipStream_t st) {
    const int64_t fit = kFillBytes / ((int64_t)D * (int)sizeof(T));
    const int64_t least = ceil_div(vocab, 1 << 21);  // a launch has fewer than 2^32 threads
    const int rows = (int)(fit < least ? least : at_most(fit, kSmall));
    const dim3 grid((int64_t)p.sum.groups * p.sum.slices + ceil_div(vocab, rows));
    if (p.sum.lanes == kWave)
        hipLaunchKernelGGL((k_embed_small<T, I, V, true>), grid, dim3(kSortThreads), 0, st, grad, tokens, n, vocab, padding,
                           D, scale, p.passes, p.bits, p.sum, rows, out);
    else
        hipLaunchKernelGGL((k_embed_small<T, I, V, false>), grid, dim3(kSortThreads), 0, st, grad, tokens, n, vocab, padding,
                           D, scale, p.passes, p.bits, p.sum, rows, out);
}

template <class T, class I>
int launch_embed_bwd(const void* grad, const void* tokens, int64_t n, int64_t vocab, int D, float scale,
                     int64_t padding, void* out_, void* ws, hipStream_t st) {
    T* out = (T*)out_;
    const int64_t total = vocab * D;
    // workgroups that fill `count` elements with zeros
    const auto filling = [](int64_t count) {
        return at_most(ceil_div(count * (int64_t)sizeof(T), kFillBytes), 1 << 20);
    };
    if (n == 0) {
        hipLaunchKernelGGL((k_fill<T>), dim3(filling(total)), dim3(kSortThreads), 0, st, out, total);
        return launch_status();
    }
    const EmbedPlan p = make_embed_plan(vocab, D, sizeof(T) == 4 ? IGS_F32 : IGS_F16, n);
    if (p.small) {
        if (D < kVec<T>)
            launch_embed_small<T, I, 1>((const T*)grad, (const I*)tokens, (int)n, vocab, padding, D, scale, p, out, st);
        else
            launch_embed_small<T, I, kVec<T>>((const T*)grad, (const I*)tokens, (int)n, vocab, padding, D, scale, p, out, st);
        return launch_status();
    }
    int *keys = (int*)ws, *pos = keys + p.padded;
    float* partial = (float*)((char*)ws + p.partial_at);
    if (!p.tiles) {
        hipLaunchKernelGGL((k_sort_one<T, I>), dim3(1 + filling(total)), dim3(kSortThreads), 0, st, (const I*)tokens, (int)n,
                           vocab, padding, p.passes, p.bits, keys, pos, out, total);
    } else {
        int *other_keys = pos + p.padded, *other_pos = other_keys + p.padded;
        int* counts = (int*)((char*)ws + p.counts_at);
        SortSource<I> src{(const I*)tokens, nullptr, nullptr, vocab, padding};
        // every launch of the sort fills its share of the rows
        const int64_t share = ceil_div(ceil_div(total, 2 * p.passes), 16) * 16;
        int64_t filled = 0;
        const auto next = [&] { return at_most(share, total - filled); };
        for (int k = 0; k < p.passes; ++k) {
            int64_t c = next();
            hipLaunchKernelGGL((k_sort_count<T, I>), dim3(p.tiles + filling(c)), dim3(kSortThreads), 0, st, src, n, p.tile,
                               p.tiles, k * p.bits, p.bits, counts, out + filled, c);
            filled += c;
            c = next();
            if (p.tile <= kSortHeld * kSortThreads)
                hipLaunchKernelGGL((k_sort_place<T, I, true>), dim3(p.tiles + filling(c)), dim3(kSortThreads), 0, st, src, n,
                                   p.tile, p.tiles, k * p.bits, p.bits, (const int*)counts, keys, pos, out + filled, c);
            else
                hipLaunchKernelGGL((k_sort_place<T, I, false>), dim3(p.tiles + filling(c)), dim3(kSortThreads), 0, st, src, n,
                                   p.tile, p.tiles, k * p.bits, p.bits, (const int*)counts, keys, pos, out + filled, c);
            filled += c;
            src = SortSource<I>{nullptr, keys, pos, vocab, padding};
            std::swap(keys, other_keys);
            std::swap(pos, other_pos);
        }
        keys = other_keys;  // where the last pass wrote
        pos = other_pos;
    }
    if (D < kVec<T>)
        launch_embed_sum<T, 1>((const T*)grad, keys, pos, n, vocab, D, scale, p, partial, out, st);
    else
        launch_embed_sum<T, kVec<T>>((const T*)grad, keys, pos, n, vocab, D, scale, p, partial, out, st);
    return launch_status();
}

template <class T>
int launch_dropout(const void* x, int64_t count, const Dropout& d, void* y, hipStream_t st) {
    constexpr int kPacks = 2;
    const int64_t packs = count / kVec<T>, groups = packs ? ceil_div(packs, kBlock * kPacks) : 1;
    hipLaunchKernelGGL((k_dropout<T, kPacks>), dim3(groups), dim3(kBlock), 0, st, (const T*)x, count, d, (T*)y);
    return launch_status();
}

// f<T, I>(args...) of an element type and a token width
#define IGS_BY_TOKENS(f, dtype, bytes, ...)                                                            \
    ((dtype) == IGS_F32   ? ((bytes) == 8 ? f<float, int64_t>(__VA_ARGS__) : f<float, int32_t>(__VA_ARGS__)) \
     : (dtype) == IGS_F16 ? ((bytes) == 8 ? f<f16, int64_t>(__VA_ARGS__) : f<f16, int32_t>(__VA_ARGS__)) \
                          : ((bytes) == 8 ? f<bf16, int64_t>(__VA_ARGS__) : f<bf16, int32_t>(__VA_ARGS__)))
}  // namespace

extern "C" {
int igs_embedding_forward(const void* weight, int64_t weight_row_stride, int dtype, int64_t vocab, int D,
                          const void* tokens, int token_bytes, int64_t count, float scale, void* out,
                          igs_stream_t stream) {
    if (!dtype_ok(dtype) || (token_bytes != 4 && token_bytes != 8)) return IGS_ERR_BAD_DTYPE;
    const int rc = embedding_shape(vocab, D, count);
    if (rc) return rc;
    if (!isfinite(scale) || weight_row_stride < 0) return IGS_ERR_BAD_ARGUMENT;
    if (count == 0) return IGS_OK;
    if (!weight || !tokens || !out) return IGS_ERR_NULL_POINTER;
    const int e = dtype_bytes(dtype);
    if (!aligned_to(weight, e) || !aligned_to(out, e) || !aligned_to(tokens, token_bytes)) return IGS_ERR_ALIGNMENT;
    return IGS_BY_TOKENS(launch_embed_fwd, dtype, token_bytes, weight, weight_row_stride, vocab, D, tokens, count,
                         scale, out, (hipStream_t)stream);
}

int igs_embedding_plan(int64_t vocab, int D, int dtype, int64_t count, igs_embedding_plan_t* plan) {
    return embedding_plan(vocab, D, dtype, count, plan);
}

int igs_embedding_backward(const void* grad_out, int dtype, const void* tokens, int token_bytes, int64_t count,
                           int64_t vocab, int D, float scale, int64_t padding_idx, void* grad_weight, void* ws,
                           size_t ws_bytes, igs_stream_t stream) {
    if (token_bytes != 4 && token_bytes != 8) return IGS_ERR_BAD_DTYPE;
    igs_embedding_plan_t p;
    const int rc = embedding_plan(vocab, D, dtype, count, &p);
    if (rc) return rc;
    if (!isfinite(scale) || padding_idx < -1 || padding_idx >= vocab) return IGS_ERR_BAD_ARGUMENT;
    if (!grad_weight || (count && (!grad_out || !tokens)) || (p.ws_bytes && !ws)) return IGS_ERR_NULL_POINTER;
    if (ws_bytes < p.ws_bytes) return IGS_ERR_WORKSPACE;
    const int e = dtype_bytes(dtype);
    if (!aligned_to(ws, 16) || !aligned_to(grad_out, e) || !aligned_to(grad_weight, e) ||
        !aligned_to(tokens, token_bytes))
        return IGS_ERR_ALIGNMENT;
    return IGS_BY_TOKENS(launch_embed_bwd, dtype, token_bytes, grad_out, tokens, count, vocab, D, scale, padding_idx,
                         grad_weight, ws, (hipStream_t)stream);
}

int igs_dropout(const void* x, int dtype, int64_t count, int threshold, uint64_t seed, const uint64_t* seed_device,
                uint64_t offset, void* y, igs_stream_t stream) {
    if (!dtype_ok(dtype)) return IGS_ERR_BAD_DTYPE;
    if (count < 0 || count >= (int64_t)1 << 34) return IGS_ERR_BAD_SHAPE;
    Dropout d;
    const int rc = make_dropout(threshold, seed, seed_device, offset, &d);
    if (rc) return rc;
    if (count == 0) return IGS_OK;
    if (!x || !y) return IGS_ERR_NULL_POINTER;
    const int e = dtype_bytes(dtype);
    if (!aligned_to(x, e) || !aligned_to(y, e)) return IGS_ERR_ALIGNMENT;
    hipStream_t st = (hipStream_t)stream;
    return dtype == IGS_F32   ? launch_dropout<float>(x, count, d, y, st)
           : dtype == IGS_F16 ? launch_dropout<f16>(x, count, d, y, st)
                              : launch_dropout<bf16>(x, count, d, y, st);
}
}  // extern "C"
