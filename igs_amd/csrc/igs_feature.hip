// igs_feature.hip -- the operators in front of the module's head (the features that
// src/igs/gs2d.py:611-635 of the reference takes as given): embedding lookup with its dense gradient,
// layer norm forward and backward, dropout from a counter-based generator.  Kernels in the included
// headers, argument checks and launches here.
//
// All of them are bound by memory traffic (a few operations per element); the sums of gradients over
// rows or repeated tokens have a fixed order, so results are bit-reproducible run to run.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <atomic>
#include <utility>

#include "igs_hip.h"

namespace {
#include "igs_feature_common.h"

#include "igs_dropout.h"
#include "igs_embedding.h"
#include "igs_layer_norm.h"

constexpr int64_t kMaxCount = 0x7FFFFFFE;
constexpr int kMaxRow = 1 << 20;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t at_most(int64_t v, int64_t most) { return v < most ? v : most; }

inline int launch_status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? IGS_OK : (int)e;
}

inline bool dtype_ok(int t) { return t == IGS_F32 || t == IGS_F16 || t == IGS_BF16; }
inline int dtype_bytes(int t) { return t == IGS_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

int make_dropout(int threshold, uint64_t seed, const uint64_t* seed_device, uint64_t offset, Dropout* d) {
    if (threshold < 0 || threshold > 65536) return IGS_ERR_BAD_ARGUMENT;
    if (!aligned_to(seed_device, 8)) return IGS_ERR_ALIGNMENT;
    d->threshold = (uint32_t)threshold;
    d->factor = threshold < 65536 ? (float)(65536.0 / (65536 - threshold)) : 0.0f;
    d->seed = seed;
    d->offset = offset;
    d->seed_device = seed_device;
    return IGS_OK;
}

int embedding_shape(int64_t vocab, int D, int64_t count) {
    if (vocab < 1 || vocab > kMaxCount || D < 1 || D > kMaxRow || count < 0 || count > kMaxCount) return IGS_ERR_BAD_SHAPE;
    return IGS_OK;
}

// What the dense gradient of a lookup is made of, a function of its sizes alone.
struct EmbedPlan {
    int passes, bits;        // of the sort: digits and their width
    int tiles, tile;         // more than kSortOne tokens: tiles of so many keys
    SumShape sum;
    int64_t span;            // sorted places per group of k_embed_sum
    int64_t padded;          // elements of a key or position array
    size_t counts_at, partial_at, bytes;  // in the workspace, behind the arrays
};

#ifndef IGS_EMBED_SUM_WAVES
#define IGS_EMBED_SUM_WAVES 8192
#endif
#ifndef IGS_EMBED_FILL_BYTES
#define IGS_EMBED_FILL_BYTES (64 << 10)  // per filling workgroup
#endif

EmbedPlan make_embed_plan(int64_t vocab, int D, int dtype, int64_t n) {
    EmbedPlan p;
    int total = 0;  // bits of the largest key, vocab itself
    while (vocab >> total) ++total;
    const bool one = n <= kSortOne;
    const int most = one ? 8 : kSortBits;
    p.passes = (total + most - 1) / most;
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
    const int64_t len = ceil_div(ceil_div(waves, IGS_EMBED_SUM_WAVES), kUnroll) * kUnroll;
    s.len = (int)(len < kUnroll ? kUnroll : len);
    p.span = (int64_t)(kSumThreads / s.lanes) * s.len;
    s.groups = (int)ceil_div(n, p.span);
    p.padded = ceil_div(n, 4) * 4;
    const size_t arrays = (size_t)p.padded * sizeof(int) * (one ? 2 : 4);
    p.counts_at = (arrays + 15) & ~(size_t)15;
    p.partial_at = (p.counts_at + ((size_t)p.tiles << p.bits) * sizeof(int) + 15) & ~(size_t)15;
    p.bytes = p.partial_at + (s.groups > 1 ? (size_t)s.groups * 2 * D * sizeof(float) : 0);
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

int norm_shape(int64_t rows, int D, int dtype, int wdtype) {
    if (!dtype_ok(dtype) || (wdtype != dtype && wdtype != IGS_F32)) return IGS_ERR_BAD_DTYPE;
    if (rows < 0 || rows > kMaxCount || D < 1 || D > kMaxRow) return IGS_ERR_BAD_SHAPE;
    return IGS_OK;
}

// Compute units of the current device (of an MI355X where there is none: plans are made without a GPU too).
int device_cus() {
    static std::atomic<int> cached{0};
    int cus = cached.load(std::memory_order_relaxed);
    if (cus > 0) return cus;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) {
        (void)hipGetLastError();
        return 256;
    }
    cached.store(cus, std::memory_order_relaxed);
    return cus;
}

// How a row of D elements is laid over threads: TPR threads of NV packs of V elements.  The smallest
// arrangement that holds the row: a wave of up to 16 elements per thread, a workgroup of 256 threads of up
// to 32, one of 512 (24 or 32).  More elements cost the backward, which has x, gy, h, d, w and the two
// sums of every element in registers, its occupancy; a workgroup of 1024 threads leaves a thread too few
// registers for 16 (fp16 2053 x 8205, backward: 65 us there).
struct NormShape {
    int tpr, nv;
    bool one, is_long;  // V = 1; no arrangement holds the row
};

NormShape norm_layout(int D, int dtype) {
    const int V = 16 / dtype_bytes(dtype);
    if (D < V) return {8, 1, true, false};
    const int packs = (int)ceil_div(D, V), unit = 8 / V;  // packs of eight elements
    for (int tpr = 8; tpr <= kWave; tpr *= 2)
        if (packs <= tpr) return {tpr, 1, false, false};
    for (int nv = 2; nv <= 2 * unit; nv *= 2)
        if (packs <= kWave * nv) return {kWave, nv, false, false};
    for (int k = 1; k <= 4; ++k)
        if (packs <= 256 * k * unit) return {256, k * unit, false, false};
    for (int k = 3; k <= 4; ++k)
        if (packs <= 512 * k * unit) return {512, k * unit, false, false};
    return {kLong, 0, false, true};
}

inline int norm_rows_at_once(const NormShape& s) { return s.tpr > kBlock ? 1 : kBlock / s.tpr; }

#ifndef IGS_NORM_FWD_WGS
#define IGS_NORM_FWD_WGS 8
#endif
#ifndef IGS_NORM_BWD_WGS
#define IGS_NORM_BWD_WGS 4
#endif
// Workgroups of the norm kernels: resident at once where there are more rows than that.
int64_t norm_groups(const NormShape& s, int64_t rows, int per_cu) {
    const int64_t all = ceil_div(rows, norm_rows_at_once(s));
    return at_most(all, (int64_t)device_cus() * (s.tpr > kBlock ? (per_cu + 1) / 2 : per_cu));
}

int norm_plan(int64_t rows, int D, int dtype, int wdtype, igs_layer_norm_plan_t* p) {
    if (!p) return IGS_ERR_NULL_POINTER;
    const int rc = norm_shape(rows, D, dtype, wdtype);
    if (rc) return rc;
    const NormShape s = norm_layout(D, dtype);
    int64_t P;
    if (s.is_long) {  // row groups so that there are eight workgroups per compute unit
        P = ceil_div((int64_t)device_cus() * 8, ceil_div(D, kWave));
        P = at_most(P, ceil_div(rows, kBlock / kWave));
    } else {
        P = norm_groups(s, rows, IGS_NORM_BWD_WGS);
    }
    p->rows = rows;
    p->D = D;
    p->partials = (int32_t)P;
    p->ws_bytes = (uint64_t)P * 2 * D * sizeof(float);
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
    const bool four = ceil_div(count, 4 * per) >= 8 * (int64_t)device_cus();
    const dim3 grid(ceil_div(count, four ? 4 * per : per));
#define IGS_EMBED_FWD(VV, U)                                                                                    \
    hipLaunchKernelGGL((k_embed_fwd<T, I, VV, U>), grid, dim3(kBlock), 0, st, (const T*)weight, stride, vocab, D, \
                       (const I*)tokens, count, scale, lanes, (T*)out)
    if (D < V) {
        if (four) IGS_EMBED_FWD(1, 4);
        else IGS_EMBED_FWD(1, 1);
    } else {
        if (four) IGS_EMBED_FWD(V, 4);
        else IGS_EMBED_FWD(V, 1);
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

template <class T, class I>
int launch_embed_bwd(const void* grad, const void* tokens, int64_t n, int64_t vocab, int D, float scale,
                     int64_t padding, void* out_, void* ws, hipStream_t st) {
    const EmbedPlan p = make_embed_plan(vocab, D, sizeof(T) == 4 ? IGS_F32 : IGS_F16, n);
    T* out = (T*)out_;
    const int64_t total = vocab * D;
    // workgroups that fill `count` elements with zeros
    const auto filling = [](int64_t count) {
        return at_most(ceil_div(count * (int64_t)sizeof(T), IGS_EMBED_FILL_BYTES), 1 << 20);
    };
    if (n == 0) {
        hipLaunchKernelGGL((k_fill<T>), dim3(filling(total)), dim3(kSortThreads), 0, st, out, total);
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
            hipLaunchKernelGGL((k_sort_place<T, I>), dim3(p.tiles + filling(c)), dim3(kSortThreads), 0, st, src, n, p.tile,
                               p.tiles, k * p.bits, p.bits, (const int*)counts, keys, pos, out + filled, c);
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

// f(TPR, NV, V) as constants for the arrangement `s` of a row
template <int TPR, int NV, int V>
struct NormLayout {
    static constexpr int tpr = TPR, nv = NV, v = V;
};
template <class T, class F>
void norm_dispatch(const NormShape& s, F f) {
    constexpr int V = kVec<T>, U = 8 / V;  // packs of eight elements
    if (s.one) return f(NormLayout<8, 1, 1>());
    if (s.tpr <= kWave) {
        if (s.tpr == 8) return f(NormLayout<8, 1, V>());
        if (s.tpr == 16) return f(NormLayout<16, 1, V>());
        if (s.tpr == 32) return f(NormLayout<32, 1, V>());
        if (s.nv == 1) return f(NormLayout<64, 1, V>());
        if (s.nv == 2) return f(NormLayout<64, 2, V>());
        return f(NormLayout<64, 2 * U, V>());
    }
    if (s.tpr == 256) {
        if (s.nv == U) return f(NormLayout<256, U, V>());
        if (s.nv == 2 * U) return f(NormLayout<256, 2 * U, V>());
        if (s.nv == 3 * U) return f(NormLayout<256, 3 * U, V>());
        return f(NormLayout<256, 4 * U, V>());
    }
    if (s.nv == 3 * U) return f(NormLayout<512, 3 * U, V>());
    return f(NormLayout<512, 4 * U, V>());
}

template <class T, class W>
int launch_norm_fwd(const void* x, int64_t stride, const void* w, const void* b, int64_t rows, int D, float eps,
                    const Dropout& d, void* y, float* stats, hipStream_t st) {
    const NormShape s = norm_layout(D, sizeof(T) == 4 ? IGS_F32 : IGS_F16);
    if (s.is_long)
        hipLaunchKernelGGL((k_norm_fwd_long<T, W>), dim3(at_most(rows, 1 << 20)), dim3(kLong), 0, st, (const T*)x, stride,
                           (const W*)w, (const W*)b, rows, D, eps, d, (T*)y, stats);
    else
        norm_dispatch<T>(s, [&](auto l) {
            using L = decltype(l);
            hipLaunchKernelGGL((k_norm_fwd<T, W, L::tpr, L::nv, L::v>), dim3(norm_groups(s, rows, IGS_NORM_FWD_WGS)),
                               dim3(norm_threads(L::tpr)), 0, st, (const T*)x, stride, (const W*)w, (const W*)b, rows, D,
                               eps, d, (T*)y, stats);
        });
    return launch_status();
}

template <class T, class W>
int launch_norm_bwd(const void* gy, const void* x, int64_t stride, const void* w, const float* stats, int64_t rows,
                    int D, const Dropout& d, int partials, void* gx, void* gw, void* gb, float* part, hipStream_t st) {
    const NormShape s = norm_layout(D, sizeof(T) == 4 ? IGS_F32 : IGS_F16);
    const bool sums = gw || gb;
    if (rows && s.is_long) {
        if (gx)
            hipLaunchKernelGGL((k_norm_bwd_x_long<T, W>), dim3(at_most(rows, 1 << 20)), dim3(kLong), 0, st, (const T*)gy,
                               (const T*)x, stride, (const W*)w, stats, rows, D, d, (T*)gx);
        if (sums)
            hipLaunchKernelGGL((k_norm_bwd_w_long<T>), dim3(ceil_div(D, kWave), partials), dim3(kBlock), 0, st,
                               (const T*)gy, (const T*)x, stride, stats, rows, D, d, part);
    } else if (rows && (gx || sums)) {
        norm_dispatch<T>(s, [&](auto l) {
            using L = decltype(l);
            hipLaunchKernelGGL((k_norm_bwd<T, W, L::tpr, L::nv, L::v>), dim3(partials), dim3(norm_threads(L::tpr)), 0, st,
                               (const T*)gy, (const T*)x, stride, (const W*)w, stats, rows, D, d, (T*)gx,
                               sums ? part : (float*)nullptr);
        });
    }
    if (sums)
        hipLaunchKernelGGL((k_norm_reduce<W>), dim3(ceil_div(2 * D, kReduceCols)), dim3(kWave * kReduceWaves), 0, st,
                           (const float*)part, partials, D, (W*)gw, (W*)gb);
    return launch_status();
}

// f<T, W>(args...) of the pair of types (norm_shape has refused the others)
#define IGS_BY_TYPES(f, dtype, wdtype, ...)                                                             \
    ((dtype) == IGS_F32   ? f<float, float>(__VA_ARGS__)                                                \
     : (dtype) == IGS_F16 ? ((wdtype) == IGS_F32 ? f<f16, float>(__VA_ARGS__) : f<f16, f16>(__VA_ARGS__)) \
                          : ((wdtype) == IGS_F32 ? f<bf16, float>(__VA_ARGS__) : f<bf16, bf16>(__VA_ARGS__)))
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

int igs_layer_norm_forward(const void* x, int64_t x_row_stride, int dtype, const void* weight, const void* bias,
                           int wdtype, int64_t rows, int D, float eps, int threshold, uint64_t seed,
                           const uint64_t* seed_device, uint64_t offset, void* y, float* stats, igs_stream_t stream) {
    int rc = norm_shape(rows, D, dtype, wdtype);
    if (rc) return rc;
    if (!(eps >= 0.0f) || !isfinite(eps) || x_row_stride < 0) return IGS_ERR_BAD_ARGUMENT;
    Dropout d;
    rc = make_dropout(threshold, seed, seed_device, offset, &d);
    if (rc) return rc;
    if (rows == 0) return IGS_OK;
    if (!x || !y) return IGS_ERR_NULL_POINTER;
    const int e = dtype_bytes(dtype), we = dtype_bytes(wdtype);
    if (!aligned_to(x, e) || !aligned_to(y, e) || !aligned_to(weight, we) || !aligned_to(bias, we) ||
        !aligned_to(stats, 8))
        return IGS_ERR_ALIGNMENT;
    return IGS_BY_TYPES(launch_norm_fwd, dtype, wdtype, x, x_row_stride, weight, bias, rows, D, eps, d, y, stats,
                        (hipStream_t)stream);
}

int igs_layer_norm_plan(int64_t rows, int D, int dtype, int wdtype, igs_layer_norm_plan_t* plan) {
    return norm_plan(rows, D, dtype, wdtype, plan);
}

int igs_layer_norm_backward(const void* grad_y, const void* x, int64_t x_row_stride, int dtype, const void* weight,
                            int wdtype, const float* stats, int64_t rows, int D, int threshold, uint64_t seed,
                            const uint64_t* seed_device, uint64_t offset, void* grad_x, void* grad_weight,
                            void* grad_bias, void* ws, size_t ws_bytes, igs_stream_t stream) {
    igs_layer_norm_plan_t p;
    int rc = norm_plan(rows, D, dtype, wdtype, &p);
    if (rc) return rc;
    if (x_row_stride < 0) return IGS_ERR_BAD_ARGUMENT;
    Dropout d;
    rc = make_dropout(threshold, seed, seed_device, offset, &d);
    if (rc) return rc;
    if (rows && (!grad_y || !x || !stats)) return IGS_ERR_NULL_POINTER;
    if (p.ws_bytes && !ws && (grad_weight || grad_bias)) return IGS_ERR_NULL_POINTER;
    if (ws_bytes < p.ws_bytes && (grad_weight || grad_bias)) return IGS_ERR_WORKSPACE;
    const int e = dtype_bytes(dtype), we = dtype_bytes(wdtype);
    if (!aligned_to(grad_y, e) || !aligned_to(x, e) || !aligned_to(grad_x, e) || !aligned_to(weight, we) ||
        !aligned_to(grad_weight, we) || !aligned_to(grad_bias, we) || !aligned_to(stats, 8) || !aligned_to(ws, 16))
        return IGS_ERR_ALIGNMENT;
    return IGS_BY_TYPES(launch_norm_bwd, dtype, wdtype, grad_y, x, x_row_stride, weight, stats, rows, D, d, p.partials,
                        grad_x, grad_weight, grad_bias, (float*)ws, (hipStream_t)stream);
}
}  // extern "C"
