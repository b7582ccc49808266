// igs_norm.hip -- layer norm over rows with dropout of its result, forward and backward: arrangements of a
// row over threads, argument checks and launches around the kernels of igs_layer_norm.h.

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <atomic>

#include "igs_hip.h"

namespace {
#include "igs_feature_common.h"
#include "igs_feature_host.h"

#include "igs_layer_norm.h"

int norm_shape(int64_t rows, int D, int dtype, int wdtype) {
    if (!dtype_ok(dtype) || (wdtype != dtype && wdtype != IGS_F32)) return IGS_ERR_BAD_DTYPE;
    if (rows < 0 || rows > kMaxCount || D < 1 || D > kMaxRow) return IGS_ERR_BAD_SHAPE;
    return IGS_OK;
}

// How a row of D elements is laid over threads: TPR threads of NV packs of V elements, the smallest
// arrangement that holds the row.  A wave or 128 threads of up to 16 elements each, a workgroup of 256 threads of
// up to 32, one of 512 (24 or 32).  The backward, which has x, gy, h, d, w and the two sums of every element in
// registers, takes no more than 16 (kTwoPass elements a row); wider rows go in two kernels there.
struct NormShape {
    int tpr, nv;
    bool one, is_long;  // V = 1; no arrangement holds the row
};
constexpr int kTwoPass = 4096;

NormShape norm_layout(int D, int dtype) {
    const int V = 16 / dtype_bytes(dtype);
    if (D < V) return {8, 1, true, false};
    const int packs = (int)ceil_div(D, V), unit = 8 / V;  // packs of eight elements
    for (int tpr = 4; tpr <= kWave; tpr *= 2)
        if (packs <= tpr) return {tpr, 1, false, false};
    for (int nv = 2; nv <= 2 * unit; nv *= 2)
        if (packs <= kWave * nv) return {kWave, nv, false, false};
    if (packs <= 128 * 2 * unit) return {128, 2 * unit, false, false};
    for (int k = 2; k <= 4; ++k)
        if (packs <= 256 * k * unit) return {256, k * unit, false, false};
    for (int k = 3; k <= 4; ++k)
        if (packs <= 512 * k * unit) return {512, k * unit, false, false};
    return {kLong, 0, false, true};
}

inline int norm_rows_at_once(const NormShape& s) { return s.tpr > kBlock ? 1 : kBlock / s.tpr; }
inline int norm_elements(const NormShape& s, int dtype) { return s.one ? 1 : s.nv * (16 / dtype_bytes(dtype)); }

// Workgroups per compute unit: each loads the weights of its columns once and, in the backward, leaves a
// partial row of 2 D sums, so few workgroups that walk over many rows, but enough to keep the memory busy
// (us at 2 / 4 / 6 per compute unit, backward: bf16 32768 x 1024 40 / 45 / 50, fp32 4096 x 4096
// 46 / 57 / 69, bf16 65536 x 256 25 / 23 / 27).
constexpr int kFwdGroups = 8, kFwdGroupsWide = 2, kFwdGroups512 = 1;  // 16 elements a thread at most; more; 512 threads
constexpr int kBwdGroups = 4, kBwdGroups16 = 2;                       // 8 elements a thread at most; more
constexpr int kColsGroups = 4;                                        // of k_norm_bwd_cols
int64_t norm_fwd_groups(const NormShape& s, int64_t rows, int dtype) {
    const int per_cu = s.tpr > kBlock ? kFwdGroups512 : norm_elements(s, dtype) > 16 ? kFwdGroupsWide : kFwdGroups;
    return at_most(ceil_div(rows, norm_rows_at_once(s)), (int64_t)device_cus() * per_cu);
}
int64_t norm_bwd_groups(const NormShape& s, int64_t rows, int dtype) {
    const int per_cu = norm_elements(s, dtype) > 8 ? kBwdGroups16 : kBwdGroups;
    return at_most(ceil_div(rows, norm_rows_at_once(s)), (int64_t)device_cus() * per_cu);
}

inline int norm_slices(int D, int dtype) { return (int)ceil_div(ceil_div(D, 16 / dtype_bytes(dtype)), kWave); }

int norm_plan(int64_t rows, int D, int dtype, int wdtype, igs_layer_norm_plan_t* p) {
    if (!p) return IGS_ERR_NULL_POINTER;
    const int rc = norm_shape(rows, D, dtype, wdtype);
    if (rc) return rc;
    int64_t P, row_sums = 0;
    if (D > kTwoPass) {  // groups of rows: two rounds of loads per wave, or as many as the device holds workgroups
        P = at_most(ceil_div(rows, 2 * kRowsAhead * (kBlock / kWave)),
                    ceil_div((int64_t)device_cus() * kColsGroups, norm_slices(D, dtype)));
        row_sums = rows;
    } else {
        P = norm_bwd_groups(norm_layout(D, dtype), rows, dtype);
    }
    p->rows = rows;
    p->D = D;
    p->partials = (int32_t)P;
    p->ws_bytes = (uint64_t)P * 2 * D * sizeof(float) + row_sums * sizeof(float2);
    return IGS_OK;
}

// f(TPR, NV, V) as constants for the arrangement `s` of a row
template <int TPR, int NV, int V>
struct NormLayout {
    static constexpr int tpr = TPR, nv = NV, v = V;
};
template <class T, class F>
void norm_dispatch(const NormShape& s, F f) {  // rows of up to kTwoPass elements
    constexpr int V = kVec<T>, U = 8 / V;  // packs of eight elements
    if (s.one) return f(NormLayout<8, 1, 1>());
    if (s.tpr <= kWave) {
        if (s.tpr == 4) return f(NormLayout<4, 1, V>());
        if (s.tpr == 8) return f(NormLayout<8, 1, V>());
        if (s.tpr == 16) return f(NormLayout<16, 1, V>());
        if (s.tpr == 32) return f(NormLayout<32, 1, V>());
        if (s.nv == 1) return f(NormLayout<64, 1, V>());
        if (s.nv == 2) return f(NormLayout<64, 2, V>());
        return f(NormLayout<64, 2 * U, V>());
    }
    if (s.tpr == 128) return f(NormLayout<128, 2 * U, V>());
    return f(NormLayout<256, 2 * U, V>());
}
template <class T, class F>
void norm_dispatch_wide(const NormShape& s, F f) {  // more
    constexpr int V = kVec<T>, U = 8 / V;
    if (s.tpr == 256) {
        if (s.nv == 3 * U) return f(NormLayout<256, 3 * U, V>());
        return f(NormLayout<256, 4 * U, V>());
    }
    if (s.nv == 3 * U) return f(NormLayout<512, 3 * U, V>());
    return f(NormLayout<512, 4 * U, V>());
}

template <class T, class W>
int launch_norm_fwd(const void* x, int64_t stride, const void* w, const void* b, int64_t rows, int D, float eps,
                    const Dropout& d, void* y, float* stats, hipStream_t st) {
    constexpr int dtype = sizeof(T) == 4 ? IGS_F32 : IGS_F16;
    const NormShape s = norm_layout(D, dtype);
    // Past the caches goes y where a backward follows (bf16 131072 x 1024, forward and backward 250 us without, 240
    // with it; 249 with x instead), and x where none does (forward 98 us without, 84 with x, 95 with y).
    const bool large = rows * D * (int64_t)sizeof(T) >= kStreamBytes;
    const auto launch = [&](auto l) {
        using L = decltype(l);
        const dim3 grid(norm_fwd_groups(s, rows, dtype)), threads(norm_threads(L::tpr));
        if (large && stats)
            hipLaunchKernelGGL((k_norm_fwd<T, W, L::tpr, L::nv, L::v, true>), grid, threads, 0, st, (const T*)x, stride,
                               (const W*)w, (const W*)b, rows, D, eps, d, false, (T*)y, stats);
        else
            hipLaunchKernelGGL((k_norm_fwd<T, W, L::tpr, L::nv, L::v, false>), grid, threads, 0, st, (const T*)x, stride,
                               (const W*)w, (const W*)b, rows, D, eps, d, large, (T*)y, stats);
    };
    if (s.is_long)
        hipLaunchKernelGGL((k_norm_fwd_long<T, W>), dim3(at_most(rows, 1 << 20)), dim3(kLong), 0, st, (const T*)x, stride,
                           (const W*)w, (const W*)b, rows, D, eps, d, (T*)y, stats);
    else if (D > kTwoPass)
        norm_dispatch_wide<T>(s, launch);
    else
        norm_dispatch<T>(s, launch);
    return launch_status();
}

template <class T, class W>
int launch_norm_bwd(const void* gy, const void* x, int64_t stride, const void* w, const float* stats, int64_t rows,
                    int D, const Dropout& d, int partials, void* gx, void* gw, void* gb, void* ws, hipStream_t st) {
    constexpr int dtype = sizeof(T) == 4 ? IGS_F32 : IGS_F16;
    const bool sums = gw || gb;
    float* part = sums ? (float*)ws : nullptr;
    if (rows && D > kTwoPass) {
        float2* row_sums = (float2*)((float*)ws + (size_t)partials * 2 * D);
        if (gx)
            hipLaunchKernelGGL((k_norm_bwd_sums<T, W>), dim3(at_most(rows, (int64_t)device_cus() * 8)), dim3(kBlock), 0, st,
                               (const T*)gy, (const T*)x, stride, (const W*)w, stats, rows, D, d, row_sums);
        if (gx || sums)
            hipLaunchKernelGGL((k_norm_bwd_cols<T, W>), dim3(norm_slices(D, dtype), partials), dim3(kBlock), 0, st,
                               (const T*)gy, (const T*)x, stride, (const W*)w, stats, (const float2*)row_sums, rows, D, d,
                               (T*)gx, part);
    } else if (rows && (gx || sums)) {
        norm_dispatch<T>(norm_layout(D, dtype), [&](auto l) {
            using L = decltype(l);
            hipLaunchKernelGGL((k_norm_bwd<T, W, L::tpr, L::nv, L::v>), dim3(partials), dim3(norm_threads(L::tpr)), 0, st,
                               (const T*)gy, (const T*)x, stride, (const W*)w, stats, rows, D, d,
                               2 * rows * D * (int64_t)sizeof(T) >= kStreamBytes, (T*)gx, part);
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
}  // namespace

extern "C" {
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
    if (p.ws_bytes && !ws) return IGS_ERR_NULL_POINTER;
    if (ws_bytes < p.ws_bytes) return IGS_ERR_WORKSPACE;
    const int e = dtype_bytes(dtype), we = dtype_bytes(wdtype);
    if (!aligned_to(grad_y, e) || !aligned_to(x, e) || !aligned_to(grad_x, e) || !aligned_to(weight, we) ||
        !aligned_to(grad_weight, we) || !aligned_to(grad_bias, we) || !aligned_to(stats, 8) || !aligned_to(ws, 16))
        return IGS_ERR_ALIGNMENT;
    return IGS_BY_TYPES(launch_norm_bwd, dtype, wdtype, grad_y, x, x_row_stride, weight, stats, rows, D, d, p.partials,
                        grad_x, grad_weight, grad_bias, ws, (hipStream_t)stream);
}
}  // extern "C"
