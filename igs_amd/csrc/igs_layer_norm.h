// igs_layer_norm.h -- layer norm over rows, forward and backward, with dropout of its result.
// Included by igs_norm.hip inside its anonymous namespace.
//
//   h = (x - mean) rstd,  y = drop(h w + b);   d = drop(gy), g = d w
//   gx = rstd (g - mean g - h mean(g h)),  gw = sum_rows d h,  gb = sum_rows d
//
// Bound by memory: a row is read once and stays in registers between its sums and its result.  TPR
// threads share a row (4 to 64 lanes of a wave, 128 threads, or a workgroup of 256 or 512), NV packs of 16
// bytes each; the weights of a thread's columns stay in registers while its workgroup walks over the
// rows, the next row's loads in flight.  The last pack of a row whose length is no multiple of the
// pack is moved back to end with the row: its first elements are the neighbour's (computed twice, counted
// once).  The backward keeps the two sums over rows for a thread's columns in registers; each workgroup
// leaves one partial row of them, and k_norm_reduce adds those in a fixed order.  The loads of the next row must not meet
// other values of their registers at a branch (zeros for a row that is not there, say): the copy that joins them waits
// for the loads (bf16 32768 x 1024, backward: 48 us instead of 40).
#pragma once

// Sum of up to two values over the TPR threads of a row; across waves through `red`, two buffers used in turn, so that
// one barrier per sum is enough (a wave can be at most one sum ahead of another).
constexpr int kRedWaves = 16;  // of a workgroup, at most
template <int TPR>
struct RowSum {
    static constexpr int kWaves = TPR / kWave;
    float (*red)[2][kRedWaves];  // [turn][value][wave]
    int turn;

    __device__ __forceinline__ void operator()(float& a, float& b) {
        if constexpr (TPR <= kWave) {
            a = lanes_sum<TPR>(a);
            b = lanes_sum<TPR>(b);
        } else {
            a = lanes_sum<kWave>(a);
            b = lanes_sum<kWave>(b);
            const int wave = threadIdx.x / kWave, first = wave & ~(kWaves - 1);
            if ((threadIdx.x & (kWave - 1)) == 0) {
                red[turn][0][wave] = a;
                red[turn][1][wave] = b;
            }
            __syncthreads();
            a = b = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                a += red[turn][0][first + w];
                b += red[turn][1][first + w];
            }
            turn ^= 1;
        }
    }
    __device__ __forceinline__ void operator()(float& a) {
        if constexpr (TPR <= kWave) {
            a = lanes_sum<TPR>(a);
        } else {
            a = lanes_sum<kWave>(a);
            const int wave = threadIdx.x / kWave, first = wave & ~(kWaves - 1);
            if ((threadIdx.x & (kWave - 1)) == 0) red[turn][0][wave] = a;
            __syncthreads();
            a = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) a += red[turn][0][first + w];
            turn ^= 1;
        }
    }
};
constexpr int norm_threads(int tpr) { return tpr > kBlock ? tpr : kBlock; }

template <class T, class W, int TPR, int NV, int V, bool kStreamOut>
__global__ __launch_bounds__(norm_threads(TPR)) void k_norm_fwd(const T* __restrict__ x, int64_t stride,
                                                                const W* __restrict__ w, const W* __restrict__ b,
                                                                int64_t rows, int D, float eps, Dropout drop_, bool stream,
                                                                T* __restrict__ y, float* __restrict__ stats) {
    constexpr int kRows = norm_threads(TPR) / TPR;  // rows of a workgroup at a time
    __shared__ float red[2][2][kRedWaves];
    RowSum<TPR> row_sum{red, 0};
    const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * kRows;
    const PhiloxKey key = philox_key(drop_);
    const bool whole = D % 8 == 0, ragged = D % V != 0;
    const float inv = 1.0f / (float)D;

    int start[NV], skip[NV];  // first element of a pack, elements of it that another thread counts (V: no pack)
    float live[NV];           // 1, or 0 where there is no pack: its elements are zeros then and stay so
    float wv[NV][V], bv[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int col = (k * TPR + lane) * V;
        start[k] = col + V <= D ? col : D - V;
        skip[k] = col < D ? col - start[k] : V;
        live[k] = col < D ? 1.0f : 0.0f;
        Pack<W, V> pw, pb;
        if (skip[k] < V) {
            if (w) pw = load_pack<W, V>(w + start[k]);
            if (b) pb = load_pack<W, V>(b + start[k]);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            wv[k][j] = w ? to_f32(pw.v[j]) : 1.0f;
            bv[k][j] = b ? to_f32(pb.v[j]) : 0.0f;
        }
    }

    Pack<T, V> next[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) next[k].v[j] = from_f32<T>(0.0f);
    int64_t r0 = (int64_t)blockIdx.x * kRows;
    const auto load = [&](int64_t first) {
        const int64_t r = first + slot < rows ? first + slot : rows - 1;  // a slot behind the last row computes it again
        const T* p = x + r * stride;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (skip[k] < V) next[k] = load_pack<T, V>(p + start[k], stream);
    };
    if (r0 < rows) load(r0);
    for (; r0 < rows; r0 += step) {
        float c[NV][V];
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) c[k][j] = to_f32(next[k].v[j]);
        if (r0 + step < rows) load(r0 + step);
        if (!ragged) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) s += c[k][j];
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) s += j >= skip[k] ? c[k][j] : 0.0f;
        }
        row_sum(s);
        const float mean = s * inv;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) c[k][j] = fmaf(-mean, live[k], c[k][j]);
        s = 0.0f;
        if (!ragged) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) s = fmaf(c[k][j], c[k][j], s);
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) s = fmaf(c[k][j], j >= skip[k] ? c[k][j] : 0.0f, s);
        }
        row_sum(s);
        const float rstd = 1.0f / sqrtf(fmaf(s, inv, eps));
        const int64_t r = r0 + slot;
        if (r < rows) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (skip[k] < V) {
                    Pack<T, V> q;
#pragma unroll
                    for (int j = 0; j < V; ++j) c[k][j] = fmaf(c[k][j] * rstd, wv[k][j], bv[k][j]);
                    if (drop_.threshold) drop<V>(c[k], (uint64_t)r * D + start[k], whole, drop_, key);
#pragma unroll
                    for (int j = 0; j < V; ++j) q.v[j] = from_f32<T>(c[k][j]);
                    store_pack<kStreamOut, T, V>(y + r * D + start[k], q);
                }
            if (stats && lane == 0) {
                stats[2 * r] = mean;
                stats[2 * r + 1] = rstd;
            }
        }
    }
}

// part [gridDim.x][2][D]: a workgroup's sums over its rows of d h and of d.  gx may be NULL, and part where neither sum
// is wanted.
template <class T, class W, int TPR, int NV, int V>
__global__ __launch_bounds__(norm_threads(TPR)) void k_norm_bwd(const T* __restrict__ gy, const T* __restrict__ x,
                                                                int64_t stride, const W* __restrict__ w,
                                                                const float* __restrict__ stats, int64_t rows, int D,
                                                                Dropout drop_, bool stream, T* __restrict__ gx,
                                                                float* __restrict__ part) {
    constexpr int kRows = norm_threads(TPR) / TPR;
    __shared__ float red[2][2][kRedWaves];
    __shared__ float sums[kRows > 1 ? 2 * TPR * NV * V : 1];
    RowSum<TPR> row_sum{red, 0};
    const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * kRows;
    const PhiloxKey key = philox_key(drop_);
    const bool whole = D % 8 == 0, ragged = D % V != 0;
    const float inv = 1.0f / (float)D;

    int start[NV], skip[NV];
    float wv[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int col = (k * TPR + lane) * V;
        start[k] = col + V <= D ? col : D - V;
        skip[k] = col < D ? col - start[k] : V;
        Pack<W, V> pw;
        if (w && skip[k] < V) pw = load_pack<W, V>(w + start[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            wv[k][j] = skip[k] == V ? 0.0f : w ? to_f32(pw.v[j]) : 1.0f;
            aw[k][j] = ab[k][j] = 0.0f;
        }
    }

    Pack<T, V> nx[NV], ng[NV], zero;
#pragma unroll
    for (int j = 0; j < V; ++j) zero.v[j] = from_f32<T>(0.0f);
#pragma unroll
    for (int k = 0; k < NV; ++k) nx[k] = ng[k] = zero;  // where there is no pack they stay so, and nothing is added
    float2 ns;
    const auto load = [&](int64_t first) {
        const int64_t r = first + slot < rows ? first + slot : rows - 1;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (skip[k] < V) {
                nx[k] = load_pack<T, V>(x + r * stride + start[k], stream);
                ng[k] = load_pack<T, V>(gy + r * D + start[k], stream);
            }
        ns = reinterpret_cast<const float2*>(stats)[r];
    };
    int64_t r0 = (int64_t)blockIdx.x * kRows;
    if (r0 < rows) load(r0);
    for (; r0 < rows; r0 += step) {
        float h[NV][V], d[NV][V];
        const float mean = ns.x, rstd = ns.y;
        const int64_t r = r0 + slot;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[k][j] = (to_f32(nx[k].v[j]) - mean) * rstd;
                d[k][j] = to_f32(ng[k].v[j]);
            }
            if (drop_.threshold) drop<V>(d[k], (uint64_t)r * D + start[k], whole, drop_, key);
        }
        if (r0 + step < rows) load(r0 + step);
        float s0 = 0.0f, s1 = 0.0f;
        if (r < rows) {  // a slot behind the last row computes it again, and does not count it
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    aw[k][j] = fmaf(d[k][j], h[k][j], aw[k][j]);
                    ab[k][j] += d[k][j];
                }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) d[k][j] *= wv[k][j];
        if (!ragged) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s0 += d[k][j];
                    s1 = fmaf(d[k][j], h[k][j], s1);
                }
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float g = j >= skip[k] ? d[k][j] : 0.0f;
                    s0 += g;
                    s1 = fmaf(g, h[k][j], s1);
                }
        }
        if (!gx) continue;  // uniform
        row_sum(s0, s1);
        s0 *= inv;
        s1 *= inv;
        if (r < rows) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (skip[k] < V) {
                    Pack<T, V> q;
#pragma unroll
                    for (int j = 0; j < V; ++j) q.v[j] = from_f32<T>(rstd * (d[k][j] - fmaf(h[k][j], s1, s0)));
                    store_pack<T, V>(gx + r * D + start[k], q);
                }
        }
    }
    if (!part) return;
    float* out = part + (size_t)blockIdx.x * 2 * D;
    // the rows of a wave by lane exchange, then the workgroup's waves (TPR <= 64) or rows (128) one after the other
    if constexpr (TPR < kWave) {
#pragma unroll
        for (int m = TPR; m < kWave; m <<= 1)
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    aw[k][j] += __shfl_xor(aw[k][j], m);
                    ab[k][j] += __shfl_xor(ab[k][j], m);
                }
    }
    constexpr int kTurn = TPR < kWave ? kWave : TPR, kTurns = kRows > 1 ? kBlock / kTurn : 1;
    const int turn = threadIdx.x / kTurn, at = threadIdx.x % kTurn;
    if constexpr (kTurns > 1) {
        for (int q = kTurns - 1; q > 0; --q) {
            if (turn == q && at < TPR) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        float* p = sums + ((k * V + j) * TPR + at) * 2;
                        p[0] = q < kTurns - 1 ? p[0] + aw[k][j] : aw[k][j];
                        p[1] = q < kTurns - 1 ? p[1] + ab[k][j] : ab[k][j];
                    }
            }
            __syncthreads();
        }
    }
    if (turn == 0 && at < TPR) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j >= skip[k]) {
                    const float* p = sums + (kTurns > 1 ? ((k * V + j) * TPR + at) * 2 : 0);
                    out[start[k] + j] = kTurns > 1 ? p[0] + aw[k][j] : aw[k][j];
                    out[D + start[k] + j] = kTurns > 1 ? p[1] + ab[k][j] : ab[k][j];
                }
    }
}

// gw, gb = the column sums of part [P][2][D].  A workgroup owns 16 of the 2 D columns; each quarter of its 16 waves adds
// every 64th partial row.
constexpr int kReduceWaves = 16, kReduceCols = 16;
template <class W>
__global__ __launch_bounds__(kWave* kReduceWaves) void k_norm_reduce(const float* __restrict__ part, int P, int D,
                                                                     W* __restrict__ gw, W* __restrict__ gb) {
    __shared__ float red[kReduceWaves][kReduceCols];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t col = (int64_t)blockIdx.x * kReduceCols + (lane & (kReduceCols - 1));
    float s = 0.0f;
    if (col < 2 * (int64_t)D) {
#pragma unroll 8
        for (int p = wave * 4 + lane / kReduceCols; p < P; p += 4 * kReduceWaves) s += part[(size_t)p * 2 * D + col];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < kReduceCols) red[wave][lane] = s;
    __syncthreads();
    if (threadIdx.x < kReduceCols && col < 2 * (int64_t)D) {
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < kReduceWaves; ++k) s += red[k][lane];
        if (col < D) {
            if (gw) gw[col] = from_f32<W>(s);
        } else if (gb) {
            gb[col - D] = from_f32<W>(s);
        }
    }
}

// ---- wide rows ------------------------------------------------------------------------------------------
constexpr int kLong = 1024;

// Rows that fit no workgroup's registers: read three times, the second and third time from the caches.
template <class T, class W>
__global__ __launch_bounds__(kLong) void k_norm_fwd_long(const T* __restrict__ x, int64_t stride,
                                                         const W* __restrict__ w, const W* __restrict__ b,
                                                         int64_t rows, int D, float eps, Dropout drop_,
                                                         T* __restrict__ y, float* __restrict__ stats) {
    constexpr int V = kVec<T>;
    __shared__ float red[2][2][kRedWaves];
    RowSum<kLong> row_sum{red, 0};
    const PhiloxKey key = philox_key(drop_);
    const float inv = 1.0f / (float)D;
    const bool whole = D % 8 == 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * stride;
        float s = 0.0f;
#pragma unroll 2
        for (int col = threadIdx.x * V; col < D; col += kLong * V) {
            const int start = col + V <= D ? col : D - V;
            const Pack<T, V> q = load_pack<T, V>(xr + start);
#pragma unroll
            for (int j = 0; j < V; ++j) s += start + j >= col ? to_f32(q.v[j]) : 0.0f;
        }
        row_sum(s);
        const float mean = s * inv;
        s = 0.0f;
#pragma unroll 2
        for (int col = threadIdx.x * V; col < D; col += kLong * V) {
            const int start = col + V <= D ? col : D - V;
            const Pack<T, V> q = load_pack<T, V>(xr + start);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float c = start + j >= col ? to_f32(q.v[j]) - mean : 0.0f;
                s = fmaf(c, c, s);
            }
        }
        row_sum(s);
        const float rstd = 1.0f / sqrtf(fmaf(s, inv, eps));
#pragma unroll 2
        for (int col = threadIdx.x * V; col < D; col += kLong * V) {
            const int start = col + V <= D ? col : D - V;
            Pack<T, V> q = load_pack<T, V>(xr + start);
            Pack<W, V> pw, pb;
            if (w) pw = load_pack<W, V>(w + start);
            if (b) pb = load_pack<W, V>(b + start);
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j)
                v[j] = fmaf((to_f32(q.v[j]) - mean) * rstd, w ? to_f32(pw.v[j]) : 1.0f, b ? to_f32(pb.v[j]) : 0.0f);
            if (drop_.threshold) drop<V>(v, (uint64_t)r * D + start, whole, drop_, key);
#pragma unroll
            for (int j = 0; j < V; ++j) q.v[j] = from_f32<T>(v[j]);
            store_pack<T, V>(y + r * D + start, q);
        }
        if (stats && threadIdx.x == 0) {
            stats[2 * r] = mean;
            stats[2 * r + 1] = rstd;
        }
    }
}

// Backward of rows of more than 4096 elements, in two kernels.  Holding such a row's x, gy, weights and sums in one
// workgroup's registers leaves one or two waves per SIMD and a partial row of 2 D sums from each workgroup (fp16
// 2053 x 8205: 47 us); reading x and gy a second time, the better part of it from the last-level cache, costs less.
// sums[r] = (mean g, mean (g h)) of row r.
template <class T, class W>
__global__ __launch_bounds__(kBlock) void k_norm_bwd_sums(const T* __restrict__ gy, const T* __restrict__ x,
                                                          int64_t stride, const W* __restrict__ w,
                                                          const float* __restrict__ stats, int64_t rows, int D,
                                                          Dropout drop_, float2* __restrict__ sums) {
    constexpr int V = kVec<T>;
    __shared__ float red[2][2][kRedWaves];
    RowSum<kBlock> row_sum{red, 0};
    const PhiloxKey key = philox_key(drop_);
    const float inv = 1.0f / (float)D;
    const bool whole = D % 8 == 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mean = stats[2 * r], rstd = stats[2 * r + 1];
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll 4
        for (int col = threadIdx.x * V; col < D; col += kBlock * V) {
            const int start = col + V <= D ? col : D - V;
            const Pack<T, V> qx = load_pack<T, V>(x + r * stride + start), qg = load_pack<T, V>(gy + r * D + start);
            Pack<W, V> pw;
            if (w) pw = load_pack<W, V>(w + start);
            float d[V];
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = to_f32(qg.v[j]);
            if (drop_.threshold) drop<V>(d, (uint64_t)r * D + start, whole, drop_, key);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float g = start + j >= col ? d[j] * (w ? to_f32(pw.v[j]) : 1.0f) : 0.0f;
                s0 += g;
                s1 = fmaf(g, (to_f32(qx.v[j]) - mean) * rstd, s1);
            }
        }
        row_sum(s0, s1);
        if (threadIdx.x == 0) sums[r] = make_float2(s0 * inv, s1 * inv);
    }
}

// Workgroup (slice, group) owns 64 packs of columns, a pack per lane, and walks with four waves over every
// gridDim.y-th group of four rows, kRowsAhead of a wave's rows in flight.  part [gridDim.y][2][D].
constexpr int kRowsAhead = 4;
template <class T, class W>
__global__ __launch_bounds__(kBlock) void k_norm_bwd_cols(const T* __restrict__ gy, const T* __restrict__ x,
                                                          int64_t stride, const W* __restrict__ w,
                                                          const float* __restrict__ stats,
                                                          const float2* __restrict__ sums, int64_t rows, int D,
                                                          Dropout drop_, T* __restrict__ gx, float* __restrict__ part) {
    constexpr int V = kVec<T>, kWaves = kBlock / kWave;
    __shared__ alignas(16) float red[kWaves - 1][2][kWave][V];
    const PhiloxKey key = philox_key(drop_);
    const bool whole = D % 8 == 0;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x & (kWave - 1);
    const int col = ((int)blockIdx.x * kWave + lane) * V;
    const bool mine = col < D;
    const int start = !mine ? 0 : col + V <= D ? col : D - V;
    float wv[V], aw[V], ab[V];
    Pack<W, V> pw;
    if (w) pw = load_pack<W, V>(w + start);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        wv[j] = w ? to_f32(pw.v[j]) : 1.0f;
        aw[j] = ab[j] = 0.0f;
    }
    const int64_t step = (int64_t)gridDim.y * kWaves;
    for (int64_t r0 = (int64_t)blockIdx.y * kWaves + wave; r0 < rows; r0 += step * kRowsAhead) {
        Pack<T, V> qx[kRowsAhead], qg[kRowsAhead];
        float2 st[kRowsAhead], sm[kRowsAhead];
#pragma unroll
        for (int u = 0; u < kRowsAhead; ++u) {
            const int64_t r = r0 + u * step < rows ? r0 + u * step : r0;
            qx[u] = load_pack<T, V>(x + r * stride + start);
            qg[u] = load_pack<T, V>(gy + r * D + start);
            st[u] = reinterpret_cast<const float2*>(stats)[r];
            if (gx) sm[u] = sums[r];
        }
#pragma unroll
        for (int u = 0; u < kRowsAhead; ++u) {
            const int64_t r = r0 + u * step;
            if (r >= rows) break;  // uniform
            float d[V], h[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                d[j] = to_f32(qg[u].v[j]);
                h[j] = (to_f32(qx[u].v[j]) - st[u].x) * st[u].y;
            }
            if (drop_.threshold) drop<V>(d, (uint64_t)r * D + start, whole, drop_, key);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                aw[j] = fmaf(d[j], h[j], aw[j]);
                ab[j] += d[j];
            }
            if (gx && mine) {
                Pack<T, V> q;
#pragma unroll
                for (int j = 0; j < V; ++j) q.v[j] = from_f32<T>(st[u].y * (d[j] * wv[j] - fmaf(h[j], sm[u].y, sm[u].x)));
                store_pack<T, V>(gx + r * D + start, q);
            }
        }
    }
    if (!part) return;
    if (wave > 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            red[wave - 1][0][lane][j] = aw[j];
            red[wave - 1][1][lane][j] = ab[j];
        }
    }
    __syncthreads();
    if (wave == 0 && mine) {
        float* out = part + (size_t)blockIdx.y * 2 * D + start;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float a = aw[j], c = ab[j];
#pragma unroll
            for (int k = 0; k < kWaves - 1; ++k) {
                a += red[k][0][lane][j];
                c += red[k][1][lane][j];
            }
            if (start + j >= col) {
                out[j] = a;
                out[D + j] = c;
            }
        }
    }
}
