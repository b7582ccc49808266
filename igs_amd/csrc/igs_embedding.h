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

// ---- dense gradient: out[v,:] = scale * sum over i with tokens[i] = v of grad[i,:] ----------------------
//
// The tokens are sorted (stable, least significant digit first, positions carried along), so that equal
// tokens are neighbours and every row of the gradient is read once, by whoever holds its place in the
// sorted order; work is cut by places, not by rows of the table, so a token that fills the batch costs what
// any other does.  Tokens that reach no gradient (out of range, padding) get the key `vocab`, behind all others.
//   k_sort_one                  up to kSortOne tokens: one workgroup, keys in registers
//   k_sort_count, k_sort_place  more: per digit, counts of every tile, then each tile to its place
//   k_embed_sum                 runs of equal keys added up (and, by other workgroups of the launch, zeros
//                               into the rows that no key names); runs that cross a workgroup's border
//                               leave partial rows
//   k_embed_join                adds those
// Every sum has a fixed order; the atomics are integer counters in LDS.

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortOne = 4 * kSortThreads;
constexpr int kSortBits = 9;     // of a digit, at most
constexpr int kSortTiles = 128;  // at most: a tile's workgroup adds up the counts of all tiles itself
constexpr int kSumThreads = 512;
constexpr int kUnroll = 8;       // rows in flight per thread; keys come in groups of that many

template <class I>
__device__ __forceinline__ int token_key(I t, int64_t vocab, int64_t padding) {
    return token_ok(t, vocab) && (int64_t)t != padding ? (int)t : (int)vocab;
}

// Lanes of the wave whose digit is this lane's (`active`: the lanes that hold a key).
__device__ __forceinline__ uint64_t match_digit(int digit, int bits, bool valid) {
    uint64_t m = __ballot(valid);
    for (int b = 0; b < bits; ++b) {
        const bool set = (digit >> b) & 1;
        const uint64_t v = __ballot(set);
        m &= set ? v : ~v;
    }
    return m;
}
__device__ __forceinline__ int lanes_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// count [kSortWaves][bins]: from the keys of each wave per digit to the first place of each wave's keys;
// first[d] (in LDS): the first place of digit d.  Called by all threads.
__device__ __forceinline__ void wave_places(int* count, const int* first, int bins) {
    for (int d = threadIdx.x; d < bins; d += kSortThreads) {
        int run = first[d];
        for (int w = 0; w < kSortWaves; ++w) {
            const int c = count[w * bins + d];
            count[w * bins + d] = run;
            run += c;
        }
    }
    __syncthreads();
}
// first[d] = sum of total[d'] over d' < d, over up to 512 digits; `part` 8 ints of LDS.
__device__ __forceinline__ void digit_places(const int* total, int* first, int* part, int bins) {
    const int d = threadIdx.x, lane = d & (kWave - 1);
    int v = d < bins ? total[d] : 0, own = v;
    for (int k = 1; k < kWave; k <<= 1) {
        const int t = __shfl_up(v, k);
        if (lane >= k) v += t;
    }
    if (lane == kWave - 1 && d < 512) part[d / kWave] = v;
    __syncthreads();
    if (d < bins) {
        int before = 0;
        for (int w = 0; w < d / kWave; ++w) before += part[w];
        first[d] = before + v - own;
    }
    __syncthreads();
}
// Place of this lane's key: `place` [bins] is its wave's row of counters, moved on behind the wave's keys.
__device__ __forceinline__ int take_place(volatile int* place, int digit, int bits, bool valid) {
    const uint64_t same = match_digit(digit, bits, valid);
    const int rank = lanes_below(same);
    int at = 0;
    if (valid) {
        at = place[digit];
        if (rank == __popcll(same) - 1) place[digit] = at + rank + 1;  // the last of the equal ones; LDS keeps a wave's order
    }
    __builtin_amdgcn_wave_barrier();
    return at + rank;
}

// keys, pos [n rounded up to kUnroll, plus kUnroll]: sorted keys and their places in `tokens`; the places behind n hold
// the key `vocab` and position 0.
template <class I>
__global__ __launch_bounds__(kSortThreads) void k_sort_one(const I* __restrict__ tokens, int n, int64_t vocab,
                                                           int64_t padding, int passes, int bits, int* __restrict__ keys,
                                                           int* __restrict__ pos) {
    constexpr int kPer = kSortOne / kSortThreads, kBins = 1 << 8;
    __shared__ int count[kSortWaves * kBins], total[kBins], first[kBins], part[8], sk[kSortOne], sp[kSortOne];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), bins = 1 << bits;
    int key[kPer], at[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        at[j] = (wave * kPer + j) * kWave + lane;
        key[j] = at[j] < n ? token_key(tokens[at[j]], vocab, padding) : 0;
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * bits;
        for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) count[i] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if ((wave * kPer + j) * kWave + lane < n) atomicAdd(&count[wave * bins + ((key[j] >> shift) & (bins - 1))], 1);
        __syncthreads();
        for (int d = threadIdx.x; d < bins; d += kSortThreads) {
            int t = 0;
            for (int w = 0; w < kSortWaves; ++w) t += count[w * bins + d];
            total[d] = t;
        }
        __syncthreads();
        digit_places(total, first, part, bins);
        wave_places(count, first, bins);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const bool valid = (wave * kPer + j) * kWave + lane < n;
            const int to = take_place(count + wave * bins, (key[j] >> shift) & (bins - 1), bits, valid);
            if (valid) {
                sk[to] = key[j];
                sp[to] = at[j];
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = (wave * kPer + j) * kWave + lane;
            if (i < n) {
                key[j] = sk[i];
                at[j] = sp[i];
            }
        }
        // (the barriers of the next pass stand between these reads and its writes)
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = (wave * kPer + j) * kWave + lane;
        if (i < n) {
            keys[i] = key[j];
            pos[i] = at[j];
        }
    }
    const int end = (n + kUnroll - 1) / kUnroll * kUnroll + kUnroll;
    if (n + (int)threadIdx.x < end) {
        keys[n + threadIdx.x] = (int)vocab;
        pos[n + threadIdx.x] = 0;
    }
}

// Where a pass of the sort finds its keys: in the tokens (first pass) or where the pass before left them.
template <class I>
struct SortSource {
    const I* tokens;  // NULL after the first pass
    const int *keys, *pos;
    int64_t vocab, padding;
    __device__ __forceinline__ int key(int64_t i) const { return tokens ? token_key(tokens[i], vocab, padding) : keys[i]; }
    __device__ __forceinline__ int position(int64_t i) const { return tokens ? (int)i : pos[i]; }
};

// counts [tiles][bins] of the digits of each tile of `tile` keys.
template <class I>
__global__ __launch_bounds__(kSortThreads) void k_sort_count(SortSource<I> src, int64_t n, int tile, int shift, int bits,
                                                             int* __restrict__ counts) {
    __shared__ int count[1 << kSortBits];
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += kSortThreads) count[d] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * tile, i1 = i0 + tile < n ? i0 + tile : n;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kSortThreads) atomicAdd(&count[(src.key(i) >> shift) & (bins - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) counts[(size_t)blockIdx.x * bins + d] = count[d];
}

// Every key of a tile to its place: behind the smaller digits of all tiles, the equal digits of earlier tiles and those
// of the same tile before it.  A wave owns a contiguous sixteenth of the tile.
template <class I>
__global__ __launch_bounds__(kSortThreads) void k_sort_place(SortSource<I> src, int64_t n, int tile, int shift, int bits,
                                                             const int* __restrict__ counts, int* __restrict__ keys,
                                                             int* __restrict__ pos) {
    __shared__ int count[kSortWaves << kSortBits], total[1 << kSortBits], first[1 << kSortBits], part[8];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), bins = 1 << bits;
    const int64_t i0 = (int64_t)blockIdx.x * tile + (int64_t)wave * (tile / kSortWaves);
    const int64_t end = i0 + tile / kSortWaves, i1 = end < n ? end : n;
    for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) count[i] = 0;
    int before = 0, all = 0;
    if ((int)threadIdx.x < bins) {
#pragma unroll 8
        for (int t = 0; t < (int)gridDim.x; ++t) {
            const int c = counts[(size_t)t * bins + threadIdx.x];
            all += c;
            before += t < (int)blockIdx.x ? c : 0;
        }
        total[threadIdx.x] = all;
    }
    __syncthreads();
    for (int64_t i = i0 + lane; i < i1; i += kWave) atomicAdd(&count[wave * bins + ((src.key(i) >> shift) & (bins - 1))], 1);
    digit_places(total, first, part, bins);
    if ((int)threadIdx.x < bins) first[threadIdx.x] += before;
    __syncthreads();
    wave_places(count, first, bins);
    for (int64_t i = i0; i < i1; i += kWave) {  // wave-uniform
        const bool valid = i + lane < i1;
        const int key = valid ? src.key(i + lane) : 0;
        const int to = take_place(count + wave * bins, (key >> shift) & (bins - 1), bits, valid);
        if (valid) {
            keys[to] = key;
            pos[to] = src.position(i + lane);
        }
    }
    if (blockIdx.x == 0) {
        const int64_t last = (n + kUnroll - 1) / kUnroll * kUnroll + kUnroll;
        if (n + threadIdx.x < last) {
            keys[n + threadIdx.x] = (int)src.vocab;
            pos[n + threadIdx.x] = 0;
        }
    }
}

// First of n sorted keys that is not below v; by a whole wave, 64 probes at a time.
__device__ __forceinline__ int64_t first_not_below(const int* __restrict__ keys, int64_t n, int64_t v) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t step = (hi - lo + kWave - 1) / kWave;
        const int64_t p = lo + (int64_t)(threadIdx.x & (kWave - 1)) * step;
        const int c = __popcll(__ballot(p < hi && (int64_t)keys[p] < v));
        if (c == 0) break;
        const int64_t next = lo + (int64_t)c * step;
        lo += (int64_t)(c - 1) * step + 1;
        hi = next < hi ? next : hi;
    }
    return lo;
}

// How the sorted places are shared out.  A unit of `lanes` threads owns `len` consecutive places and a slice of
// `lanes` packs of the row; a workgroup's units are neighbours (span = units * len places).
struct SumShape {
    int lanes, slices, len;
    int groups;     // workgroups per slice
    int zero_rows;  // rows of the table per zeroing workgroup
    int packs;      // per row
};

template <class T, int V>
__device__ __forceinline__ void write_row(T* __restrict__ out, int64_t row, int D, int start, const float (&acc)[V], float scale) {
    Pack<T, V> q;
#pragma unroll
    for (int j = 0; j < V; ++j) q.v[j] = from_f32<T>(acc[j] * scale);
    store_pack<T, V>(out + row * D + start, q);
}

// partial [groups][2][D]: a workgroup's share of the run that came into it, and of the run that leaves it.
template <class T, int V>
__global__ __launch_bounds__(kSumThreads) void k_embed_sum(const T* __restrict__ grad, const int* __restrict__ keys,
                                                           const int* __restrict__ pos, int64_t n, int64_t vocab, int D,
                                                           float scale, SumShape s, float* __restrict__ partial,
                                                           T* __restrict__ out) {
    __shared__ alignas(16) float heads[kSumThreads * V], tails[kSumThreads * V];
    __shared__ int through[kSumThreads];
    const int work = s.groups * s.slices;
    if ((int)blockIdx.x >= work) {
        // ---- zeros into the rows v0 .. v0 + rows - 1 that no key names
        int* absent = through;
        int64_t* range = reinterpret_cast<int64_t*>(heads);
        const int64_t v0 = (int64_t)(blockIdx.x - work) * s.zero_rows;
        const int rows = (int)(v0 + s.zero_rows < vocab ? s.zero_rows : vocab - v0);
        if (threadIdx.x < 2 * kWave) {
            const int64_t at = first_not_below(keys, n, v0 + (threadIdx.x < kWave ? 0 : rows));
            if ((threadIdx.x & (kWave - 1)) == 0) range[threadIdx.x / kWave] = at;
        }
        __syncthreads();
        if ((int)threadIdx.x < rows) {
            int64_t lo = range[0], hi = range[1];
            const int end = (int)(hi - lo), v = (int)(v0 + threadIdx.x);
            const int64_t last = hi;
            while (lo < hi) {
                const int64_t mid = lo + (hi - lo) / 2;
                if (keys[mid] < v) lo = mid + 1;
                else hi = mid;
            }
            absent[threadIdx.x] = end == 0 || lo == last || keys[lo] != v;
        }
        __syncthreads();
        Pack<T, V> zero;
#pragma unroll
        for (int j = 0; j < V; ++j) zero.v[j] = from_f32<T>(0.0f);
        const unsigned packs = (unsigned)s.packs;
        for (unsigned p = threadIdx.x; p < (unsigned)rows * packs; p += kSumThreads) {
            const unsigned r = p / packs;
            if (!absent[r]) continue;
            const int col = (int)(p - r * packs) * V;
            store_pack<T, V>(out + (v0 + r) * D + (col + V <= D ? col : D - V), zero);
        }
        return;
    }
    const int lane = threadIdx.x & (s.lanes - 1), unit = threadIdx.x / s.lanes, units = kSumThreads / s.lanes;
    const int group = (int)blockIdx.x / s.slices, slice = (int)blockIdx.x - group * s.slices;
    const int col = (slice * s.lanes + lane) * V;
    const bool mine = col < D;
    const int start = !mine ? 0 : col + V <= D ? col : D - V;
    const int64_t i0 = ((int64_t)group * units + unit) * s.len, i1 = i0 + s.len < n ? i0 + s.len : n;
    float acc[V];
    int key = (int)vocab;
    bool came = false, goes_on = false, open = false;
    if (i0 < i1) {
        key = keys[i0];
        came = i0 > 0 && keys[i0 - 1] == key;  // the run began before this unit's places
        goes_on = i1 < n && keys[i1] == keys[i1 - 1];
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = 0.0f;
        bool head = came;
        for (int64_t i = i0; i < i1; i += kUnroll) {
            int k[kUnroll];
            Pack<T, V> g[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                k[u] = i + u < i1 ? keys[i + u] : (int)vocab;
                if (mine && k[u] != (int)vocab) g[u] = load_pack<T, V>(grad + (int64_t)pos[i + u] * D + start);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (i + u < i1 && k[u] != key) {  // a run ends
                    if (head) {
#pragma unroll
                        for (int j = 0; j < V; ++j) heads[threadIdx.x * V + j] = acc[j];
                        head = false;
                    } else if (mine) {
                        write_row<T, V>(out, key, D, start, acc, scale);
                    }
                    key = k[u];
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
                }
                if (mine && k[u] != (int)vocab)
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[j] += to_f32(g[u].v[j]);
            }
        }
        // the last run
        if (head) {
#pragma unroll
            for (int j = 0; j < V; ++j) heads[threadIdx.x * V + j] = acc[j];
        } else if (goes_on) {
            open = true;
#pragma unroll
            for (int j = 0; j < V; ++j) tails[threadIdx.x * V + j] = acc[j];
        } else if (mine && key != (int)vocab) {
            write_row<T, V>(out, key, D, start, acc, scale);
        }
        if (lane == 0) through[unit] = head && goes_on;
    }
    __syncthreads();
    if (key == (int)vocab && !came) return;
    // runs that cross units: whoever they begin in adds them up
    if (unit == 0 && came && mine) {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = heads[threadIdx.x * V + j];
        for (int u = 0; u + 1 < units && through[u]; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += heads[((u + 1) * s.lanes + lane) * V + j];
#pragma unroll
        for (int j = 0; j < V; ++j) partial[(size_t)group * 2 * D + start + j] = acc[j];
    }
    if (open && mine && key != (int)vocab) {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = tails[threadIdx.x * V + j];
        int u = unit;
        bool on = true;
        while (on && u + 1 < units) {
            ++u;
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += heads[(u * s.lanes + lane) * V + j];
            on = through[u];
        }
        if (!on) write_row<T, V>(out, key, D, start, acc, scale);
        else
#pragma unroll
            for (int j = 0; j < V; ++j) partial[((size_t)group * 2 + 1) * D + start + j] = acc[j];
    }
}

// Runs that cross workgroups of k_embed_sum: workgroup (group, slice) adds up the run that leaves that group, if it
// began there.  span: places per group.
template <class T, int V>
__global__ __launch_bounds__(kSumThreads) void k_embed_join(const int* __restrict__ keys, int64_t n, int64_t vocab, int D,
                                                            float scale, SumShape s, int64_t span,
                                                            const float* __restrict__ partial, T* __restrict__ out) {
    __shared__ float sums[kSumThreads * V];
    const int group = (int)blockIdx.x / s.slices, slice = (int)blockIdx.x - group * s.slices;
    const int64_t i0 = (int64_t)group * span, i1 = i0 + span;
    if (i1 >= n) return;
    const int key = keys[i1 - 1];
    if (key == (int)vocab || keys[i1] != key) return;
    if (i0 > 0 && keys[i0] == key && keys[i0 - 1] == key) return;  // began earlier
    const int lane = threadIdx.x & (s.lanes - 1), unit = threadIdx.x / s.lanes, units = kSumThreads / s.lanes;
    const int col = (slice * s.lanes + lane) * V;
    const bool mine = col < D;
    const int start = !mine ? 0 : col + V <= D ? col : D - V;
    // following groups that the run comes into
    int more = 0;
    for (;;) {
        const int64_t g = (int64_t)group + 1 + more + (threadIdx.x & (kWave - 1));
        const int c = __popcll(__ballot(g * span < n && keys[g * span < n ? g * span : 0] == key));
        more += c;
        if (c < kWave) break;
    }
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    if (mine)
#pragma unroll 4
        for (int g = unit; g <= more; g += units) {
            const float* p = partial + ((size_t)(group + g) * 2 + (g == 0 ? 1 : 0)) * D + start;
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += p[j];
        }
#pragma unroll
    for (int j = 0; j < V; ++j) sums[threadIdx.x * V + j] = acc[j];
    __syncthreads();
    if (unit == 0 && mine) {
        for (int u = 1; u < units && u <= more; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += sums[(u * s.lanes + lane) * V + j];
        write_row<T, V>(out, key, D, start, acc, scale);
    }
}
