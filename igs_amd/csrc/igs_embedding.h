// igs_embedding.h -- embedding lookup with scaling and its dense gradient.  Included by
// igs_feature.hip inside its anonymous namespace.
#pragma once

template <class I>
__device__ __forceinline__ bool token_ok(I t, int64_t vocab) {
    return (int64_t)t >= 0 && (int64_t)t < vocab;
}

// out[i,:] = scale * weight[tokens[i],:].  `lanes` threads (a power of two, at most a workgroup) share a
// token and walk its row in packs of V elements; the last pack of a row of another length is moved back
// to end with the row.  Rows of fewer elements than a pack go with V = 1.  A thread has the packs of U
// tokens in flight: a single gather per thread leaves the memory idle between id, row and store.
template <class T, class I, int V, int U, bool kStream>
__global__ __launch_bounds__(kBlock) void k_embed_fwd(const T* __restrict__ weight, int64_t stride, int64_t vocab,
                                                      int D, const I* __restrict__ tokens, int64_t count,
                                                      float scale, int lanes, T* __restrict__ out) {
    const int per = kBlock / lanes, slot = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
    for (int64_t i = (int64_t)blockIdx.x * (per * U) + slot; i < count; i += (int64_t)gridDim.x * (per * U)) {
        const T* src[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = i + u * per;
            const I t = at < count ? tokens[at] : (I)0;
            ok[u] = token_ok(t, vocab);
            src[u] = weight + (ok[u] ? (int64_t)t : 0) * stride;
        }
        for (int d = lane * V; d < D; d += lanes * V) {
            const int col = d + V <= D ? d : D - V;
            Pack<T, V> q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = load_pack<T, V>(src[u] + col);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = i + u * per;
                if (at >= count) break;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    q[u].v[j] = ok[u] ? from_f32<T>(to_f32(q[u].v[j]) * scale) : from_f32<T>(__builtin_nanf(""));
                store_pack<kStream, T, V>(out + at * D + col, q[u]);
            }
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
//   k_embed_sum                 runs of equal keys added up; runs that cross a workgroup's border leave
//                               partial rows
//   k_embed_join                adds those
//   k_embed_small               all of it, for few tokens
// us of the whole gradient at the borders, this side / the other (a table of 8192 rows, uniform tokens, device time):
//   kSmall    one launch / three   1024 tokens: fp32 x 64 12.9 / 14.6, fp16 x 333 12.2 / 13.6, fp32 x 1024 13.0 / 16.3;
//                                  513: 10.0 / 12.7, 11.7 / 13.4, 12.6 / 15.4; one token in all 1024 places 25.6 / 16.8
//   kSortOne  one workgroup / tiles   8192 tokens: 24.7 / 25.5, 25.4 / 26.3, 34.6 / 35.7; 4097: 20.1 / 25.2, 20.6 / 25.7,
//                                  25.9 / 30.6; and 8193, in tiles: fp16 x 333 26.1, fp32 x 1024 35.9
// The sort waits on memory and keeps few compute units busy; the other workgroups of its launches fill the
// table's gradient with zeros meanwhile, so that k_embed_sum writes the rows that tokens name and no more.
// Every sum has a fixed order; the atomics are integer counters in LDS.

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortPer = 8;  // keys per thread of the one-workgroup sort, at most
constexpr int kSortOne = kSortPer * kSortThreads;
constexpr int kSortBits = 9;     // of a digit, at most
constexpr int kSortHeld = 4;     // keys per thread that a tile's workgroup keeps in registers
constexpr int kSortTiles = 128;  // at most: a tile's workgroup adds up the counts of all tiles itself
constexpr int kSumThreads = 512;
constexpr int kUnroll = 8;  // rows in a group of loads

template <class I>
__device__ __forceinline__ int token_key(I t, int64_t vocab, int64_t padding) {
    return token_ok(t, vocab) && (int64_t)t != padding ? (int)t : (int)vocab;
}

// Lanes of the wave with this lane's digit, among those that hold a key (`valid`).  Per bit: the lanes where it is set, as
// a scalar, and two three-input operations, m & ~(set ^ mine).
__device__ __forceinline__ uint64_t match_digit(int digit, int bits, bool valid) {
    const uint64_t all = __ballot(valid);
    int lo = (int)(uint32_t)all, hi = (int)(uint32_t)(all >> 32);
#pragma unroll
    for (int b = 0; b < kSortBits; ++b) {
        if (b >= bits) break;  // uniform
        const int mine = (int)((uint32_t)digit << (31 - b)) >> 31;
        const uint64_t set = __ballot(mine != 0);
        lo = __builtin_amdgcn_bitop3_b32(lo, (int)(uint32_t)set, mine, 0x90);
        hi = __builtin_amdgcn_bitop3_b32(hi, (int)(uint32_t)(set >> 32), mine, 0x90);
    }
    return (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo;
}
__device__ __forceinline__ int lanes_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// From count [kSortWaves][bins], the keys of each wave per digit, and before[d], the equal digits of earlier tiles
// (NULL: none), to the first place of each wave's keys.  all[d]: keys of digit d in all tiles (NULL: this workgroup's).
// `part`: 8 ints of LDS.  Up to 512 digits, one per thread.  Called by all threads, with count complete.
__device__ __forceinline__ void wave_places(int* count, const int* before, const int* all, int* part, int bins) {
    const int d = threadIdx.x, lane = d & (kWave - 1);
    int c[kSortWaves], own = 0;
    if (d < bins) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) c[w] = count[w * bins + d];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) own += c[w];
        if (all) own = all[d];
    }
    int v = own;  // inclusive sums over the digits of a wave
    if (d < 512) {
#pragma unroll
        for (int k = 1; k < kWave; k <<= 1) {
            const int t = __shfl_up(v, k);
            if (lane >= k) v += t;
        }
        if (lane == kWave - 1) part[d / kWave] = v;
    }
    __syncthreads();
    if (d < bins) {
        int run = v - own + (before ? before[d] : 0);
        for (int w = 0; w < d / kWave; ++w) run += part[w];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            count[w * bins + d] = run;
            run += c[w];
        }
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

// Zeros into `count` elements by `groups` workgroups of kSortThreads, this one being `group`.
template <class T>
__device__ __forceinline__ void fill_zero(T* __restrict__ out, int64_t count, int group, int groups) {
    constexpr int V = kVec<T>;
    const int64_t packs = count / V;
    Pack<T, V> zero;
#pragma unroll
    for (int j = 0; j < V; ++j) zero.v[j] = from_f32<T>(0.0f);
    for (int64_t p = (int64_t)group * kSortThreads + threadIdx.x; p < packs; p += (int64_t)groups * kSortThreads)
        store_pack<T, V>(out + p * V, zero);
    if (group == 0 && (int64_t)threadIdx.x < count - packs * V) out[packs * V + threadIdx.x] = from_f32<T>(0.0f);
}
template <class T>
__global__ __launch_bounds__(kSortThreads) void k_fill(T* __restrict__ out, int64_t count) {
    fill_zero(out, count, blockIdx.x, gridDim.x);
}

// The sort within one workgroup: up to kPer keys per thread, left sorted in sk and their positions in sp.  `count`:
// kSortWaves << bits ints, `part` 8 ints of LDS.
template <int kPer, class I>
__device__ __forceinline__ void sort_here(const I* __restrict__ tokens, int n, int64_t vocab, int64_t padding, int passes,
                                          int bits, int* count, int* part, int* sk, int* sp) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), bins = 1 << bits;
    const int per = (n + kSortThreads - 1) / kSortThreads;  // a wave owns 64 per consecutive keys
    int* own = count + wave * bins;
    int key[kPer], at[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = (wave * per + j) * kWave + lane;
        at[j] = j < per && i < n ? i : -1;
        key[j] = at[j] >= 0 ? token_key(tokens[i], vocab, padding) : 0;
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * bits;
        if (p > 0) {
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (at[j] >= 0) {
                    const int i = (wave * per + j) * kWave + lane;
                    key[j] = sk[i];
                    at[j] = sp[i];
                }
        }
        for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) count[i] = 0;
        __syncthreads();
        int off[kPer];  // among the wave's equal digits; the counters end as the wave's counts
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j < per) off[j] = take_place(own, (key[j] >> shift) & (bins - 1), bits, at[j] >= 0);  // uniform
        __syncthreads();
        wave_places(count, nullptr, nullptr, part, bins);
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (at[j] >= 0) {
                const int to = own[(key[j] >> shift) & (bins - 1)] + off[j];
                sk[to] = key[j];
                sp[to] = at[j];
            }
        __syncthreads();
    }
}

// keys, pos [n]: sorted keys and their places in `tokens`.  The workgroups behind the first fill out.
template <class T, class I>
__global__ __launch_bounds__(kSortThreads) void k_sort_one(const I* __restrict__ tokens, int n, int64_t vocab,
                                                           int64_t padding, int passes, int bits, int* __restrict__ keys,
                                                           int* __restrict__ pos, T* __restrict__ out, int64_t out_count) {
    __shared__ int count[kSortWaves << kSortBits], part[8], sk[kSortOne], sp[kSortOne];
    if (blockIdx.x > 0) return fill_zero(out, out_count, blockIdx.x - 1, gridDim.x - 1);
    sort_here<kSortPer>(tokens, n, vocab, padding, passes, bits, count, part, sk, sp);
    for (int i = threadIdx.x; i < n; i += kSortThreads) {
        keys[i] = sk[i];
        pos[i] = sp[i];
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

// counts [tiles][bins] of the digits of each tile of `tile` keys.  The workgroups behind the tiles fill out.
template <class T, class I>
__global__ __launch_bounds__(kSortThreads) void k_sort_count(SortSource<I> src, int64_t n, int tile, int tiles, int shift,
                                                             int bits, int* __restrict__ counts, T* __restrict__ out,
                                                             int64_t out_count) {
    __shared__ int count[1 << kSortBits];
    if ((int)blockIdx.x >= tiles) return fill_zero(out, out_count, blockIdx.x - tiles, gridDim.x - tiles);
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += kSortThreads) count[d] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * tile, i1 = i0 + tile < n ? i0 + tile : n;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kSortThreads) atomicAdd(&count[(src.key(i) >> shift) & (bins - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) counts[(size_t)blockIdx.x * bins + d] = count[d];
}

// Every key of a tile to its place: behind the smaller digits of all tiles, the equal digits of earlier tiles and those
// of the same tile before it.  A wave owns a contiguous sixteenth of the tile.  The two halves of the workgroup add up
// the counts of every other tile.  kHeld: a wave's keys fit kSortHeld registers and are read once, before anything is
// waited for.  The workgroups behind the tiles fill out.
template <class T, class I, bool kHeld>
__global__ __launch_bounds__(kSortThreads) void k_sort_place(SortSource<I> src, int64_t n, int tile, int tiles, int shift,
                                                             int bits, const int* __restrict__ counts,
                                                             int* __restrict__ keys, int* __restrict__ pos,
                                                             T* __restrict__ out, int64_t out_count) {
    __shared__ int count[kSortWaves << kSortBits], all[2 << kSortBits], before[2 << kSortBits], part[8];
    if ((int)blockIdx.x >= tiles) return fill_zero(out, out_count, blockIdx.x - tiles, gridDim.x - tiles);
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), bins = 1 << bits;
    const int64_t i0 = (int64_t)blockIdx.x * tile + (int64_t)wave * (tile / kSortWaves);
    const int64_t end = i0 + tile / kSortWaves, i1 = end < n ? end : n;
    int key[kSortHeld], at[kSortHeld];
    if (kHeld) {
#pragma unroll
        for (int j = 0; j < kSortHeld; ++j) {
            const int64_t i = i0 + j * kWave + lane;
            at[j] = -1;
            if (i < i1) {
                key[j] = src.key(i);
                at[j] = src.position(i);
            } else {
                key[j] = 0;
            }
        }
    }
    for (int i = threadIdx.x; i < kSortWaves * bins; i += kSortThreads) count[i] = 0;
    const int half = threadIdx.x >> kSortBits, d = threadIdx.x & ((1 << kSortBits) - 1);
    int sum = 0, earlier = 0;
    if (d < bins) {
        for (int t0 = half; t0 < tiles; t0 += 32) {
            int c[16];
#pragma unroll
            for (int t = 0; t < 16; ++t) c[t] = t0 + 2 * t < tiles ? counts[(size_t)(t0 + 2 * t) * bins + d] : 0;
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                sum += c[t];
                earlier += t0 + 2 * t < (int)blockIdx.x ? c[t] : 0;
            }
        }
        all[(half << kSortBits) + d] = sum;
        before[(half << kSortBits) + d] = earlier;
    }
    __syncthreads();
    if (half == 0 && d < bins) {
        all[d] += all[(1 << kSortBits) + d];
        before[d] += before[(1 << kSortBits) + d];
    }
    int* own = count + wave * bins;
    int off[kSortHeld];  // among the wave's equal digits; the counters end as the wave's counts
    if (kHeld) {
#pragma unroll
        for (int j = 0; j < kSortHeld; ++j)
            if (i0 + j * kWave < i1) off[j] = take_place(own, (key[j] >> shift) & (bins - 1), bits, at[j] >= 0);
    } else {
        for (int64_t i = i0 + lane; i < i1; i += kWave) atomicAdd(&own[(src.key(i) >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    wave_places(count, before, all, part, bins);
    if (kHeld) {
#pragma unroll
        for (int j = 0; j < kSortHeld; ++j)
            if (at[j] >= 0) {
                const int to = own[(key[j] >> shift) & (bins - 1)] + off[j];
                keys[to] = key[j];
                pos[to] = at[j];
            }
    } else {
        for (int64_t i = i0; i < i1; i += kWave) {  // wave-uniform
            const bool valid = i + lane < i1;
            const int k = valid ? src.key(i + lane) : 0;
            const int to = take_place(own, (k >> shift) & (bins - 1), bits, valid);
            if (valid) {
                keys[to] = k;
                pos[to] = src.position(i + lane);
            }
        }
    }
}

// How the sorted places are shared out.  A unit of `lanes` threads owns `len` consecutive places and a slice of
// `lanes` packs of the row; a workgroup's units are neighbours (span = units * len places).
struct SumShape {
    int lanes, slices, len;
    int groups;   // workgroups per slice
    bool stream;  // the upstream gradient is read past the caches
};

template <class T, int V>
__device__ __forceinline__ void write_row(T* __restrict__ out, int64_t row, int D, int start, const float (&acc)[V], float scale) {
    Pack<T, V> q;
#pragma unroll
    for (int j = 0; j < V; ++j) q.v[j] = from_f32<T>(acc[j] * scale);
    store_pack<T, V>(out + row * D + start, q);
}

// partial [groups][2][D]: a workgroup's share of the run that came into it, and of the run that leaves it.
// kWide: a unit is a whole wave, so its keys and positions are scalars.  Keys and positions of up to `lanes` places are
// read at once, one per lane; the rows of the next kUnroll places are in flight while those of the last are added.
// heads, tails: kThreads * V floats, through: kThreads / 8 ints of LDS.
// kAlone: there is one group, so that no run leaves it.
template <class T, int V, bool kWide, int kThreads, bool kAlone>
__device__ __forceinline__ void sum_places(const T* __restrict__ grad, const int* keys, const int* pos, int64_t n,
                                           int64_t vocab, int D, float scale, const SumShape& s, int group, int slice,
                                           float* heads, float* tails, int* through, float* __restrict__ partial,
                                           T* __restrict__ out) {
    const int lanes = kWide ? kWave : s.lanes;
    const int lane = threadIdx.x & (lanes - 1), unit = threadIdx.x / lanes, units = kThreads / lanes;
    const int col = (slice * lanes + lane) * V;
    const bool mine = col < D;
    const int start = !mine ? 0 : col + V <= D ? col : D - V;
    const int64_t i0 = ((int64_t)group * units + unit) * s.len, i1 = i0 + s.len < n ? i0 + s.len : n;
    const int none = (int)vocab;
    float acc[V];
    int key = none;
    bool came = false, open = false;
    if (i0 < i1) {
        const auto of = [&](int v, int place) {
            return kWide ? __builtin_amdgcn_readlane(v, place) : __shfl(v, (int)(threadIdx.x & (kWave - 1) & ~(lanes - 1)) + place);
        };
        came = i0 > 0 && keys[i0 - 1] == keys[i0];  // the run began before this unit's places
        const bool goes_on = i1 < n && keys[i1] == keys[i1 - 1];
        bool head = came;
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = 0.0f;
        for (int64_t b = i0; b < i1; b += lanes) {
            const int places = (int)(i1 - b < lanes ? i1 - b : lanes);
            int kv = none, pv = 0;
            if (lane < places) {
                kv = keys[b + lane];
                pv = pos[b + lane];
            }
            if (b == i0) key = of(kv, 0);
            const auto load = [&](Pack<T, V> (&g)[kUnroll], int q) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    if (q + u >= places) break;
                    const int k = of(kv, q + u), i = of(pv, q + u);  // all lanes of the unit: one of them holds the values
                    if (k != none && mine) g[u] = load_pack<T, V>(grad + (int64_t)i * D + start, s.stream);
                }
            };
            const auto add = [&](const Pack<T, V> (&g)[kUnroll], int q) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    if (q + u >= places) break;
                    const int k = of(kv, q + u);
                    if (k != key) {  // a run ends
                        if (head) {
#pragma unroll
                            for (int j = 0; j < V; ++j) heads[threadIdx.x * V + j] = acc[j];
                            head = false;
                        } else if (mine) {
                            write_row<T, V>(out, key, D, start, acc, scale);
                        }
                        key = k;
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[j] = 0.0f;
                    }
                    if (k != none && mine)
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[j] += to_f32(g[u].v[j]);
                }
            };
            Pack<T, V> ga[kUnroll], gb[kUnroll];
            load(ga, 0);
            for (int q = 0; q < places; q += 2 * kUnroll) {
                load(gb, q + kUnroll);
                add(ga, q);
                load(ga, q + 2 * kUnroll);
                add(gb, q + kUnroll);
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
        } else if (mine && key != none) {
            write_row<T, V>(out, key, D, start, acc, scale);
        }
        if (lane == 0) through[unit] = head && goes_on;
    }
    __syncthreads();
    // runs that cross units: whoever they begin in adds them up
    if (!kAlone && unit == 0 && came && mine) {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = heads[threadIdx.x * V + j];
        for (int u = 0; u + 1 < units && through[u]; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += heads[((u + 1) * lanes + lane) * V + j];
#pragma unroll
        for (int j = 0; j < V; ++j) partial[(size_t)group * 2 * D + start + j] = acc[j];
    }
    if (open && mine && key != none) {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = tails[threadIdx.x * V + j];
        int u = unit;
        bool on = true;
        while (on && u + 1 < units) {
            ++u;
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += heads[(u * lanes + lane) * V + j];
            on = through[u];
        }
        if (kAlone || !on) write_row<T, V>(out, key, D, start, acc, scale);
        else
#pragma unroll
            for (int j = 0; j < V; ++j) partial[((size_t)group * 2 + 1) * D + start + j] = acc[j];
    }
}

template <class T, int V, bool kWide>
__global__ __launch_bounds__(kSumThreads) void k_embed_sum(const T* __restrict__ grad, const int* __restrict__ keys,
                                                           const int* __restrict__ pos, int64_t n, int64_t vocab, int D,
                                                           float scale, SumShape s, float* __restrict__ partial,
                                                           T* __restrict__ out) {
    __shared__ alignas(16) float heads[kSumThreads * V], tails[kSumThreads * V];
    __shared__ int through[kSumThreads / 8];
    const int group = (int)blockIdx.x / s.slices, slice = (int)blockIdx.x - group * s.slices;
    sum_places<T, V, kWide, kSumThreads, false>(grad, keys, pos, n, vocab, D, scale, s, group, slice, heads, tails, through,
                                         partial, out);
}

// First of n sorted keys behind `at` that differs from the one before `at` (at itself for at = 0, n at most).
__device__ __forceinline__ int run_border(const int* keys, int n, int at) {
    if (at <= 0) return 0;
    if (at >= n) return n;
    const int key = keys[at - 1];
    int lo = at, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (keys[mid] == key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Few tokens (up to kSmall): the whole gradient in one launch and without a workspace, a small step being bound by its
// launches (1024 tokens of 8192 x 1024 in fp32: 13 us, 16 in three launches).  Workgroup (group, slice)
// sorts all tokens for itself and adds up the runs that begin in its group's places; the workgroups behind those
// each look all tokens up for `zero_rows` rows of the table and write zeros into the rows that none names.  A run is not
// shared among workgroups here: one token in all 1024 places takes 26 us (17 in three launches), which bounds kSmall.
constexpr int kSmall = kSortThreads;
template <class T, class I, int V, bool kWide>
__global__ __launch_bounds__(kSortThreads) void k_embed_small(const T* __restrict__ grad, const I* __restrict__ tokens,
                                                              int n, int64_t vocab, int64_t padding, int D, float scale,
                                                              int passes, int bits, SumShape s, int zero_rows,
                                                              T* __restrict__ out) {
    __shared__ alignas(16) float heads[kSortThreads * V], tails[kSortThreads * V];
    __shared__ int count[kSortWaves << kSortBits], through[kSortThreads / 8], part[8], sk[kSmall], sp[kSmall];
    const int work = s.groups * s.slices;
    if ((int)blockIdx.x < work) {
        sort_here<1>(tokens, n, vocab, padding, passes, bits, count, part, sk, sp);
        const int group = (int)blockIdx.x / s.slices, slice = (int)blockIdx.x - group * s.slices;
        const int units = kSortThreads / (kWide ? kWave : s.lanes), span = units * s.len;
        const int i0 = run_border(sk, n, group * span), i1 = run_border(sk, n, (group + 1) * span);
        if (i0 < i1) {
            s.len = ((i1 - i0 + units - 1) / units + kUnroll - 1) / kUnroll * kUnroll;
            sum_places<T, V, kWide, kSortThreads, true>(grad, sk + i0, sp + i0, i1 - i0, vocab, D, scale, s, 0, slice,
                                                        heads, tails, through, nullptr, out);
        }
        return;
    }
    int* named = sk;
    const int64_t v0 = (int64_t)(blockIdx.x - work) * zero_rows;
    const int rows = (int)(v0 + zero_rows < vocab ? zero_rows : vocab - v0);
    for (int r = threadIdx.x; r < rows; r += kSortThreads) named[r] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSortThreads) {
        const int64_t r = (int64_t)token_key(tokens[i], vocab, padding) - v0;
        if (r >= 0 && r < rows) named[r] = 1;
    }
    __syncthreads();
    Pack<T, V> zero;
#pragma unroll
    for (int j = 0; j < V; ++j) zero.v[j] = from_f32<T>(0.0f);
    const unsigned packs = (unsigned)((D + V - 1) / V);
    for (unsigned p = threadIdx.x; p < (unsigned)rows * packs; p += kSortThreads) {
        const unsigned r = p / packs;
        if (named[r]) continue;
        const int col = (int)(p - r * packs) * V;
        store_pack<T, V>(out + (v0 + r) * D + (col + V <= D ? col : D - V), zero);
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
