// Rows of a learned table by integer id, scaled, and the gradient of the table, for gfx950.
//
//   out[n] = scale * table[ids[n]]            d_table[v] = scale * sum over {n : ids[n] = v} of d_out[n]
//
// The forward pass is a gather bound by memory.  The gradient is formed without atomics, so that equal inputs give equal
// bits and a row that most of the batch asks for (one image's code in a whole ray batch, a frequent token) costs no more
// than its bytes: the positions are sorted by id with a stable radix sort (ids that take no gradient -- out of range, or
// the padding row -- sort behind all others as id V), and every row of d_table is then written exactly once, zeros
// included, from the run of sorted positions that its id owns:
//   - each aligned chunk of 64 sorted positions that lies inside one run is summed into a partial row;
//   - runs of at least 128 positions are summed by a workgroup, from their whole chunks' partials and the positions at
//     both ends; shorter ones by a few lanes from d_out itself.
// Sums are held in float, in an order that the ids alone decide, and rounded once.
#include <algorithm>

#include "typed.h"

namespace nerf {

constexpr int EMB_CHUNK = 64;        // sorted positions of a partial row
constexpr int EMB_LONG = 128;        // runs from this length on contain at least one whole chunk
constexpr int EMB_CANDIDATES = 16;   // chunks whose long run, if one starts there, one workgroup sums

constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64, SORT_ITEMS = 8;
constexpr int SORT_TILE = SORT_THREADS * SORT_ITEMS;   // keys that a workgroup ranks at once
constexpr int SORT_BITS = 10, SORT_DIGITS = 1 << SORT_BITS;

// ---- forward ---------------------------------------------------------------------------------------------------
template <class T, int VEC, class ID>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const T* __restrict__ table, int64_t V, int D, const ID* __restrict__ ids, int64_t N,
                                                            float scale, int l_lanes, T* __restrict__ out) {
    const int lanes = 1 << l_lanes, vectors = D / VEC;
    const int64_t step = (int64_t)gridDim.x * (256 >> l_lanes);
    for (int64_t n = (int64_t)blockIdx.x * (256 >> l_lanes) + (threadIdx.x >> l_lanes); n < N; n += step) {
        const int64_t id = (int64_t)ids[n];
        const bool good = id >= 0 && id < V;
        for (int i = (threadIdx.x & (lanes - 1)) + (int)blockIdx.y * lanes; i < vectors; i += lanes * (int)gridDim.y) {
            float v[VEC];
            if (good) {
                load_run<VEC>(table + id * D + (int64_t)i * VEC, v);
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[k] *= scale;
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[k] = __builtin_nanf("");
            }
            store_run<VEC>(out + n * D + (int64_t)i * VEC, v);
        }
    }
}

// ---- stable radix sort of (id, position) -------------------------------------------------------------------------
template <class ID>
__device__ __forceinline__ unsigned sort_key(ID id, int64_t V, int64_t padding) {
    const int64_t i = (int64_t)id;
    return (unsigned)((i >= 0 && i < V && i != padding) ? i : V);
}

// Ranks of a tile's keys by their digit, equal digits in the order of the keys.  Wave w holds the keys
// w * 64 * ITEMS + r * 64 + lane; count[w][digit] is the wave's own, so a round needs no atomics: lanes with the same
// digit find each other by ballots, take their ranks from the old count, and the last of them writes the new one.
// On return rank[r] is the key's place within its wave and digit, and after digit_starts() count[w][d] is where the
// wave's keys of digit d start in the sorted tile.
__device__ __forceinline__ void rank_in_wave(const unsigned (&key)[SORT_ITEMS], const bool (&on)[SORT_ITEMS], int shift, int bits,
                                             volatile unsigned* __restrict__ count, unsigned (&rank)[SORT_ITEMS]) {
    const unsigned mask = (1u << bits) - 1u;
    const unsigned long long below = (1ull << (threadIdx.x & 63)) - 1ull;
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
        const unsigned d = (key[r] >> shift) & mask;
        unsigned long long same = __ballot(on[r]);
        for (int b = 0; b < bits; ++b) {
            const bool bit = (d >> b) & 1u;
            const unsigned long long set = __ballot(bit);
            same &= bit ? set : ~set;
        }
        rank[r] = 0;
        if (on[r]) {
            const unsigned old = count[d];
            rank[r] = old + (unsigned)__popcll(same & below);
            if ((same >> (threadIdx.x & 63)) == 1ull) count[d] = old + (unsigned)__popcll(same);   // the highest of them
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Exclusive sum over the workgroup's 1024 threads.
__device__ __forceinline__ unsigned block_exclusive(unsigned v, unsigned* __restrict__ s_wave) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned inc = v;
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
    }
    if (lane == 63) s_wave[wave] = inc;
    __syncthreads();
    unsigned base = 0;
    for (int w = 0; w < wave; ++w) base += s_wave[w];
    __syncthreads();
    return base + inc - v;
}

// count[w][d] -> where the keys of wave w and digit d start in the sorted tile (thread d does digit d); returns the
// number of keys of the thread's digit and, in `start`, where they begin.
__device__ __forceinline__ unsigned digit_starts(unsigned (*__restrict__ count)[SORT_DIGITS], unsigned* __restrict__ s_wave, unsigned& start) {
    unsigned total = 0;
    for (int w = 0; w < SORT_WAVES; ++w) total += count[w][threadIdx.x];
    start = block_exclusive(total, s_wave);
    unsigned at = start;
    for (int w = 0; w < SORT_WAVES; ++w) {
        const unsigned c = count[w][threadIdx.x];
        count[w][threadIdx.x] = at;
        at += c;
    }
    return total;
}

// Up to SORT_TILE keys: every pass in one workgroup, the pairs changing places through LDS.
template <class ID>
__global__ __launch_bounds__(SORT_THREADS) void sort_small_kernel(const ID* __restrict__ ids, int n, int64_t V, int64_t padding, int passes, int bits,
                                                                  unsigned* __restrict__ keys, unsigned* __restrict__ vals) {
    __shared__ unsigned s_count[SORT_WAVES][SORT_DIGITS];
    __shared__ unsigned s_key[SORT_TILE];
    __shared__ unsigned short s_val[SORT_TILE];
    __shared__ unsigned s_wave[SORT_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int items = (n + SORT_THREADS - 1) / SORT_THREADS;   // rounds in use: the tile is packed to the front of every wave
    unsigned key[SORT_ITEMS], rank[SORT_ITEMS], val[SORT_ITEMS];
    bool on[SORT_ITEMS];
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
        const int i = wave * 64 * items + r * 64 + lane;
        on[r] = r < items && i < n;
        key[r] = on[r] ? sort_key(ids[i], V, padding) : 0u;
        val[r] = (unsigned)i;
    }
    for (int p = 0; p < passes; ++p) {
        for (int i = threadIdx.x; i < SORT_WAVES * SORT_DIGITS; i += SORT_THREADS) (&s_count[0][0])[i] = 0u;
        __syncthreads();
        rank_in_wave(key, on, p * bits, bits, s_count[wave], rank);
        __syncthreads();
        unsigned start;
        digit_starts(s_count, s_wave, start);
        __syncthreads();
        const unsigned mask = (1u << bits) - 1u;
#pragma unroll
        for (int r = 0; r < SORT_ITEMS; ++r) {
            if (on[r]) {
                const unsigned to = s_count[wave][(key[r] >> (p * bits)) & mask] + rank[r];
                s_key[to] = key[r];
                s_val[to] = (unsigned short)val[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_ITEMS; ++r) {
            const int i = wave * 64 * items + r * 64 + lane;
            if (on[r]) {
                key[r] = s_key[i];
                val[r] = s_val[i];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
        const int i = wave * 64 * items + r * 64 + lane;
        if (on[r]) {
            keys[i] = key[r];
            vals[i] = val[r];
        }
    }
}

// More keys: per pass, the digits of every tile are counted, the counts summed over the tiles in front, and the tiles
// ranked and scattered.  table: [tiles][digits], then [digits] totals.
template <class ID, bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(const ID* __restrict__ ids, const unsigned* __restrict__ keys, int64_t n, int64_t V,
                                                                  int64_t padding, int shift, int bits, unsigned* __restrict__ table) {
    __shared__ unsigned s_count[SORT_DIGITS];
    const int digits = 1 << bits;
    for (int i = threadIdx.x; i < digits; i += SORT_THREADS) s_count[i] = 0u;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_TILE;
    for (int r = 0; r < SORT_ITEMS; ++r) {
        const int64_t i = base + r * SORT_THREADS + threadIdx.x;
        if (i < n) {
            const unsigned key = FIRST ? sort_key(ids[i], V, padding) : keys[i];
            atomicAdd(&s_count[(key >> shift) & (digits - 1)], 1u);   // whole numbers: the order does not matter
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < digits; i += SORT_THREADS) table[(int64_t)blockIdx.x * digits + i] = s_count[i];
}

// Exclusive sums along the tiles, 64 digits per workgroup, the tiles cut into one stretch per wave.
__global__ __launch_bounds__(SORT_THREADS) void sort_prefix_kernel(unsigned* __restrict__ table, int tiles, int digits) {
    __shared__ unsigned s_sum[SORT_WAVES][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = blockIdx.x * 64 + lane;
    const int per = (tiles + SORT_WAVES - 1) / SORT_WAVES, begin = min(wave * per, tiles), end = min(begin + per, tiles);
    unsigned sum = 0;
    if (d < digits)
#pragma unroll 8
        for (int t = begin; t < end; ++t) sum += table[(int64_t)t * digits + d];
    s_sum[wave][lane] = sum;
    __syncthreads();
    unsigned at = 0, total = 0;
    for (int w = 0; w < SORT_WAVES; ++w) {
        if (w < wave) at += s_sum[w][lane];
        total += s_sum[w][lane];
    }
    if (d < digits) {
#pragma unroll 8
        for (int t = begin; t < end; ++t) {
            const unsigned c = table[(int64_t)t * digits + d];
            table[(int64_t)t * digits + d] = at;
            at += c;
        }
        if (wave == 0) table[(int64_t)tiles * digits + d] = total;
    }
}

template <class ID, bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void sort_scatter_kernel(const ID* __restrict__ ids, const unsigned* __restrict__ keys, const unsigned* __restrict__ vals,
                                                                    int64_t n, int64_t V, int64_t padding, int shift, int bits, const unsigned* __restrict__ table,
                                                                    int tiles, unsigned* __restrict__ keys_out, unsigned* __restrict__ vals_out) {
    __shared__ unsigned s_count[SORT_WAVES][SORT_DIGITS];
    __shared__ unsigned s_to[SORT_DIGITS];   // what a rank in the sorted tile lacks to its place in the output, per digit
    __shared__ unsigned s_wave[SORT_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << bits;
    const int64_t base = (int64_t)blockIdx.x * SORT_TILE + wave * 64 * SORT_ITEMS;
    unsigned key[SORT_ITEMS], rank[SORT_ITEMS];
    bool on[SORT_ITEMS];
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
        const int64_t i = base + r * 64 + lane;
        on[r] = i < n;
        key[r] = on[r] ? (FIRST ? sort_key(ids[i], V, padding) : keys[i]) : 0u;
    }
    for (int i = threadIdx.x; i < SORT_WAVES * SORT_DIGITS; i += SORT_THREADS) (&s_count[0][0])[i] = 0u;
    __syncthreads();
    rank_in_wave(key, on, shift, bits, s_count[wave], rank);
    __syncthreads();
    unsigned start;
    digit_starts(s_count, s_wave, start);
    // where the digit starts in the whole output, and what the tiles in front hold of it
    const unsigned total = (int)threadIdx.x < digits ? table[(int64_t)tiles * digits + threadIdx.x] : 0u;
    const unsigned first = block_exclusive(total, s_wave);
    if ((int)threadIdx.x < digits) s_to[threadIdx.x] = first + table[(int64_t)blockIdx.x * digits + threadIdx.x] - start;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
        if (on[r]) {
            const unsigned d = (key[r] >> shift) & (unsigned)(digits - 1);
            const unsigned to = s_count[wave][d] + rank[r] + s_to[d];
            const int64_t i = base + r * 64 + lane;
            keys_out[to] = key[r];
            vals_out[to] = FIRST ? (unsigned)i : vals[i];
        }
    }
}

// ---- sums over the runs --------------------------------------------------------------------------------------------
// Lanes of a group on one row: LR lanes of VEC elements, column tile blockIdx.y.
template <int VEC>
struct RowLanes {
    int lanes, group, c;
    bool on;
    int64_t col;
    __device__ __forceinline__ RowLanes(int l_lanes, int D) {
        lanes = 1 << l_lanes;
        group = threadIdx.x >> l_lanes;
        c = threadIdx.x & (lanes - 1);
        const int64_t v = (int64_t)blockIdx.y * lanes + c;
        col = v * VEC;
        on = col < D;
    }
};

template <class T, int VEC>
__device__ __forceinline__ void add_row(const T* __restrict__ d_out, int64_t row, int D, int64_t col, float (&sum)[VEC]) {
    float v[VEC];
    load_run<VEC>(d_out + row * D + col, v);
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum[k] += v[k];
}

template <class T, int VEC>
__global__ __launch_bounds__(256) void embedding_partial_kernel(const T* __restrict__ d_out, int D, const unsigned* __restrict__ keys,
                                                                const unsigned* __restrict__ vals, int64_t chunks, unsigned V, int l_lanes,
                                                                float* __restrict__ part) {
    const int64_t chunk = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (chunk >= chunks) return;
    const unsigned key = keys[chunk * EMB_CHUNK];
    if (key >= V || keys[chunk * EMB_CHUNK + EMB_CHUNK - 1] != key) return;
    const int lane = threadIdx.x & 63;
    const RowLanes<VEC> w(l_lanes, D);
    const int groups = 64 >> l_lanes, group = lane >> l_lanes;
    float sum[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
#pragma unroll 4
    for (int i = group; i < EMB_CHUNK; i += groups) {
        if (w.on) add_row<T, VEC>(d_out, vals[chunk * EMB_CHUNK + i], D, w.col, sum);
    }
    for (int d = w.lanes; d < 64; d <<= 1)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += __shfl_xor(sum[k], d, 64);
    if (group == 0 && w.on) store_run<VEC>(part + chunk * D + w.col, sum);
}

__device__ __forceinline__ int64_t lower_bound(const unsigned* __restrict__ keys, int64_t n, unsigned key) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Blocks [0, long_blocks): the long runs whose first aligned position is one of the block's candidates.
// The others: `rows` rows each.
template <class T, int VEC>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const T* __restrict__ d_out, int D, const unsigned* __restrict__ keys,
                                                             const unsigned* __restrict__ vals, int64_t N, int64_t V, float scale, int l_lanes, int rows,
                                                             int64_t long_blocks, const float* __restrict__ part, T* __restrict__ d_table) {
    __shared__ int64_t s_lo[257];
    __shared__ float s_sum[256 * VEC];
    const RowLanes<VEC> w(l_lanes, D);
    const int groups = 256 >> l_lanes;
    if ((int64_t)blockIdx.x < long_blocks) {
        if (threadIdx.x < EMB_CANDIDATES) {
            const int64_t at = ((int64_t)blockIdx.x * EMB_CANDIDATES + threadIdx.x) * EMB_CHUNK;
            int64_t lo = -1, hi = -1;
            // a run of EMB_LONG that starts in the chunk before `at` or at it holds the whole chunk from `at` on
            if (at + EMB_CHUNK <= N) {
                const unsigned key = keys[at];
                if (key < (unsigned)V && keys[at + EMB_CHUNK - 1] == key && (at == 0 || keys[at - EMB_CHUNK] != key)) {
                    lo = lower_bound(keys, at, key);
                    hi = at + lower_bound(keys + at, N - at, key + 1u);
                    if (hi - lo < EMB_LONG) lo = -1;
                }
            }
            s_lo[threadIdx.x] = lo;
            s_lo[EMB_CANDIDATES + threadIdx.x] = hi;
        }
        __syncthreads();
        for (int q = 0; q < EMB_CANDIDATES; ++q) {
            const int64_t lo = s_lo[q], hi = s_lo[EMB_CANDIDATES + q];
            if (lo < 0) continue;
            const int64_t first = (lo + EMB_CHUNK - 1) / EMB_CHUNK, last = hi / EMB_CHUNK;   // whole chunks
            const int64_t head = first * EMB_CHUNK - lo, tail = hi - last * EMB_CHUNK;
            float sum[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
            if (w.on) {
#pragma unroll 4
                for (int64_t i = w.group; i < head + tail; i += groups)
                    add_row<T, VEC>(d_out, vals[i < head ? lo + i : last * EMB_CHUNK + (i - head)], D, w.col, sum);
#pragma unroll 8
                for (int64_t i = first + w.group; i < last; i += groups) add_row<float, VEC>(part, i, D, w.col, sum);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < VEC; ++k) s_sum[threadIdx.x * VEC + k] = sum[k];
            __syncthreads();
            if (w.group == 0 && w.on) {
                for (int g = 1; g < groups; ++g)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) sum[k] += s_sum[(g * w.lanes + w.c) * VEC + k];
#pragma unroll
                for (int k = 0; k < VEC; ++k) sum[k] *= scale;
                store_run<VEC>(d_table + (int64_t)keys[lo] * D + w.col, sum);
            }
        }
        return;
    }
    const int64_t v0 = ((int64_t)blockIdx.x - long_blocks) * rows;
    for (int i = threadIdx.x; i <= rows; i += 256) s_lo[i] = lower_bound(keys, N, (unsigned)min(v0 + i, V));
    __syncthreads();
    if (!w.on) return;
    for (int q = w.group; q < rows && v0 + q < V; q += groups) {
        const int64_t lo = s_lo[q], hi = s_lo[q + 1];
        if (hi - lo >= EMB_LONG) continue;
        float sum[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
#pragma unroll 4
        for (int64_t i = lo; i < hi; ++i) add_row<T, VEC>(d_out, vals[i], D, w.col, sum);
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] *= scale;
        store_run<VEC>(d_table + (v0 + q) * D + w.col, sum);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
struct EmbWork {                       // the workspace, cut into arrays that start on 256-byte boundaries
    int passes, bits;
    int64_t tiles, chunks;
    size_t keys[2], vals[2], table, part, bytes;
};

static EmbWork embedding_work(int64_t N, int64_t V, int D) {
    EmbWork w;
    int bits = 1;
    while ((1ll << bits) < V + 1) ++bits;
    w.passes = (int)ceil_div(bits, SORT_BITS);
    w.bits = (int)ceil_div(bits, w.passes);
    w.tiles = ceil_div(N, SORT_TILE);
    w.chunks = N / EMB_CHUNK;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    for (int k = 0; k < 2; ++k) {
        const bool used = k == 0 || w.tiles > 1;
        w.keys[k] = take(used ? 4 * N : 0);
        w.vals[k] = take(used ? 4 * N : 0);
    }
    w.table = take(w.tiles > 1 ? 4ull * (w.tiles + 1) << w.bits : 0);
    w.part = take(N >= EMB_LONG ? 4ull * w.chunks * D : 0);
    w.bytes = at;
    return w;
}

static int vector_of(int D, int size) {   // elements per lane: the widest power of two that divides a row, 16 bytes at most
    int v = 16 / size;
    while (D % v) v >>= 1;
    return v;
}

// f(integral_constant VEC) for the vector that a row of D elements of T allows
template <class T, class F>
static int with_vector(int D, F&& f) {
    const int v = vector_of(D, sizeof(T));
    if (v == 1) return f(std::integral_constant<int, 1>{});
    if (v == 2) return f(std::integral_constant<int, 2>{});
    if (sizeof(T) == 4 || v == 4) return f(std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, sizeof(T) == 4 ? 4 : 8>{});
}

static int lanes_log2(int vectors) {
    int l = 0;
    while (l < 6 && (1 << l) < vectors) ++l;
    return l;
}

template <class T, class ID>
static int embedding_fwd_typed(const T* table, int64_t V, int D, const ID* ids, int64_t N, float scale, T* out, hipStream_t stream) {
    return with_vector<T>(D, [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        const int l = lanes_log2(D / VEC);
        const int64_t blocks = std::min<int64_t>(ceil_div(N, 256 >> l), 1 << 20);   // a launch holds fewer than 2^32 threads
        // few rows: their columns are spread over workgroups too
        const int wide = (int)std::min<int64_t>(ceil_div(D / VEC, 1 << l), std::max<int64_t>(1, ceil_div(1024, blocks)));
        hipLaunchKernelGGL((embedding_fwd_kernel<T, VEC, ID>), dim3((unsigned)blocks, wide), dim3(256), 0, stream, table, V, D, ids, N, scale, l, out);
        return check_launch("nerf_embedding_fwd");
    });
}

template <class ID>
static int embedding_sort(const ID* ids, int64_t N, int64_t V, int64_t padding, const EmbWork& w, char* work, const unsigned** keys, const unsigned** vals,
                          hipStream_t stream) {
    unsigned* k[2] = {reinterpret_cast<unsigned*>(work + w.keys[0]), reinterpret_cast<unsigned*>(work + w.keys[1])};
    unsigned* v[2] = {reinterpret_cast<unsigned*>(work + w.vals[0]), reinterpret_cast<unsigned*>(work + w.vals[1])};
    if (w.tiles <= 1) {
        hipLaunchKernelGGL((sort_small_kernel<ID>), dim3(1), dim3(SORT_THREADS), 0, stream, ids, (int)N, V, padding, w.passes, w.bits, k[0], v[0]);
        *keys = k[0];
        *vals = v[0];
        return check_launch("nerf_embedding_bwd(sort)");
    }
    unsigned* table = reinterpret_cast<unsigned*>(work + w.table);
    int from = 0;
    for (int p = 0; p < w.passes; ++p) {
        const int to = p == 0 ? 0 : 1 - from, shift = p * w.bits;
        const dim3 grid((unsigned)w.tiles), block(SORT_THREADS);
        if (p == 0) hipLaunchKernelGGL((sort_count_kernel<ID, true>), grid, block, 0, stream, ids, nullptr, N, V, padding, shift, w.bits, table);
        else hipLaunchKernelGGL((sort_count_kernel<ID, false>), grid, block, 0, stream, ids, k[from], N, V, padding, shift, w.bits, table);
        hipLaunchKernelGGL(sort_prefix_kernel, dim3((unsigned)ceil_div(1 << w.bits, 64)), block, 0, stream, table, (int)w.tiles, 1 << w.bits);
        if (p == 0)
            hipLaunchKernelGGL((sort_scatter_kernel<ID, true>), grid, block, 0, stream, ids, nullptr, nullptr, N, V, padding, shift, w.bits, table, (int)w.tiles,
                               k[to], v[to]);
        else
            hipLaunchKernelGGL((sort_scatter_kernel<ID, false>), grid, block, 0, stream, ids, k[from], v[from], N, V, padding, shift, w.bits, table,
                               (int)w.tiles, k[to], v[to]);
        if (int rc = check_launch("nerf_embedding_bwd(sort)")) return rc;
        from = to;
    }
    *keys = k[from];
    *vals = v[from];
    return NERF_OK;
}

template <class T>
static int embedding_sums(const T* d_out, int64_t N, int64_t V, int D, const unsigned* keys, const unsigned* vals, float scale, const EmbWork& w, char* work,
                          T* d_table, hipStream_t stream) {
    return with_vector<T>(D, [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        const int l = lanes_log2(D / VEC);
        const unsigned col_tiles = (unsigned)ceil_div(D / VEC, 1 << l);
        float* part = reinterpret_cast<float*>(work + w.part);
        int64_t long_blocks = 0;
        if (N >= EMB_LONG) {
            hipLaunchKernelGGL((embedding_partial_kernel<T, VEC>), dim3((unsigned)ceil_div(w.chunks, 4), col_tiles), dim3(256), 0, stream, d_out, D, keys, vals,
                               w.chunks, (unsigned)V, l, part);
            if (int rc = check_launch("nerf_embedding_bwd(partial)")) return rc;
            long_blocks = ceil_div(w.chunks, EMB_CANDIDATES);
        }
        const int at_once = 256 >> l;
        const int rounds = (int)std::max<int64_t>(1, std::min<int64_t>(256 / at_once, V * col_tiles / (2048ll * at_once)));
        const int rows = at_once * rounds;
        const int64_t blocks = long_blocks + ceil_div(V, rows);
        NERF_REQUIRE(blocks < (1ll << 31), "nerf_embedding_bwd: too many workgroups");
        hipLaunchKernelGGL((embedding_rows_kernel<T, VEC>), dim3((unsigned)blocks, col_tiles), dim3(256), 0, stream, d_out, D, keys, vals, N, V, scale, l, rows,
                           long_blocks, part, d_table);
        return check_launch("nerf_embedding_bwd(rows)");
    });
}

static int embedding_check(const char* who, int64_t V, int D, int type, int64_t N, const void* ids, int ids_bytes) {
    NERF_REQUIRE(V >= 0 && D >= 0 && N >= 0, "%s: V=%lld D=%d N=%lld", who, (long long)V, D, (long long)N);
    NERF_REQUIRE(V < 0x7fffffffll && N < 0x7fffffffll, "%s: at most 2^31 - 2 rows and ids", who);
    NERF_REQUIRE(known_type(type), "%s: type %d", who, type);
    NERF_REQUIRE(ids_bytes == 4 || ids_bytes == 8, "%s: ids of %d bytes", who, ids_bytes);
    NERF_REQUIRE(N == 0 || ids, "%s: null ids", who);
    NERF_REQUIRE(((uintptr_t)ids & (uintptr_t)(ids_bytes - 1)) == 0, "%s: ids must be aligned to their size", who);
    NERF_REQUIRE(ceil_div(D, 64) < 65536, "%s: rows of %d elements", who, D);
    return NERF_OK;
}

}  // namespace nerf

using namespace nerf;

extern "C" int nerf_embedding_fwd(const void* table, int type, int64_t V, int D, const void* ids, int ids_bytes, int64_t N, float scale, void* out,
                                  void* stream) {
    const char* who = "nerf_embedding_fwd";
    if (int rc = embedding_check(who, V, D, type, N, ids, ids_bytes)) return rc;
    if (N == 0 || D == 0) return NERF_OK;
    NERF_REQUIRE((table || V == 0) && out, "%s: null pointer", who);
    NERF_REQUIRE(aligned16(table) && aligned16(out), "%s: pointers must be 16-byte aligned", who);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if (ids_bytes == 8)
            return embedding_fwd_typed(static_cast<const T*>(table), V, D, static_cast<const int64_t*>(ids), N, scale, static_cast<T*>(out), (hipStream_t)stream);
        return embedding_fwd_typed(static_cast<const T*>(table), V, D, static_cast<const int32_t*>(ids), N, scale, static_cast<T*>(out), (hipStream_t)stream);
    });
}

extern "C" size_t nerf_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int D) {
    if (N <= 0 || V <= 0 || D <= 0) return 0;
    return embedding_work(N, V, D).bytes;
}

extern "C" int nerf_embedding_bwd(const void* d_out, int type, const void* ids, int ids_bytes, int64_t N, int64_t V, int D, float scale, int64_t padding_idx,
                                  void* d_table, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "nerf_embedding_bwd";
    if (int rc = embedding_check(who, V, D, type, N, ids, ids_bytes)) return rc;
    if (V == 0 || D == 0) return NERF_OK;
    NERF_REQUIRE((d_out || N == 0) && d_table, "%s: null pointer", who);
    NERF_REQUIRE(aligned16(d_out) && aligned16(d_table) && aligned16(workspace), "%s: pointers must be 16-byte aligned", who);
    NERF_REQUIRE(workspace_bytes >= nerf_embedding_bwd_workspace_bytes(N, V, D) && (workspace || N == 0), "%s: workspace of %zu bytes, %zu needed", who,
                 workspace_bytes, nerf_embedding_bwd_workspace_bytes(N, V, D));
    const EmbWork w = embedding_work(N, V, D);
    const unsigned *keys = nullptr, *vals = nullptr;
    if (N > 0) {
        const int rc = ids_bytes == 8 ? embedding_sort(static_cast<const int64_t*>(ids), N, V, padding_idx, w, static_cast<char*>(workspace), &keys, &vals, (hipStream_t)stream)
                                      : embedding_sort(static_cast<const int32_t*>(ids), N, V, padding_idx, w, static_cast<char*>(workspace), &keys, &vals, (hipStream_t)stream);
        if (rc) return rc;
    }
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return embedding_sums(static_cast<const T*>(d_out), N, V, D, keys, vals, scale, w, static_cast<char*>(workspace), static_cast<T*>(d_table), (hipStream_t)stream);
    });
}
