// Rows of a learned table by integer id, scaled, and the gradient of the table, for gfx950.
//
//   out[n] = scale * table[ids[n]]            d_table[v] = scale * sum over {n : ids[n] = v} of d_out[n]
//
// The forward pass is a gather bound by memory.  The gradient is formed without atomics, so that equal inputs give equal
// bits and a row that most of the batch asks for (one image's code in a whole ray batch, a frequent token) costs no more
// than its bytes: the positions are sorted by id with a stable radix sort (ids that take no gradient -- out of range, or
// the padding row -- sort behind all others as id V).  The sorted positions are cut into chunks of equal size, whatever
// runs of equal ids they hold, one wave each, so that the work is even however skewed the ids are:
//   - a wave adds up its chunk's rows, run by run.  A run that lies inside the chunk is finished and written; the
//     stretches of runs that cross the chunk's borders are left as partial rows, at most two a chunk;
//   - a second launch joins the partial rows of each run that crosses chunks.
// The rows that no id names are zeros: the whole table is cleared by workgroups of the sorting launches, which fill the
// compute units that the sort leaves idle.
// Rows of one vector (a hash grid's two features) are moved instead of sorted: see the buckets below.
// Sums are held in float, in an order that the ids alone decide, and rounded once.
#include <algorithm>

#include "typed.h"

namespace nerf {

constexpr int JOIN_THREADS = 512;
constexpr int JOIN_CHUNKS = 64;      // most chunks whose crossing runs one workgroup joins

constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
// Keys that a workgroup ranks at once: 4 a thread with more than SORT_MANY of them, else 1, so that more workgroups share the
// ranking.  16384 ids of 50021 rows of 64 float: 37 us with 4, 34 with 1 (most of them a few ids: 42 and 37); 2^17 49 and 48;
// 2^20 121 and 142.
constexpr int SORT_ITEMS = 4, SORT_TILE = SORT_THREADS * SORT_ITEMS;
constexpr int64_t SORT_MANY = 1 << 17;
constexpr int sort_items(int64_t n) { return n > SORT_MANY ? SORT_ITEMS : 1; }
constexpr int SORT_BITS = 10, SORT_DIGITS = 1 << SORT_BITS;
// Up to SORT_TILE keys are sorted by one workgroup in one launch.  More keys a workgroup (16384, 16 a thread) were slower than
// several tiles: 6000 ids of 1000 rows 30 us against 24, 16384 36 against 25, of 50021 rows 46 against 40.
// Up to so many tiles the scattering workgroups count all tiles' digits themselves, a launch a pass less (4 us for the host):
// 8 tiles 19.7 us against 21.5 (8192 ids of 2^19 rows of two floats), 21 and 22 (of 40 rows; 28 and 24 where a few ids are most).
constexpr int SORT_OWN_TILES = 8;
// Up to so many tiles they sum the counts of the tiles in front themselves.  Against a launch of its own for that: 64 tiles 42
// us and 44 (65536 ids of 50021 rows of 64 float), 27 and 25 (of 2^19 rows of two floats), 128 tiles 54 and 47, 36 and 25.
constexpr int SORT_FEW_TILES = 48;
constexpr unsigned NO_KEY = 0xffffffffu;

// ---- forward ---------------------------------------------------------------------------------------------------
// A group of lanes per row, 16 bytes a lane where the row divides into them.  Bound by the reads of the rows and the writes
// where those are long (65536 rows of 1024 bfloat16 out of 50021: 44 us, 6.1 TB/s, above a copy's rate, since some rows come
// from the caches again), by the lines that a row of a few bytes touches where they are short (2^20 rows of two floats out of
// 2^19: 11.6 us for 21 MB of ids, rows and outputs).  Four rows a group at a time were no faster (1 % on either side of it).
template <class T, int VEC, class ID>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const T* __restrict__ table, int64_t V, int D, const ID* __restrict__ ids, int64_t N,
                                                            float scale, int l_lanes, T* __restrict__ out) {
    const int lanes = 1 << l_lanes, vectors = D / VEC, at_once = 256 >> l_lanes, first = (threadIdx.x & (lanes - 1)) + (int)blockIdx.y * lanes;
    for (int64_t n = (int64_t)blockIdx.x * at_once + (threadIdx.x >> l_lanes); n < N; n += (int64_t)gridDim.x * at_once) {
        const int64_t id = (int64_t)ids[n];
        for (int i = first; i < vectors; i += lanes * (int)gridDim.y) {
            float v[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = __builtin_nanf("");
            if (id >= 0 && id < V) load_run<VEC>(table + id * D + (int64_t)i * VEC, v);
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] *= scale;
            store_run<VEC>(out + n * D + (int64_t)i * VEC, v);
        }
    }
}

// Zeros over the table's gradient, 16 bytes a store: workgroup `block` of `blocks`, 1024 threads each.
__device__ __forceinline__ void clear_table(char* __restrict__ p, int64_t bytes, int64_t block, int64_t blocks) {
    const int64_t wide = bytes >> 4;
    for (int64_t i = block * 1024 + threadIdx.x; i < wide; i += blocks * 1024) reinterpret_cast<uint4*>(p)[i] = uint4{0u, 0u, 0u, 0u};
    if (block == 0 && (int64_t)threadIdx.x < bytes - (wide << 4)) p[(wide << 4) + threadIdx.x] = 0;
}

__global__ __launch_bounds__(1024) void clear_kernel(char* __restrict__ p, int64_t bytes) { clear_table(p, bytes, blockIdx.x, gridDim.x); }

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
template <int ITEMS, int WAVES, int DIGITS>
__device__ __forceinline__ void rank_in_wave(const unsigned (&key)[ITEMS], const bool (&on)[ITEMS], int shift, int bits, unsigned (&count)[WAVES][DIGITS],
                                             unsigned (&rank)[ITEMS]) {
    const unsigned mask = (1u << bits) - 1u;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned long long below = (1ull << lane) - 1ull;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const unsigned d = (key[r] >> shift) & mask;
        unsigned long long same = __ballot(on[r]);
        unsigned lo = (unsigned)same, hi = (unsigned)(same >> 32);
        for (int b = 0; b < bits; ++b) {   // four vector instructions a bit: this loop is what ranking costs
            const int m = (int)(d << (31 - b)) >> 31;   // all ones where the bit is set
            const unsigned long long set = __ballot(m != 0);
            lo &= ~((unsigned)set ^ (unsigned)m);
            hi &= ~((unsigned)(set >> 32) ^ (unsigned)m);
        }
        same = (unsigned long long)hi << 32 | lo;
        rank[r] = 0;
        if (on[r]) {
            const unsigned old = count[wave][d];
            rank[r] = old + (unsigned)__popcll(same & below);
            if ((same >> lane) == 1ull) count[wave][d] = old + (unsigned)__popcll(same);   // the highest of them
        }
        // the next round reads what other lanes of this wave have just written: LDS keeps a wave's accesses in order,
        // the compiler has to as well
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
    }
}

// Exclusive sum over the workgroup's threads.
template <int WAVES>
__device__ __forceinline__ unsigned block_exclusive(unsigned v, unsigned (&s_wave)[WAVES]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
    }
    if (lane == 63) s_wave[wave] = inc;
    __syncthreads();
    unsigned base = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) base += w < wave ? s_wave[w] : 0u;
    __syncthreads();
    return base + inc - v;
}

// count[w][d] -> where the keys of wave w and digit d start in the sorted tile (thread d does digit d); `start`: where
// the digit's keys begin.
template <int DIGITS>
__device__ __forceinline__ void digit_starts(unsigned (&count)[SORT_WAVES][DIGITS], unsigned (&s_wave)[SORT_WAVES], int digits, unsigned& start) {
    const int d = threadIdx.x;
    unsigned c[SORT_WAVES], total = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
        c[w] = d < digits ? count[w][d] : 0u;
        total += c[w];
    }
    start = block_exclusive(total, s_wave);
    unsigned at = start;
    if (d < digits) {
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            count[w][d] = at;
            at += c[w];
        }
    }
}

template <int DIGITS>
__device__ __forceinline__ void clear_counts(unsigned (&count)[SORT_WAVES][DIGITS], int digits) {
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w)
        if ((int)threadIdx.x < digits) count[w][threadIdx.x] = 0u;
}

// One tile: every pass in one workgroup, the pairs changing places through LDS.
template <class ID, int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void sort_small_kernel(const ID* __restrict__ ids, int n, int64_t V, int64_t padding, int passes, int bits,
                                                                  uint2* __restrict__ sorted, char* __restrict__ clear, int64_t clear_bytes) {
    if (blockIdx.x > 0) {
        clear_table(clear, clear_bytes, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    __shared__ unsigned s_count[SORT_WAVES][SORT_DIGITS];
    __shared__ unsigned s_key[SORT_THREADS * ITEMS];
    __shared__ unsigned short s_val[SORT_THREADS * ITEMS];
    __shared__ unsigned s_wave[SORT_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int items = (n + SORT_THREADS - 1) / SORT_THREADS;   // rounds in use: the tile is packed to the front of every wave
    unsigned key[ITEMS], rank[ITEMS], val[ITEMS];
    bool on[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int i = wave * 64 * items + r * 64 + lane;
        on[r] = r < items && i < n;
        key[r] = on[r] ? sort_key(ids[i], V, padding) : 0u;
        val[r] = (unsigned)i;
    }
    for (int p = 0; p < passes; ++p) {
        clear_counts(s_count, 1 << bits);
        __syncthreads();
        rank_in_wave(key, on, p * bits, bits, s_count, rank);
        __syncthreads();
        unsigned start;
        digit_starts(s_count, s_wave, 1 << bits, start);
        __syncthreads();
        const unsigned mask = (1u << bits) - 1u;
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            if (on[r]) {
                const unsigned to = s_count[wave][(key[r] >> (p * bits)) & mask] + rank[r];
                s_key[to] = key[r];
                s_val[to] = (unsigned short)val[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ITEMS; ++r) {
            const int i = wave * 64 * items + r * 64 + lane;
            if (on[r]) {
                key[r] = s_key[i];
                val[r] = s_val[i];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int i = wave * 64 * items + r * 64 + lane;
        if (on[r]) sorted[i] = uint2{key[r], val[r]};
    }
}

// More keys: per pass, the digits of every tile are counted, the counts summed over the tiles in front, and the tiles
// ranked and scattered.  table: [tiles][digits], then [digits] totals.  With few tiles the scattering workgroups count
// or sum themselves: a launch or two less.
template <class ID, bool FIRST, int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(const ID* __restrict__ ids, const uint2* __restrict__ from, int64_t n, int64_t V,
                                                                  int64_t padding, int shift, int bits, unsigned limit, int tiles, unsigned* __restrict__ table,
                                                                  char* __restrict__ clear, int64_t clear_bytes) {
    if ((int)blockIdx.x >= tiles) {
        clear_table(clear, clear_bytes, blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    __shared__ unsigned s_count[SORT_DIGITS];
    const int digits = 1 << bits;
    for (int i = threadIdx.x; i < digits; i += SORT_THREADS) s_count[i] = 0u;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ITEMS);
    for (int r = 0; r < ITEMS; ++r) {
        const int64_t i = base + r * SORT_THREADS + threadIdx.x;
        if (i < n) {
            const unsigned key = FIRST ? sort_key(ids[i], V, padding) : from[i].x;
            if (key < limit) atomicAdd(&s_count[(key >> shift) & (digits - 1)], 1u);   // whole numbers: the order does not matter
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

// How many keys of digit threadIdx.x there are in all (total) and in the tiles in front of this one (front).  With the sums of
// sort_prefix_kernel (SUMMED), with the tiles' counts (COUNTED), or from the keys themselves: key_at(i), NO_KEY where there is
// none, counted in s_total and s_front [digits].
enum { SORT_SUMMED, SORT_COUNTED, SORT_UNCOUNTED };
template <int ITEMS, class F>
__device__ __forceinline__ void digit_counts(int mode, const unsigned* __restrict__ table, int tiles, int digits, int shift, unsigned (&s_total)[SORT_DIGITS],
                                             unsigned (&s_front)[SORT_DIGITS], const F& key_at, unsigned& total, unsigned& front) {
    const int d = threadIdx.x;
    total = front = 0;
    if (mode == SORT_UNCOUNTED) {
        s_total[d] = s_front[d] = 0u;
        __syncthreads();
        for (int t = 0; t < tiles; ++t) {
            unsigned key[ITEMS];
#pragma unroll
            for (int r = 0; r < ITEMS; ++r) key[r] = key_at((int64_t)t * (SORT_THREADS * ITEMS) + r * SORT_THREADS + d);
#pragma unroll
            for (int r = 0; r < ITEMS; ++r) {
                if (key[r] == NO_KEY) continue;
                const unsigned digit = (key[r] >> shift) & (unsigned)(digits - 1);
                atomicAdd(&s_total[digit], 1u);   // whole numbers: the order does not matter
                if (t < (int)blockIdx.x) atomicAdd(&s_front[digit], 1u);
            }
        }
        __syncthreads();
        if (d < digits) {
            total = s_total[d];
            front = s_front[d];
        }
    } else if (d < digits) {
        if (mode == SORT_SUMMED) {
            total = table[(int64_t)tiles * digits + d];
            front = table[(int64_t)blockIdx.x * digits + d];
        } else {
#pragma unroll 8
            for (int t = 0; t < tiles; ++t) {
                const unsigned n_t = table[(int64_t)t * digits + d];
                total += n_t;
                front += t < (int)blockIdx.x ? n_t : 0u;
            }
        }
    }
}

// The tile is put in order in LDS first, so that neighbouring lanes write neighbouring places of the output.  Bound by the
// chain of loads, ballots and barriers of one workgroup a tile: 8 us up to 256 tiles (2^20 keys 12 us, 16 MB moved).
template <class ID, bool FIRST, int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void sort_scatter_kernel(const ID* __restrict__ ids, const uint2* __restrict__ from, int64_t n, int64_t V, int64_t padding,
                                                                    int shift, int bits, const unsigned* __restrict__ table, int tiles, int mode,
                                                                    uint2* __restrict__ to, char* __restrict__ clear, int64_t clear_bytes) {
    if ((int)blockIdx.x >= tiles) {
        clear_table(clear, clear_bytes, blockIdx.x - tiles, gridDim.x - tiles);
        return;
    }
    __shared__ unsigned s_count[SORT_WAVES][SORT_DIGITS];
    __shared__ unsigned s_to[SORT_DIGITS];   // what a rank in the sorted tile lacks to its place in the output, per digit
    __shared__ unsigned s_wave[SORT_WAVES];
    __shared__ uint2 s_pair[(SORT_THREADS * ITEMS)];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << bits;
    const int64_t tile = (int64_t)blockIdx.x * (SORT_THREADS * ITEMS);
    unsigned key[ITEMS], val[ITEMS], rank[ITEMS];
    bool on[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int64_t i = tile + (wave * ITEMS + r) * 64 + lane;
        on[r] = i < n;
        key[r] = val[r] = 0u;
        if (on[r]) {
            if (FIRST) {
                key[r] = sort_key(ids[i], V, padding);
                val[r] = (unsigned)i;
            } else {
                const uint2 pair = from[i];
                key[r] = pair.x;
                val[r] = pair.y;
            }
        }
    }
    unsigned total, front;
    digit_counts<ITEMS>(mode, table, tiles, digits, shift, s_to, s_count[0], [&](int64_t i) { return i >= n ? NO_KEY : FIRST ? sort_key(ids[i], V, padding) : from[i].x; }, total, front);
    __syncthreads();
    clear_counts(s_count, digits);
    __syncthreads();
    rank_in_wave(key, on, shift, bits, s_count, rank);
    __syncthreads();
    unsigned start;
    digit_starts(s_count, s_wave, digits, start);
    const unsigned first = block_exclusive(total, s_wave);
    if ((int)threadIdx.x < digits) s_to[threadIdx.x] = first + front - start;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
        if (on[r]) s_pair[s_count[wave][(key[r] >> shift) & (unsigned)(digits - 1)] + rank[r]] = uint2{key[r], val[r]};
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int i = r * SORT_THREADS + (int)threadIdx.x;
        if (tile + i < n) {
            const uint2 pair = s_pair[i];
            to[(unsigned)i + s_to[(pair.x >> shift) & (unsigned)(digits - 1)]] = pair;
        }
    }
}

// ---- sums over the runs --------------------------------------------------------------------------------------------
struct EmbSums {
    const uint2* sorted;    // (id, position) in the order of the ids
    int64_t N, V;
    int D, l_lanes;         // log2 of the lanes on a row
    int l_chunk;            // log2 of the positions of a chunk
    int col_tiles;          // column tiles of a row: 64 lanes cover one
    int64_t chunks;
    int join_chunks;        // chunks whose crossing runs one workgroup of the join looks after
    float scale;
    float* part;            // [chunks][2][D]: the stretch of the run that comes in from the chunk in front, and of the run that starts here and goes on
};

// A wave holds 64 / lanes sorted positions at a time, one per group of lanes, and adds them up by a scan that stops where
// the id changes; what the last group holds is carried into the next round.  The rows of ROUNDS rounds are under way at
// once.  WHOLE: all 64 lanes on one row -- the id is the wave's, and nothing changes lanes.  Bound by the reads of the rows,
// and by their latency where there are few: 65536 rows of 32 float 6.8 us (8 MB), 16384 of 1024 bfloat16 15 us (34 MB).
template <class T, int VEC, bool WHOLE>
__global__ __launch_bounds__(256) void embedding_sums_kernel(EmbSums p, const T* __restrict__ d_out, T* __restrict__ d_table) {
    constexpr int ROUNDS = 8;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), chunk = id / p.col_tiles;
    if (chunk >= p.chunks) return;
    const int l_lanes = WHOLE ? 6 : p.l_lanes;
    const int lane = threadIdx.x & 63, lanes = 1 << l_lanes, groups = 64 >> l_lanes, group = lane >> l_lanes, c = lane & (lanes - 1);
    const int64_t col = ((id - chunk * p.col_tiles) * lanes + c) * VEC;
    const bool on = col < p.D;
    const int64_t base = chunk << p.l_chunk, end = min(base + (1ll << p.l_chunk), p.N);
    const unsigned before = base > 0 ? p.sorted[base - 1].x : NO_KEY, after = end < p.N ? p.sorted[end].x : NO_KEY;
    const unsigned V = (unsigned)p.V;
    float* __restrict__ part = p.part + chunk * 2 * p.D + col;

    const auto write = [&](unsigned key, const float (&v)[VEC], bool goes_on) {
        if (!on) return;
        if (key == before) {
            store_run<VEC>(part, v);
        } else if (goes_on) {
            store_run<VEC>(part + p.D, v);
        } else {
            float out[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) out[k] = v[k] * p.scale;
            store_run<VEC>(d_table + (int64_t)key * p.D + col, out);
        }
    };

    unsigned carry_key = NO_KEY;
    float carry[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) carry[k] = 0.0f;
    for (int64_t at = base; at < end; at += ROUNDS * groups) {
        unsigned key[ROUNDS];
        float row[ROUNDS][VEC];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int64_t i = at + r * groups + group;
            uint2 pair{NO_KEY, 0u};
            if (i < end) pair = p.sorted[i];
            key[r] = pair.x >= V ? NO_KEY : pair.x;   // ids that take no gradient
            if (WHOLE) key[r] = (unsigned)__builtin_amdgcn_readfirstlane((int)key[r]);
#pragma unroll
            for (int k = 0; k < VEC; ++k) row[r][k] = 0.0f;
            if (on && key[r] != NO_KEY) load_run<VEC>(d_out + (int64_t)pair.y * p.D + col, row[r]);
        }
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            if (at + r * groups >= end) break;
            const unsigned k = key[r];
            if (WHOLE) {
                if (k != carry_key) {
                    if (carry_key != NO_KEY) write(carry_key, carry, false);
                    carry_key = k;
#pragma unroll
                    for (int q = 0; q < VEC; ++q) carry[q] = row[r][q];
                } else {
#pragma unroll
                    for (int q = 0; q < VEC; ++q) carry[q] += row[r][q];
                }
                continue;
            }
            float v[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) v[q] = row[r][q];
            for (int d = 1; d < groups; d <<= 1) {
                const bool take = __shfl_up(k, d << l_lanes, 64) == k && group >= d;
#pragma unroll
                for (int q = 0; q < VEC; ++q) {
                    const float o = __shfl_up(v[q], d << l_lanes, 64);
                    if (take) v[q] += o;
                }
            }
            if (carry_key != NO_KEY && __shfl(k, c, 64) != carry_key && group == 0) write(carry_key, carry, false);   // it ended with the last round
            if (k == carry_key) {
#pragma unroll
                for (int q = 0; q < VEC; ++q) v[q] += carry[q];
            }
            const unsigned next = __shfl_down(k, lanes, 64);
            if (group + 1 < groups && next != k && k != NO_KEY) write(k, v, false);
            const int last = 64 - lanes + c;
            carry_key = __shfl(k, last, 64);
#pragma unroll
            for (int q = 0; q < VEC; ++q) carry[q] = __shfl(v[q], last, 64);
        }
    }
    if (carry_key != NO_KEY && group == 0) write(carry_key, carry, carry_key == after);
}

// The runs that cross chunks: a run belongs to the chunk that it starts in.  Those over a few chunks are joined by a
// group of lanes each, longer ones by the whole workgroup.  A few dependent reads long whatever there is to join: 7 us where
// there is little, 13 for 40 runs over some fifty chunks each.
template <class T, int VEC>
__global__ __launch_bounds__(JOIN_THREADS) void embedding_join_kernel(EmbSums p, T* __restrict__ d_table) {
    constexpr int FEW = 16;   // against 8: runs over 8 to 15 chunks 39 us and 52 (262144 ids of 1000 rows), shorter ones 0.7 us more
    __shared__ int s_over[JOIN_CHUNKS];       // chunks that the run goes on over, FEW: at least so many; 0: none starts here
    __shared__ unsigned s_key[JOIN_CHUNKS];
    __shared__ int s_count[JOIN_THREADS / 64];
    __shared__ float s_sum[JOIN_THREADS * VEC];
    const int64_t first = (int64_t)blockIdx.x * p.join_chunks;
    // a run goes on into a chunk that starts with its id
    const auto start_key = [&](int64_t chunk) { return chunk < p.chunks ? p.sorted[chunk << p.l_chunk].x : NO_KEY; };
    if ((int)threadIdx.x < p.join_chunks) {
        const int64_t chunk = first + threadIdx.x, end = (chunk + 1) << p.l_chunk;
        int over = 0;
        if (end < p.N) {
            const unsigned key = p.sorted[end - 1].x, next = p.sorted[end].x, before = chunk == 0 ? NO_KEY : p.sorted[(chunk << p.l_chunk) - 1].x;
            unsigned starts[FEW - 1];
#pragma unroll
            for (int k = 0; k < FEW - 1; ++k) starts[k] = start_key(chunk + 2 + k);
            if (key < (unsigned)p.V && next == key && before != key) {
                over = 1;
#pragma unroll
                for (int k = 0; k < FEW - 1; ++k) over += over == k + 1 && starts[k] == key;
            }
            s_key[threadIdx.x] = key;
        }
        s_over[threadIdx.x] = over;
    }
    __syncthreads();
    const int lanes = 1 << p.l_lanes, groups = JOIN_THREADS >> p.l_lanes, group = threadIdx.x >> p.l_lanes, c = threadIdx.x & (lanes - 1);
    const int64_t col = ((int64_t)blockIdx.y * lanes + c) * VEC;
    const bool on = col < p.D;
    const float* __restrict__ part = p.part + col;
    const auto add = [&](int64_t chunk, int64_t i, float (&sum)[VEC]) {
        float v[VEC];
        load_run<VEC>(part + (i * 2 + (i == chunk ? 1 : 0)) * p.D, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] += v[k];
    };
    const auto finish = [&](unsigned key, float (&sum)[VEC]) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] *= p.scale;
        store_run<VEC>(d_table + (int64_t)key * p.D + col, sum);
    };
    if (on) {
        for (int q = group; q < p.join_chunks; q += groups) {
            const int over = s_over[q];
            if (over == 0 || over == FEW) continue;
            const int64_t chunk = first + q;
            float sum[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
#pragma unroll 4
            for (int64_t i = chunk; i <= chunk + over; ++i) add(chunk, i, sum);
            finish(s_key[q], sum);
        }
    }
    for (int q = 0; q < p.join_chunks; ++q) {
        if (s_over[q] != FEW) continue;
        const int64_t chunk = first + q;
        // the last chunk that the run goes on into, by JOIN_THREADS probes a round: in [lo, hi)
        int64_t lo = chunk + FEW, hi = p.chunks;
        while (hi - lo > 1) {
            const int64_t step = (hi - lo - 1 + JOIN_THREADS - 1) / JOIN_THREADS, at = lo + (threadIdx.x + 1) * step;
            const int in_wave = __popcll(__ballot(at < hi && start_key(at) == s_key[q]));
            __syncthreads();
            if ((threadIdx.x & 63) == 0) s_count[threadIdx.x >> 6] = in_wave;
            __syncthreads();
            int through = 0;
            for (int k = 0; k < JOIN_THREADS / 64; ++k) through += s_count[k];
            lo += through * step;
            hi = min(hi, lo + step);
        }
        const int64_t last = lo;
        float sum[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
        if (on) {
#pragma unroll 8
            for (int64_t i = chunk + group; i <= last; i += groups) add(chunk, i, sum);
        }
        const int used = (int)min((int64_t)groups, last - chunk + 1);   // groups that hold something
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VEC; ++k) s_sum[threadIdx.x * VEC + k] = sum[k];
        __syncthreads();
        if (group == 0 && on) {
#pragma unroll 4
            for (int g = 1; g < used; ++g)
#pragma unroll
                for (int k = 0; k < VEC; ++k) sum[k] += s_sum[(g * lanes + c) * VEC + k];
            finish(s_key[q], sum);
        }
    }
}

// ---- narrow rows -------------------------------------------------------------------------------------------------------
// Rows of up to 16 bytes.  Sorted whole, each position costs two moves of a pair and then a read of its row from anywhere
// (2^20 rows of 8 bytes: 19 us of 70 for that alone).  Here the rows themselves are moved, once and as they are read, in order
// of their ids' upper bits: a bucket holds the rows of 2^low neighbouring ids, in the order of their positions.  A workgroup
// then puts up to BUCKET_SEG rows of a bucket in order in LDS and adds up each id's run; it writes all of its bucket's part of
// the table, so that nothing is cleared.  A bucket of more rows -- ids are often far from even -- is cut into segments, whose
// sums a last launch adds in order.  2^20 positions over 2^19 rows of two floats: 38 us, sorted whole 66; 16384: 27 and 38;
// most of them a few ids: 51 and 77.  (Up to 1023 rows one pass sorts them, and the two ways take the same time.)
constexpr int BUCKETS = 1024, BUCKET_BITS = 10, BUCKET_LOW = 5;   // 2^5 ids to a bucket at least
constexpr int BUCKET_WAVES = 4, BUCKET_THREADS = 64 * BUCKET_WAVES, BUCKET_ITEMS = 8, BUCKET_SEG = BUCKET_THREADS * BUCKET_ITEMS;
constexpr int BUCKET_MOST_BITS = 20;
constexpr unsigned BUCKET_RUN = 128;   // rows of one id that a lane adds up by itself; of more, a wave

template <class T, int VEC>
constexpr int row_words() { return (int)(sizeof(T) * VEC + 3) / 4; }

// A row as it lies in memory, in words, and back.
template <class T, int VEC>
__device__ __forceinline__ void row_load(const T* __restrict__ p, unsigned (&w)[row_words<T, VEC>()]) {
    const Run<T, VEC> r = *reinterpret_cast<const Run<T, VEC>*>(p);
    if constexpr (sizeof(T) * VEC == 2) w[0] = __builtin_bit_cast(unsigned short, r.v[0]);
    else __builtin_memcpy(w, &r, sizeof(r));
}
template <class T, int VEC>
__device__ __forceinline__ float row_value(const unsigned* w, int k) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[k]);
    else return (float)__builtin_bit_cast(T, (unsigned short)(w[k / 2] >> (k & 1) * 16));
}

template <class T, int VEC, class ID, int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void bucket_scatter_kernel(const ID* __restrict__ ids, int64_t n, int64_t V, int64_t padding, int low,
                                                                      unsigned* __restrict__ table, int tiles, int mode, const T* __restrict__ d_out,
                                                                      unsigned* __restrict__ to) {
    constexpr int W = row_words<T, VEC>(), ITEM = 1 + W;
    __shared__ unsigned s_count[SORT_WAVES][BUCKETS];
    __shared__ unsigned s_to[BUCKETS];   // as in sort_scatter_kernel
    __shared__ unsigned s_wave[SORT_WAVES];
    __shared__ unsigned s_item[(SORT_THREADS * ITEMS) * ITEM];
    __shared__ int s_held;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t tile = (int64_t)blockIdx.x * (SORT_THREADS * ITEMS);
    unsigned key[ITEMS], rank[ITEMS], row[ITEMS][W];
    bool on[ITEMS];
    if (threadIdx.x == 0) s_held = 0;
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int64_t i = tile + (wave * ITEMS + r) * 64 + lane;
        key[r] = i < n ? sort_key(ids[i], V, padding) : (unsigned)V;
        on[r] = key[r] < (unsigned)V;
#pragma unroll
        for (int k = 0; k < W; ++k) row[r][k] = 0u;
        if (i < n) row_load<T, VEC>(d_out + i * VEC, row[r]);
    }
    unsigned total, front;
    const auto key_at = [&](int64_t i) {
        const unsigned k = i < n ? sort_key(ids[i], V, padding) : (unsigned)V;
        return k < (unsigned)V ? k : NO_KEY;
    };
    digit_counts<ITEMS>(mode, table, tiles, BUCKETS, low, s_to, s_count[0], key_at, total, front);
    if (mode != SORT_SUMMED && blockIdx.x == 0) table[(int64_t)tiles * BUCKETS + threadIdx.x] = total;   // for the sums
    __syncthreads();
    clear_counts(s_count, BUCKETS);
    __syncthreads();
    rank_in_wave(key, on, low, BUCKET_BITS, s_count, rank);
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int held = __popcll(__ballot(on[r]));
        if (lane == 0) atomicAdd(&s_held, held);
    }
    __syncthreads();
    unsigned start;
    digit_starts(s_count, s_wave, BUCKETS, start);
    const unsigned first = block_exclusive(total, s_wave);
    s_to[threadIdx.x] = first + front - start;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        if (on[r]) {
            unsigned* const at = s_item + (s_count[wave][key[r] >> low] + rank[r]) * ITEM;
            at[0] = key[r];
#pragma unroll
            for (int k = 0; k < W; ++k) at[1 + k] = row[r][k];
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
        const int i = r * SORT_THREADS + (int)threadIdx.x;
        if (i < s_held) {
            const unsigned* const from = s_item + i * ITEM;
            unsigned* const at = to + (int64_t)((unsigned)i + s_to[from[0] >> low]) * ITEM;
#pragma unroll
            for (int k = 0; k < ITEM; ++k) at[k] = from[k];
        }
    }
}

struct BucketSums {
    const unsigned* total;   // [BUCKETS] rows
    const unsigned* items;
    float* part;             // [segments][2^low][D]
    int64_t V;
    int low, buckets;
    float scale;
};
__device__ __forceinline__ unsigned bucket_segments(const BucketSums& p, int q, unsigned rows) {
    return q < p.buckets ? max(1u, (rows + BUCKET_SEG - 1) / BUCKET_SEG) : 0u;
}

// A workgroup: one segment.
template <class T, int VEC>
__global__ __launch_bounds__(BUCKET_THREADS) void bucket_sums_kernel(BucketSums p, T* __restrict__ d_table) {
    constexpr int W = row_words<T, VEC>(), ITEM = 1 + W, PER = BUCKETS / BUCKET_THREADS;
    __shared__ unsigned s_count[BUCKET_WAVES][BUCKETS];
    __shared__ unsigned s_row[BUCKET_SEG * W];
    __shared__ unsigned s_start[BUCKETS + 1];
    __shared__ unsigned s_wave[BUCKET_WAVES];
    __shared__ unsigned s_bucket, s_segment, s_first, s_rows;
    __shared__ unsigned s_long[BUCKET_SEG / BUCKET_RUN], s_longs;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // which segment of which bucket: buckets hold their segments one after the other
    if (threadIdx.x == 0) {
        s_bucket = NO_KEY;
        s_longs = 0;
    }
    unsigned rows[PER], segments[PER], all_rows = 0, all_segments = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int q = (int)threadIdx.x * PER + k;
        rows[k] = p.total[q];
        segments[k] = bucket_segments(p, q, rows[k]);
        all_rows += rows[k];
        all_segments += segments[k];
    }
    unsigned first = block_exclusive(all_rows, s_wave), segment = block_exclusive(all_segments, s_wave);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        if (blockIdx.x >= segment && blockIdx.x < segment + segments[k]) {
            s_bucket = threadIdx.x * PER + k;
            s_segment = blockIdx.x - segment;
            s_first = first;
            s_rows = rows[k];
        }
        first += rows[k];
        segment += segments[k];
    }
    for (int i = threadIdx.x; i < BUCKET_WAVES * BUCKETS; i += BUCKET_THREADS) s_count[0][i] = 0u;
    __syncthreads();
    if (s_bucket == NO_KEY) return;   // more workgroups than segments
    const int skip = (int)s_segment * BUCKET_SEG, n = min(BUCKET_SEG, (int)s_rows - skip), ids = 1 << p.low;
    const bool whole = s_rows <= BUCKET_SEG;
    const unsigned* const items = p.items + ((int64_t)s_first + skip) * ITEM;
    const int rounds = (n + BUCKET_THREADS - 1) / BUCKET_THREADS;   // in use: the rows are packed to the front of every wave
    unsigned key[BUCKET_ITEMS], rank[BUCKET_ITEMS], row[BUCKET_ITEMS][W];
    bool on[BUCKET_ITEMS];
#pragma unroll
    for (int r = 0; r < BUCKET_ITEMS; ++r) {
        const int i = wave * 64 * rounds + r * 64 + lane;
        on[r] = r < rounds && i < n;
        key[r] = 0u;
#pragma unroll
        for (int k = 0; k < W; ++k) row[r][k] = 0u;
        if (on[r]) {
            key[r] = items[(int64_t)i * ITEM] & (unsigned)(ids - 1);
#pragma unroll
            for (int k = 0; k < W; ++k) row[r][k] = items[(int64_t)i * ITEM + 1 + k];
        }
    }
    rank_in_wave(key, on, 0, p.low, s_count, rank);
    __syncthreads();
    unsigned held = 0, c[PER][BUCKET_WAVES];
#pragma unroll
    for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int w = 0; w < BUCKET_WAVES; ++w) {
            c[k][w] = s_count[w][threadIdx.x * PER + k];
            held += c[k][w];
        }
    unsigned at = block_exclusive(held, s_wave);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        s_start[threadIdx.x * PER + k] = at;
#pragma unroll
        for (int w = 0; w < BUCKET_WAVES; ++w) {
            s_count[w][threadIdx.x * PER + k] = at;
            at += c[k][w];
        }
    }
    if (threadIdx.x == BUCKET_THREADS - 1) s_start[BUCKETS] = at;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < BUCKET_ITEMS; ++r) {
        if (on[r]) {
#pragma unroll
            for (int k = 0; k < W; ++k) s_row[(s_count[wave][key[r]] + rank[r]) * W + k] = row[r][k];
        }
    }
    __syncthreads();
    const auto finish = [&](unsigned id, float (&sum)[VEC]) {
        if (whole) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] *= p.scale;
            store_run<VEC>(d_table + (((int64_t)s_bucket << p.low) + id) * VEC, sum);
        } else {
            store_run<VEC>(p.part + ((int64_t)blockIdx.x * ids + id) * VEC, sum);
        }
    };
    const int here = (int)min((int64_t)ids, p.V - ((int64_t)s_bucket << p.low));   // ids that are rows of the table
    for (int id = threadIdx.x; id < here; id += BUCKET_THREADS) {
        const unsigned begin = s_start[id], end = s_start[id + 1];
        if (end - begin > BUCKET_RUN) {
            s_long[atomicAdd(&s_longs, 1u)] = id;   // each is added up by itself: their order does not matter
            continue;
        }
        float sum[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
#pragma unroll 4
        for (unsigned i = begin; i < end; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += row_value<T, VEC>(s_row + i * W, k);
        finish(id, sum);
    }
    __syncthreads();
    for (unsigned q = wave; q < s_longs; q += BUCKET_WAVES) {
        const unsigned id = s_long[q], end = s_start[id + 1];
        float sum[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
        for (unsigned i = s_start[id] + lane; i < end; i += 64)
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += row_value<T, VEC>(s_row + i * W, k);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1)
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += __shfl_xor(sum[k], d, 64);
        if (lane == 0) finish(id, sum);
    }
}

// The buckets of several segments: JOIN_IDS ids a workgroup, JOIN_PARTS stretches of the segments side by side.
constexpr int JOIN_IDS = 256, JOIN_PARTS = 1024 / JOIN_IDS;
template <class T, int VEC>
__global__ __launch_bounds__(1024) void bucket_join_kernel(BucketSums p, T* __restrict__ d_table) {
    __shared__ unsigned s_wave[SORT_WAVES];
    __shared__ unsigned s_first;
    __shared__ float s_sum[JOIN_PARTS][JOIN_IDS][VEC];
    const unsigned q = blockIdx.x;
    const unsigned mine = bucket_segments(p, (int)q, p.total[q]);
    if (mine == 1) return;
    const unsigned first = block_exclusive(bucket_segments(p, (int)threadIdx.x, p.total[threadIdx.x]), s_wave);
    if (threadIdx.x == q) s_first = first;
    __syncthreads();
    const int slot = threadIdx.x & (JOIN_IDS - 1), stretch = threadIdx.x / JOIN_IDS, ids = 1 << p.low, id = (int)blockIdx.y * JOIN_IDS + slot;
    const int64_t v = ((int64_t)q << p.low) + id;
    const bool on = id < ids && v < p.V;
    const unsigned per = (mine + JOIN_PARTS - 1) / JOIN_PARTS, begin = min(stretch * per, mine), end = min(begin + per, mine);
    float sum[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
    if (on) {
#pragma unroll 8
        for (unsigned i = begin; i < end; ++i) {
            float x[VEC];
            load_run<VEC>(p.part + ((int64_t)(s_first + i) * ids + id) * VEC, x);
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] += x[k];
        }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) s_sum[stretch][slot][k] = sum[k];
    __syncthreads();
    if (stretch > 0 || !on) return;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        for (int j = 1; j < JOIN_PARTS; ++j) sum[k] += s_sum[j][slot][k];
        sum[k] *= p.scale;
    }
    store_run<VEC>(d_table + v * VEC, sum);
}

// ---- host ------------------------------------------------------------------------------------------------------------
static int vector_of(int D, int size) {   // elements per lane: the widest power of two that divides a row, 16 bytes at most
    int v = 16 / size;
    while (D % v) v >>= 1;
    return v;
}

static int lanes_log2(int vectors) {
    int l = 0;
    while (l < 6 && (1 << l) < vectors) ++l;
    return l;
}

struct EmbWork {                       // the workspace, cut into arrays that start on 256-byte boundaries
    int passes, bits;
    int64_t tiles;
    size_t pairs[2], table, part, bytes;
};

// log2 of the positions of a chunk: 32 positions or four rounds of a wave, whichever is more, which keeps the two partial
// rows of a chunk (8 bytes an element, written and read) a small part of its rows' bytes; down to 8 or four rounds while that
// leaves too few waves to hide the reads.  50021 rows of 1024 bfloat16: 4096 ids 28 us with 8 positions, 33 with 16, 42 with
// 32; 16384 ids 49, 52 and 59, or where a few ids are most of them 65, 60 and 63; 65536 ids 90, 76 and 72.
constexpr int SUM_WAVES = 2048;
static int chunk_log2(int64_t N, int l_lanes, int col_tiles) {
    int l = std::max(5, 8 - l_lanes);
    while (l > std::max(3, 8 - l_lanes) && ceil_div(N, 1ll << l) * col_tiles < SUM_WAVES) --l;
    return l;
}

static EmbWork embedding_work(int64_t N, int64_t V, int D) {
    EmbWork w;
    int bits = 1;
    while ((1ll << bits) < V + 1) ++bits;
    const bool small = N <= SORT_TILE;
    w.passes = (int)ceil_div(bits, SORT_BITS);
    w.bits = (int)ceil_div(bits, w.passes);
    w.tiles = small ? 1 : ceil_div(N, SORT_THREADS * sort_items(N));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    w.pairs[0] = take(8 * N);
    w.pairs[1] = take(small ? 0 : 8 * N);
    w.table = take(small ? 0 : 4ull * (w.tiles + 1) << w.bits);
    // chunks hold 32 positions or more, or 8 or more while they are fewer than twice SUM_WAVES
    w.part = take(N > 8 ? 8ull * D * (size_t)std::max(ceil_div(N, 32), std::min<int64_t>(ceil_div(N, 8), 2 * SUM_WAVES)) : 0);
    w.bytes = at;
    return w;
}

// Narrow rows: one vector each, more ids than one tile, more rows than one pass sorts by, few enough for the buckets.  (2048 ids
// of 2^19 rows of two floats: 18 us, sorted by one workgroup 22.)
static bool embedding_narrow(int64_t N, int64_t V, int D, int size) { return N > SORT_THREADS && V >= SORT_DIGITS && V <= 1ll << BUCKET_MOST_BITS && vector_of(D, size) == D; }

struct NarrowWork {
    int low, buckets;
    int64_t tiles, segments;   // segments: at most
    size_t table, items, part, bytes;
};
static NarrowWork narrow_work(int64_t N, int64_t V, int D) {   // for elements of any size
    NarrowWork w;
    w.low = BUCKET_LOW;
    while (BUCKETS << w.low < V) ++w.low;
    w.buckets = (int)ceil_div(V, 1 << w.low);
    w.tiles = ceil_div(N, SORT_THREADS * sort_items(N));
    w.segments = w.buckets + N / BUCKET_SEG;
    w.table = 0;
    w.items = 4ull * (w.tiles + 1) * BUCKETS;
    w.part = w.items + (4ull * (1 + std::min(D, 4)) * N + 255) / 256 * 256;   // a row of more than four elements has 16-bit ones
    w.bytes = w.part + (4ull * D * w.segments << w.low);
    return w;
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

static int sort_mode(int64_t tiles) { return tiles > SORT_FEW_TILES ? SORT_SUMMED : tiles > SORT_OWN_TILES ? SORT_COUNTED : SORT_UNCOUNTED; }

// f(integral_constant ITEMS)
template <class F>
static void with_items(int64_t N, F&& f) {
    if (sort_items(N) == 1) f(std::integral_constant<int, 1>{});
    else f(std::integral_constant<int, SORT_ITEMS>{});
}

template <class ID>
static int embedding_sort(const ID* ids, int64_t N, int64_t V, int64_t padding, const EmbWork& w, char* work, char* clear, int64_t clear_bytes,
                          const uint2** sorted, hipStream_t stream) {
    // workgroups that clear: 16 KB each while that leaves them one to a compute unit or fewer, then more
    const auto clearing = [](int64_t bytes) { return (unsigned)std::min<int64_t>(1024, ceil_div(bytes, 16384)); };
    uint2* pairs[2] = {reinterpret_cast<uint2*>(work + w.pairs[0]), reinterpret_cast<uint2*>(work + w.pairs[1])};
    if (N <= SORT_TILE) {   // one workgroup
        const auto launch = [&](auto items) {
            hipLaunchKernelGGL((sort_small_kernel<ID, decltype(items)::value>), dim3(1 + clearing(clear_bytes)), dim3(SORT_THREADS), 0, stream, ids, (int)N, V, padding, w.passes,
                               w.bits, pairs[0], clear, clear_bytes);
        };
        if (N <= SORT_THREADS) launch(std::integral_constant<int, 1>{});
        else launch(std::integral_constant<int, SORT_ITEMS>{});
        *sorted = pairs[0];
        return check_launch("nerf_embedding_bwd(sort)");
    }
    unsigned* table = reinterpret_cast<unsigned*>(work + w.table);
    const int mode = sort_mode(w.tiles);
    // The launches share the clearing of a large table, by the time that they take for themselves: a count one part, a scatter
    // two.  (50021 rows of 1024 bfloat16, 102 MB, 16384 ids, two passes: 38 us with all of it beside the first launch, 35 so.)
    const int parts = (mode == SORT_UNCOUNTED ? 2 : 3) * w.passes;
    const int64_t part = std::max<int64_t>((ceil_div(clear_bytes, parts) + 15) / 16 * 16, 8 << 20);
    int64_t cleared = 0;
    const auto share = [&](int n) {   // the next n parts to clear
        const int64_t bytes = std::min(n * part, clear_bytes - cleared);
        cleared += bytes;
        return bytes;
    };
    int from = 0;
    for (int p = 0; p < w.passes; ++p) {
        const int to = p == 0 ? 0 : 1 - from, shift = p * w.bits;
        const dim3 block(SORT_THREADS);
        const auto pass = [&](auto first, auto items) {
            constexpr bool FIRST = decltype(first)::value;
            constexpr int ITEMS = decltype(items)::value;
            char* at = clear + cleared;
            int64_t bytes = mode == SORT_UNCOUNTED ? 0 : share(1);
            if (mode != SORT_UNCOUNTED)
                hipLaunchKernelGGL((sort_count_kernel<ID, FIRST, ITEMS>), dim3((unsigned)w.tiles + clearing(bytes)), block, 0, stream, ids, (const uint2*)pairs[from], N, V, padding,
                                   shift, w.bits, NO_KEY, (int)w.tiles, table, at, bytes);
            if (mode == SORT_SUMMED)
                hipLaunchKernelGGL(sort_prefix_kernel, dim3((unsigned)ceil_div(1 << w.bits, 64)), block, 0, stream, table, (int)w.tiles, 1 << w.bits);
            at = clear + cleared;
            bytes = share(2);
            hipLaunchKernelGGL((sort_scatter_kernel<ID, FIRST, ITEMS>), dim3((unsigned)w.tiles + clearing(bytes)), block, 0, stream, ids, (const uint2*)pairs[from], N, V, padding,
                               shift, w.bits, table, (int)w.tiles, mode, pairs[to], at, bytes);
        };
        with_items(N, [&](auto items) {
            if (p == 0) pass(std::true_type{}, items);
            else pass(std::false_type{}, items);
        });
        if (int rc = check_launch("nerf_embedding_bwd(sort)")) return rc;
        from = to;
    }
    *sorted = pairs[from];
    return NERF_OK;
}

template <class T>
static int embedding_sums(const T* d_out, int64_t N, int64_t V, int D, const uint2* sorted, float scale, const EmbWork& w, char* work,
                          T* d_table, hipStream_t stream) {
    return with_vector<T>(D, [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        EmbSums p;
        p.sorted = sorted; p.N = N; p.V = V; p.D = D; p.scale = scale;
        p.l_lanes = lanes_log2(D / VEC);
        p.col_tiles = (int)ceil_div(D / VEC, 1 << p.l_lanes);
        p.l_chunk = chunk_log2(N, p.l_lanes, p.col_tiles);
        p.chunks = ceil_div(N, 1 << p.l_chunk);
        p.join_chunks = std::min(JOIN_CHUNKS, 2 * (JOIN_THREADS >> p.l_lanes));
        p.part = reinterpret_cast<float*>(work + w.part);
        const int64_t blocks = ceil_div(p.chunks * p.col_tiles, 4);
        NERF_REQUIRE(blocks < (1ll << 24), "nerf_embedding_bwd: too many workgroups");   // a launch holds fewer than 2^32 threads
        if (p.l_lanes == 6) hipLaunchKernelGGL((embedding_sums_kernel<T, VEC, true>), dim3((unsigned)blocks), dim3(256), 0, stream, p, d_out, d_table);
        else hipLaunchKernelGGL((embedding_sums_kernel<T, VEC, false>), dim3((unsigned)blocks), dim3(256), 0, stream, p, d_out, d_table);
        if (int rc = check_launch("nerf_embedding_bwd(sums)")) return rc;
        if (p.chunks <= 1) return NERF_OK;
        hipLaunchKernelGGL((embedding_join_kernel<T, VEC>), dim3((unsigned)ceil_div(p.chunks, p.join_chunks), (unsigned)p.col_tiles), dim3(JOIN_THREADS), 0, stream, p,
                           d_table);
        return check_launch("nerf_embedding_bwd(join)");
    });
}

template <class T, class ID>
static int embedding_narrow_bwd(const T* d_out, const ID* ids, int64_t N, int64_t V, int D, float scale, int64_t padding, char* work, T* d_table, hipStream_t stream) {
    return with_vector<T>(D, [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        const NarrowWork w = narrow_work(N, V, D);
        unsigned* const table = reinterpret_cast<unsigned*>(work + w.table);
        unsigned* const at = reinterpret_cast<unsigned*>(work + w.items);
        const BucketSums p{table + w.tiles * BUCKETS, at, reinterpret_cast<float*>(work + w.part), V, w.low, w.buckets, scale};
        const dim3 tiles((unsigned)w.tiles), block(SORT_THREADS);
        const int mode = sort_mode(w.tiles);
        with_items(N, [&](auto items) {
            constexpr int ITEMS = decltype(items)::value;
            if (mode != SORT_UNCOUNTED)
                hipLaunchKernelGGL((sort_count_kernel<ID, true, ITEMS>), tiles, block, 0, stream, ids, (const uint2*)nullptr, N, V, padding, w.low, BUCKET_BITS, (unsigned)V, (int)w.tiles,
                                   table, (char*)nullptr, int64_t(0));
            if (mode == SORT_SUMMED)
                hipLaunchKernelGGL(sort_prefix_kernel, dim3(BUCKETS / 64), block, 0, stream, table, (int)w.tiles, BUCKETS);
            hipLaunchKernelGGL((bucket_scatter_kernel<T, VEC, ID, ITEMS>), tiles, block, 0, stream, ids, N, V, padding, w.low, table, (int)w.tiles, mode, d_out, at);
        });
        if (int rc = check_launch("nerf_embedding_bwd(buckets)")) return rc;
        hipLaunchKernelGGL((bucket_sums_kernel<T, VEC>), dim3((unsigned)w.segments), dim3(BUCKET_THREADS), 0, stream, p, d_table);
        hipLaunchKernelGGL((bucket_join_kernel<T, VEC>), dim3((unsigned)w.buckets, (unsigned)ceil_div(1 << w.low, JOIN_IDS)), dim3(1024), 0, stream, p, d_table);
        return check_launch("nerf_embedding_bwd(bucket sums)");
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
    const size_t bytes = embedding_work(N, V, D).bytes;
    return embedding_narrow(N, V, D, 4) || embedding_narrow(N, V, D, 2) ? std::max(bytes, narrow_work(N, V, D).bytes) : bytes;
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
    const int64_t clear_bytes = V * D * (type == NERF_F32 ? 4 : 2);
    if (N == 0) {
        hipLaunchKernelGGL(clear_kernel, dim3((unsigned)std::min<int64_t>(1024, ceil_div(clear_bytes, 16384))), dim3(1024), 0, (hipStream_t)stream,
                           static_cast<char*>(d_table), clear_bytes);
        return check_launch(who);
    }
    char* const work = static_cast<char*>(workspace);
    if (embedding_narrow(N, V, D, type == NERF_F32 ? 4 : 2)) {
        return with_type(type, [&](auto t) {
            using T = decltype(t);
            if (ids_bytes == 8)
                return embedding_narrow_bwd(static_cast<const T*>(d_out), static_cast<const int64_t*>(ids), N, V, D, scale, padding_idx, work, static_cast<T*>(d_table), (hipStream_t)stream);
            return embedding_narrow_bwd(static_cast<const T*>(d_out), static_cast<const int32_t*>(ids), N, V, D, scale, padding_idx, work, static_cast<T*>(d_table), (hipStream_t)stream);
        });
    }
    const EmbWork w = embedding_work(N, V, D);
    char* const clear = static_cast<char*>(d_table);
    const uint2* sorted = nullptr;
    const int rc = ids_bytes == 8 ? embedding_sort(static_cast<const int64_t*>(ids), N, V, padding_idx, w, work, clear, clear_bytes, &sorted, (hipStream_t)stream)
                                  : embedding_sort(static_cast<const int32_t*>(ids), N, V, padding_idx, w, work, clear, clear_bytes, &sorted, (hipStream_t)stream);
    if (rc) return rc;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return embedding_sums(static_cast<const T*>(d_out), N, V, D, sorted, scale, w, work, static_cast<T*>(d_table), (hipStream_t)stream);
    });
}
