// Gated linear recurrence along a sequence or a ray, and its gradient, for gfx950.
//
//   h_i = a_i h_{i-1} + w_i x_i,   w_i = 1, or 1 - a_i ("blend": with the samples taken last to first this is
//   back-to-front alpha compositing of any number of channels, a_i = 1 - alpha_i).
//
// A stretch of steps acts on the state it is entered with as h -> A h + X (A the product of its gates), and two
// stretches compose, (A2 A1, A2 X1 + X2).  So every thread takes K consecutive steps of VEC channels into registers and
// forms (A, X) of them; a scan over the time slices of the group (lanes, then waves) gives each thread the state it
// starts from; and the thread replays its steps from there -- every output comes from the recurrence itself, only the
// states between slices from the composed form.  The state is held in float whatever the types of gate and x are.
//
// Gradient, with r_i what reaches h_i from the steps behind it: g_i = dh_i + r_i, r_{i-1} = a_i g_i, d x_i = w_i g_i,
// d a_i = g_i h_{i-1} (blend: g_i (h_{i-1} - x_i)), summed over the channels that share the gate.  r is the same kind of
// recurrence from the other end, with the same products A.  h is recomputed from x and the state the tile was entered
// with (kept in float by the forward pass): x costs the bytes that a saved h would, and h is not rounded on the way.
//
// Where there are few sequences and many steps the time axis is spread over workgroups as well, in one of two ways:
// segments, whose (A, X) a pass of its own finds first; or, with enough columns for it to keep the memory busy, tiles in a
// chain, each of which finds the state it is entered with from what the tiles in front of it (in the backward pass: behind
// it) have published: one pass over the data.
//
// Layout: x [B,T,C], gate [B,T,G]; the C/G = P channels of a gate are neighbours.  G = C: one "unit" of C columns per
// batch entry; G < C: one unit of P columns per (batch entry, gate).  A workgroup of 256 threads is cut into groups of
// CL x S threads: CL lanes side by side on the columns of a unit (VEC each), S slices of K steps.  Both passes are
// bound by memory: the forward pass moves gate + x + h once, the backward pass gate, x, dh in and d_gate, d_x out.  16384 rays
// x 192 x 32 float, one gate a step: 141 us for 818 MB and 240 for 1.23 GB, 5.8 and 5.1 TB/s, against 5.1 for a large copy.
#include <algorithm>

#include "typed.h"

namespace nerf {

// steps per thread, by the gates that a thread holds for a step
constexpr int scan_steps(int gates) { return gates > 1 ? 4 : 8; }
constexpr int SCAN_THREADS = 256;
constexpr int SCAN_COLS = 64;      // most columns of a unit that one workgroup takes side by side
constexpr int SCAN_CHANNELS = 1 << 17;   // most channels
// Workgroups to aim for along the time axis, in segments.  65536 x 64 float: 28 us, with 512 21, with 2048 27; x 128 bfloat16
// 28, 28 and 46, backward 37, 38 and 51; x 256 backward 62, 67 and 66.
constexpr int SCAN_WANT_BLOCKS = 1024;
constexpr int CHAIN_GROUP = 32;    // tiles of the chain between two published states
constexpr int CHAIN_BLOCKS = 8;    // fewest chains side by side

struct ScanShape {
    int64_t B, T;
    int C, G, P;            // channels, gates, channels per unit
    int units_per_b;        // 1 (a gate per channel) or G
    int vec, steps, lcl, ls;   // elements per lane, steps per thread, log2 of CL and of S
    int col_tiles;          // column tiles of a unit
    int64_t unit_tiles;     // B * units_per_b * col_tiles, below 2^32
    int64_t blocks;         // workgroups that hold them, below 2^24
    int tile_steps;         // S * K
    int64_t tiles;          // time tiles
    int64_t segments, seg_tiles;   // the time axis is cut into segments of seg_tiles tiles when there are few workgroups
};

static int log2_up(int64_t n) {
    int l = 0;
    while ((1ll << l) < n) ++l;
    return l;
}

// A function of the sizes alone: the backward pass finds the forward pass's tiles again.
static ScanShape scan_shape(int64_t B, int64_t T, int C, int G, int steps = 0) {
    ScanShape s;
    s.B = B; s.T = T; s.C = C; s.G = G;
    s.units_per_b = G == C ? 1 : G;
    s.P = C / s.units_per_b;
    // Two or three channels of a gate: a lane takes them all (65536 x 192 x 3 float, one gate a step: 78 us, a lane a channel 112,
    // backward 115 and 157; x 2 55 and 105), in dense pieces where it can (see scan_fwd_kernel).  Of another even number two (x 6 159 and 192; 39475 x 17 x 100 in ten gates 156
    // and 249; 4096 x 192 x 250 bfloat16 in five 288 and 296, backward 430 and 504).
    s.vec = s.P % 4 == 0 ? 4 : G != C && s.P <= 3 ? s.P : G != C && s.P % 2 == 0 ? 2 : 1;
    s.steps = steps ? steps : scan_steps(G == C ? s.vec : 1);
    s.lcl = log2_up(std::min<int64_t>(ceil_div(s.P, s.vec), SCAN_COLS / s.vec));
    s.ls = std::min(log2_up(ceil_div(T, s.steps)), 8 - s.lcl);
    s.col_tiles = (int)ceil_div(s.P, (int64_t)s.vec << s.lcl);
    s.unit_tiles = B * s.units_per_b * s.col_tiles;
    const int per_block = SCAN_THREADS >> (s.lcl + s.ls);
    s.blocks = ceil_div(s.unit_tiles, per_block);
    s.tile_steps = s.steps << s.ls;
    s.tiles = ceil_div(T, s.tile_steps);
    // few workgroups: cut the time axis (a second pass over gate and x, or gate and dh, finds the states between segments)
    const int64_t want = std::min<int64_t>(s.tiles, ceil_div(SCAN_WANT_BLOCKS, s.blocks));
    s.seg_tiles = ceil_div(s.tiles, std::max<int64_t>(1, want));
    s.segments = ceil_div(s.tiles, s.seg_tiles);
    return s;
}

// Steps per thread of the forward pass in a chain: long tiles, as many steps as the registers hold beside four workgroups on
// a compute unit -- 16 of 16 bits (65536 x 1024 bfloat16 111 us, with 8 129; 8 x 2048 x 1024 24 and 28; 65536 x 1024 with
// eight gates in float 68 and 89).
constexpr int CHAIN_STEPS = 8, CHAIN_STEPS_16BIT = 16;
// Whether the tiles of a pass form chains: a workgroup holds one tile of one chain, there are enough chains (a chain advances
// by a group of tiles in 2 to 4 us), and they are long enough to be worth clearing their words first.
// 65536 steps of bfloat16 with float32 gates, chain against segments: 1024 channels (16 chains) 141 against 179 us, 512 (8)
// 70 against 78, 256 (4) 42 against 43; 2048 of float32 347 against 526; 8 x 2048 x 1024 of bfloat16 24 against 32.  Backward
// (see there) 512 channels 133 against 131, 256 73 against 62.
static bool scan_chained(const ScanShape& s, int steps = CHAIN_STEPS) {
    return s.segments > 1 && s.lcl + s.ls == 8 && s.blocks >= CHAIN_BLOCKS && s.T >= 4ll * ((int64_t)steps << s.ls);
}

// What a chain's tiles publish, in 8-byte words of a value and a mark: per workgroup column block and tile the (A, X) of
// up to SCAN_COLS columns, per group of tiles the states it is entered with; and the next tile to take.
struct ChainWork {
    int64_t tickets, words, states, bytes;   // offsets
};
static ChainWork chain_work(const ScanShape& s) {
    ChainWork w;
    w.tickets = 0;
    w.words = 128 * s.blocks;
    w.states = w.words + s.blocks * s.tiles * (SCAN_COLS * 16);
    w.bytes = w.states + s.blocks * ceil_div(s.tiles, CHAIN_GROUP) * (SCAN_COLS * 8);
    return w;
}

struct ScanArgs {
    ScanShape s;
    const void* gate;
    const void* x;
    const float* state;    // [B,C] or null (zeros)
    int reverse, blend;
    void* h;
    float* last;           // [B,C] or null
    float* carry;          // [tiles - 1][B,C]: the state every tile (of the backward pass) but the first is entered with; null: not kept
    int l_carry;           // log2 of that tile's steps
    unsigned long long* chain_words;    // a chain's published (A, X), states and tickets
    unsigned long long* chain_states;
    unsigned* chain_tickets;
    float* agg;            // [2][segments][B,C]: A and X (backward: A and R) of the segments
    // backward
    const void* d_h;       // null: zeros
    const float* d_last;   // null: zeros
    void* d_gate;
    void* d_x;
    float* d_state;
    float* d_gate_part;    // [col_tiles][B,T,G] where a gate's channels take more than one column tile
};

// A h + X.  A state of exactly zero stays without effect however large the product of the gates has become.
__device__ __forceinline__ float scan_apply(float A, float h, float X) { return h == 0.0f ? X : fmaf(A, h, X); }

// Workgroup -> column block and segment, in 32 bits: a launch holds fewer than 2^24 workgroups.
__device__ __forceinline__ unsigned scan_segment(const ScanShape& s, unsigned& block) {
    block = blockIdx.x;
    if (s.segments == 1) return 0;
    const unsigned seg = blockIdx.x / (unsigned)s.blocks;
    block -= seg * (unsigned)s.blocks;
    return seg;
}

// Where a thread stands: its columns and its slice.
template <int VEC>
struct ScanPlace {
    int CL, S, SW, NW;          // lanes on columns, slices, slices of the group in one wave, waves of the group
    int c, sl, slw, lane, first_wave;
    bool on, in_unit;           // has columns; stands in a unit, with or without columns of it
    int64_t b;
    int j;                      // first column, in [0, C)
    int64_t g;                  // gate of a shared unit
    int64_t bc;                 // b * C + j
    int col_tile;
    // Where the workgroup's first unit lies, and how far from it the slice's first step does, in [B,T,C] and [B,T,G]
    // (elements; at most 2^30 bytes: 2048 rows of at most SCAN_CHANNELS channels, or 4096 of 16 bits).
    int64_t b0, j0, g0;
    unsigned x_off, g_off;

    __device__ __forceinline__ explicit ScanPlace(const ScanShape& s, unsigned block, int reverse) {
        const int tid = threadIdx.x;
        CL = 1 << s.lcl;
        S = 1 << s.ls;
        SW = min(S, 64 >> s.lcl);
        NW = S / SW;
        lane = tid & 63;
        c = tid & (CL - 1);
        sl = (tid >> s.lcl) & (S - 1);
        slw = sl & (SW - 1);
        const int q = tid >> (s.lcl + s.ls);
        first_wave = NW > 1 ? (tid >> 6) & ~(NW - 1) : 0;
        const unsigned ut = (unsigned)block * (SCAN_THREADS >> (s.lcl + s.ls)) + q;
        unsigned u = ut, in_b = 0;
        col_tile = 0;
        if (s.col_tiles > 1) {
            u = ut / (unsigned)s.col_tiles;
            col_tile = (int)(ut - u * s.col_tiles);
        }
        if (s.units_per_b > 1) {
            const unsigned all = u;
            u = all / (unsigned)s.units_per_b;
            in_b = all - u * s.units_per_b;
        }
        b = u;
        g = in_b;
        const unsigned ut0 = block * (SCAN_THREADS >> (s.lcl + s.ls)), u0 = s.col_tiles > 1 ? ut0 / (unsigned)s.col_tiles : ut0;
        b0 = s.units_per_b > 1 ? u0 / (unsigned)s.units_per_b : u0;
        g0 = s.units_per_b > 1 ? u0 - (unsigned)b0 * s.units_per_b : 0;
        j0 = g0 * s.P + (int64_t)(ut0 - u0 * s.col_tiles) * CL * VEC;
        const int col = (col_tile * CL + c) * VEC;
        in_unit = (int64_t)ut < s.unit_tiles;
        on = in_unit && col < s.P;
        j = (int)g * s.P + col;
        bc = b * s.C + j;
        const unsigned row = (unsigned)(b - b0) * (unsigned)s.T + (unsigned)(reverse ? (S - 1 - sl) * s.steps + s.steps - 1 : sl * s.steps);
        x_off = row * (unsigned)s.C + (unsigned)(j - (int)j0);
        g_off = s.G == s.C ? x_off : row * (unsigned)s.G + (unsigned)(g - g0);
    }
    // element that x_off (g_off) counts from, for a tile: its first row in memory
    __device__ __forceinline__ int64_t row0(const ScanShape& s, int64_t tile, int reverse) const {
        return b0 * s.T + (reverse ? s.T - (tile + 1) * s.tile_steps : tile * s.tile_steps);
    }
    __device__ __forceinline__ int64_t x0(const ScanShape& s, int64_t tile, int reverse) const { return row0(s, tile, reverse) * s.C + j0; }
    __device__ __forceinline__ int64_t gate0(const ScanShape& s, int64_t tile, int reverse) const {
        return s.G == s.C ? x0(s, tile, reverse) : row0(s, tile, reverse) * s.G + g0;
    }
    // place of step i (in the order of the recurrence) of this thread's columns in a [B,T,C] array / of its gate; from one
    // step to the next it moves by step(C) / step(G)
    __device__ __forceinline__ int64_t at(const ScanShape& s, int64_t i, int reverse) const {
        return (b * s.T + (reverse ? s.T - 1 - i : i)) * s.C + j;
    }
    __device__ __forceinline__ int64_t gate_at(const ScanShape& s, int64_t i, int reverse) const {
        // one gate for the unit, or the columns' own
        return s.G == s.C ? at(s, i, reverse) : (b * s.T + (reverse ? s.T - 1 - i : i)) * s.G + g;
    }
    // steps of the slice that starts at i0 and exist
    __device__ __forceinline__ int count(const ScanShape& s, int64_t i0) const {
        return !on || i0 >= s.T ? 0 : (int)min((int64_t)s.steps, s.T - i0);
    }
    __device__ __forceinline__ int count_in_unit(const ScanShape& s, int64_t i0) const {
        return !in_unit || i0 >= s.T ? 0 : (int)min((int64_t)s.steps, s.T - i0);
    }
};

// Reads from an address that is the same for all lanes on, at 32-bit offsets of the lanes' own, in bytes, below BUFFER_END.
// An offset of BUFFER_END or more reads zeros: steps that do not exist need no branch, and addresses no 64-bit arithmetic.
// (Writes go by ordinary addresses: after a 16-byte buffer store with an offset in a scalar register the compiler lets the
// stored registers be overwritten while they are still being read.)
constexpr unsigned BUFFER_END = 0x7fffffffu, BUFFER_NONE = 0x80000000u;
using Buffer = __amdgpu_buffer_rsrc_t;
__device__ __forceinline__ Buffer buffer(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)BUFFER_END, 4 << 15 | 7 << 12);   // 32-bit words
}
typedef unsigned Words2 __attribute__((ext_vector_type(2)));
typedef unsigned Words3 __attribute__((ext_vector_type(3)));
typedef unsigned Words4 __attribute__((ext_vector_type(4)));
// N elements of T as they lie in memory
template <class T, int N>
__device__ __forceinline__ void buffer_load(Buffer p, unsigned off, unsigned (&w)[(sizeof(T) * N + 3) / 4]) {
    constexpr int BYTES = sizeof(T) * N;
    if constexpr (BYTES == 2) {
        w[0] = __builtin_amdgcn_raw_buffer_load_b16(p, off, 0, 0);
    } else if constexpr (BYTES == 4) {
        w[0] = __builtin_amdgcn_raw_buffer_load_b32(p, off, 0, 0);
    } else if constexpr (BYTES == 6) {
        const unsigned lo = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(p, off, 0, 0), hi = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(p, off + 2, 0, 0);
        w[0] = lo | hi << 16;
        w[1] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(p, off + 4, 0, 0);
    } else if constexpr (BYTES == 8) {
        const Words2 q = __builtin_amdgcn_raw_buffer_load_b64(p, off, 0, 0);
        w[0] = q.x; w[1] = q.y;
    } else if constexpr (BYTES == 12) {
        const Words3 q = __builtin_amdgcn_raw_buffer_load_b96(p, off, 0, 0);
        w[0] = q.x; w[1] = q.y; w[2] = q.z;
    } else {
        static_assert(BYTES == 16, "");
        const Words4 q = __builtin_amdgcn_raw_buffer_load_b128(p, off, 0, 0);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    }
}
// K steps of the thread's columns as they lie in memory, in registers.  The conversion to float is done at each use: a
// value is used two or three times, and kept as it is it takes half the registers where its type has 16 bits.
template <class T, int N, int K>
struct Steps {
    static constexpr int WORDS = (sizeof(T) * N + 3) / 4;
    unsigned w[K][WORDS];
    __device__ __forceinline__ float operator()(int k, int v) const {
        if (N == 1) v = 0;   // one gate for all columns
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[k][v]);
        else return (float)__builtin_bit_cast(T, (unsigned short)(w[k][v / 2] >> (v & 1) * 16));
    }
    // `count` of the K steps exist; the others read `fill`.
    __device__ __forceinline__ void load(const T* __restrict__ p, int64_t step, int count, float fill) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Run<T, N> r;
#pragma unroll
            for (int v = 0; v < N; ++v) r.v[v] = (T)fill;
            if (k < count) r = *reinterpret_cast<const Run<T, N>*>(p + k * step);
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < WORDS; ++i) w[k][i] = __builtin_bit_cast(unsigned, r.v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < WORDS; ++i) {
                    w[k][i] = __builtin_bit_cast(unsigned short, r.v[2 * i]);
                    if (2 * i + 1 < N) w[k][i] |= (unsigned)__builtin_bit_cast(unsigned short, r.v[2 * i + 1 < N ? 2 * i + 1 : 0]) << 16;
                }
            }
        }
    }
    // The same through a buffer, the first step at off, the next ones `step` bytes on (modulo 2^32).
    __device__ __forceinline__ void load(Buffer p, unsigned off, unsigned step, int count, float fill) {
#pragma unroll
        for (int k = 0; k < K; ++k) buffer_load<T, N>(p, k < count ? off + k * step : BUFFER_NONE, w[k]);
        if (fill != 0.0f && count < K) {   // (zeros were read)
            unsigned bits;
            if constexpr (sizeof(T) == 4) bits = __float_as_uint(fill);
            else bits = 0x10001u * __builtin_bit_cast(unsigned short, (T)fill);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < WORDS; ++i) w[k][i] = k < count ? w[k][i] : bits;
        }
    }
    // All K steps where they are one piece of memory of K * N elements, from its lowest address, a multiple of 16 bytes.
    __device__ __forceinline__ void load_dense(const T* __restrict__ p, int reverse) {
        constexpr int ALL = K * N * sizeof(T) / 4;
        unsigned word[ALL];
#pragma unroll
        for (int i = 0; i < ALL; i += 4) {
            const uint4 q = *reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned*>(p) + i);
            word[i] = q.x; word[i + 1] = q.y; word[i + 2] = q.z; word[i + 3] = q.w;
        }
        const auto half = [&](int e) { return word[e / 2] >> (e & 1) * 16 & 0xffffu; };
        const auto take = [&](int k, int from) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                if constexpr (sizeof(T) == 4) {
                    w[k][i] = word[from * N + i];
                } else {
                    w[k][i] = half(from * N + 2 * i);
                    if (2 * i + 1 < N) w[k][i] |= half(from * N + 2 * i + 1) << 16;
                }
            }
        };
        if (reverse) {
#pragma unroll
            for (int k = 0; k < K; ++k) take(k, K - 1 - k);
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) take(k, k);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[k][i] = 0u;
    }
    // What was formed from the values so far is formed again from here on.  Without this the compiler keeps the products
    // of the first sweep over the steps for the second, which costs more in occupancy than the instructions it saves
    // (backward kernel, shared gate, float: 191 registers against 128).
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < WORDS; ++i) asm volatile("" : "+v"(w[k][i]));
    }
};

// The K steps' outputs as one piece of memory.
template <class T, int K, int N>
__device__ __forceinline__ void store_dense(T* __restrict__ p, int reverse, const float (&v)[K][N]) {
    const auto value = [&](int e) { return (T)(reverse ? v[K - 1 - e / N][e % N] : v[e / N][e % N]); };
    constexpr int ALL = K * N * sizeof(T) / 4;
    unsigned word[ALL];
#pragma unroll
    for (int i = 0; i < ALL; ++i) {
        if constexpr (sizeof(T) == 4) word[i] = __builtin_bit_cast(unsigned, value(i));
        else word[i] = __builtin_bit_cast(unsigned short, value(2 * i)) | (unsigned)__builtin_bit_cast(unsigned short, value(2 * i + 1)) << 16;
    }
#pragma unroll
    for (int i = 0; i < ALL; i += 4)
        *reinterpret_cast<uint4*>(reinterpret_cast<unsigned*>(p) + i) = uint4{word[i], word[i + 1], word[i + 2], word[i + 3]};
}

// Everywhere below: A [GV], one product for all VEC columns of a lane where they share a gate (GV = 1), else one each.
template <int GV>
__device__ __forceinline__ constexpr int scan_gate(int v) { return GV == 1 ? 0 : v; }

// The value of another lane, by its number; beyond the wave's ends it wraps, for lanes that do not use it.
__device__ __forceinline__ float lane_get(int lane, float v) {
    return __int_as_float(__builtin_amdgcn_ds_bpermute(lane << 2, __float_as_int(v)));
}

// Inclusive scan of (A, X) over the slices that the wave holds of the group; UP: from the first slice, else from the last.
template <bool UP, int VEC, int GV>
__device__ __forceinline__ void scan_wave(const ScanPlace<VEC>& w, float (&A)[GV], float (&X)[VEC]) {
    for (int d = 1; d < w.SW; d <<= 1) {
        const bool take = UP ? w.slw >= d : w.slw + d < w.SW;
        const int from = w.lane + (UP ? -d : d) * w.CL;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float px = lane_get(from, X[v]);
            if (take) X[v] = scan_apply(A[scan_gate<GV>(v)], px, X[v]);
        }
#pragma unroll
        for (int g = 0; g < GV; ++g) {
            const float pa = lane_get(from, A[g]);
            if (take) A[g] *= pa;
        }
    }
}

// The waves' own (A, X) where a group has several: s_a, s_x [waves][SCAN_COLS] of this exchange's own, written here and
// read behind the barrier.
template <bool UP, int VEC, int GV>
__device__ __forceinline__ void scan_exchange(const ScanPlace<VEC>& w, const float (&A)[GV], const float (&X)[VEC], float (*s_a)[SCAN_COLS], float (*s_x)[SCAN_COLS]) {
    if (w.NW == 1) return;
    if (w.slw == (UP ? w.SW - 1 : 0)) {   // its inclusive value is the wave's
#pragma unroll
        for (int g = 0; g < GV; ++g) s_a[threadIdx.x >> 6][w.c * VEC + g] = A[g];
#pragma unroll
        for (int v = 0; v < VEC; ++v) s_x[threadIdx.x >> 6][w.c * VEC + v] = X[v];
    }
    __syncthreads();
}

// From the inclusive wave scan (A, X), exchanged, and the state `carry` that the tile is entered with (the same in all
// slices of a column): `in` = the state this slice is entered with, `carry` = the state the tile is left with.
template <bool UP, int VEC, int GV>
__device__ __forceinline__ void scan_carry(const ScanPlace<VEC>& w, const float (&A)[GV], const float (&X)[VEC], float (&carry)[VEC], float (&in)[VEC],
                                           float (*s_a)[SCAN_COLS], float (*s_x)[SCAN_COLS]) {
    float from[VEC], pa[GV];
    if (w.NW > 1) {
        const int mine = (threadIdx.x >> 6) - w.first_wave;
#pragma unroll
        for (int v = 0; v < VEC; ++v) from[v] = carry[v];
#pragma unroll 1
        for (int n = 0; n < w.NW; ++n) {
            const int k = UP ? n : w.NW - 1 - n;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if (k == mine) from[v] = carry[v];
                carry[v] = scan_apply(s_a[w.first_wave + k][w.c * VEC + scan_gate<GV>(v)], carry[v], s_x[w.first_wave + k][w.c * VEC + v]);
            }
        }
    } else {
        const int last = (w.lane & ~(w.CL * w.SW - 1)) + (UP ? (w.SW - 1) * w.CL : 0) + w.c;
#pragma unroll
        for (int g = 0; g < GV; ++g) pa[g] = lane_get(last, A[g]);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            from[v] = carry[v];
            carry[v] = scan_apply(pa[scan_gate<GV>(v)], carry[v], lane_get(last, X[v]));
        }
    }
    const bool first = UP ? w.slw == 0 : w.slw == w.SW - 1;
    const int beside = w.lane + (UP ? -w.CL : w.CL);
#pragma unroll
    for (int g = 0; g < GV; ++g) pa[g] = lane_get(beside, A[g]);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        const float px = lane_get(beside, X[v]);
        in[v] = first ? from[v] : scan_apply(pa[scan_gate<GV>(v)], from[v], px);
    }
}

template <int VEC, int GV>
__device__ __forceinline__ void scan_identity(float (&A)[GV], float (&X)[VEC]) {
#pragma unroll
    for (int g = 0; g < GV; ++g) A[g] = 1.0f;
#pragma unroll
    for (int v = 0; v < VEC; ++v) X[v] = 0.0f;
}
// (A, X) <- first (A, X), then (A2, X2)
template <int VEC, int GV>
__device__ __forceinline__ void scan_append(float (&A)[GV], float (&X)[VEC], const float (&A2)[GV], const float (&X2)[VEC]) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) X[v] = scan_apply(A2[scan_gate<GV>(v)], X[v], X2[v]);
#pragma unroll
    for (int g = 0; g < GV; ++g) A[g] *= A2[g];
}

// The state a segment is entered with, from `carry` = what the recurrence starts from: the (A, X) of the segments in
// front of it (UP) or behind it, a stretch of them per slice, joined like the slices of a tile.
template <bool UP, int GV, int VEC>
__device__ __forceinline__ void scan_fold(const ScanArgs& p, const ScanPlace<VEC>& w, int64_t seg, float (*s_a)[SCAN_COLS], float (*s_x)[SCAN_COLS], float (&carry)[VEC]) {
    const int64_t first = UP ? 0 : seg + 1, n = UP ? seg : p.s.segments - 1 - seg, BC = p.s.B * p.s.C;
    if (n == 0) return;
    const int64_t per = (n + w.S - 1) >> p.s.ls, begin = w.sl * per, end = min(begin + per, n);
    float A[GV], X[VEC], in[VEC];
    scan_identity(A, X);
    if (w.on) {
#pragma unroll 4
        for (int64_t i = begin; i < end; ++i) {
            const int64_t k = first + (UP ? i : end - 1 - (i - begin));
            float A_k[GV], X_k[VEC];
            load_run<GV>(p.agg + k * BC + w.bc, A_k);   // (of the same value for all columns of a gate the first)
            load_run<VEC>(p.agg + (p.s.segments + k) * BC + w.bc, X_k);
            scan_append(A, X, A_k, X_k);
        }
    }
    scan_wave<UP>(w, A, X);
    scan_exchange<UP>(w, A, X, s_a, s_x);
    scan_carry<UP>(w, A, X, carry, in, s_a, s_x);
}

// APART: f(true_type) or f(false_type), one branch around a sweep over the steps; else f(blend != 0), a select per step --
// two sweeps take registers, which is dear where a thread holds many values (backward kernel, float, four columns of a
// shared gate: 306 us against 269 for 65536 x 192 x 8; one column gains, 52 us against 43 for x 1).
template <bool APART, class F>
__device__ __forceinline__ void by_blend(int blend, F&& f) {
    if (!APART) f(blend != 0);
    else if (blend) f(std::true_type{});
    else f(std::false_type{});
}
__device__ __forceinline__ float scan_step(bool blend, float a, float h, float x) { return fmaf(a, h, blend ? (1.0f - a) * x : x); }

// (A, X) of the thread's K steps; x is multiplied by its weight first if the recurrence blends.
template <int VEC, int K, class GT, int GV, class XT>
__device__ __forceinline__ void scan_local(const Steps<GT, GV, K>& a, const Steps<XT, VEC, K>& x, int blend, float (&A)[GV], float (&X)[VEC]) {
    scan_identity(A, X);
    by_blend<(K < 16)>(blend, [&](auto blends) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) X[v] = scan_step(blends, a(k, v), X[v], x(k, v));
#pragma unroll
            for (int g = 0; g < GV; ++g) A[g] *= a(k, g);
        }
    });
}
// (A, R) of the same steps from the other end: r_{i-1} = a_i (dh_i + r_i)
template <int VEC, int K, class GT, int GV, class XT>
__device__ __forceinline__ void scan_local_back(const Steps<GT, GV, K>& a, const Steps<XT, VEC, K>& dh, float (&A)[GV], float (&R)[VEC]) {
    scan_identity(A, R);
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) R[v] = a(k, v) * (dh(k, v) + R[v]);
#pragma unroll
        for (int g = 0; g < GV; ++g) A[g] *= a(k, g);
    }
}

// ---- chains -----------------------------------------------------------------------------------------------------
// The tiles of a chain are taken in order, by ticket, so that whatever a tile waits for belongs to tiles that have been
// taken before it and are running or done: the first tile of a chain that is not done waits for nothing, and every wait
// ends.  A tile publishes its (A, X); the last one of each group of CHAIN_GROUP publishes the state the next group is
// entered with; so a state is at most CHAIN_GROUP - 1 compositions, always the same ones in the same order, behind a
// published one, and the chain advances by groups and not by tiles.  A word carries its own mark beside the value: it is
// read until the mark is there, and no order between words is needed.
constexpr int CHAIN_PATIENCE = 1 << 20;   // reads of a word; a chain that is cut short by a fault elsewhere gives NaN and not a hang

__device__ __forceinline__ void chain_put(unsigned long long* p, float v) {
    __hip_atomic_store(p, 1ull << 32 | __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Every read of a word that is not there yet goes to memory: they are kept few.  SLEEP: units of 64 clocks between reads.
template <int N, int SLEEP>
__device__ __forceinline__ void chain_get(const unsigned long long* p, int stride, float (&v)[N]) {
    unsigned long long word[N];
#pragma unroll 1
    for (int spin = 0;; ++spin) {
        bool there = true;
#pragma unroll
        for (int i = 0; i < N; ++i) word[i] = __hip_atomic_load(p + i * stride, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int i = 0; i < N; ++i) there = there && word[i] >> 32;
        if (there) break;
        if (spin == CHAIN_PATIENCE) {
#pragma unroll
            for (int i = 0; i < N; ++i) word[i] = 0x7fc00000u;
            break;
        }
        __builtin_amdgcn_s_sleep(SLEEP);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float((unsigned)word[i]);
}

__device__ __forceinline__ int64_t chain_ticket(const ScanArgs& p, int64_t chain) {
    __shared__ unsigned s_ticket;
    if (threadIdx.x == 0) s_ticket = atomicAdd(p.chain_tickets + chain * 32, 1u);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane((int)s_ticket);   // the whole workgroup's: kept out of the vector registers
}

// Where a tile's words and its group's state lie.  Word i of a lane lies i * CL words on, so that the lanes of a slice read
// and write whole lines: nothing of this is kept in a cache, and every line touched is a transfer of its own.
template <int VEC>
struct ChainPlace {
    int64_t group;
    int k;                        // place in the group
    unsigned long long *words;    // of the group's first tile
    unsigned long long *states;
    __device__ __forceinline__ ChainPlace(const ScanArgs& p, const ScanPlace<VEC>& w, int64_t chain, int64_t order) {
        group = order / CHAIN_GROUP;
        k = (int)(order % CHAIN_GROUP);
        words = p.chain_words + (chain * p.s.tiles + group * CHAIN_GROUP) * (2 * SCAN_COLS) + w.c;
        states = p.chain_states + (chain * ((p.s.tiles + CHAIN_GROUP - 1) / CHAIN_GROUP) + group) * SCAN_COLS + w.c;
    }
};

// Publishes the (A, X) of the order-th tile of the chain.  The waves' have been exchanged through s_a and s_x.
template <int GV, bool UP, int VEC>
__device__ __forceinline__ void chain_publish(const ScanArgs& p, const ScanPlace<VEC>& w, int64_t chain, int64_t order, float (*s_a)[SCAN_COLS], float (*s_x)[SCAN_COLS]) {
    const ChainPlace<VEC> at(p, w, chain, order);
    if (w.sl != 0 || at.k == CHAIN_GROUP - 1) return;
    float A[GV], X[VEC];
    scan_identity(A, X);
    for (int i = 0; i < w.NW; ++i) {
        const int n = UP ? i : w.NW - 1 - i;
        float A_n[GV], X_n[VEC];
#pragma unroll
        for (int g = 0; g < GV; ++g) A_n[g] = s_a[n][w.c * VEC + g];
#pragma unroll
        for (int v = 0; v < VEC; ++v) X_n[v] = s_x[n][w.c * VEC + v];
        scan_append(A, X, A_n, X_n);
    }
    unsigned long long* const to = at.words + at.k * (2 * SCAN_COLS);
#pragma unroll
    for (int g = 0; g < GV; ++g) chain_put(to + g * w.CL, A[g]);
#pragma unroll
    for (int v = 0; v < VEC; ++v) chain_put(to + (GV + v) * w.CL, X[v]);
}

// `state`: what the recurrence starts from -> what this tile is entered with.  s_part is [CHAIN_GROUP][2][SCAN_COLS].
// Everything that can be composed without the group's state is composed before it is waited for, and the last tile of a
// group hands the next group's state on as soon as it has its own: between two groups lie a read, a product and a write.
template <int GV, bool UP, int VEC>
__device__ __forceinline__ void chain_state(const ScanArgs& p, const ScanPlace<VEC>& w, int64_t chain, int64_t order, float (*s_a)[SCAN_COLS], float (*s_x)[SCAN_COLS],
                                            float (*s_part)[2][SCAN_COLS], float (&state)[VEC]) {
    const ChainPlace<VEC> at(p, w, chain, order);
    const int k = at.k, col = w.c * VEC;
    const bool hands_on = w.sl == w.S - 1 && k == CHAIN_GROUP - 1 && order + 1 < p.s.tiles;
#pragma unroll 1
    for (int q = w.sl; q < k; q += w.S) {
        float ax[GV + VEC];
        chain_get<GV + VEC, 8>(at.words + q * (2 * SCAN_COLS), w.CL, ax);
#pragma unroll
        for (int g = 0; g < GV; ++g) s_part[q][0][col + g] = ax[g];
#pragma unroll
        for (int v = 0; v < VEC; ++v) s_part[q][1][col + v] = ax[GV + v];
    }
    __syncthreads();
    float A[GV], X[VEC];
    const auto append = [&](const float* a_n, const float* x_n) {
        float A_n[GV], X_n[VEC];
#pragma unroll
        for (int g = 0; g < GV; ++g) A_n[g] = a_n[col + g];
#pragma unroll
        for (int v = 0; v < VEC; ++v) X_n[v] = x_n[col + v];
        scan_append(A, X, A_n, X_n);
    };
    scan_identity(A, X);
#pragma unroll 2
    for (int q = 0; q < k; ++q) append(s_part[q][0], s_part[q][1]);
    float A_in[GV], X_in[VEC];
#pragma unroll
    for (int g = 0; g < GV; ++g) A_in[g] = A[g];
#pragma unroll
    for (int v = 0; v < VEC; ++v) X_in[v] = X[v];
    if (hands_on) {   // this tile too
#pragma unroll 1
        for (int i = 0; i < w.NW; ++i) append(s_a[UP ? i : w.NW - 1 - i], s_x[UP ? i : w.NW - 1 - i]);
    }
    const auto hand_on = [&](const float (&h)[VEC]) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) chain_put(at.states + SCAN_COLS + v * w.CL, scan_apply(A[scan_gate<GV>(v)], h[v], X[v]));
    };
    if (at.group > 0) {
        if (w.sl == w.S - 1) {   // the slice that has the fewest tiles to wait for
            float h[VEC];
            if (!hands_on && w.c == 0) {   // one lane waits
                float first[1];
                chain_get<1, 4>(at.states, 0, first);
            }
            chain_get<VEC, 1>(at.states, w.CL, h);
            if (hands_on) hand_on(h);
#pragma unroll
            for (int v = 0; v < VEC; ++v) s_part[CHAIN_GROUP - 1][0][col + v] = h[v];
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; ++v) state[v] = s_part[CHAIN_GROUP - 1][0][col + v];
    } else if (hands_on) {
        hand_on(state);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) state[v] = scan_apply(A_in[scan_gate<GV>(v)], state[v], X_in[v]);
}

// (A, X) of whole segments -- all but the last one -- or, BACK, (A, R) of all but the first.  Nothing is written per step,
// so a slice takes one stretch of the segment and goes through it alone; the slices are joined once at the end.
// Bound by the reads (65536 x 1024 bfloat16 with float32 gates: 402 MB at 4.5 TB/s, what reads alone reach here).
template <class GT, class XT, int VEC, int GV, bool BACK>
__global__ __launch_bounds__(SCAN_THREADS) void scan_segments_kernel(ScanArgs p) {
    constexpr int K = scan_steps(GV);
    __shared__ float s_a[4][SCAN_COLS], s_x[4][SCAN_COLS];
    const ScanShape& s = p.s;
    unsigned block;
    const int64_t seg = scan_segment(s, block) + (BACK ? 1 : 0);
    const ScanPlace<VEC> w(s, block, p.reverse);
    const int64_t rounds = min(s.seg_tiles, s.tiles - seg * s.seg_tiles);
    const int64_t begin = seg * s.seg_tiles * s.tile_steps + w.sl * rounds * K;   // of the slice's stretch
    const int64_t x_step = p.reverse ? -(int64_t)s.C : s.C, gate_step = p.reverse ? -(int64_t)s.G : s.G;
    float A[GV], X[VEC];
    scan_identity(A, X);
    Steps<GT, GV, K> a, a_next;
    Steps<XT, VEC, K> x, x_next;
    const auto fetch = [&](int64_t n, Steps<GT, GV, K>& to_a, Steps<XT, VEC, K>& to_x) {
        const int64_t i0 = begin + (BACK ? rounds - 1 - n : n) * K;
        const int count = w.count(s, i0);
        to_a.load(static_cast<const GT*>(p.gate) + w.gate_at(s, i0, p.reverse), gate_step, count, 1.0f);   // a stretch may be long: whole addresses
        if (BACK && !p.d_h) to_x.clear();
        else to_x.load(static_cast<const XT*>(BACK ? p.d_h : p.x) + w.at(s, i0, p.reverse), x_step, count, 0.0f);
    };
    fetch(0, a_next, x_next);
    for (int64_t n = 0; n < rounds; ++n) {
        a = a_next;
        x = x_next;
        if (n + 1 < rounds) fetch(n + 1, a_next, x_next);   // under way while these steps are summed
        float A_now[GV], X_now[VEC];
        if (BACK) scan_local_back(a, x, A_now, X_now);
        else scan_local(a, x, p.blend, A_now, X_now);
        scan_append(A, X, A_now, X_now);
    }
    scan_wave<!BACK>(w, A, X);   // the last slice (BACK: the first) of a wave holds the wave's
    const auto write = [&] {
        const int64_t BC = s.B * s.C;
        float A_all[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) A_all[v] = A[scan_gate<GV>(v)];
        store_run<VEC>(p.agg + seg * BC + w.bc, A_all);
        store_run<VEC>(p.agg + (s.segments + seg) * BC + w.bc, X);
    };
    if (w.NW == 1) {
        if (w.on && w.slw == (BACK ? 0 : w.SW - 1)) write();
        return;
    }
    scan_exchange<!BACK>(w, A, X, s_a, s_x);
    if (w.on && w.sl == 0) {
        scan_identity(A, X);
        for (int k = 0; k < w.NW; ++k) {
            const int from = w.first_wave + (BACK ? w.NW - 1 - k : k);
            float A_k[GV], X_k[VEC];
#pragma unroll
            for (int g = 0; g < GV; ++g) A_k[g] = s_a[from][w.c * VEC + g];
#pragma unroll
            for (int v = 0; v < VEC; ++v) X_k[v] = s_x[from][w.c * VEC + v];
            scan_append(A, X, A_k, X_k);
        }
        write();
    }
}

// Whether a kernel reads through buffers: with four columns to a lane (16384 x 192 x 32 bfloat16, one gate a step, backward:
// 164 us, by ordinary addresses 250).  With one column lanes without any still make their requests: 65536 x 192 x 5 float took
// 245 us so against 198 forward and 429 against 377 backward, 65536 x 64 x 4 in dense pieces 50 against 47 backward.
template <int VEC, bool DENSE>
constexpr bool scan_buffers() { return VEC == 4 && !DENSE; }

// DENSE: a lane has all channels of a sequence and its steps are one piece of memory (few channels, the rays of a picture):
// they move 16 bytes at a time.  65536 rays x 192 x 3 float: 78 us, step by step (193 samples) 103; x 2 55 and 93, x 1 26 and
// 70.  (Backward 115 and 179, 80 and 144, 47 and 122.)
template <class GT, class XT, int VEC, int GV, int K, bool CHAIN, bool DENSE>
__global__ __launch_bounds__(SCAN_THREADS, CHAIN ? 4 : 1) void scan_fwd_kernel(ScanArgs p) {
    __shared__ float s_a[2][4][SCAN_COLS], s_x[2][4][SCAN_COLS], s_part[CHAIN ? CHAIN_GROUP : 1][2][SCAN_COLS];
    const ScanShape& s = p.s;
    unsigned block;
    const int64_t BC = s.B * s.C, segment = scan_segment(s, block), seg = CHAIN ? chain_ticket(p, block) : segment;
    const ScanPlace<VEC> w(s, block, p.reverse);
    const int64_t t_begin = CHAIN ? seg : seg * s.seg_tiles, t_end = CHAIN ? seg + 1 : min(t_begin + s.seg_tiles, s.tiles);
    float carry[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = 0.0f;
    if (w.on) {
        if (p.state) load_run<VEC>(p.state + w.bc, carry);
    }
    if (!CHAIN) scan_fold<true, GV>(p, w, seg, s_a[~t_begin & 1], s_x[~t_begin & 1], carry);
    const int64_t x_step = p.reverse ? -(int64_t)s.C : s.C, gate_step = p.reverse ? -(int64_t)s.G : s.G;
    const int64_t low = p.reverse ? K - 1 : 0;   // rows from a slice's first step to the one that lies first in memory
    Steps<GT, GV, K> a, a_next;
    Steps<XT, VEC, K> x, x_next;
    const auto fetch = [&](int64_t tile, Steps<GT, GV, K>& to_a, Steps<XT, VEC, K>& to_x) {
        const int64_t i0 = tile * s.tile_steps + w.sl * K;
        const int count = tile < t_end ? w.count(s, i0) : 0;
        if constexpr (scan_buffers<VEC, DENSE>()) {
            to_a.load(buffer(static_cast<const GT*>(p.gate) + w.gate0(s, tile, p.reverse)), w.g_off * sizeof(GT), (unsigned)gate_step * sizeof(GT), count, 1.0f);
            to_x.load(buffer(static_cast<const XT*>(p.x) + w.x0(s, tile, p.reverse)), w.x_off * sizeof(XT), (unsigned)x_step * sizeof(XT), count, 0.0f);
        } else {
            const GT* __restrict__ gate_from = static_cast<const GT*>(p.gate) + w.gate_at(s, i0, p.reverse);
            const XT* __restrict__ x_from = static_cast<const XT*>(p.x) + w.at(s, i0, p.reverse);
            if constexpr (DENSE) {
                if (count == K) {
                    to_a.load_dense(gate_from - low * s.G, p.reverse);
                    to_x.load_dense(x_from - low * s.C, p.reverse);
                    return;
                }
            }
            to_a.load(gate_from, gate_step, count, 1.0f);
            to_x.load(x_from, x_step, count, 0.0f);
        }
    };
    // the next tile is under way while this one is scanned -- where a thread holds few steps: with a shared gate it holds
    // twice as many, and the registers are worth more as a fourth workgroup on the compute unit
    constexpr bool AHEAD = GV > 1 && !CHAIN;
    if (AHEAD) fetch(t_begin, a_next, x_next);
    for (int64_t tile = t_begin; tile < t_end; ++tile) {
        if (AHEAD) {
            a = a_next;
            x = x_next;
            if (tile + 1 < t_end) fetch(tile + 1, a_next, x_next);
        } else {
            fetch(tile, a, x);
        }
        const int64_t i0 = tile * s.tile_steps + w.sl * K;
        const int count = w.count(s, i0);
        float A[GV], X[VEC], h[VEC];
        scan_local(a, x, p.blend, A, X);
        scan_wave<true>(w, A, X);
        scan_exchange<true>(w, A, X, s_a[tile & 1], s_x[tile & 1]);
        if (CHAIN) {
            chain_publish<GV, true>(p, w, block, tile, s_a[tile & 1], s_x[tile & 1]);
            chain_state<GV, true>(p, w, block, tile, s_a[tile & 1], s_x[tile & 1], s_part, carry);
        }
        scan_carry<true>(w, A, X, carry, h, s_a[tile & 1], s_x[tile & 1]);
        if (p.carry && count > 0 && i0 > 0 && (i0 & ((1 << p.l_carry) - 1)) == 0) store_run<VEC>(p.carry + ((i0 >> p.l_carry) - 1) * BC + w.bc, h);
        a.forget();
        x.forget();
        XT* __restrict__ out = static_cast<XT*>(p.h) + w.at(s, i0, p.reverse);
        float piece[DENSE ? K : 1][VEC];
        by_blend<(K < 16)>(p.blend, [&](auto blends) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    h[v] = scan_step(blends, a(k, v), h[v], x(k, v));
                    if (DENSE) piece[DENSE ? k : 0][v] = h[v];
                }
                if (!DENSE && k < count) store_run<VEC>(out + k * x_step, h);
            }
        });
        if constexpr (DENSE) {
            if (count == K) {
                store_dense(out - low * s.C, p.reverse, piece);
            } else {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (k < count) store_run<VEC>(out + k * x_step, piece[k]);
            }
        }
    }
    if (p.last && t_end == s.tiles && w.on && w.sl == 0) store_run<VEC>(p.last + w.bc, carry);
}

// Sums of the K steps' values over the CL lanes of a slice, and their place in the gate's gradient.  While there are
// several values to a lane, neighbours split them: each hands half of its values on and adds what it is handed -- 7
// exchanges for 8 values over 8 lanes instead of 24.
template <class GT, int VEC, int K>
__device__ __forceinline__ void scan_gate_sums(const ScanArgs& p, const ScanPlace<VEC>& w, float (&sum)[K][1], int count, GT* __restrict__ da_out, int64_t gate_at,
                                               int64_t gate_step) {
    static_assert(K == 8, "three halvings");
    int first = 0, d = 1;   // the lane's values are of the steps first, first + 1, ...
#pragma unroll
    for (int n = K / 2; n > 0; n >>= 1) {
        if (d < w.CL) {
            const bool upper = w.c & d;
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const float give = upper ? sum[j][0] : sum[j + n][0], keep = upper ? sum[j + n][0] : sum[j][0];
                sum[j][0] = keep + lane_get(w.lane ^ d, give);
            }
            first += upper ? n : 0;
            d <<= 1;
        }
    }
    const int held = K / d;
    bool writes = true;
    for (; d < w.CL; d <<= 1) {
        sum[0][0] += lane_get(w.lane ^ d, sum[0][0]);
        writes = writes && !(w.c & d);
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const int k = first + j;
        if (j < held && writes && k < count) {
            if (p.s.col_tiles == 1) da_out[k * gate_step] = (GT)sum[j][0];
            else p.d_gate_part[(int64_t)w.col_tile * p.s.B * p.s.T * p.s.G + gate_at + k * gate_step] = sum[j][0];
        }
    }
}

// CHAIN: the stretch from the other end is formed and published before the states from the front are scanned, which then
// goes on while the other tiles' stretches arrive (published behind it: 283 us against 246 for 65536 x 1024 bfloat16 with
// float32 gates, 281 in segments; 2048 of float32 622, 576 and 772; 8 x 16384 x 512 bfloat16, eight gates, 127, 124 and 142).
template <class GT, class XT, int VEC, int GV, bool CHAIN, bool DENSE>
__global__ __launch_bounds__(SCAN_THREADS, CHAIN ? 4 : 1) void scan_bwd_kernel(ScanArgs p) {
    constexpr int K = scan_steps(GV);
    __shared__ float s_a[2][4][SCAN_COLS], s_x[2][4][SCAN_COLS], s_b[2][4][SCAN_COLS], s_r[2][4][SCAN_COLS],
        s_part[CHAIN ? CHAIN_GROUP : 1][2][SCAN_COLS];
    const ScanShape& s = p.s;
    unsigned block;
    const int64_t BC = s.B * s.C, segment = scan_segment(s, block), order = CHAIN ? chain_ticket(p, block) : 0, seg = CHAIN ? s.tiles - 1 - order : segment;
    const ScanPlace<VEC> w(s, block, p.reverse);
    const int64_t t_begin = CHAIN ? seg : seg * s.seg_tiles, t_end = CHAIN ? seg + 1 : min(t_begin + s.seg_tiles, s.tiles);
    const bool shared_gate = s.G != s.C;
    float r_carry[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) r_carry[v] = 0.0f;
    if (w.on) {
        if (p.d_last) load_run<VEC>(p.d_last + w.bc, r_carry);
    }
    if (!CHAIN) scan_fold<false, GV>(p, w, seg, s_b[t_end & 1], s_r[t_end & 1], r_carry);
    const int64_t x_step = p.reverse ? -(int64_t)s.C : s.C, gate_step = p.reverse ? -(int64_t)s.G : s.G;
    const int64_t low = p.reverse ? K - 1 : 0;
    // (the next tile under way as in the forward pass was slower here: 151 registers against 119, 240 us against 215 for a
    // bfloat16 sequence of 65536 x 1024)
    for (int64_t tile = t_end - 1; tile >= t_begin; --tile) {
        const int64_t i0 = tile * s.tile_steps + w.sl * K, at = w.at(s, i0, p.reverse), gate_at = w.gate_at(s, i0, p.reverse);
        const int count = w.count(s, i0);
        Steps<GT, GV, K> a;
        Steps<XT, VEC, K> x, dh;
        float A[GV], X[VEC], h[VEC], r[VEC], carry[VEC];
        const bool whole = DENSE && count == K;
        if constexpr (scan_buffers<VEC, DENSE>()) {
            const int64_t x0 = w.x0(s, tile, p.reverse);
            const unsigned x_next = (unsigned)x_step * sizeof(XT);
            a.load(buffer(static_cast<const GT*>(p.gate) + w.gate0(s, tile, p.reverse)), w.g_off * sizeof(GT), (unsigned)gate_step * sizeof(GT), count, 1.0f);
            x.load(buffer(static_cast<const XT*>(p.x) + x0), w.x_off * sizeof(XT), x_next, count, 0.0f);
            if (p.d_h) dh.load(buffer(static_cast<const XT*>(p.d_h) + x0), w.x_off * sizeof(XT), x_next, count, 0.0f);
            else dh.clear();
        } else {
            const GT* __restrict__ gate_from = static_cast<const GT*>(p.gate) + gate_at;
            const XT* __restrict__ x_from = static_cast<const XT*>(p.x) + at;
            const XT* __restrict__ dh_from = static_cast<const XT*>(p.d_h) + at;
            if constexpr (DENSE) {
                if (whole) {
                    a.load_dense(gate_from - low * s.G, p.reverse);
                    x.load_dense(x_from - low * s.C, p.reverse);
                    if (p.d_h) dh.load_dense(dh_from - low * s.C, p.reverse);
                    else dh.clear();
                }
            }
            if (!whole) {
                a.load(gate_from, gate_step, count, 1.0f);
                x.load(x_from, x_step, count, 0.0f);
                if (p.d_h) dh.load(dh_from, x_step, count, 0.0f);
                else dh.clear();
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) carry[v] = 0.0f;
        if (w.on) {
            if (tile > 0) load_run<VEC>(p.carry + (tile - 1) * BC + w.bc, carry);
            else if (p.state) load_run<VEC>(p.state + w.bc, carry);
        }
        const auto back = [&](float (&A_b)[GV], float (&R)[VEC]) {   // the tile's stretch from the other end
            scan_local_back(a, dh, A_b, R);
            scan_wave<false>(w, A_b, R);
            scan_exchange<false>(w, A_b, R, s_b[tile & 1], s_r[tile & 1]);
        };
        float A_b[GV], R[VEC];
        if (CHAIN) {   // others wait for it: first of all
            back(A_b, R);
            chain_publish<GV, false>(p, w, block, order, s_b[tile & 1], s_r[tile & 1]);
            a.forget();
        }
        scan_local(a, x, p.blend, A, X);
        scan_wave<true>(w, A, X);
        scan_exchange<true>(w, A, X, s_a[tile & 1], s_x[tile & 1]);
        scan_carry<true>(w, A, X, carry, h, s_a[tile & 1], s_x[tile & 1]);
        a.forget();
        if (CHAIN) chain_state<GV, false>(p, w, block, order, s_b[tile & 1], s_r[tile & 1], s_part, r_carry);
        else back(A_b, R);
        scan_carry<false>(w, A_b, R, r_carry, r, s_b[tile & 1], s_r[tile & 1]);
        a.forget();
        x.forget();
        dh.forget();
        XT* __restrict__ dx_out = static_cast<XT*>(p.d_x) + at;
        GT* __restrict__ da_out = static_cast<GT*>(p.d_gate) + gate_at;
        float dx_piece[DENSE ? K : 1][VEC], da_sum[K][1];
        by_blend<VEC == 1>(p.blend, [&](auto blends) {
            const bool blend = blends;
            float beside[K][VEC];   // what multiplies g in the gradient of the gate
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    beside[k][v] = blend ? h[v] - x(k, v) : h[v];
                    h[v] = scan_step(blend, a(k, v), h[v], x(k, v));
                }
#pragma unroll
            for (int k = K - 1; k >= 0; --k) {
                float da[VEC], dx[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float ak = a(k, v), g = dh(k, v) + r[v];
                    da[v] = g * beside[k][v];
                    dx[v] = blend ? (1.0f - ak) * g : g;
                    r[v] = ak * g;
                    if (DENSE) dx_piece[DENSE ? k : 0][v] = dx[v];
                }
                if (!DENSE && p.d_x && k < count) store_run<VEC>(dx_out + k * x_step, dx);
                da_sum[k][0] = da[0];
                if (GV == 1) {
#pragma unroll
                    for (int v = 1; v < VEC; ++v) da_sum[k][0] += da[v];
                } else if (p.d_gate && k < count) {
                    store_run<VEC>(da_out + k * gate_step, da);
                }
            }
        });
        if constexpr (DENSE) {
            if (whole) {
                if (p.d_x) store_dense(dx_out - low * s.C, p.reverse, dx_piece);
                if (p.d_gate) store_dense(da_out - low * s.G, p.reverse, da_sum);
            } else {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (p.d_x && k < count) store_run<VEC>(dx_out + k * x_step, dx_piece[k]);
            }
        }
        if constexpr (GV == 1) {
            if (whole || !p.d_gate) continue;
            if (!shared_gate) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (k < count) da_out[k * gate_step] = (GT)da_sum[k][0];
            } else {
                scan_gate_sums(p, w, da_sum, w.count_in_unit(s, i0), da_out, gate_at, gate_step);   // lanes without columns write too
            }
        }
    }
    if (p.d_state && t_begin == 0 && w.on && w.sl == 0) store_run<VEC>(p.d_state + w.bc, r_carry);
}

// ---- one step ------------------------------------------------------------------------------------------------------
// A single step (the next token of every sequence) is element by element, whatever the channels divide into: four of them a
// thread, the gate of element i of [B,C] at i / P.  Bound by memory, small calls by the launch: 64 x 2048 bfloat16 with state
// 2.7 us, as tiles 4.2; 65536 x 1023 float 137 and 460 (5.9 TB/s), x 100 in ten gates 10 and 73, x 256 backward 67 and 79.
constexpr int ONE_ELEMENTS = 4;

template <class GT, class XT>
__global__ __launch_bounds__(SCAN_THREADS) void scan_one_fwd_kernel(ScanArgs p) {
    constexpr int N = ONE_ELEMENTS;
    const unsigned n = (unsigned)(p.s.B * p.s.C), i = (blockIdx.x * SCAN_THREADS + threadIdx.x) * N;
    if (i >= n) return;
    const GT* __restrict__ gate = static_cast<const GT*>(p.gate);
    const XT* __restrict__ x = static_cast<const XT*>(p.x);
    XT* __restrict__ out = static_cast<XT*>(p.h);
    const unsigned P = p.s.G == p.s.C ? 1u : (unsigned)p.s.P;
    if (i + N <= n) {
        float a[N], v[N], h[N] = {};
        load_run<N>(x + i, v);
        if (p.state) load_run<N>(p.state + i, h);
        if (P == 1) {
            load_run<N>(gate + i, a);
        } else {
            unsigned q = i / P, r = i - q * P;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                a[k] = (float)gate[q];
                if (++r == P) {
                    r = 0;
                    ++q;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) h[k] = scan_step(p.blend != 0, a[k], h[k], v[k]);
        store_run<N>(out + i, h);
        if (p.last) store_run<N>(p.last + i, h);
    } else {
        for (unsigned e = i; e < n; ++e) {
            const float h = scan_step(p.blend != 0, (float)gate[e / P], p.state ? p.state[e] : 0.0f, (float)x[e]);
            out[e] = (XT)h;
            if (p.last) p.last[e] = h;
        }
    }
}

// A gate for each channel.
template <class GT, class XT>
__global__ __launch_bounds__(SCAN_THREADS) void scan_one_bwd_kernel(ScanArgs p) {
    constexpr int N = ONE_ELEMENTS;
    const unsigned n = (unsigned)(p.s.B * p.s.C), i = (blockIdx.x * SCAN_THREADS + threadIdx.x) * N;
    if (i >= n) return;
    const GT* __restrict__ gate = static_cast<const GT*>(p.gate);
    const XT* __restrict__ x = static_cast<const XT*>(p.x);
    const XT* __restrict__ d_h = static_cast<const XT*>(p.d_h);
    const auto gradients = [&](float a, float v, float h, float g, float& da, float& dx, float& ds) {
        da = g * (p.blend ? h - v : h);
        dx = p.blend ? (1.0f - a) * g : g;
        ds = a * g;
    };
    if (i + N <= n) {
        float a[N], v[N], h[N] = {}, g[N] = {}, r[N] = {}, da[N], dx[N], ds[N];
        load_run<N>(gate + i, a);
        load_run<N>(x + i, v);
        if (p.state) load_run<N>(p.state + i, h);
        if (d_h) load_run<N>(d_h + i, g);
        if (p.d_last) load_run<N>(p.d_last + i, r);
#pragma unroll
        for (int k = 0; k < N; ++k) gradients(a[k], v[k], h[k], g[k] + r[k], da[k], dx[k], ds[k]);
        if (p.d_gate) store_run<N>(static_cast<GT*>(p.d_gate) + i, da);
        if (p.d_x) store_run<N>(static_cast<XT*>(p.d_x) + i, dx);
        if (p.d_state) store_run<N>(p.d_state + i, ds);
    } else {
        for (unsigned e = i; e < n; ++e) {
            float da, dx, ds;
            gradients((float)gate[e], (float)x[e], p.state ? p.state[e] : 0.0f, (d_h ? (float)d_h[e] : 0.0f) + (p.d_last ? p.d_last[e] : 0.0f), da, dx, ds);
            if (p.d_gate) static_cast<GT*>(p.d_gate)[e] = (GT)da;
            if (p.d_x) static_cast<XT*>(p.d_x)[e] = (XT)dx;
            if (p.d_state) p.d_state[e] = ds;
        }
    }
}

// d_gate = the sum over the column tiles, in their order
template <class GT>
__global__ __launch_bounds__(256) void scan_gate_sum_kernel(const float* __restrict__ part, int col_tiles, int64_t n, GT* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float sum = 0.0f;
    for (int k = 0; k < col_tiles; ++k) sum += part[(int64_t)k * n + i];
    out[i] = (GT)sum;
}

enum { SCAN_FWD, SCAN_BWD };

__global__ __launch_bounds__(256) void chain_clear_kernel(uint4* __restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = uint4{0u, 0u, 0u, 0u};
}

template <class GT, class XT, int VEC, int GV, int K, bool BACK = false>
static int scan_chain_launch(ScanArgs p, const char* who, hipStream_t stream) {
    p.s = scan_shape(p.s.B, p.s.T, p.s.C, p.s.G, K);
    const ChainWork work = chain_work(p.s);
    char* const at = reinterpret_cast<char*>(p.agg);
    p.chain_tickets = reinterpret_cast<unsigned*>(at + work.tickets);
    p.chain_words = reinterpret_cast<unsigned long long*>(at + work.words);
    p.chain_states = reinterpret_cast<unsigned long long*>(at + work.states);
    hipLaunchKernelGGL(chain_clear_kernel, dim3((unsigned)std::min<int64_t>(2048, ceil_div(work.bytes, 4096))), dim3(256), 0, stream,
                       reinterpret_cast<uint4*>(at), work.bytes / 16);
    if (int rc = check_launch(who)) return rc;
    if constexpr (BACK)
        hipLaunchKernelGGL((scan_bwd_kernel<GT, XT, VEC, GV, true, false>), dim3((unsigned)(p.s.blocks * p.s.tiles)), dim3(SCAN_THREADS), 0, stream, p);
    else
        hipLaunchKernelGGL((scan_fwd_kernel<GT, XT, VEC, GV, K, true, false>), dim3((unsigned)(p.s.blocks * p.s.tiles)), dim3(SCAN_THREADS), 0, stream, p);
    return check_launch(who);
}

// Where a gate's channels take several column tiles: the tiles' sums.
template <class GT>
static int scan_gate_total(const ScanArgs& p, const char* who, hipStream_t stream) {
    const ScanShape& s = p.s;
    if (!p.d_gate || s.G == s.C || s.col_tiles == 1) return NERF_OK;
    const int64_t n = s.B * s.T * s.G;
    hipLaunchKernelGGL((scan_gate_sum_kernel<GT>), dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, stream, p.d_gate_part, s.col_tiles, n, static_cast<GT*>(p.d_gate));
    return check_launch(who);
}

template <class GT, class XT, int VEC, int GV>
static int scan_launch(const ScanArgs& p, int dir, const char* who, hipStream_t stream) {
    if (dir == SCAN_FWD && scan_chained(p.s)) {
        if constexpr (sizeof(XT) == 2 && (GV == 1 || sizeof(GT) == 2)) {
            if (scan_chained(p.s, CHAIN_STEPS_16BIT)) return scan_chain_launch<GT, XT, VEC, GV, CHAIN_STEPS_16BIT>(p, who, stream);
        }
        return scan_chain_launch<GT, XT, VEC, GV, CHAIN_STEPS>(p, who, stream);
    }
    const ScanShape& s = p.s;
    if (dir == SCAN_BWD && scan_chained(s, scan_steps(GV))) {
        if (int rc = scan_chain_launch<GT, XT, VEC, GV, scan_steps(GV), true>(p, who, stream)) return rc;
        return scan_gate_total<GT>(p, who, stream);
    }
    if (s.segments > 1) {
        const dim3 grid((unsigned)(s.blocks * (s.segments - 1)));
        if (dir == SCAN_FWD) hipLaunchKernelGGL((scan_segments_kernel<GT, XT, VEC, GV, false>), grid, dim3(SCAN_THREADS), 0, stream, p);
        else hipLaunchKernelGGL((scan_segments_kernel<GT, XT, VEC, GV, true>), grid, dim3(SCAN_THREADS), 0, stream, p);
        if (int rc = check_launch(who)) return rc;
    }
    const dim3 grid((unsigned)(s.blocks * s.segments));
    bool dense = false;
    if constexpr (GV == 1) {
        dense = s.C == VEC && s.G == 1 && s.T * VEC * sizeof(XT) % 16 == 0 && s.T * sizeof(GT) % 16 == 0;
        if (dense && dir == SCAN_FWD) hipLaunchKernelGGL((scan_fwd_kernel<GT, XT, VEC, 1, scan_steps(1), false, true>), grid, dim3(SCAN_THREADS), 0, stream, p);
        else if (dense) hipLaunchKernelGGL((scan_bwd_kernel<GT, XT, VEC, 1, false, true>), grid, dim3(SCAN_THREADS), 0, stream, p);
    }
    if (!dense && dir == SCAN_FWD) hipLaunchKernelGGL((scan_fwd_kernel<GT, XT, VEC, GV, scan_steps(GV), false, false>), grid, dim3(SCAN_THREADS), 0, stream, p);
    else if (!dense) hipLaunchKernelGGL((scan_bwd_kernel<GT, XT, VEC, GV, false, false>), grid, dim3(SCAN_THREADS), 0, stream, p);
    if (int rc = check_launch(who)) return rc;
    return dir == SCAN_BWD ? scan_gate_total<GT>(p, who, stream) : NERF_OK;
}

template <class GT, class XT>
static int scan_run_typed(const ScanArgs& p, int dir, const char* who, hipStream_t stream) {
    if (p.s.T == 1 && p.s.B * p.s.C < 1ll << 31 && (dir == SCAN_FWD || p.s.G == p.s.C)) {
        const dim3 grid((unsigned)ceil_div(p.s.B * p.s.C, SCAN_THREADS * ONE_ELEMENTS));
        if (dir == SCAN_FWD) hipLaunchKernelGGL((scan_one_fwd_kernel<GT, XT>), grid, dim3(SCAN_THREADS), 0, stream, p);
        else hipLaunchKernelGGL((scan_one_bwd_kernel<GT, XT>), grid, dim3(SCAN_THREADS), 0, stream, p);
        return check_launch(who);
    }
    if (p.s.vec == 1) return scan_launch<GT, XT, 1, 1>(p, dir, who, stream);
    if (p.s.vec == 2) return scan_launch<GT, XT, 2, 1>(p, dir, who, stream);
    if (p.s.vec == 3) return scan_launch<GT, XT, 3, 1>(p, dir, who, stream);
    return p.s.G == p.s.C ? scan_launch<GT, XT, 4, 4>(p, dir, who, stream) : scan_launch<GT, XT, 4, 1>(p, dir, who, stream);
}

static int scan_run(const ScanArgs& p, int gate_type, int x_type, int dir, const char* who, hipStream_t stream) {
    return with_type(x_type, [&](auto xt) {
        using XT = decltype(xt);
        return gate_type == NERF_F32 ? scan_run_typed<float, XT>(p, dir, who, stream) : scan_run_typed<XT, XT>(p, dir, who, stream);
    });
}

// Floats of the workspace that hold what the workgroups along the time axis tell each other (a multiple of 4).
static size_t scan_states_floats(const ScanShape& s, bool backward) {
    if (scan_chained(s, backward ? s.steps : CHAIN_STEPS)) return (size_t)chain_work(backward ? s : scan_shape(s.B, s.T, s.C, s.G, CHAIN_STEPS)).bytes / 4;
    return s.segments > 1 ? (size_t)(2 * s.segments * ceil_div(s.B * s.C, 4) * 4) : 0;
}

static int scan_check(const char* who, int64_t B, int64_t T, int C, int G, int gate_type, int x_type) {
    NERF_REQUIRE(B >= 0 && T >= 0 && C >= 0 && G >= 0, "%s: B=%lld T=%lld C=%d G=%d", who, (long long)B, (long long)T, C, G);
    NERF_REQUIRE(C == 0 || (G > 0 && C % G == 0), "%s: %d gates do not divide %d channels", who, G, C);
    NERF_REQUIRE(known_type(x_type) && (gate_type == NERF_F32 || gate_type == x_type), "%s: gate type %d with x type %d", who, gate_type, x_type);
    NERF_REQUIRE(C <= SCAN_CHANNELS, "%s: %d channels, at most %d", who, C, SCAN_CHANNELS);
    if (B == 0 || T == 0 || C == 0) return NERF_OK;
    NERF_REQUIRE(B <= (1ll << 40) && T <= (1ll << 40) && B * (double)T * C < 9e17, "%s: too large", who);
    const ScanShape s = scan_shape(B, T, C, G);
    // a launch holds fewer than 2^32 threads; one joins the sums of a shared gate's column tiles (more than 64 channels a gate),
    // a thread each
    NERF_REQUIRE(s.blocks * (scan_chained(s) ? s.tiles : s.segments) < (1ll << 24) && (G == C || s.col_tiles == 1 || B * (double)T * G < (double)(1ll << 32)),
                 "%s: too many workgroups", who);
    return NERF_OK;
}

}  // namespace nerf

using namespace nerf;

extern "C" size_t nerf_linear_scan_carry_floats(int64_t B, int64_t T, int C, int G) {
    if (B <= 0 || T <= 0 || C <= 0 || G <= 0 || C % G) return 0;
    return (size_t)((scan_shape(B, T, C, G).tiles - 1) * B * C);
}

extern "C" size_t nerf_linear_scan_workspace_floats(int64_t B, int64_t T, int C, int G, int backward) {
    if (B <= 0 || T <= 0 || C <= 0 || G <= 0 || C % G) return 0;
    const ScanShape s = scan_shape(B, T, C, G);
    size_t n = scan_states_floats(s, backward);
    if (backward && G != C && s.col_tiles > 1) n += (size_t)s.col_tiles * (size_t)(B * T * G);
    return n;
}

extern "C" int nerf_linear_scan_fwd(const void* gate, int gate_type, const void* x, int x_type, const float* state, int64_t B,
                                    int64_t T, int C, int G, int reverse, int blend, void* h, float* last, float* carry,
                                    float* workspace, void* stream) {
    const char* who = "nerf_linear_scan_fwd";
    if (int rc = scan_check(who, B, T, C, G, gate_type, x_type)) return rc;
    if (B == 0 || C == 0) return NERF_OK;
    NERF_REQUIRE(T > 0, "%s: a sequence of no steps", who);
    NERF_REQUIRE(gate && x && h, "%s: null pointer", who);
    NERF_REQUIRE(aligned16(gate) && aligned16(x) && aligned16(state) && aligned16(h) && aligned16(last) && aligned16(carry) && aligned16(workspace),
                 "%s: pointers must be 16-byte aligned", who);
    ScanArgs p{};
    p.s = scan_shape(B, T, C, G);
    p.l_carry = log2_up(p.s.tile_steps);
    NERF_REQUIRE(workspace || nerf_linear_scan_workspace_floats(B, T, C, G, 0) == 0, "%s: null workspace", who);
    p.gate = gate; p.x = x; p.state = state; p.reverse = reverse != 0; p.blend = blend != 0;
    p.h = h; p.last = last; p.carry = carry; p.agg = workspace;
    return scan_run(p, gate_type, x_type, SCAN_FWD, who, (hipStream_t)stream);
}

extern "C" int nerf_linear_scan_bwd(const void* gate, int gate_type, const void* x, int x_type, const float* state, const float* carry,
                                    const void* d_h, const float* d_last, int64_t B, int64_t T, int C, int G, int reverse, int blend,
                                    void* d_gate, void* d_x, float* d_state, float* workspace, void* stream) {
    const char* who = "nerf_linear_scan_bwd";
    if (int rc = scan_check(who, B, T, C, G, gate_type, x_type)) return rc;
    if (B == 0 || C == 0) return NERF_OK;
    NERF_REQUIRE(T > 0, "%s: a sequence of no steps", who);
    NERF_REQUIRE(gate && x, "%s: null pointer", who);
    NERF_REQUIRE(aligned16(gate) && aligned16(x) && aligned16(state) && aligned16(carry) && aligned16(d_h) && aligned16(d_last) && aligned16(d_gate) &&
                     aligned16(d_x) && aligned16(d_state) && aligned16(workspace),
                 "%s: pointers must be 16-byte aligned", who);
    ScanArgs p{};
    p.s = scan_shape(B, T, C, G);
    p.l_carry = log2_up(p.s.tile_steps);
    NERF_REQUIRE(carry || p.s.tiles == 1, "%s: null carry (the forward pass keeps it)", who);
    NERF_REQUIRE(workspace || nerf_linear_scan_workspace_floats(B, T, C, G, 1) == 0, "%s: null workspace", who);
    p.gate = gate; p.x = x; p.state = state; p.reverse = reverse != 0; p.blend = blend != 0;
    p.carry = const_cast<float*>(carry);
    p.d_h = d_h; p.d_last = d_last; p.d_gate = d_gate; p.d_x = d_x; p.d_state = d_state;
    p.agg = workspace;
    p.d_gate_part = workspace ? workspace + scan_states_floats(p.s, true) : nullptr;
    return scan_run(p, gate_type, x_type, SCAN_BWD, who, (hipStream_t)stream);
}
