// Element types of the operators that take more than float32: storage in float, bf16 or f16, arithmetic in float.
#pragma once
#include "common.h"

namespace nerf {

// N consecutive elements, aligned as an array of them that starts on a 16-byte boundary is.
template <class T, int N>
struct __attribute__((aligned((sizeof(T) * N) & -(sizeof(T) * N)))) Run {
    T v[N];
};

// N consecutive elements as one load / store (the address is a multiple of N elements).
template <int N, class T>
__device__ __forceinline__ void load_run(const T* __restrict__ p, float (&out)[N]) {
    const Run<T, N> r = *reinterpret_cast<const Run<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)r.v[i];
}
// Rounds to nearest even (the conversion instructions of the chip).
template <int N, class T>
__device__ __forceinline__ void store_run(T* __restrict__ p, const float (&v)[N]) {
    Run<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = (T)v[i];
    *reinterpret_cast<Run<T, N>*>(p) = r;
}

inline bool known_type(int type) { return type == NERF_F32 || type == NERF_BF16 || type == NERF_F16; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// f(T{}) with the storage type that `type` names.
template <class F>
inline int with_type(int type, F&& f) {
    if (type == NERF_F32) return f(float{});
    if (type == NERF_BF16) return f(__bf16{});
    return f(_Float16{});
}

}  // namespace nerf
