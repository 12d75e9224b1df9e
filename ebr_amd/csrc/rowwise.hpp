// What the row-wise kernels of the token ends and of the group norm share: accumulation types, 16-byte vectors, sums and
// maxima over a wave or a part of one.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ebr_block.h"

namespace ebr_row {

template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };

// N consecutive elements, loaded and stored whole (N * sizeof(T) a power of two, at most 16 bytes, and so aligned).
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T e[N]; };

template <typename T, int N> __device__ __forceinline__ Pack<T, N> ldp(const T* p) {
    return *reinterpret_cast<const Pack<T, N>*>(p);
}
template <typename T, int N> __device__ __forceinline__ void stp(T* p, const Pack<T, N>& v) {
    *reinterpret_cast<Pack<T, N>*>(p) = v;
}

// Elements as they lie in memory: held as elements, each of 16 bits would have a register of its own.
template <int BYTES> struct Words { using type = uint4; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<4> { using type = uint32_t; };
template <> struct Words<2> { using type = uint16_t; };
template <typename T, int VEC, typename W> __device__ __forceinline__ Pack<T, VEC> unpacked(W w) {
    Pack<T, VEC> v;
    static_assert(sizeof(v) == sizeof(w), "the words of a pack");
    __builtin_memcpy(&v, &w, sizeof(v));
    return v;
}

// N elements of T from or to memory of which 16 bytes (or all of them, where fewer) are aligned, as whole vectors.
template <typename T, int N, typename A> __device__ __forceinline__ void load_wide(const T* p, A (&x)[N]) {
    constexpr int V = N * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += V) {
        const Pack<T, V> v = ldp<T, V>(p + i);
#pragma unroll
        for (int e = 0; e < V; ++e) x[i + e] = (A)v.e[e];
    }
}
template <typename A, int N> __device__ __forceinline__ void store_wide(A* p, const A (&x)[N]) {
    constexpr int V = N * (int)sizeof(A) > 16 ? 16 / (int)sizeof(A) : N;
#pragma unroll
    for (int i = 0; i < N; i += V) {
        Pack<A, V> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.e[e] = x[i + e];
        stp<A, V>(p + i, v);
    }
}

// As store_wide, past the caches: for what nothing reads soon.
template <typename A, int N> __device__ __forceinline__ void store_past(A* p, const A (&x)[N]) {
    constexpr int V = N * (int)sizeof(A) > 16 ? 16 / (int)sizeof(A) : N;
    if constexpr (V * sizeof(A) == 16) {
        using W = uint32_t __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < N; i += V) {
            W w;
            __builtin_memcpy(&w, &x[i], 16);
            __builtin_nontemporal_store(w, reinterpret_cast<W*>(p + i));
        }
    } else {
        store_wide<A, N>(p, x);
    }
}

// Over aligned parts of W lanes of a wave.
template <int W, typename A> __device__ __forceinline__ A lanes_sum(A v) {
#pragma unroll
    for (int m = W / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    return v;
}

static inline int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? EBR_OK : EBR_ERR_HIP_BASE + (int)e;
}

static inline bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

constexpr int64_t MAX_BLOCKS = ((int64_t)1 << 24) - 1;  // of 256 threads: a launch holds fewer than 2^32 threads
static inline unsigned blocks_for(int64_t n, int64_t per) {
    const int64_t want = (n + per - 1) / per;
    return (unsigned)(want < MAX_BLOCKS ? want : MAX_BLOCKS);
}

}  // namespace ebr_row
