// Device helpers shared by the training operators (embedding.hip,
// window_scores.hip, preference.hip): element types, vector access, node
// loads.  Every value is computed in float32 and rounded once, to nearest even,
// where it is stored.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "mlxc_train.h"

namespace mlxc {

// An element type: its storage, and its conversions from and to float32.
struct F32 {
    using S = float;
    static __device__ __forceinline__ float load(S x) { return x; }
    static __device__ __forceinline__ S store(float x) { return x; }
};
struct BF16 {
    using S = uint16_t;
    static __device__ __forceinline__ float load(S x) {
        return __builtin_bit_cast(float, static_cast<uint32_t>(x) << 16);
    }
    static __device__ __forceinline__ S store(float x) {
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
    }
};
struct F16 {
    using S = _Float16;
    static __device__ __forceinline__ float load(S x) { return static_cast<float>(x); }
    static __device__ __forceinline__ S store(float x) { return static_cast<_Float16>(x); }
};

// N elements that one memory instruction moves (at most 16 bytes).
template <typename S, int N>
struct alignas(sizeof(S) * N) Pack {
    S v[N];
};

template <typename E, int N>
__device__ __forceinline__ void load_pack(float (&x)[N], const typename E::S* p) {
    const Pack<typename E::S, N> k = *reinterpret_cast<const Pack<typename E::S, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = E::load(k.v[i]);
}

template <typename E, int N>
__device__ __forceinline__ void store_pack(typename E::S* p, const float (&x)[N]) {
    Pack<typename E::S, N> k;
#pragma unroll
    for (int i = 0; i < N; ++i) k.v[i] = E::store(x[i]);
    *reinterpret_cast<Pack<typename E::S, N>*>(p) = k;
}

// A store past the caches, for what the call does not read again.
template <typename S, int N>
__device__ __forceinline__ void stream_pack(S* p, const Pack<S, N>& k) {
    constexpr int kBytes = sizeof(S) * N;
    if constexpr (kBytes == 16) {
        typedef uint32_t Words __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(__builtin_bit_cast(Words, k), reinterpret_cast<Words*>(p));
    } else if constexpr (kBytes == 8) {
        __builtin_nontemporal_store(__builtin_bit_cast(uint64_t, k), reinterpret_cast<uint64_t*>(p));
    } else if constexpr (kBytes == 4) {
        __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, k), reinterpret_cast<uint32_t*>(p));
    } else {
        *p = k.v[0];
    }
}

// Nodes of a call: int64 or int32, num_rows of them valid.
struct Nodes {
    const void* p;
    int64_t num_rows;
    bool wide;  // int64
};

// Node i, or -1 where there is none; a node outside [0, num_rows) other than
// -1 is none either and sets bad.
__device__ __forceinline__ int64_t node_at(const Nodes& n, int64_t i, bool& bad) {
    const int64_t v = n.wide ? static_cast<const int64_t*>(n.p)[i]
                             : static_cast<int64_t>(static_cast<const int32_t*>(n.p)[i]);
    if (static_cast<uint64_t>(v) < static_cast<uint64_t>(n.num_rows)) return v;
    bad |= v != -1;
    return -1;
}

__device__ __forceinline__ void report_bad(bool bad, int64_t* status) {
    if (bad && status)
        atomicOr(reinterpret_cast<unsigned long long*>(status),
                 static_cast<unsigned long long>(MLXC_STATUS_BAD_NODE));
}

}  // namespace mlxc
