// Maps in their stored type (fp32, bf16, fp16) and as fp32 registers: the maps of the normalisation, dropout and adapter
// kernels may be kept in 16 bits; every sum over them is fp32.
#pragma once
#include "common.h"

constexpr int DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2;

typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

template <class T> struct dtype_of;
template <> struct dtype_of<float> { static constexpr int value = DT_F32; };
template <> struct dtype_of<__bf16> { static constexpr int value = DT_BF16; };
template <> struct dtype_of<_Float16> { static constexpr int value = DT_F16; };

// V elements as they are stored, in W dwords.
template <class T, int V> struct Raw {
    static constexpr int W = V * (int)sizeof(T) / 4;
    unsigned w[W];
};

// From / to an address of element alignment: rows of odd length put a vector anywhere, and global memory takes unaligned
// 16-byte accesses on this part. STREAM: a map that is read once (group norm: 94 us against 103 at the sizes below; with it on
// rows that other blocks read again, 64 tokens beside a 4096 x 4096 projection went from 24 to 28).
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
    typedef unsigned Vec __attribute__((ext_vector_type(Raw<T, V>::W), aligned(sizeof(T))));
    Vec q;
    if constexpr (STREAM) q = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(p));
    else q = *reinterpret_cast<const Vec*>(p);
    Raw<T, V> r;
#pragma unroll
    for (int i = 0; i < Raw<T, V>::W; ++i) r.w[i] = q[i];
    return r;
}

template <class T>
__device__ __forceinline__ unsigned bits_of(T v) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(unsigned, v);
    else return (unsigned)__builtin_bit_cast(unsigned short, v);
}

// the first n of V elements; the rest is zero and not read (their loads repeat the last element's: independent loads instead of
// a chain of conditions that waits for each)
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p, int n) {
    if (n >= V) return load_raw<T, V, STREAM>(p);
    Raw<T, V> r;
    constexpr int E = 4 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < Raw<T, V>::W; ++i) r.w[i] = 0;
    if (n <= 0) return r;
    unsigned e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = bits_of<T>(p[min(i, n - 1)]);
#pragma unroll
    for (int i = 0; i < V; ++i) r.w[i / E] |= (i < n ? e[i] : 0u) << (16 * (i % E));
    return r;
}

template <class T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&o)[V]) {
#pragma unroll
    for (int i = 0; i < Raw<T, V>::W; ++i) {
        if constexpr (sizeof(T) == 4) {
            o[i] = __builtin_bit_cast(float, r.w[i]);
        } else if constexpr (dtype_of<T>::value == DT_BF16) {
            o[2 * i] = __builtin_bit_cast(float, r.w[i] << 16);
            o[2 * i + 1] = __builtin_bit_cast(float, r.w[i] & 0xffff0000u);
        } else {
            const f16x2 h = __builtin_bit_cast(f16x2, r.w[i]);
            o[2 * i] = (float)h[0];
            o[2 * i + 1] = (float)h[1];
        }
    }
}

template <class T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float (&v)[V]) {
    Raw<T, V> r;
#pragma unroll
    for (int i = 0; i < Raw<T, V>::W; ++i) {
        if constexpr (sizeof(T) == 4) r.w[i] = __builtin_bit_cast(unsigned, v[i]);
        else r.w[i] = bits_of<T>((T)v[2 * i]) | bits_of<T>((T)v[2 * i + 1]) << 16;
    }
    return r;
}

// STREAM: a result that is as large as the maps it comes from - it goes past the caches and leaves them to what is read (group
// norm backward at 10 x 32 x 1024 x 64 fp32: 103 us against 123; dropout of 210 M bf16 elements: 139 against 147). Not for
// parts that the next launch reads.
template <class T, int V, bool STREAM = true>
__device__ __forceinline__ void store_raw(T* p, const Raw<T, V>& r, int n) {
    if (n >= V) {
        typedef unsigned Vec __attribute__((ext_vector_type(Raw<T, V>::W), aligned(sizeof(T))));
        Vec q;
#pragma unroll
        for (int i = 0; i < Raw<T, V>::W; ++i) q[i] = r.w[i];
        if constexpr (STREAM) __builtin_nontemporal_store(q, reinterpret_cast<Vec*>(p));
        else *reinterpret_cast<Vec*>(p) = q;
        return;
    }
    constexpr int E = 4 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < Raw<T, V>::W; ++i)
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (i * E + j < n) {
                if constexpr (sizeof(T) == 4) p[i] = __builtin_bit_cast(T, r.w[i]);
                else p[i * E + j] = __builtin_bit_cast(T, (unsigned short)(r.w[i] >> (16 * j)));
            }
}

template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void load_part(const T* p, int n, float (&o)[V]) { unpack<T, V>(load_raw<T, V, STREAM>(p, n), o); }

template <class T, int V, bool STREAM = true>
__device__ __forceinline__ void store_part(T* p, int n, const float (&v)[V]) { store_raw<T, V, STREAM>(p, pack<T, V>(v), n); }

// Zeroes the elements of a vector whose bit is 0.
template <class T, int V>
__device__ __forceinline__ void keep_raw(Raw<T, V>& r, unsigned bits) {
#pragma unroll
    for (int i = 0; i < Raw<T, V>::W; ++i) {
        if constexpr (sizeof(T) == 4) r.w[i] = (bits >> i & 1u) ? r.w[i] : 0u;
        else r.w[i] &= ((bits >> (2 * i) & 1u) ? 0xffffu : 0u) | ((bits >> (2 * i + 1) & 1u) ? 0xffff0000u : 0u);
    }
}
