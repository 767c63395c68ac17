// Dropout masks from a counter: whether element e of a client stays is a function of (client seed, step, site, e) alone,
// so no mask is stored, the backward pass draws it again, and a node's masks do not depend on which nodes share its card.
//
// Generator: Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011;
// 7 is the smallest count that passes the authors' BigCrush runs). Block e / 4 has the counter (e / 4, site, step low,
// step high) and the key (seed low, seed high); element e takes its word e % 4 and is dropped where that word is below
// round(p 2^32). A round is two 32 x 32 -> 64 bit products (quarter rate): ten rounds instead of seven made the bf16
// stream slower (dropout.hip has both times).
#pragma once
#include "common.h"

struct P2pflDrop {
    const long long* seeds;      // [K] one per client (null: no dropout)
    const long long* step;       // [1] read on the device: a captured graph draws new masks when it is advanced
    unsigned site;               // tells apart the dropouts of one step
    unsigned threshold;          // round(p 2^32)
    int all;                     // p == 1: nothing stays
    float scale;                 // 1 / (1 - p)
};

struct DropKey {
    unsigned k0 = 0, k1 = 0, site = 0, s0 = 0, s1 = 0;
    DropKey() = default;
    __device__ __forceinline__ DropKey(const P2pflDrop& d, int client) {
        const unsigned long long k = (unsigned long long)d.seeds[client], s = (unsigned long long)d.step[0];
        k0 = (unsigned)k; k1 = (unsigned)(k >> 32); site = d.site; s0 = (unsigned)s; s1 = (unsigned)(s >> 32);
    }
};

constexpr int PHILOX_ROUNDS = 7;

__device__ __forceinline__ void philox4(const DropKey& key, unsigned block, unsigned (&out)[4]) {
    unsigned c0 = block, c1 = key.site, c2 = key.s0, c3 = key.s1, k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < PHILOX_ROUNDS; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c1 = (unsigned)b;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    out[0] = c0; out[1] = c1; out[2] = c2; out[3] = c3;
}

// Bit i: element e + i of the client stays, i < V (V a multiple of 4; elements of a client < 2^34).
template <int V>
__device__ __forceinline__ unsigned keep_bits(const P2pflDrop& d, const DropKey& key, unsigned long long e) {
    unsigned bits = 0;
    const unsigned sh = (unsigned)e & 3u, first = (unsigned)(e >> 2);
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        unsigned w[4];
        philox4(key, first + q, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) bits |= (unsigned)(w[j] >= d.threshold) << (4 * q + j);
    }
    if (sh) {                    // the vector straddles one more block
        unsigned w[4];
        philox4(key, first + V / 4, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) bits |= (unsigned)(w[j] >= d.threshold) << (V + j);
        bits >>= sh;
    }
    return d.all ? 0u : bits & ((1u << V) - 1u);
}

// keep_bits of I vectors, `step` elements apart, in registers; one copy of the generator's code per 32 of them.
template <int V, int I>
struct KeepRows {
    static constexpr int PER = 32 / V, WORDS = (I + PER - 1) / PER;
    unsigned w[WORDS];
    __device__ __forceinline__ void draw(const P2pflDrop& d, const DropKey& key, unsigned long long e, unsigned long long step, int rows) {
#pragma unroll
        for (int q = 0; q < WORDS; ++q) {
            unsigned t = 0;
#pragma unroll 1
            for (int j = 0; j < PER; ++j)
                if (q * PER + j < rows) t |= keep_bits<V>(d, key, e + step * (q * PER + j)) << (j * V);
            w[q] = t;
        }
    }
    __device__ __forceinline__ unsigned operator[](int i) const { return w[i / PER] >> (i % PER * V) & (unsigned)((1ull << V) - 1); }
};

// A dropped element is zero whatever it held (infinities and NaN too); a kept one is scaled by 1 / (1 - p).
template <int V>
__device__ __forceinline__ void drop_vec(const P2pflDrop& d, unsigned bits, float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (bits >> i & 1u) ? v[i] * d.scale : 0.f;
}
template <int V>
__device__ __forceinline__ void drop_vec(const P2pflDrop& d, const DropKey& key, unsigned long long e, float (&v)[V]) {
    drop_vec<V>(d, keep_bits<V>(d, key, e), v);
}
