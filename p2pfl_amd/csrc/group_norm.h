// Group normalisation with residual, activation and dropout over channels-last maps [K, N, S, C] of K clients:
//
//   z = (x - mean_g) rstd_g w_c + b_c (+ res),   y = drop(act(z)),   mean / var over the S x C/G elements of (k, n, g)
//   dz = drop(dy) act'(z),  dres = dz,  db_c = sum dz,  dw_c = sum dz xhat,  t = dz w
//   dx = rstd (t - mean_g(t) - xhat mean_g(t xhat))
//
// Both passes are memory-bound: the floor is one read of every input map and one write of every output map. A block owns
// a slab of whole groups (CW channels of one sample) and keeps it in registers between the statistics and the result, so
// nothing is read twice; the mean is taken first and the squares around it (no cancellation for maps far from zero). A
// slab that does not fit is cut into row chunks: their statistics go through scratch memory, are joined in a fixed
// order (Chan, Golub, LeVeque 1979), and the maps are read a second time.
//
// Thread layout of a block: VC = ceil(CW / V) vector columns x RPP rows per pass, so a thread keeps its channels over all
// rows: affine parameters and per-channel sums live in registers. No atomics: every sum has a fixed order.
//
// One translation unit per type of the maps (group_norm_f32.hip, ...); group_norm.hip has the entry points.
#pragma once
#include <type_traits>
#include "typed.h"
#include "philox.h"

namespace {

struct GnMap { void* p; long sk, sn, ss; };       // element strides of client, sample and position; channels are dense

}  // namespace

struct P2pflGroupNorm {
    GnMap x, y, res, dy, dx, dres;                // p null: absent
    const float* w; long w_cs;
    const float* b; long b_cs;
    float* mean; float* rstd;                     // [K][N][G]
    float* dw; long dw_cs;
    float* db; long db_cs;
    float* scratch; long scratch_len;
    P2pflDrop drop;
    int K, N, S, C, G, act, dtype;
    float eps;
};

namespace {

constexpr int ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3;

// NaN passes through relu and its gradient, as in torch.
__device__ __forceinline__ float act_of(float z, const int act) {
    switch (act) {
        case ACT_RELU: return z <= 0.f ? 0.f : z;
        case ACT_SILU: return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));        // (the reciprocal is exact to 1 ulp)
        case ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    }
    return z;
}

template <int V>
__device__ __forceinline__ void act_all(float (&z)[V], int act) {     // (the choice outside the loop: one branch a vector)
    switch (act) {
        case ACT_RELU:
#pragma unroll
            for (int v = 0; v < V; ++v) z[v] = act_of(z[v], ACT_RELU);
            break;
        case ACT_SILU:
#pragma unroll
            for (int v = 0; v < V; ++v) z[v] = act_of(z[v], ACT_SILU);
            break;
        case ACT_GELU:
#pragma unroll
            for (int v = 0; v < V; ++v) z[v] = act_of(z[v], ACT_GELU);
            break;
    }
}

__device__ __forceinline__ float dact_of(float z, int act) {
    switch (act) {
        case ACT_RELU: return z <= 0.f ? 0.f : 1.f;
        case ACT_SILU: { const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z)); return s * (1.f + z * (1.f - s)); }
        case ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
    }
    return 1.f;
}

__device__ __forceinline__ float rsqrt_of(float v) { return __builtin_amdgcn_rsqf(v); }       // exact to 1 ulp

// How the maps are cut: slabs of gpb groups (cw channels), chunks of `rows` rows.
struct Cut { int gpb, slabs, chunks, rows, nt, iters; };

template <int V>
struct Place {
    int k, n, slab, chunk, g0, ng, c0, cw, vc, rpp, col, row, nv, c;
    long kn;
    bool on;
    __device__ __forceinline__ Place(const P2pflGroupNorm& a, const Cut& cut) {
        unsigned id = blockIdx.x, q = id;         // (32-bit divisions: a grid has less than 2^32 blocks)
        if (cut.chunks > 1) q = id / (unsigned)cut.chunks;
        chunk = (int)(id - q * (unsigned)cut.chunks);
        id = q;
        if (cut.slabs > 1) q = id / (unsigned)cut.slabs;
        slab = (int)(id - q * (unsigned)cut.slabs);
        kn = q;
        k = (int)(q / (unsigned)a.N); n = (int)(q - (unsigned)k * (unsigned)a.N);
        const int cpg = a.C / a.G;
        g0 = slab * cut.gpb;
        ng = min(cut.gpb, a.G - g0);
        c0 = g0 * cpg; cw = ng * cpg;
        vc = (cut.gpb * cpg + V - 1) / V;
        rpp = blockDim.x / (unsigned)vc;
        row = threadIdx.x / (unsigned)vc; col = threadIdx.x - row * vc;
        nv = max(0, min(V, cw - col * V));         // this thread's channels (a short last vector, or a short last slab)
        c = c0 + col * V;
        on = row < rpp && nv > 0;
    }
    // a thread's rows of a map: row i of the block is `step` elements behind row i - 1
    template <class T>
    struct Walk {
        T* p; long step;
        __device__ __forceinline__ T* operator[](int i) const { return p + i * step; }
    };
    template <class T>
    __device__ __forceinline__ Walk<T> walk(const GnMap& m, int s0) const {
        return {reinterpret_cast<T*>(m.p) + k * m.sk + n * m.sn + (s0 + row) * m.ss + c, rpp * m.ss};
    }
    __device__ __forceinline__ unsigned long long element(const P2pflGroupNorm& a, int s) const {
        return ((unsigned long long)n * a.S + s) * a.C + c;
    }
};

// Sums of NQ per-thread, per-channel values over the block's rows: ch[q * vc * V + channel of the slab]. `red`: LDS of
// NQ * blockDim.x * V floats. All threads call it; ch may be read after the return.
template <int V, int NQ>
__device__ __forceinline__ void channel_sums(float (&s)[NQ][V], const Place<V>& p, float* red, float* ch) {
    const int cwp = p.vc * V;
    int slots = p.rpp, slot = p.row;
    bool writes = p.row < p.rpp;
    if (p.vc <= 64 && (p.vc & (p.vc - 1)) == 0) {            // lanes of one column are vc apart: add them in the wave first
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int v = 0; v < V; ++v)
                for (int off = 32; off >= p.vc; off >>= 1) s[q][v] += __shfl_xor(s[q][v], off, 64);
        slots = blockDim.x >> 6;
        slot = threadIdx.x >> 6;
        writes = (threadIdx.x & 63) < p.vc;
    }
    if (writes) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int v = 0; v < V; ++v) red[(q * slots + slot) * cwp + p.col * V + v] = s[q][v];
    }
    __syncthreads();
    const int items = NQ * cwp, share = blockDim.x / items;
    if (share >= 2 && slots >= 8) {                          // few channels, many rows: several threads per channel first
        const int item = threadIdx.x % items, first = threadIdx.x / items, q = item / cwp;
        float t = 0.f;
        if (first < share)
#pragma unroll 4
            for (int j = first; j < slots; j += share) t += red[(q * slots + j) * cwp + item - q * cwp];
        __syncthreads();
        if (first < share) red[first * items + item] = t;
        __syncthreads();
        if ((int)threadIdx.x < items) {
            t = 0.f;
#pragma unroll 4
            for (int j = 0; j < share; ++j) t += red[j * items + item];
            ch[item] = t;
        }
    } else {
        for (int i = threadIdx.x; i < items; i += blockDim.x) {
            const int q = i / cwp, c = i - q * cwp;
            float t = 0.f;
#pragma unroll 8
            for (int j = 0; j < slots; ++j) t += red[(q * slots + j) * cwp + c];
            ch[i] = t;
        }
    }
    __syncthreads();
}

// out[g] = sum over the cpg channels of group g of f(channel of the slab); a wave per group.
template <class F>
__device__ __forceinline__ void group_sums(int ng, int cpg, float* out, F f) {
    const int lane = threadIdx.x & 63;
    for (int g = threadIdx.x >> 6; g < ng; g += blockDim.x >> 6) {
        float t = 0.f;
        for (int c = lane; c < cpg; c += 64) t += f(g * cpg + c);
        t = wave_reduce_sum(t);
        if (lane == 0) out[g] = t;
    }
    __syncthreads();
}

// LDS of a block, in floats: red | ch | per-group values (2)
__host__ __device__ inline long lds_floats(int nq, int V, int nt, int vc, int gpb) { return (long)nq * nt * V + (long)nq * vc * V + 2L * gpb; }

// Which elements of a thread's rows dropout keeps (drawn while the rows are on their way).
template <int V, int I>
__device__ __forceinline__ void gn_draw(const P2pflGroupNorm& a, const Place<V>& p, int s0, int left, KeepRows<V, I>& keep) {
    if (a.drop.seeds)
        keep.draw(a.drop, DropKey(a.drop, p.k), p.element(a, s0 + p.row), (unsigned long long)p.rpp * a.C,
                  left > 0 ? (left + p.rpp - 1) / p.rpp : 0);
}

// y of a thread's rows from x (by row), the mean, w rstd and b of its channels.
template <class T, int V, int I, class X>
__device__ __forceinline__ void gn_finish(const P2pflGroupNorm& a, const Place<V>& p, int s0, int left, const float (&mu)[V],
                                          const float (&wa)[V], const float (&bb)[V], const KeepRows<V, I>& keep, X x_of) {
    const auto py = p.template walk<T>(a.y, s0);
    const auto pr = p.template walk<const T>(a.res, s0);
    const bool drops = a.drop.seeds != nullptr, res = a.res.p != nullptr;
#pragma unroll
    for (int i = 0; i < I; ++i) {
        if (i * p.rpp < left) {
            float x[V], r[V];
            unpack<T, V>(x_of(i), x);
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = (x[v] - mu[v]) * wa[v] + bb[v];
            if (res) {
                load_part<T, V, true>(pr[i], p.nv, r);
#pragma unroll
                for (int v = 0; v < V; ++v) x[v] += r[v];
            }
            act_all<V>(x, a.act);
            if (drops) drop_vec<V>(a.drop, keep[i], x);
            store_part<T, V>(py[i], p.nv, x);
        }
    }
}

// Statistics of a slab chunk held in registers, then its result (SPLIT: only the chunk's statistics, to scratch).
template <class T, int V, int I, bool SPLIT>
__global__ __launch_bounds__(1024) void gn_fwd_kernel(P2pflGroupNorm a, Cut cut) {
    extern __shared__ float lds[];
    const Place<V> p(a, cut);
    const int cpg = a.C / a.G;
    const int s0 = p.chunk * cut.rows, s1 = min(a.S, s0 + cut.rows);
    float* red = lds;
    float* ch = red + blockDim.x * V;
    float* gv = ch + p.vc * V;                     // [2][gpb]
    const auto px = p.template walk<const T>(a.x, s0);
    const int left = p.on ? s1 - s0 - p.row : 0;   // rows of this thread: those i * rpp < left
    Raw<T, V> raw[I];
    float sum[1][V], wa[V], bb[V];
    int group[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {                  // (loaded here: used only once the sums are there)
        const bool in = p.on && v < p.nv;
        wa[v] = in && a.w && !SPLIT ? a.w[p.k * a.w_cs + p.c + v] : 1.f;
        bb[v] = in && a.b && !SPLIT ? a.b[p.k * a.b_cs + p.c + v] : 0.f;
        group[v] = in ? (p.col * V + v) / cpg : 0;
        sum[0][v] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
        if (i * p.rpp < left) raw[i] = load_raw<T, V, !SPLIT>(px[i], p.nv);
    }
    KeepRows<V, I> keep;
    if constexpr (!SPLIT) gn_draw<V, I>(a, p, s0, left, keep);
#pragma unroll
    for (int i = 0; i < I; ++i) {
        if (i * p.rpp < left) {
            float x[V];
            unpack<T, V>(raw[i], x);
#pragma unroll
            for (int v = 0; v < V; ++v) sum[0][v] += x[v];
        }
    }
    channel_sums<V, 1>(sum, p, red, ch);
    group_sums(p.ng, cpg, gv, [&](int c) { return ch[c]; });
    const float inv = 1.f / ((float)(s1 - s0) * (float)cpg);
    float mu[V];
#pragma unroll
    for (int v = 0; v < V; ++v) mu[v] = v < p.nv ? gv[group[v]] * inv : 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) sum[0][v] = 0.f;
#pragma unroll
    for (int i = 0; i < I; ++i) {
        if (i * p.rpp < left) {
            float x[V];
            unpack<T, V>(raw[i], x);
#pragma unroll
            for (int v = 0; v < V; ++v) { const float d = x[v] - mu[v]; sum[0][v] += v < p.nv ? d * d : 0.f; }
        }
    }
    channel_sums<V, 1>(sum, p, red, ch);
    float* m2 = gv + cut.gpb;
    group_sums(p.ng, cpg, m2, [&](int c) { return ch[c]; });
    if constexpr (SPLIT) {
        for (int g = threadIdx.x; g < p.ng; g += blockDim.x) {
            float* o = a.scratch + ((p.kn * cut.chunks + p.chunk) * a.G + p.g0 + g) * 2;
            o[0] = gv[g] * inv;
            o[1] = m2[g];
        }
        return;
    }
    for (int g = threadIdx.x; g < p.ng; g += blockDim.x) {
        if (a.mean) a.mean[p.kn * a.G + p.g0 + g] = gv[g] * inv;
        if (a.rstd) a.rstd[p.kn * a.G + p.g0 + g] = rsqrt_of(m2[g] * inv + a.eps);
    }
    if (!p.on) return;
#pragma unroll
    for (int v = 0; v < V; ++v) wa[v] *= v < p.nv ? rsqrt_of(m2[group[v]] * inv + a.eps) : 0.f;
    gn_finish<T, V, I>(a, p, s0, left, mu, wa, bb, keep, [&](int i) { return raw[i]; });
}

// Joins the chunks' (mean, sum of squares around it) of every group of a sample in the order of the chunks.
__global__ __launch_bounds__(64) void gn_join_kernel(P2pflGroupNorm a, Cut cut, float* mean, float* rstd) {
    const long i = (long)blockIdx.x * 64 + threadIdx.x;
    if (i >= (long)a.K * a.N * a.G) return;
    const long kn = i / a.G;
    const int g = (int)(i - kn * a.G), cpg = a.C / a.G;
    float n = 0.f, m = 0.f, q = 0.f;
    for (int c = 0; c < cut.chunks; ++c) {
        const float* o = a.scratch + ((kn * cut.chunks + c) * a.G + g) * 2;
        const float nc = (float)(min(a.S, (c + 1) * cut.rows) - c * cut.rows) * (float)cpg;
        const float d = o[0] - m, t = n + nc;
        m += d * (nc / t);
        q += o[1] + d * d * (n * nc / t);
        n = t;
    }
    mean[i] = m;
    rstd[i] = rsqrt_of(q / n + a.eps);
}

// The result from known statistics (second read of a slab that was cut into chunks).
template <class T, int V, int I>
__global__ __launch_bounds__(1024) void gn_apply_kernel(P2pflGroupNorm a, Cut cut, const float* mean, const float* rstd) {
    const Place<V> p(a, cut);
    if (!p.on) return;
    const int cpg = a.C / a.G;
    const int s0 = p.chunk * cut.rows, s1 = min(a.S, s0 + cut.rows);
    float mu[V], wa[V], bb[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const bool in = v < p.nv;
        const long g = p.kn * a.G + (p.c + (in ? v : 0)) / cpg;
        mu[v] = mean[g];
        wa[v] = in ? (a.w ? a.w[p.k * a.w_cs + p.c + v] : 1.f) * rstd[g] : 0.f;
        bb[v] = in && a.b ? a.b[p.k * a.b_cs + p.c + v] : 0.f;
    }
    const auto px = p.template walk<const T>(a.x, s0);
    KeepRows<V, I> keep;
    gn_draw<V, I>(a, p, s0, s1 - s0 - p.row, keep);
    gn_finish<T, V, I>(a, p, s0, s1 - s0 - p.row, mu, wa, bb, keep, [&](int i) { return load_raw<T, V, true>(px[i], p.nv); });
}

// ------------------------------------------------------------------------------------------------ backward
// relu goes by the given result where there is one (its sign holds the dropout too: a dropped element is zero there), else by
// the value before it, which the residual belongs to.
// Of a thread's channels: mean, rstd and the factor rstd w of x - mean in z, and b.
template <int V>
__device__ __forceinline__ void gn_params(const P2pflGroupNorm& a, const Place<V>& p, float (&mu)[V], float (&rs)[V], float (&rw)[V],
                                          float (&bb)[V]) {
    const int cpg = a.C / a.G;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const bool in = p.on && v < p.nv;
        const long g = in ? p.kn * a.G + (p.c + v) / cpg : 0;
        mu[v] = in ? a.mean[g] : 0.f;
        rs[v] = in ? a.rstd[g] : 0.f;
        rw[v] = in ? (a.w ? a.w[p.k * a.w_cs + p.c + v] : 1.f) * rs[v] : 0.f;
        bb[v] = in && a.b ? a.b[p.k * a.b_cs + p.c + v] : 0.f;
    }
}

// What a thread keeps of a row between the sums and the result, as stored: x, and dy with the elements zeroed that dropout or relu's
// given result take out (exact; the factor 1 / (1 - p) comes in again when it is used).
template <class T, int V>
struct GnRows {
    typename Place<V>::template Walk<const T> x, dy, y, res;
    int nv;
    bool by_y, drops, has_res;                    // relu by the given result; dropout; a residual that z needs
    __device__ __forceinline__ GnRows(const P2pflGroupNorm& a, const Place<V>& p, int s0)
        : x(p.template walk<const T>(a.x, s0)), dy(p.template walk<const T>(a.dy, s0)), y(p.template walk<const T>(a.y, s0)),
          res(p.template walk<const T>(a.res, s0)), nv(p.nv), by_y(a.act == ACT_RELU && a.y.p), drops(a.drop.seeds != nullptr),
          has_res(a.res.p && a.act != ACT_NONE && !by_y) {}
    template <bool STREAM>                        // (chunked slabs: read once more)
    __device__ __forceinline__ void load(int i, Raw<T, V>& xv, Raw<T, V>& g) const {
        xv = load_raw<T, V, STREAM>(x[i], nv);
        g = load_raw<T, V, STREAM>(dy[i], nv);
        if (by_y) {
            float r[V];
            load_part<T, V, STREAM>(y[i], nv, r);
            unsigned keep = 0;
#pragma unroll
            for (int v = 0; v < V; ++v) keep |= (unsigned)!(r[v] <= 0.f) << v;
            keep_raw<T, V>(g, keep);
        }
    }
    // dz and x - mean of row i from that
    __device__ __forceinline__ void dz_of(const P2pflGroupNorm& a, int i, const Raw<T, V>& xv, const Raw<T, V>& g, const float (&mu)[V],
                                          const float (&rw)[V], const float (&bb)[V], float (&d)[V], float (&dz)[V]) const {
        unpack<T, V>(xv, d);
        unpack<T, V>(g, dz);
#pragma unroll
        for (int v = 0; v < V; ++v) d[v] -= mu[v];
        if (drops) {
#pragma unroll
            for (int v = 0; v < V; ++v) dz[v] *= a.drop.scale;
        }
        if (a.act == ACT_NONE || by_y) return;
        float z[V];
#pragma unroll
        for (int v = 0; v < V; ++v) z[v] = d[v] * rw[v] + bb[v];
        if (has_res) {
            float r[V];
            load_part<T, V>(res[i], nv, r);
#pragma unroll
            for (int v = 0; v < V; ++v) z[v] += r[v];
        }
        switch (a.act) {
            case ACT_RELU:
#pragma unroll
                for (int v = 0; v < V; ++v) dz[v] = z[v] <= 0.f ? 0.f : dz[v];
                break;
            case ACT_SILU:
#pragma unroll
                for (int v = 0; v < V; ++v) dz[v] *= dact_of(z[v], ACT_SILU);
                break;
            case ACT_GELU:
#pragma unroll
                for (int v = 0; v < V; ++v) dz[v] *= dact_of(z[v], ACT_GELU);
                break;
        }
    }
};

// dx = rstd w dz - rstd m1 - (x - mean) rstd^2 m2 (and dres = dz) of a thread's rows; m1, m2: the group means of t and t xhat.
template <class T, int V, int I, class X>
__device__ __forceinline__ void gn_bwd_finish(const P2pflGroupNorm& a, const Place<V>& p, const GnRows<T, V>& in, int s0, int left,
                                              const float (&mu)[V], const float (&rw)[V], const float (&bb)[V], const float* g1,
                                              const float* g2, X row_of) {
    const int cpg = a.C / a.G;
    const float inv = 1.f / ((float)a.S * (float)cpg);
    float c1[V], c2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int gi = v < p.nv ? (p.col * V + v) / cpg : 0;
        const float rs = a.rstd[p.kn * a.G + p.g0 + gi];
        c1[v] = rs * (g1[gi] * inv);
        c2[v] = rs * (rs * (g2[gi] * inv));
    }
    const auto pdx = p.template walk<T>(a.dx, s0), pdres = p.template walk<T>(a.dres, s0);
#pragma unroll
    for (int i = 0; i < I; ++i) {
        if (i * p.rpp < left) {
            float d[V], dz[V];
            Raw<T, V> x, g;
            row_of(i, x, g);
            in.dz_of(a, i, x, g, mu, rw, bb, d, dz);
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] = dz[v] * rw[v] - c1[v] - d[v] * c2[v];
            if (a.dres.p) store_part<T, V>(pdres[i], p.nv, dz);
            store_part<T, V>(pdx[i], p.nv, d);
        }
    }
}

// Per-channel sums of (dz, dz xhat) over a chunk, and (whole slabs) dx from them. `part`: [K N][chunks][2][C].
template <class T, int V, int I, bool SPLIT>
__global__ __launch_bounds__(1024) void gn_bwd_kernel(P2pflGroupNorm a, Cut cut, float* part) {
    extern __shared__ float lds[];
    const Place<V> p(a, cut);
    const int cpg = a.C / a.G;
    const int s0 = p.chunk * cut.rows, s1 = min(a.S, s0 + cut.rows), left = p.on ? s1 - s0 - p.row : 0;
    const int cwp = p.vc * V;
    float* red = lds;
    float* ch = red + 2 * blockDim.x * V;
    float* gv = ch + 2 * cwp;
    const GnRows<T, V> in(a, p, s0);
    Raw<T, V> x[I], g[I];
#pragma unroll
    for (int i = 0; i < I; ++i)
        if (i * p.rpp < left) in.template load<!SPLIT>(i, x[i], g[i]);
    if (in.drops) {
        KeepRows<V, I> keep;
        gn_draw<V, I>(a, p, s0, left, keep);
#pragma unroll
        for (int i = 0; i < I; ++i) keep_raw<T, V>(g[i], keep[i]);
    }
    float mu[V], rs[V], rw[V], bb[V];
    gn_params<V>(a, p, mu, rs, rw, bb);
    float sum[2][V];
#pragma unroll
    for (int v = 0; v < V; ++v) sum[0][v] = sum[1][v] = 0.f;
#pragma unroll
    for (int i = 0; i < I; ++i) {
        if (i * p.rpp < left) {
            float d[V], dz[V];
            in.dz_of(a, i, x[i], g[i], mu, rw, bb, d, dz);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                sum[0][v] += v < p.nv ? dz[v] : 0.f;
                sum[1][v] += v < p.nv ? dz[v] * d[v] : 0.f;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sum[1][v] *= rs[v];
    channel_sums<V, 2>(sum, p, red, ch);
    float* o = part + (p.kn * cut.chunks + p.chunk) * 2 * a.C + p.c0;
    for (int i = threadIdx.x; i < p.cw; i += blockDim.x) { o[i] = ch[i]; o[a.C + i] = ch[cwp + i]; }
    if constexpr (!SPLIT) {
        auto w_of = [&](int c) { return a.w ? a.w[p.k * a.w_cs + p.c0 + c] : 1.f; };
        group_sums(p.ng, cpg, gv, [&](int c) { return ch[c] * w_of(c); });
        group_sums(p.ng, cpg, gv + cut.gpb, [&](int c) { return ch[cwp + c] * w_of(c); });
        if (p.on) gn_bwd_finish<T, V, I>(a, p, in, s0, left, mu, rw, bb, gv, gv + cut.gpb,
                                         [&](int i, Raw<T, V>& xv, Raw<T, V>& dv) { xv = x[i]; dv = g[i]; });
    }
}

// Chunked slabs: sums over the chunks, [K N][2][C].
__global__ __launch_bounds__(256) void gn_bwd_join_kernel(P2pflGroupNorm a, int chunks, const float* part, float* whole) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x, row = 2L * a.C;
    if (i >= (long)a.K * a.N * row) return;
    const long kn = i / row, c = i - kn * row;
    float t = 0.f;
    for (int j = 0; j < chunks; ++j) t += part[(kn * chunks + j) * row + c];
    whole[i] = t;
}

template <class T, int V, int I>
__global__ __launch_bounds__(1024) void gn_bwd_apply_kernel(P2pflGroupNorm a, Cut cut, const float* whole) {
    extern __shared__ float lds[];                 // [2][gpb]
    const Place<V> p(a, cut);
    const int cpg = a.C / a.G;
    const int s0 = p.chunk * cut.rows, s1 = min(a.S, s0 + cut.rows);
    const float* h = whole + p.kn * 2 * a.C + p.c0;
    auto w_of = [&](int c) { return a.w ? a.w[p.k * a.w_cs + p.c0 + c] : 1.f; };
    group_sums(p.ng, cpg, lds, [&](int c) { return h[c] * w_of(c); });
    group_sums(p.ng, cpg, lds + cut.gpb, [&](int c) { return h[a.C + c] * w_of(c); });
    if (!p.on) return;
    float mu[V], rs[V], rw[V], bb[V];
    gn_params<V>(a, p, mu, rs, rw, bb);
    const GnRows<T, V> in(a, p, s0);
    KeepRows<V, I> keep;
    gn_draw<V, I>(a, p, s0, s1 - s0 - p.row, keep);
    gn_bwd_finish<T, V, I>(a, p, in, s0, s1 - s0 - p.row, mu, rw, bb, lds, lds + cut.gpb,
                           [&](int i, Raw<T, V>& xv, Raw<T, V>& dv) {
                               in.template load<true>(i, xv, dv);
                               if (in.drops) keep_raw<T, V>(dv, keep[i]);
                           });
}

// dw, db: the samples' per-channel sums, four interleaved runs of samples added in order (dw null: only db, and the other way
// round).
__global__ __launch_bounds__(256) void gn_param_grads_kernel(P2pflGroupNorm a, const float* whole) {
    __shared__ float sums[4][2][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6, c = blockIdx.x * 64 + lane, k = blockIdx.y;
    const long row = 2L * a.C;
    float sb = 0.f, sw = 0.f;
    if (c < a.C) {
        const float* h = whole + (long)k * a.N * row + c;
        int n = run;
        for (; n + 12 < a.N; n += 16) {
            const float *h0 = h + n * row, *h1 = h0 + 4 * row, *h2 = h1 + 4 * row, *h3 = h2 + 4 * row;
            const float b0 = h0[0], b1 = h1[0], b2 = h2[0], b3 = h3[0], w0 = h0[a.C], w1 = h1[a.C], w2 = h2[a.C], w3 = h3[a.C];
            sb = (((sb + b0) + b1) + b2) + b3;
            sw = (((sw + w0) + w1) + w2) + w3;
        }
        for (; n < a.N; n += 4) { sb += h[n * row]; sw += h[n * row + a.C]; }
    }
    sums[run][0][lane] = sb;
    sums[run][1][lane] = sw;
    __syncthreads();
    if (run != 0 || c >= a.C) return;
    if (a.db) a.db[k * a.db_cs + c] = (sums[0][0][lane] + sums[1][0][lane]) + (sums[2][0][lane] + sums[3][0][lane]);
    if (a.dw) a.dw[k * a.dw_cs + c] = (sums[0][1][lane] + sums[1][1][lane]) + (sums[2][1][lane] + sums[3][1][lane]);
}

// ------------------------------------------------------------------------------------------------ host
inline int cdiv(long a, long b) { return (int)((a + b - 1) / b); }

// Vector of a slab: 16 bytes; 8 for 16-bit maps so narrow that a row is one short vector.
inline int vec_of(const P2pflGroupNorm& a) { return a.dtype == DT_F32 ? 4 : a.C <= 4 ? 4 : 8; }

// Channels of a slab: what keeps the reduction buffers of a block within 64 KB of LDS. A group has to fit.
constexpr int MAX_CHANNELS = 2048;

// How the maps are cut: slabs of whole groups that a block can hold, of at least 128 bytes of a row
// - a cache line; blocks of half lines reach half the rate - or, for tall maps, 64; as narrow as that allows while there are
// fewer than two blocks per CU, else of up to 16 KB. A slab that no block can hold is cut into chunks of rows.
struct Limits { int threads, tall_threads, hold; };      // of a block; of one that holds a tall slab; vectors a thread holds

inline Cut cut_with(const P2pflGroupNorm& a, int V, int gpb, int nt, int most_iters) {
    Cut c{};
    const int vc = cdiv((long)gpb * (a.C / a.G), V);
    c.gpb = gpb;
    c.slabs = cdiv(a.G, gpb);
    c.nt = max(nt, cdiv(vc, 64) * 64);
    const int rpp = c.nt / vc;
    c.iters = 1;
    while (c.iters < most_iters && (long)c.iters * rpp < a.S) c.iters *= 2;
    c.rows = c.iters * rpp;
    c.chunks = cdiv(a.S, c.rows);
    return c;
}

Cut cut_of(const P2pflGroupNorm& a, int V, Limits lim) {
    const int cpg = a.C / a.G, size = a.dtype == DT_F32 ? 4 : 2;
    int step = 1;                                  // groups that fill whole vectors
    while ((long)step * cpg % V && step < V) step *= 2;
    const int most = max(1, min(a.G, MAX_CHANNELS / cpg));
    auto at_least = [&](int bytes) { return min(most, cdiv(cdiv(bytes, (long)cpg * size), step) * step); };
    for (int bytes = 128; bytes >= 64; bytes /= 2) {
        int gpb = at_least(bytes);
        while (gpb < most && (long)a.S * gpb * cpg * size * 2 <= 16384 && (long)a.K * a.N * cdiv(a.G, 2 * gpb) >= 512) gpb = min(most, 2 * gpb);
        const long vectors = (long)a.S * cdiv((long)gpb * cpg, V);
        // four vectors a thread; one, where the blocks are too few to hide what a vector costs
        const long each = (long)a.K * a.N * cdiv(a.G, gpb) >= 512 ? 4 : 1;
        const int nt = (int)min((long)lim.threads, max(1L, (vectors + 64 * each - 1) / (64 * each)) * 64);
        Cut c = cut_with(a, V, gpb, nt, lim.hold);
        if (c.chunks > 1 && lim.tall_threads > lim.threads) c = cut_with(a, V, gpb, lim.tall_threads, lim.hold);
        if (c.chunks == 1) return c;
    }
    return cut_with(a, V, most, lim.threads, 8);
}

// Forward: two blocks of 512 threads with sixteen 16-byte vectors each in 128 registers fill a CU; a tall slab takes 1024. Backward:
// 1024 threads with x and dy of eight 16-byte (fp32) or sixteen 8-byte vectors, again in 128 registers - sixteen waves a CU
// cover each other's exponentials (eight waves with twice the vectors, both with stores through the caches: 359 us against 332 at
// 50 x 32 x 1024 x 64 bf16, silu and dropout; 10 x 32 x 1024 x 64 fp32, relu and residual: 129 against 120. With stores past
// the caches the sixteen waves take 275 and 94.)
constexpr Limits FWD{512, 1024, 16};
inline Limits backward_limits(const P2pflGroupNorm& a) { return {1024, 1024, a.dtype == DT_F32 ? 8 : 16}; }
constexpr int BWD_THREADS = 1024, BWD_VECTOR = 4;

template <int MOST, class F>
int by_iters(int iters, F f) {
    switch (iters) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 4: return f(std::integral_constant<int, 4>());
        case 8: return f(std::integral_constant<int, 8>());
        case 16: if constexpr (MOST == 16) return f(std::integral_constant<int, 16>());
    }
    return -2;
}

template <class T, int V>
int forward(const P2pflGroupNorm& a, hipStream_t st) {
    const Cut c = cut_of(a, V, FWD);
    const int vc = cdiv((long)c.gpb * (a.C / a.G), V);
    const long blocks = (long)a.K * a.N * c.slabs * c.chunks;
    if (a.C / a.G > MAX_CHANNELS || blocks * c.nt > 0xffffffffL) return -3;      // (a grid has less than 2^32 threads)
    const size_t lds = lds_floats(1, V, c.nt, vc, c.gpb) * sizeof(float);
    return by_iters<16>(c.iters, [&](auto n) {
        constexpr int I = decltype(n)::value;
        if (c.chunks == 1) {
            gn_fwd_kernel<T, V, I, false><<<(unsigned)blocks, c.nt, lds, st>>>(a, c);
            return (int)hipGetLastError();
        }
        const long kng = (long)a.K * a.N * a.G;
        if (a.scratch_len < 2 * kng * c.chunks + 2 * kng) return -5;
        float* mean = a.mean ? a.mean : a.scratch + 2 * kng * c.chunks;
        float* rstd = a.rstd ? a.rstd : a.scratch + 2 * kng * c.chunks + kng;
        gn_fwd_kernel<T, V, I, true><<<(unsigned)blocks, c.nt, lds, st>>>(a, c);
        gn_join_kernel<<<cdiv(kng, 64), 64, 0, st>>>(a, c, mean, rstd);
        gn_apply_kernel<T, V, I><<<(unsigned)blocks, c.nt, 0, st>>>(a, c, mean, rstd);
        return (int)hipGetLastError();
    });
}

int param_grads(const P2pflGroupNorm& a, const float* whole, hipStream_t st) {
    if (a.dw || a.db)
        for (int k0 = 0; k0 < a.K; k0 += 65535) {                // (the y dimension of a grid ends at 65535)
            P2pflGroupNorm ak = a;
            if (ak.dw) ak.dw += k0 * a.dw_cs;
            if (ak.db) ak.db += k0 * a.db_cs;
            gn_param_grads_kernel<<<dim3(cdiv(a.C, 64), min(65535, a.K - k0)), 256, 0, st>>>(ak, whole + (long)k0 * a.N * 2 * a.C);
        }
    return (int)hipGetLastError();
}

template <class T, int V>
int backward(const P2pflGroupNorm& a, hipStream_t st) {
    const Cut c = cut_of(a, V, backward_limits(a));
    const int vc = cdiv((long)c.gpb * (a.C / a.G), V);
    const long blocks = (long)a.K * a.N * c.slabs * c.chunks;
    if (a.C / a.G > MAX_CHANNELS || blocks * c.nt > 0xffffffffL) return -3;      // (a grid has less than 2^32 threads)
    const long whole_len = (long)a.K * a.N * 2 * a.C;
    if (a.scratch_len < whole_len * (c.chunks > 1 ? c.chunks + 1 : 1)) return -5;
    float* whole = a.scratch;
    float* part = c.chunks > 1 ? a.scratch + whole_len : whole;
    const size_t lds = lds_floats(2, V, c.nt, vc, c.gpb) * sizeof(float);
    const int rc = by_iters<sizeof(T) == 4 ? 8 : 16>(c.iters, [&](auto n) {
        constexpr int I = decltype(n)::value;
        if (c.chunks == 1) {
            gn_bwd_kernel<T, V, I, false><<<(unsigned)blocks, c.nt, lds, st>>>(a, c, whole);
            return 0;
        }
        gn_bwd_kernel<T, V, I, true><<<(unsigned)blocks, c.nt, lds, st>>>(a, c, part);
        gn_bwd_join_kernel<<<cdiv(whole_len, 256), 256, 0, st>>>(a, c.chunks, part, whole);
        gn_bwd_apply_kernel<T, V, I><<<(unsigned)blocks, c.nt, 2 * c.gpb * sizeof(float), st>>>(a, c, whole);
        return 0;
    });
    return rc ? rc : param_grads(a, whole, st);
}

// Reduction buffer, per-channel sums and the values of up to MAX_CHANNELS groups in 64 KB of LDS.
static_assert(4 * (FWD.tall_threads * 8 + MAX_CHANNELS + 2 * MAX_CHANNELS) <= 65536, "forward LDS");
static_assert(4 * (2 * BWD_THREADS * BWD_VECTOR + 2 * MAX_CHANNELS + 2 * MAX_CHANNELS) <= 65536, "backward LDS");
static_assert(MAX_CHANNELS / BWD_VECTOR <= BWD_THREADS && MAX_CHANNELS / 4 <= FWD.threads, "columns of a slab");

}  // namespace

// What a type's translation unit offers to the entry points.
template <class T> int group_norm_pass(const P2pflGroupNorm& a, bool backwards, hipStream_t st);

#ifdef GROUP_NORM_TYPE
template <> int group_norm_pass<GROUP_NORM_TYPE>(const P2pflGroupNorm& a, bool backwards, hipStream_t st) {
    typedef GROUP_NORM_TYPE T;
    if (backwards) return backward<T, BWD_VECTOR>(a, st);
    if constexpr (sizeof(T) == 2)
        if (vec_of(a) == 8) return forward<T, 8>(a, st);
    return forward<T, 4>(a, st);
}
#endif
