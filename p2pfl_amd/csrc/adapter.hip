// Low-rank adapters of K clients beside one shared projection W [Out, In]:
//
//   forward   u = s drop(x) A_k^T          y  = x W^T + b + u B_k^T
//   dgrad     v = s dy B_k                 dx = dy W + drop'(v A_k)
//   wgrad     dA_k = v^T drop(x)           dB_k = dy^T u
//
// for the rows of client k; the rows of a client are consecutive (row_ptr, or K equal blocks), rows behind the last client
// have no adapter. u and v are fp32 and kept for the weight gradients.
//
// The shared product is one matrix product over the rows of ALL clients: W is read once, not once per client. The adapters
// enter it as a few more steps of the same matrix instructions - for every client with rows in a tile, R columns of u against
// B_k, selected into that client's rows (a client whose adapter holds NaN does not reach its neighbours) - so y is written
// once.
//
// Precision: bf16 / fp16 maps multiply on their own matrix instructions with fp32 accumulation, u rounded to the map's type
// only as an operand of that last product. fp32 maps are decomposed EXACTLY into three bf16 terms on the way into LDS and
// multiplied as six bf16 products (dropped cross terms <= 2^-24 of a product; common.h).
#include <type_traits>
#include "typed.h"
#include "philox.h"

struct P2pflAdapter {
    const void* x; long x_cs, x_rs;               // [T] rows of In: client stride (equal blocks) and row stride
    const void* w; long w_rs;                     // [Out] rows of In
    const void* bias;                             // [Out] or null
    const void* la; long la_cs;                   // forward: A [K][R][In];  dgrad: B transposed, [K][R][Out]
    const void* lb; long lb_cs;                   // forward: B [K][Out][R]; dgrad: A transposed, [K][In][R]
    float* u;                                     // [T][R]
    void* y; long y_cs, y_rs;                     // [T] rows of Out
    const int* row_ptr;                           // [K + 1], or null: client k has rows k B .. (k + 1) B - 1
    P2pflDrop drop;                               // of x (forward: in the shrink product), of the adapters' part of y (dgrad)
    int drop_out;
    int K, T, B, In, Out, R, dtype;
    float scale;
};

namespace {

// ------------------------------------------------------------------------------------------------ rows and clients
struct Rows {
    const int* ptr; int K, T, B;
    __device__ __forceinline__ Rows(const P2pflAdapter& a) : ptr(a.row_ptr), K(a.K), T(a.T), B(a.B) {}
    // whatever row_ptr holds, a client's rows are inside [0, T]
    __device__ __forceinline__ int lo(int k) const { return ptr ? min(max(ptr[k], 0), T) : k * B; }
    __device__ __forceinline__ int hi(int k) const { return ptr ? min(max(ptr[k + 1], lo(k)), T) : (k + 1) * B; }
    // the first client that ends behind this row (K: none)
    __device__ __forceinline__ int first_ending_after(int row) const {
        if (!ptr) return B > 0 ? min(row / B, K) : K;
        int a = 0, b = K;
        while (a < b) {
            const int m = (a + b) >> 1;
            if (ptr[m + 1] > row) b = m; else a = m + 1;
        }
        return a;
    }
    // client of a row, or -1
    __device__ __forceinline__ int client(int row) const {
        const int k = first_ending_after(row);
        return k < K && row >= lo(k) && row < hi(k) ? k : -1;
    }
};

__device__ __forceinline__ long row_offset(int row, int B, long cs, long rs) {
    return B > 0 ? (long)(row / B) * cs + (long)(row % B) * rs : (long)row * rs;
}

// ------------------------------------------------------------------------------------------------ transposition
// [batch][rows][cols] -> [batch][cols][rows], 64 x 64 tiles through LDS.
template <class U>
__global__ __launch_bounds__(256) void transpose_kernel(const U* __restrict__ src, long s_cs, long s_rs, U* __restrict__ dst, int rows,
                                                        int cols) {
    __shared__ U tile[64][64 + 4 / sizeof(U)];
    const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64, k = blockIdx.z;
    src += k * s_cs;
    dst += (long)k * rows * cols;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int r = ty; r < 64; r += 4)
        if (r0 + r < rows && c0 + tx < cols) tile[r][tx] = src[(long)(r0 + r) * s_rs + c0 + tx];
    __syncthreads();
    for (int c = ty; c < 64; c += 4)
        if (c0 + c < cols && r0 + tx < rows) dst[(long)(c0 + c) * rows + r0 + tx] = tile[tx][c];
}

template <class U>
int transpose(const void* src, long s_cs, long s_rs, void* dst, int batch, int rows, int cols, hipStream_t s) {
    if (batch > 65535 || (rows + 63) / 64 > 65535) return -3;
    transpose_kernel<U><<<dim3((cols + 63) / 64, (rows + 63) / 64, batch), 256, 0, s>>>((const U*)src, s_cs, s_rs, (U*)dst, rows, cols);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ u = s drop(x) A^T
// A block: 16 rows of ONE client x 16 ranks; its waves split the reduction and are added through LDS in a fixed order.
// MFMA 16x16x32 (16-bit maps) / four 16x16x4 (fp32): lane l holds row (or rank) l & 15, columns 8 (l >> 4) .. + 7 / 4 (l >> 4)
// .. + 3 of a step, straight from global memory: 64 contiguous bytes of a row per step.
constexpr int SHRINK_WAVES = 8;

template <class T> struct Shrink;
template <> struct Shrink<float> {
    static constexpr int V = 4, STEP = 16;
    __device__ static f32x4 mma(const Raw<float, 4>& a, const Raw<float, 4>& b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, a.w[i]), __builtin_bit_cast(float, b.w[i]), c, 0, 0, 0);
        return c;
    }
};
template <> struct Shrink<__bf16> {
    static constexpr int V = 8, STEP = 32;
    __device__ static f32x4 mma(const Raw<__bf16, 8>& a, const Raw<__bf16, 8>& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Shrink<_Float16> {
    static constexpr int V = 8, STEP = 32;
    __device__ static f32x4 mma(const Raw<_Float16, 8>& a, const Raw<_Float16, 8>& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Zeroes the dropped elements of a vector; the factor 1 / (1 - p) is applied to the sum.
template <class T, int V>
__device__ __forceinline__ void keep_raw(Raw<T, V>& r, unsigned bits) {
#pragma unroll
    for (int i = 0; i < Raw<T, V>::W; ++i) {
        if constexpr (sizeof(T) == 4) r.w[i] = (bits >> i & 1u) ? r.w[i] : 0u;
        else r.w[i] &= ((bits >> (2 * i) & 1u) ? 0xffffu : 0u) | ((bits >> (2 * i + 1) & 1u) ? 0xffff0000u : 0u);
    }
}

// The tile of 16 rows with this number, counted over the clients' own tiles: (client, first row, last row); false: none.
// Ragged clients: every block counts the tiles of the clients before it.
__device__ __forceinline__ bool find_tile(const Rows& rows, int id, int& k, int& r0, int& r1) {
    if (!rows.ptr) {
        const int per = (rows.B + 15) / 16;
        k = per ? id / per : rows.K;
        if (k >= rows.K) return false;
        r0 = k * rows.B + (id % per) * 16;
        r1 = min(r0 + 16, (k + 1) * rows.B);
        return true;
    }
    int before = 0;
    const int lane = threadIdx.x & 63;
    for (int k0 = 0; k0 < rows.K; k0 += 64) {
        const int kk = k0 + lane;
        const int n = kk < rows.K ? (rows.hi(kk) - rows.lo(kk) + 15) / 16 : 0;
        int inc = n;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int t = __shfl_up(inc, off, 64);
            if (lane >= off) inc += t;
        }
        const int total = __shfl(inc, 63, 64);
        if (id < before + total) {
            const unsigned long long hit = __ballot(before + inc > id);
            const int l = __ffsll((long long)hit) - 1;
            const int first = before + __shfl(inc - n, l, 64);
            k = k0 + l;
            r0 = rows.lo(k) + (id - first) * 16;
            r1 = min(r0 + 16, rows.hi(k));
            return true;
        }
        before += total;
    }
    return false;
}

template <class T>
__global__ __launch_bounds__(64 * SHRINK_WAVES) void shrink_kernel(P2pflAdapter a) {
    constexpr int V = Shrink<T>::V, STEP = Shrink<T>::STEP;
    __shared__ float part[SHRINK_WAVES][16][17];
    const Rows rows(a);
    int k, r0, r1;
    if (!find_tile(rows, blockIdx.x, k, r0, r1)) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i16 = lane & 15, h = lane >> 4;
    const int row = r0 + i16, rank = blockIdx.y * 16 + i16;
    const T* x = (const T*)a.x + (row < r1 ? row_offset(row, a.B, a.x_cs, a.x_rs) : 0);
    const T* la = (const T*)a.la + k * a.la_cs + (long)min(rank, a.R - 1) * a.In;
    const bool drops = a.drop.seeds != nullptr && !a.drop_out;
    const DropKey key = drops ? DropKey(a.drop, k) : DropKey();
    const unsigned long long e0 = (unsigned long long)(row - rows.lo(k)) * a.In;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int c = wave * STEP; c < a.In; c += SHRINK_WAVES * STEP) {
        const int i = c + h * V, n = max(0, min(V, a.In - i));
        Raw<T, V> xv = load_raw<T, V>(x + i, row < r1 ? n : 0);
        const Raw<T, V> av = load_raw<T, V>(la + i, rank < a.R ? n : 0);
        if (drops) keep_raw<T, V>(xv, keep_bits<V>(a.drop, key, e0 + i));
        acc = Shrink<T>::mma(xv, av, acc);
    }
    // lane l holds rank l & 15 of rows 4 (l >> 4) .. + 3
#pragma unroll
    for (int j = 0; j < 4; ++j) part[wave][4 * h + j][i16] = acc[j];
    __syncthreads();
    if (threadIdx.x < 256) {
        const int rr = threadIdx.x >> 4, q = threadIdx.x & 15, rk = blockIdx.y * 16 + q;
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < SHRINK_WAVES; ++w) t += part[w][rr][q];
        if (r0 + rr < r1 && rk < a.R) a.u[(long)(r0 + rr) * a.R + rk] = t * a.scale * (drops ? a.drop.scale : 1.f);
    }
}

// u of the rows without a client.
__global__ __launch_bounds__(256) void shrink_free_kernel(P2pflAdapter a) {
    const Rows rows(a);
    for (int row = blockIdx.x * 256 + threadIdx.x; row < a.T; row += gridDim.x * 256)
        if (rows.client(row) < 0)
            for (int r = 0; r < a.R; ++r) a.u[(long)row * a.R + r] = 0.f;
}

template <class T>
int shrink(const P2pflAdapter& a, hipStream_t s) {
    const long tiles = a.row_ptr ? (long)a.T / 16 + a.K : (long)a.K * ((a.B + 15) / 16);
    if (tiles > 0)
        shrink_kernel<T><<<dim3((unsigned)tiles, (a.R + 15) / 16), 64 * SHRINK_WAVES, 0, s>>>(a);
    if (a.row_ptr) shrink_free_kernel<<<min(1024, (a.T + 255) / 256), 256, 0, s>>>(a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ the shared product
// C^T tiles: the matrix instruction's rows are columns of y (rows of W), its columns are rows of x, so a lane holds four
// consecutive elements of a row of y: one vector store, one Philox block.
template <class T> struct Terms { typedef T E; static constexpr int N = 1; };
template <> struct Terms<float> { typedef __bf16 E; static constexpr int N = 3; };

__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <class E> struct Frag;
template <> struct Frag<__bf16> { typedef bf16x8 type; };
template <> struct Frag<_Float16> { typedef f16x8 type; };

// 8 elements on their way into LDS: as stored, or (fp32) as three bf16 terms.
template <class T> struct Piece {
    Raw<T, 8> r;
    __device__ __forceinline__ void load(const T* p, int n) { r = load_raw<T, 8>(p, n); }
    __device__ __forceinline__ void set(const float (&v)[8]) { r = pack<T, 8>(v); }
    template <class F> __device__ __forceinline__ void store(T* lds, int) const { *reinterpret_cast<F*>(lds) = __builtin_bit_cast(F, r); }
};
template <> struct Piece<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p, int n) {
        float a[4], b[4];
        load_part<float, 4>(p, n, a);
        load_part<float, 4>(p + 4, n - 4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    }
    __device__ __forceinline__ void set(const float (&s)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = s[i];
    }
    template <class F> __device__ __forceinline__ void store(__bf16* lds, int plane) const {
        bf16x8 t[3];
        split_bf16x8<3>(v, t);
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<bf16x8*>(lds + i * plane) = t[i];
    }
};

template <class T, int BM, int BN, int BK>
__global__ __launch_bounds__(256) void shared_kernel(P2pflAdapter a) {
    typedef typename Terms<T>::E E;
    typedef typename Frag<E>::type F;
    constexpr int NS = Terms<T>::N, LDK = BK + 8, KC = BK / 8;
    constexpr int TM = BM / 2, TN = BN / 2, RM = TM / 32, RN = TN / 32;
    constexpr int PX = BM * KC / 256, PW = BN * KC / 256;
    __shared__ E xs[NS][BM * LDK], ws[NS][BN * LDK];
    const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;            // rows of x, rows of W
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
    const int wm = (wave >> 1) * TM, wn = (wave & 1) * TN;
    const Rows rows(a);
    f32x16 acc[RN][RM];
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
        for (int j = 0; j < RM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    Piece<T> px[PX], pw[PW];
    auto put = [&]() {
#pragma unroll
        for (int i = 0; i < PX; ++i) {
            const int c = threadIdx.x + i * 256;
            px[i].template store<F>(&xs[0][(c / KC) * LDK + (c % KC) * 8], BM * LDK);
        }
#pragma unroll
        for (int i = 0; i < PW; ++i) {
            const int c = threadIdx.x + i * 256;
            pw[i].template store<F>(&ws[0][(c / KC) * LDK + (c % KC) * 8], BN * LDK);
        }
    };
    auto multiply = [&](f32x16 (&acc)[RN][RM]) {
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
            F xf[NS][RM], wf[NS][RN];
#pragma unroll
            for (int t = 0; t < NS; ++t) {
#pragma unroll
                for (int j = 0; j < RM; ++j) xf[t][j] = *reinterpret_cast<const F*>(&xs[t][(wm + j * 32 + r32) * LDK + kk * 16 + h * 8]);
#pragma unroll
                for (int i = 0; i < RN; ++i) wf[t][i] = *reinterpret_cast<const F*>(&ws[t][(wn + i * 32 + r32) * LDK + kk * 16 + h * 8]);
            }
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int t = 0; s + t < NS; ++t)
#pragma unroll
                    for (int i = 0; i < RN; ++i)
#pragma unroll
                        for (int j = 0; j < RM; ++j) acc[i][j] = mma32(wf[s][i], xf[t][j], acc[i][j]);
        }
    };

    // the adapters, client by client
    for (int k = rows.first_ending_after(m0); k < a.K; ++k) {
        const int lo = rows.lo(k), hi = rows.hi(k);
        if (lo >= m0 + BM) break;
        if (hi <= m0 || lo >= hi) continue;
        f32x16 own[RN][RM];
#pragma unroll
        for (int i = 0; i < RN; ++i)
#pragma unroll
            for (int j = 0; j < RM; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) own[i][j][e] = 0.f;
        const bool here = lo < m0 + wm + TM && hi > m0 + wm;       // the wave has rows of this client
        for (int r0 = 0; r0 < a.R; r0 += BK) {
#pragma unroll
            for (int i = 0; i < PX; ++i) {
                const int c = threadIdx.x + i * 256, row = m0 + c / KC, r = r0 + (c % KC) * 8;
                float v[8];
                const bool mine = row >= lo && row < hi;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = mine && r + j < a.R ? a.u[(long)row * a.R + r + j] : 0.f;
                px[i].set(v);
            }
#pragma unroll
            for (int i = 0; i < PW; ++i) {
                const int c = threadIdx.x + i * 256, col = n0 + c / KC, r = r0 + (c % KC) * 8;
                const int n = col < a.Out ? max(0, min(8, a.R - r)) : 0;
                pw[i].load((const T*)a.lb + (n ? k * a.lb_cs + (long)col * a.R + r : 0), n);
            }
            __syncthreads();
            put();
            __syncthreads();
            if (here) multiply(own);
        }
        if (!here) continue;
#pragma unroll
        for (int j = 0; j < RM; ++j) {
            const int row = m0 + wm + j * 32 + r32;
            const bool mine = row >= lo && row < hi;
#pragma unroll
            for (int i = 0; i < RN; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = mine ? own[i][j][e] : acc[i][j][e];
        }
    }
    if (a.drop_out && a.drop.seeds) {             // the adapters' part alone is in the accumulators
#pragma unroll
        for (int j = 0; j < RM; ++j) {
            const int row = m0 + wm + j * 32 + r32;
            const int k = row < a.T ? rows.client(row) : -1;
            if (k < 0) continue;
            const DropKey key(a.drop, k);
            const unsigned long long e0 = (unsigned long long)(row - rows.lo(k)) * a.Out;
#pragma unroll
            for (int i = 0; i < RN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const unsigned bits = keep_bits<4>(a.drop, key, e0 + n0 + wn + i * 32 + 8 * q + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = (bits >> e & 1u) ? acc[i][j][4 * q + e] * a.drop.scale : 0.f;
                }
        }
    }

    long xo[PX], wo[PW];
#pragma unroll
    for (int i = 0; i < PX; ++i) {
        const int row = m0 + (threadIdx.x + i * 256) / KC;
        xo[i] = row < a.T ? row_offset(row, a.B, a.x_cs, a.x_rs) : -1;
    }
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        const int col = n0 + (threadIdx.x + i * 256) / KC;
        wo[i] = col < a.Out ? (long)col * a.w_rs : -1;
    }
    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < PX; ++i) {
            const int c = k0 + ((threadIdx.x + i * 256) % KC) * 8, n = xo[i] < 0 ? 0 : max(0, min(8, a.In - c));
            px[i].load((const T*)a.x + (n ? xo[i] + c : 0), n);
        }
#pragma unroll
        for (int i = 0; i < PW; ++i) {
            const int c = k0 + ((threadIdx.x + i * 256) % KC) * 8, n = wo[i] < 0 ? 0 : max(0, min(8, a.In - c));
            pw[i].load((const T*)a.w + (n ? wo[i] + c : 0), n);
        }
    };
    fetch(0);
    for (int k0 = 0; k0 < a.In; k0 += BK) {
        __syncthreads();
        put();
        __syncthreads();
        if (k0 + BK < a.In) fetch(k0 + BK);
        multiply(acc);
    }

#pragma unroll
    for (int j = 0; j < RM; ++j) {
        const int row = m0 + wm + j * 32 + r32;
        if (row >= a.T) continue;
        T* y = (T*)a.y + row_offset(row, a.B, a.y_cs, a.y_rs);
#pragma unroll
        for (int i = 0; i < RN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = n0 + wn + i * 32 + 8 * q + 4 * h, n = min(4, a.Out - col);
                if (n <= 0) continue;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = acc[i][j][4 * q + e] + (a.bias && e < n ? (float)((const T*)a.bias)[col + e] : 0.f);
                store_part<T, 4>(y + col, n, v);
            }
    }
}

template <class T>
int shared_product(const P2pflAdapter& a, hipStream_t s) {
    constexpr int BK = sizeof(T) == 4 ? 16 : 64;
    const dim3 grid((a.Out + 127) / 128, (a.T + 127) / 128);
    shared_kernel<T, 128, 128, BK><<<grid, 256, 0, s>>>(a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ weight gradients
// out[k][wide][rank] or [k][rank][wide] = sum over the rows of client k of map[row][wide] * low[row][rank]: memory-bound (the
// map is read once per 64 ranks), so the products stay on fp32 MFMA whatever the map's type: exact operands, u and v are not rounded.
// MFMA 16x16x4: lane l brings V consecutive columns of row l >> 4 of a step, instruction j multiplies column j of each lane.
struct WgradArgs {
    const void* map; long cs, rs;
    const float* low;
    float* out; long out_cs;
    int wide, ranks_first, drops;
};

template <class T, int RT>
__global__ __launch_bounds__(256) void adapter_wgrad_kernel(P2pflAdapter a, WgradArgs ga, WgradArgs gb, int blocks_a) {
    constexpr int V = 16 / sizeof(T);
    const bool first = (int)blockIdx.x < blocks_a;
    const WgradArgs g = first ? ga : gb;
    const int tile = (first ? blockIdx.x : blockIdx.x - blocks_a) * 4 + (threadIdx.x >> 6);
    const int k = blockIdx.y, rank0 = blockIdx.z * 16 * RT;
    const int lane = threadIdx.x & 63, i16 = lane & 15, h = lane >> 4;
    const int c = tile * 16 * V + i16 * V, n = max(0, min(V, g.wide - c));
    const Rows rows(a);
    const int lo = rows.lo(k), hi = rows.hi(k);
    const bool drops = g.drops && a.drop.seeds;
    const DropKey key = drops ? DropKey(a.drop, k) : DropKey();
    f32x4 acc[RT][V];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int r = lo; r < hi; r += 4) {
        const int row = r + h;
        const bool in = row < hi;
        Raw<T, V> m = load_raw<T, V>((const T*)g.map + (in && n ? row_offset(row, a.B, g.cs, g.rs) + c : 0), in ? n : 0);
        if (drops) keep_raw<T, V>(m, keep_bits<V>(a.drop, key, (unsigned long long)(row - lo) * g.wide + c));
        float mv[V], lv[RT];
        unpack<T, V>(m, mv);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int rank = rank0 + 16 * t + i16;
            lv[t] = in && rank < a.R ? g.low[(long)row * a.R + rank] : 0.f;
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int v = 0; v < V; ++v)
                acc[t][v] = __builtin_amdgcn_mfma_f32_16x16x4f32(lv[t], mv[v], acc[t][v], 0, 0, 0);
    }
    const float f = drops ? a.drop.scale : 1.f;
    float* out = g.out + k * g.out_cs;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {              // lane l: ranks 4 (l >> 4) + e, columns c .. c + V - 1
            const int rank = rank0 + 16 * t + 4 * h + e;
            if (rank >= a.R) continue;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < n) out[g.ranks_first ? (long)rank * g.wide + c + v : (long)(c + v) * a.R + rank] = acc[t][v][e] * f;
        }
}

template <class T>
int weight_gradients(const P2pflAdapter& a, const WgradArgs& ga, const WgradArgs& gb, hipStream_t s) {
    constexpr int V = 16 / sizeof(T), COLS = 4 * 16 * V;
    const int blocks_a = ga.out ? (ga.wide + COLS - 1) / COLS : 0, blocks_b = gb.out ? (gb.wide + COLS - 1) / COLS : 0;
    if (a.K > 65535) return -3;
    if (blocks_a + blocks_b == 0) return 0;
    if (a.R <= 16) adapter_wgrad_kernel<T, 1><<<dim3(blocks_a + blocks_b, a.K, 1), 256, 0, s>>>(a, ga, gb, blocks_a);
    else adapter_wgrad_kernel<T, 2><<<dim3(blocks_a + blocks_b, a.K, (a.R + 31) / 32), 256, 0, s>>>(a, ga, gb, blocks_a);
    return (int)hipGetLastError();
}

template <class F>
int by_type(int dtype, F f) {
    switch (dtype) {
        case DT_F32: return f(float());
        case DT_BF16: return f(__bf16());
        case DT_F16: return f(_Float16());
    }
    return -2;
}

inline long floats_of(long elements, int dtype) { return dtype == DT_F32 ? elements : (elements + 1) / 2; }

}  // namespace

P2PFL_API int p2pfl_adapter_linear_fwd(const P2pflAdapter* a, void* stream) {
    if (a->T <= 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    return by_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        const int rc = shrink<T>(*a, s);
        return rc ? rc : shared_product<T>(*a, s);
    });
}

// Floats of scratch memory of the data gradient: W, A and B transposed.
P2PFL_API long p2pfl_adapter_linear_dgrad_scratch(int K, int In, int Out, int R, int dtype) {
    return floats_of((long)In * Out, dtype) + floats_of((long)K * R * In, dtype) + floats_of((long)K * R * Out, dtype) + 12;
}

// As the forward pass with dy for x and the roles of A and B exchanged: `a` holds x = dy, In = the projection's outputs, Out =
// its inputs, w [In][Out] as stored, la = B [K][In][R], lb = A [K][R][Out].
P2PFL_API int p2pfl_adapter_linear_dgrad(const P2pflAdapter* a0, float* scratch, long scratch_len, void* stream) {
    P2pflAdapter a = *a0;
    if (a.T <= 0) return 0;
    if (scratch_len < p2pfl_adapter_linear_dgrad_scratch(a.K, a.In, a.Out, a.R, a.dtype)) return -5;
    hipStream_t s = (hipStream_t)stream;
    auto up = [](long n) { return (n + 3) / 4 * 4; };
    float* wt = scratch;                                             // [Out][In]
    float* bt = wt + up(floats_of((long)a.In * a.Out, a.dtype));     // B transposed: [K][R][In]
    float* at = bt + up(floats_of((long)a.K * a.R * a.In, a.dtype)); // A transposed: [K][Out][R]
    auto all = [&](auto u) {
        typedef decltype(u) U;
        int rc = transpose<U>(a.w, 0, a.w_rs, wt, 1, a.In, a.Out, s);
        if (!rc && a.K) rc = transpose<U>(a.la, a.la_cs, a.R, bt, a.K, a.In, a.R, s);
        if (!rc && a.K) rc = transpose<U>(a.lb, a.lb_cs, a.Out, at, a.K, a.R, a.Out, s);
        return rc;
    };
    int rc = a.dtype == DT_F32 ? all(0u) : all((unsigned short)0);
    if (rc) return rc;
    a.w = wt; a.w_rs = a.In;
    a.la = bt; a.la_cs = (long)a.R * a.In;
    a.lb = at; a.lb_cs = (long)a.R * a.Out;
    a.drop_out = 1;
    return by_type(a.dtype, [&](auto t) {
        typedef decltype(t) T;
        const int r = shrink<T>(a, s);
        return r ? r : shared_product<T>(a, s);
    });
}

// dA (null: not wanted) and dB. `a` as in the forward pass, with y = dy and u; v beside it.
P2PFL_API int p2pfl_adapter_linear_wgrad(const P2pflAdapter* a, const float* v, float* dla, long dla_cs, float* dlb, long dlb_cs,
                                         void* stream) {
    if (a->K <= 0) return 0;
    const WgradArgs ga{a->x, a->x_cs, a->x_rs, v, dla, dla_cs, a->In, 1, 1};
    const WgradArgs gb{a->y, a->y_cs, a->y_rs, a->u, dlb, dlb_cs, a->Out, 0, 0};
    return by_type(a->dtype, [&](auto t) { return weight_gradients<decltype(t)>(*a, ga, gb, (hipStream_t)stream); });
}
