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
// Precision: bf16 / fp16 maps multiply on their own matrix instructions with fp32 accumulation. u stays fp32 but as an operand of
// that last product beside many rows: there it is two terms of the map's type (16 or 22 bits), brought into that type's range by a
// power of two per row and 32 ranks, which comes out of the accumulators again - u of any finite size is an operand. fp32 maps are
// decomposed into three bf16 terms on the way into LDS (exactly, between 2^-109 and the largest bf16, 3.389e38) and multiplied as six
// bf16 products (dropped cross terms <= 2^-24 of a product; common.h). An element beyond that, or an infinite one, makes the results
// that it enters infinite or NaN, and so does, in every type, an infinite element of B beside the two terms of u (A, in the data
// gradient); up to 64 rows are multiplied as they are.
//
// One translation unit per type of the rows (adapter_f32.hip, adapter_bf16.hip, adapter_f16.hip); adapter.hip has the entry points.
#pragma once
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
        while (b - a > 4) {                        // fifths: four independent loads per round trip
            const int q = (b - a) / 5, m1 = a + q, m2 = m1 + q, m3 = m2 + q, m4 = m3 + q;
            const int p1 = ptr[m1 + 1], p2 = ptr[m2 + 1], p3 = ptr[m3 + 1], p4 = ptr[m4 + 1];
            if (p1 > row) b = m1;
            else if (p2 > row) { a = m1 + 1; b = m2; }
            else if (p3 > row) { a = m2 + 1; b = m3; }
            else if (p4 > row) { a = m3 + 1; b = m4; }
            else a = m4 + 1;
        }
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

// ------------------------------------------------------------------------------------------------ loads into LDS
// One 16-byte load per lane straight into LDS: lane l's bytes land at lds + 16 l (`lds` is the same for the whole wave).
__device__ __forceinline__ void to_lds16(const void* p, void* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)lds,
                                     16, 0, 0);
}

// The block's barrier without the waits of __syncthreads: nothing moves across it, loads into LDS stay under way.
__device__ __forceinline__ void bare_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// all but the LEFT youngest loads of the wave are in
template <int LEFT = 0>
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt((LEFT & 15) | 7 << 4 | 15 << 8 | (LEFT >> 4) << 14); }
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 0 << 8 | 3 << 14); }

// ------------------------------------------------------------------------------------------------ u = s drop(x) A^T
// A block: 16 or 32 rows of ONE client x up to 64 ranks; its waves split the reduction and are added through LDS in a fixed
// order. MFMA 16x16x32 (16-bit maps) / four 16x16x4 (fp32): lane l holds row (or rank) l & 15, columns 8 (l >> 4) .. + 7 /
// 4 (l >> 4) .. + 3 of a step, straight from global memory. 32 rows where clients have that many: a block brings A_k in from
// L2 once more, and that is half of what it reads at rank 32.
constexpr int SHRINK_WAVES = 8;

template <class T> struct Shrink;
template <> struct Shrink<float> {
    static constexpr int V = 4;
    __device__ static f32x4 mma(const Raw<float, 4>& a, const Raw<float, 4>& b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, a.w[i]), __builtin_bit_cast(float, b.w[i]), c, 0, 0, 0);
        return c;
    }
};
template <> struct Shrink<__bf16> {
    static constexpr int V = 8;
    __device__ static f32x4 mma(const Raw<__bf16, 8>& a, const Raw<__bf16, 8>& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Shrink<_Float16> {
    static constexpr int V = 8;
    __device__ static f32x4 mma(const Raw<_Float16, 8>& a, const Raw<_Float16, 8>& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// acc[m][t] += rows of x[t] times rows of w[m] over this wave's units of [unit0, unit1) of the reduction. A unit is 256
// contiguous bytes of every row in four steps of 64 bytes, so a wave moves whole cache lines; units go round the block's
// waves. Blocks start at different units (`turn`): rows of a power-of-two length would otherwise ask the same memory channels
// everywhere at once.
template <class T> constexpr int unit_of() { return 16 * Shrink<T>::V; }

template <class T, int WAVES, int MT, int NT, class F>
__device__ __forceinline__ void stream_rows(const T* const (&w)[MT], const T* const (&x)[NT], int In, int unit0, int unit1, int turn,
                                            f32x4 (&acc)[MT][NT], F drop) {
    constexpr int V = Shrink<T>::V, STEP = 4 * V, UNIT = unit_of<T>();
    const int wave = threadIdx.x >> 6, h = (threadIdx.x & 63) >> 4;
    const int units = unit1 - unit0;
    for (int i = wave; i < units; i += WAVES) {
        const int u = unit0 + (i + turn) % units, c = u * UNIT + h * V;
        Raw<T, V> wv[MT][4], xv[NT][4];
        if ((u + 1) * UNIT <= In) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) wv[m][j] = load_raw<T, V>(w[m] + c + j * STEP);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) xv[t][j] = load_raw<T, V>(x[t] + c + j * STEP);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = max(0, min(V, In - c - j * STEP)), at = n ? c + j * STEP : 0;
#pragma unroll
                for (int m = 0; m < MT; ++m) wv[m][j] = load_raw<T, V>(w[m] + at, n);
#pragma unroll
                for (int t = 0; t < NT; ++t) xv[t][j] = load_raw<T, V>(x[t] + at, n);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int t = 0; t < NT; ++t) drop(xv[t][j], t, c + j * STEP);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[m][t] = Shrink<T>::mma(xv[t][j], wv[m][j], acc[m][t]);
        }
    }
}

// The tile of `tr` rows with this number, counted over the clients' own tiles: (client, first row, last row); false: none.
// Ragged clients: every block counts the tiles of the clients before it.
__device__ __forceinline__ bool find_tile(const Rows& rows, int tr, int id, int& k, int& r0, int& r1) {
    if (!rows.ptr) {
        const int per = (rows.B + tr - 1) / tr;
        k = per ? id / per : rows.K;
        if (k >= rows.K) return false;
        r0 = k * rows.B + (id % per) * tr;
        r1 = min(r0 + tr, (k + 1) * rows.B);
        return true;
    }
    int before = 0;
    const int lane = threadIdx.x & 63;
    for (int k0 = 0; k0 < rows.K; k0 += 64) {
        const int kk = k0 + lane;
        const int n = kk < rows.K ? (rows.hi(kk) - rows.lo(kk) + tr - 1) / tr : 0;
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
            r0 = rows.lo(k) + (id - first) * tr;
            r1 = min(r0 + tr, rows.hi(k));
            return true;
        }
        before += total;
    }
    return false;
}

// Blocks of a launch that compute u: client tiles x rank tiles x parts of the reduction, then the rows without a client.
struct ShrinkGrid {
    int tiles, ranks, parts, free;
    __host__ __device__ int blocks() const { return tiles * ranks * parts + free; }
};

constexpr int FREE_ROWS = 512;

ShrinkGrid shrink_grid(const P2pflAdapter& a, int tile_rows, int tile_ranks, int parts) {
    const int tiles = a.row_ptr ? a.T / tile_rows + a.K : a.K * ((a.B + tile_rows - 1) / tile_rows);
    return {tiles, (a.R + tile_ranks - 1) / tile_ranks, parts, a.row_ptr ? (a.T + FREE_ROWS - 1) / FREE_ROWS : 0};
}

// 16 MT ranks x 16 NT rows. `u`: [parts][T][R]; `sums`: LDS of WAVES * 16 NT * (16 MT + 1) floats.
template <class T, int WAVES, int MT, int NT>
__device__ __forceinline__ void shrink_block(const P2pflAdapter& a, const ShrinkGrid& grid, int id, float* u, float* sums) {
    constexpr int V = Shrink<T>::V, PITCH = 16 * MT + 1;
    const Rows rows(a);
    if (id >= grid.tiles * grid.ranks * grid.parts) {                 // zero u where no client is
        const int first = (id - grid.tiles * grid.ranks * grid.parts) * FREE_ROWS;
        for (int row = first + threadIdx.x; row < min(a.T, first + FREE_ROWS); row += 64 * WAVES)
            if (rows.client(row) < 0)
                for (int p = 0; p < grid.parts; ++p)
                    for (int r = 0; r < a.R; ++r) u[((long)p * a.T + row) * a.R + r] = 0.f;
        return;
    }
    const int part = id % grid.parts, rank0 = id / grid.parts % grid.ranks * 16 * MT;
    int k, r0, r1;
    if (!find_tile(rows, 16 * NT, id / (grid.parts * grid.ranks), k, r0, r1)) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i16 = lane & 15, h = lane >> 4;
    // rows and ranks behind the last compute on a copy of the last one; they are not stored
    const T *x[NT], *la[MT];
    unsigned long long e0[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = min(r0 + 16 * t + i16, r1 - 1);
        x[t] = (const T*)a.x + row_offset(row, a.B, a.x_cs, a.x_rs);
        e0[t] = (unsigned long long)(row - rows.lo(k)) * a.In;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) la[m] = (const T*)a.la + k * a.la_cs + (long)min(rank0 + 16 * m + i16, a.R - 1) * a.In;
    const bool drops = a.drop.seeds != nullptr && !a.drop_out;
    const DropKey key = drops ? DropKey(a.drop, k) : DropKey();
    const int units = (a.In + unit_of<T>() - 1) / unit_of<T>();
    const int u0 = (int)((long)units * part / grid.parts), u1 = (int)((long)units * (part + 1) / grid.parts);
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (drops)
        stream_rows<T, WAVES, MT, NT>(la, x, a.In, u0, u1, id, acc,
                                      [&](Raw<T, V>& v, int t, int c) { keep_raw<T, V>(v, keep_bits<V>(a.drop, key, e0[t] + c)); });
    else
        stream_rows<T, WAVES, MT, NT>(la, x, a.In, u0, u1, id, acc, [](Raw<T, V>&, int, int) {});
    // lane l holds rank l & 15 of rows 4 (l >> 4) .. + 3
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[(wave * 16 * NT + 16 * t + 4 * h + j) * PITCH + 16 * m + i16] = acc[m][t][j];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NT * 16 * MT; i += 64 * WAVES) {
        const int rr = i / (16 * MT), q = i % (16 * MT), rk = rank0 + q;
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) t += sums[(w * 16 * NT + rr) * PITCH + q];
        if (r0 + rr < r1 && rk < a.R) u[((long)part * a.T + r0 + rr) * a.R + rk] = t * a.scale * (drops ? a.drop.scale : 1.f);
    }
}

// The same sums where rows start on 16 bytes: whole cache lines go straight into LDS, 512 bytes of every row per stage and DEPTH
// stages in turn, and a wave multiplies 64 bytes of each. (From global memory to registers a wave asks for 64 bytes of sixteen
// rows at once, half a line each: 39 us against 27 for 8192 bf16 rows of 4096 at rank 32.)
// Layout: a row is 32 pieces of 16 bytes, piece q of row r in slot q ^ (r & 15); a wave's load fills two rows.
template <class T, int MT, int NT, int DEPTH>
__global__ __launch_bounds__(64 * SHRINK_WAVES, MT == 4 ? 2 : 4) void shrink_aligned_kernel(P2pflAdapter a, ShrinkGrid grid) {
    constexpr int V = Shrink<T>::V, PIECES = 32, COLS = PIECES * V, LINES = 16 * (MT + NT), PITCH = 16 * MT + 1;
    constexpr int LOADS = LINES / 2 / SHRINK_WAVES;
    static_assert(LOADS * 2 * SHRINK_WAVES == LINES, "loads of a stage");
    __shared__ __attribute__((aligned(16))) T ring[DEPTH][LINES * COLS];
    static_assert(sizeof(ring) >= sizeof(float) * SHRINK_WAVES * 16 * NT * PITCH, "sums");
    const Rows rows(a);
    const int own = grid.tiles * grid.ranks;
    float* sums = reinterpret_cast<float*>(&ring[0][0]);
    if ((int)blockIdx.x >= own) {                                     // (the zeros of rows without a client)
        shrink_block<T, SHRINK_WAVES, MT, NT>(a, grid, blockIdx.x, a.u, sums);
        return;
    }
    const int rank0 = blockIdx.x % grid.ranks * 16 * MT;
    int k, r0, r1;
    if (!find_tile(rows, 16 * NT, blockIdx.x / grid.ranks, k, r0, r1)) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i16 = lane & 15, h = lane >> 4;
    const T *p[LOADS];                             // lines of a stage: 16 NT rows of x, 16 MT rows of A
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int line = (wave * LOADS + i) * 2 + (lane >> 5);
        p[i] = (line < 16 * NT ? (const T*)a.x + row_offset(min(r0 + line, r1 - 1), a.B, a.x_cs, a.x_rs)
                               : (const T*)a.la + k * a.la_cs + (long)min(rank0 + line - 16 * NT, a.R - 1) * a.In) +
               ((lane & 31) ^ (line & 15)) * V;
    }
    const T *x[NT], *la[MT];
    unsigned long long e0[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = min(r0 + 16 * t + i16, r1 - 1);
        x[t] = (const T*)a.x + row_offset(row, a.B, a.x_cs, a.x_rs);
        e0[t] = (unsigned long long)(row - rows.lo(k)) * a.In;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) la[m] = (const T*)a.la + k * a.la_cs + (long)min(rank0 + 16 * m + i16, a.R - 1) * a.In;
    const bool drops = a.drop.seeds != nullptr && !a.drop_out;
    const DropKey key = drops ? DropKey(a.drop, k) : DropKey();
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int stages = a.In / COLS;
    auto fetch = [&](int s) {
        const int at = min(s, stages - 1);         // (behind the last stage: that one again, unused)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) to_lds16(p[i] + (long)at * COLS, &ring[s % DEPTH][(wave * LOADS + i) * 2 * COLS]);
    };
    if (stages > 0) {
#pragma unroll
        for (int s = 0; s < DEPTH - 1; ++s) fetch(s);
        for (int s = 0; s < stages; ++s) {
            wait_loads<(DEPTH - 2) * LOADS>();
            wait_lds();
            bare_barrier();
            fetch(s + DEPTH - 1);
            const T* at = &ring[s % DEPTH][0];
            const int piece = 4 * wave + h;
            Raw<T, V> xv[NT], av[MT];
#pragma unroll
            for (int t = 0; t < NT; ++t) xv[t] = *reinterpret_cast<const Raw<T, V>*>(at + (16 * t + i16) * COLS + (piece ^ i16) * V);
#pragma unroll
            for (int m = 0; m < MT; ++m) av[m] = *reinterpret_cast<const Raw<T, V>*>(at + (16 * (NT + m) + i16) * COLS + (piece ^ i16) * V);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (drops) keep_raw<T, V>(xv[t], keep_bits<V>(a.drop, key, e0[t] + (long)s * COLS + piece * V));
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m][t] = Shrink<T>::mma(xv[t], av[m], acc[m][t]);
            }
        }
        wait_loads<>();
        wait_lds();
        bare_barrier();
    }
    const int units = (a.In + unit_of<T>() - 1) / unit_of<T>();       // the last columns (a unit is half a stage)
    stream_rows<T, SHRINK_WAVES, MT, NT>(la, x, a.In, 2 * stages, units, 0, acc, [&](Raw<T, V>& v, int t, int c) {
        if (drops) keep_raw<T, V>(v, keep_bits<V>(a.drop, key, e0[t] + c));
    });
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[(wave * 16 * NT + 16 * t + 4 * h + j) * PITCH + 16 * m + i16] = acc[m][t][j];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * NT * 16 * MT; i += 64 * SHRINK_WAVES) {
        const int rr = i / (16 * MT), q = i % (16 * MT), rk = rank0 + q;
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < SHRINK_WAVES; ++w) t += sums[(w * 16 * NT + rr) * PITCH + q];
        if (r0 + rr < r1 && rk < a.R) a.u[(long)(r0 + rr) * a.R + rk] = t * a.scale * (drops ? a.drop.scale : 1.f);
    }
}

template <class T, int MT, int NT>
__global__ __launch_bounds__(64 * SHRINK_WAVES) void shrink_kernel(P2pflAdapter a, ShrinkGrid grid) {
    __shared__ float sums[SHRINK_WAVES * 16 * NT * (16 * MT + 1)];
    shrink_block<T, SHRINK_WAVES, MT, NT>(a, grid, blockIdx.x, a.u, sums);
}

template <class T, int MT, int NT>
int shrink_as(const P2pflAdapter& a, hipStream_t s) {
    const ShrinkGrid g = shrink_grid(a, 16 * NT, 16 * MT, 1);
    constexpr int DEPTH = MT == 4 ? 3 : MT + NT == 2 ? 4 : MT + NT == 3 ? 3 : 2;     // two blocks per CU where they fit
    const bool aligned = ((size_t)a.x | (size_t)a.la) % 16 == 0 && (a.x_rs | a.x_cs | a.la_cs | a.In) * sizeof(T) % 16 == 0;
    if (g.blocks() <= 0) return 0;
    if (aligned) shrink_aligned_kernel<T, MT, NT, DEPTH><<<g.blocks(), 64 * SHRINK_WAVES, 0, s>>>(a, g);
    else shrink_kernel<T, MT, NT><<<g.blocks(), 64 * SHRINK_WAVES, 0, s>>>(a, g);
    return (int)hipGetLastError();
}

template <class T>
int shrink(const P2pflAdapter& a, hipStream_t s) {
    // 32 rows only where that still leaves a block for every CU
    const bool tall = (long)a.T >= 32L * a.K && a.T >= 32 * 192;
    if (a.R <= 16) return tall ? shrink_as<T, 1, 2>(a, s) : shrink_as<T, 1, 1>(a, s);
    if (a.R <= 32) return tall ? shrink_as<T, 2, 2>(a, s) : shrink_as<T, 2, 1>(a, s);
    return tall ? shrink_as<T, 4, 2>(a, s) : shrink_as<T, 4, 1>(a, s);
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to 64 rows: the product reads W once and is bound by that. One CU takes in about 32 bytes per ns, so every byte that
// reaches it twice counts: a wave keeps 64 rows of W x all rows of x per unit in registers and the reduction is split over
// blocks until the chip is full. The blocks of u run in the same launch; join_kernel adds the parts of both.
constexpr int SKINNY_ROWS = 64, SKINNY_WAVES = 4, SKINNY_COLS = 64;

template <class T, int NT>
__global__ __launch_bounds__(64 * SKINNY_WAVES) void skinny_kernel(P2pflAdapter a, ShrinkGrid grid, float* __restrict__ low,
                                                                   float* __restrict__ base, int parts) {
    constexpr int V = Shrink<T>::V, MT = SKINNY_COLS / 16;
    __shared__ float sums[SKINNY_WAVES][NT * 16][SKINNY_COLS + 1];
    if ((int)blockIdx.x < grid.blocks()) {
        shrink_block<T, SKINNY_WAVES, 1, 1>(a, grid, blockIdx.x, low, &sums[0][0][0]);
        return;
    }
    const int id = blockIdx.x - grid.blocks(), part = id % parts, o0 = id / parts * SKINNY_COLS;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i16 = lane & 15, h = lane >> 4;
    const T *w[MT], *x[NT];
    f32x4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m) w[m] = (const T*)a.w + (long)min(o0 + m * 16 + i16, a.Out - 1) * a.w_rs;
#pragma unroll
    for (int t = 0; t < NT; ++t) {                 // rows behind the last: a copy of it, not stored
        x[t] = (const T*)a.x + row_offset(min(t * 16 + i16, a.T - 1), a.B, a.x_cs, a.x_rs);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int units = (a.In + unit_of<T>() - 1) / unit_of<T>();
    stream_rows<T, SKINNY_WAVES, MT, NT>(w, x, a.In, (int)((long)units * part / parts), (int)((long)units * (part + 1) / parts),
                                         id / parts, acc, [](Raw<T, V>&, int, int) {});
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[wave][t * 16 + 4 * h + j][m * 16 + i16] = acc[m][t][j];
    __syncthreads();
    base += (long)part * a.T * a.Out;
    for (int i = threadIdx.x; i < NT * 16 * SKINNY_COLS; i += 64 * SKINNY_WAVES) {
        const int r = i / SKINNY_COLS, q = i % SKINNY_COLS;
        float t = 0.f;
#pragma unroll
        for (int v = 0; v < SKINNY_WAVES; ++v) t += sums[v][r][q];
        if (r < a.T && o0 + q < a.Out) base[(long)r * a.Out + o0 + q] = t;
    }
}

// y = the parts of the shared product + bias + drop(u B^T): a thread per column of y and ROWS rows of it, which keeps its row of
// B_k in registers while the rows are one client's. `low`: the parts of u (null: u is whole), added up by every block of a row
// and stored by its first.
constexpr int JOIN_RANKS = 32;

template <class T, int ROWS>
__global__ __launch_bounds__(256) void join_kernel(P2pflAdapter a, const float* __restrict__ low, int low_parts,
                                                   const float* __restrict__ base, int parts) {
    __shared__ float us[ROWS][JOIN_RANKS];
    __shared__ int ks[ROWS];
    const int o = blockIdx.y * 256 + threadIdx.x, row0 = blockIdx.x * ROWS;
    const Rows rows(a);
    float t[ROWS], sum[ROWS];
    if (threadIdx.x < ROWS) ks[threadIdx.x] = row0 + threadIdx.x < a.T ? rows.client(row0 + threadIdx.x) : -1;
    const float bias = a.bias && o < a.Out ? (float)((const T*)a.bias)[o] : 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) sum[i] = t[i] = 0.f;
    if (o < a.Out)
        for (int p = 0; p < parts; ++p) {
            float v[ROWS];
#pragma unroll
            for (int i = 0; i < ROWS; ++i) v[i] = base[((long)p * a.T + min(row0 + i, a.T - 1)) * a.Out + o];
#pragma unroll
            for (int i = 0; i < ROWS; ++i) t[i] += v[i];
        }
    for (int r0 = 0; r0 < a.R; r0 += JOIN_RANKS) {
        const int nr = min(JOIN_RANKS, a.R - r0);
        __syncthreads();
        for (int i = threadIdx.x; i < ROWS * JOIN_RANKS; i += 256) {
            const int row = row0 + i / JOIN_RANKS, r = i % JOIN_RANKS;
            float v = 0.f;
            if (row < a.T && r < nr) {
                const long at = (long)row * a.R + r0 + r;
                if (low) {
                    for (int p = 0; p < low_parts; ++p) v += low[(long)p * a.T * a.R + at];
                    if (blockIdx.y == 0) a.u[at] = v;
                } else {
                    v = a.u[at];
                }
            }
            us[i / JOIN_RANKS][r] = v;
        }
        __syncthreads();
        if (o >= a.Out) continue;
        int have = -1;
        float b[JOIN_RANKS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int k = ks[i];
            if (k < 0) continue;
            if (k != have) {
                const T* p = (const T*)a.lb + k * a.lb_cs + (long)o * a.R + r0;
#pragma unroll
                for (int j = 0; j < JOIN_RANKS; j += 4)
                    load_part<T, 4>(p + (j < nr ? j : 0), max(0, nr - j), reinterpret_cast<float (&)[4]>(b[j]));
                have = k;
            }
#pragma unroll
            for (int j = 0; j < JOIN_RANKS; ++j) if (j < nr) sum[i] += us[i][j] * b[j];
        }
    }
    if (o >= a.Out) return;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i, k = ks[i];
        if (row >= a.T) continue;
        if (k >= 0 && a.drop_out && a.drop.seeds) {
            const unsigned long long e = (unsigned long long)(row - rows.lo(k)) * a.Out + o;
            const unsigned bits = keep_bits<4>(a.drop, DropKey(a.drop, k), e & ~3ull);
            sum[i] = (bits >> (e & 3u) & 1u) ? sum[i] * a.drop.scale : 0.f;
        }
        ((T*)a.y + row_offset(row, a.B, a.y_cs, a.y_rs))[o] = (T)(t[i] + bias + sum[i]);
    }
}

template <class T>
void join(const P2pflAdapter& a, const float* low, int low_parts, const float* base, int parts, hipStream_t s) {
    const int cols = (a.Out + 255) / 256;
    if (a.T <= SKINNY_ROWS) join_kernel<T, 1><<<dim3(a.T, cols), 256, 0, s>>>(a, low, low_parts, base, parts);
    else join_kernel<T, 8><<<dim3((a.T + 7) / 8, cols), 256, 0, s>>>(a, low, low_parts, base, parts);
}

// y = the parts + bias, where the parts hold everything else.
template <class T>
__global__ __launch_bounds__(256) void add_parts_kernel(P2pflAdapter a, const float* __restrict__ base, int parts) {
    const long groups = (a.Out + 3) / 4, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= groups * a.T) return;
    const int row = (int)(i / groups), col = (int)(i % groups) * 4, n = min(4, a.Out - col);
    float t[4], v[4];
    load_part<float, 4>(base + (long)row * a.Out + col, n, t);
    for (int p = 1; p < parts; ++p) {
        load_part<float, 4>(base + ((long)p * a.T + row) * a.Out + col, n, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += v[e];
    }
    if (a.bias) {
        load_part<T, 4>((const T*)a.bias + col, n, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] += v[e];
    }
    store_part<T, 4>((T*)a.y + row_offset(row, a.B, a.y_cs, a.y_rs) + col, n, t);
}

template <class T>
void add_parts(const P2pflAdapter& a, const float* base, int parts, hipStream_t s) {
    const long threads = (long)((a.Out + 3) / 4) * a.T;
    add_parts_kernel<T><<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(a, base, parts);
}

// Parts of the two reductions: blocks to fill the chip, at least one unit for every wave.
struct SkinnyParts { int base, low; };

SkinnyParts skinny_parts(const P2pflAdapter& a) {
    const int unit = a.dtype == DT_F32 ? unit_of<float>() : unit_of<__bf16>(), units = (a.In + unit - 1) / unit;
    const int tiles = (a.Out + SKINNY_COLS - 1) / SKINNY_COLS;
    const int most = min(8, max(1, units / SKINNY_WAVES));
    return {max(1, min(most, 512 / tiles)), most >= 4 ? 4 : 1};
}

template <class T>
int few_rows(const P2pflAdapter& a, float* scratch, hipStream_t s) {
    const SkinnyParts parts = skinny_parts(a);
    const ShrinkGrid g = shrink_grid(a, 16, 16, parts.low);
    float* low = scratch;
    float* base = scratch + (long)parts.low * a.T * a.R;
    const int blocks = g.blocks() + parts.base * ((a.Out + SKINNY_COLS - 1) / SKINNY_COLS);
    if (a.T <= 16) skinny_kernel<T, 1><<<blocks, 64 * SKINNY_WAVES, 0, s>>>(a, g, low, base, parts.base);
    else if (a.T <= 32) skinny_kernel<T, 2><<<blocks, 64 * SKINNY_WAVES, 0, s>>>(a, g, low, base, parts.base);
    else skinny_kernel<T, 4><<<blocks, 64 * SKINNY_WAVES, 0, s>>>(a, g, low, base, parts.base);
    join<T>(a, low, parts.low, base, parts.base, s);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ the shared product
// C^T tiles: the matrix instruction's rows are columns of y (rows of W), its columns are rows of x, so a lane holds four
// consecutive elements of a row of y: one vector store, one Philox block.
template <class T> struct Terms { typedef T E; static constexpr int N = 1; };
template <> struct Terms<float> { typedef __bf16 E; static constexpr int N = 3; };

template <class E> struct Frag;
template <> struct Frag<__bf16> { typedef bf16x8 type; };
template <> struct Frag<_Float16> { typedef f16x8 type; };

// 8 elements on their way into LDS: as stored, or (fp32) as three bf16 terms.
template <class T> struct Piece {
    Raw<T, 8> r;
    __device__ __forceinline__ void load(const T* p, int n) { r = load_raw<T, 8>(p, n); }
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
    template <class F> __device__ __forceinline__ void store(__bf16* lds, int plane) const {
        bf16x8 t[3];
        split_bf16x8<3>(v, t);
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<bf16x8*>(lds + i * plane) = t[i];
    }
};

// The power of two that takes a row's ranks, eight in each of four neighbouring lanes, below 2^15: v 2^-shift. (The finite ones:
// an infinite u is its own product.)
__device__ __forceinline__ int row_shift(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, __builtin_isfinite(v[j]) ? fabsf(v[j]) : 0.f);
    m = fmaxf(m, __shfl_xor(m, 1, 64));
    m = fmaxf(m, __shfl_xor(m, 2, 64));
    return __builtin_amdgcn_frexp_expf(m) - 15;
}

// Tile of a block. Blocks go round the eight XCDs, each with an L2 of its own: an XCD gets one run of tiles, in groups of
// four rows of tiles, so that what its blocks read together (4 + 8 tiles of x and W for 32 blocks) is shared in its L2.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int& m, int& n) {
    constexpr int XCDS = 8, GROUP = 4;
    const int total = tiles_m * tiles_n, base = total / XCDS, more = total % XCDS, xcd = id % XCDS;
    const int t = xcd * base + min(xcd, more) + id / XCDS;
    const int group = t / (GROUP * tiles_n), first = group * GROUP, rows = min(GROUP, tiles_m - first), in = t - first * tiles_n;
    m = first + in % rows;
    n = in / rows;
}

// ------------------------------------------------------------------------------------------------ many aligned 16-bit rows
// 16-bit maps whose rows start on 16 bytes go from global memory into LDS without passing through registers, in two stages of
// 64 columns of the reduction that take turns. 64 columns are the 128 bytes of a cache line: loads of half lines reach 7 TB/s
// into LDS over the chip, of whole lines 12 TB/s (four stages of 32 columns were bound by that).
//
// Layout of a stage: a row is eight 16-byte pieces; piece q of row r lies in slot q ^ (r / 2 & 7), so sixteen lanes that read
// one piece of sixteen rows touch all 64 banks once. A wave's load fills 8 rows; its lanes' addresses are exchanged to match.
//
// Tiles of 256 x 256 run on eight waves, two per SIMD, half a step apart: while one wave of a SIMD multiplies (32 instructions
// of 16x16x32), the other reads its operands from LDS and starts the next stage's loads. All waves in step: 259 us at
// 8192 x 4096 x 4096, this way 219 (1.25 PFLOP/s).
constexpr int STAGE = 64;

__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ int slot_of(int row, int piece) { return row * STAGE + (piece ^ (row >> 1 & 7)) * 8; }

// `base` null: y. Otherwise part blockIdx % parts of the product without the bias, fp32 [parts][T][Out]; `tailed`: with the
// adapters.
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void wide_kernel(P2pflAdapter a, float* __restrict__ base, int parts, int tailed) {
    typedef typename Frag<T>::type F;
    constexpr int NT = 64 * WM * WN, WAVES = WM * WN;
    constexpr bool APART = WAVES == 8;            // the halves of the block half a step apart
    constexpr int TM = BM / WM, TN = BN / WN, RM = TM / 16, RN = TN / 16;
    constexpr int LX = BM / 8 / WAVES, LW = BN / 8 / WAVES;           // loads of a wave per stage
    static_assert(LX * 8 * WAVES == BM && LW * 8 * WAVES == BN, "tile");
    // (objects of their own: the compiler then sees that a stage being loaded is not the one being read, and does not wait for it)
    __shared__ T xs0[BM * STAGE], xs1[BM * STAGE], ws0[BN * STAGE], ws1[BN * STAGE];
    __shared__ T xs2[APART ? 8 : BM * STAGE], xs3[APART ? 8 : BM * STAGE], ws2[APART ? 8 : BN * STAGE], ws3[APART ? 8 : BN * STAGE];
    const int part = blockIdx.x % parts;
    int tm, tn;
    tile_of(blockIdx.x / parts, (a.T + BM - 1) / BM, (a.Out + BN - 1) / BN, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;                            // rows of x, rows of W
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r16 = lane & 15, h = lane >> 4;
    const int wm = wave / WN * TM, wn = wave % WN * TN;
    const Rows rows(a);
    f32x4 acc[RN][RM];
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
        for (int j = 0; j < RM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // The adapters, 32 ranks at a time: the tile's rows of u once (a row is one client's) in two terms of the map's type, then B_k of
    // up to six clients per round, two in each of the other stages' memory. Parts of the reduction share the clients out.
    if (tailed) {
        constexpr int CLIENTS = 6;
        __shared__ int todo[64][3], found, more;  // clients with rows here among 64: client, its rows
        __shared__ int shifts[BM];                // of the rows of u
        const int k_first = rows.first_ending_after(m0);
        for (int r0 = 0; r0 < a.R; r0 += 32) {
            __syncthreads();
            for (int c = threadIdx.x; c < BM * 4; c += NT) {
                const int row = m0 + c / 4, r = r0 + c % 4 * 8;
                float v[8], l[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = row < a.T && r + j < a.R ? a.u[(long)row * a.R + r + j] : 0.f;
                const int shift = row_shift(v);
                if (c % 4 == 0) shifts[c / 4] = shift;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = __builtin_ldexpf(v[j], -shift);
                    l[j] = __builtin_isinf(v[j]) ? 0.f : v[j] - (float)(T)v[j];
                }
                *reinterpret_cast<F*>(&xs0[slot_of(c / 4, c % 4)]) = __builtin_bit_cast(F, pack<T, 8>(v));
                *reinterpret_cast<F*>(&xs0[slot_of(c / 4, 4 + c % 4)]) = __builtin_bit_cast(F, pack<T, 8>(l));
            }
            for (int kb = k_first; kb < a.K; kb += 64) {
                if (threadIdx.x < 64) {
                    const int k = kb + lane, lo = k < a.K ? rows.lo(k) : a.T, hi = k < a.K ? rows.hi(k) : a.T;
                    const bool here = lo < m0 + BM && hi > m0 && lo < hi && k < a.K && k % parts == part;
                    const unsigned long long all = __ballot(here);
                    if (here) {
                        const int at = __popcll(all & ((1ull << lane) - 1));
                        todo[at][0] = k; todo[at][1] = lo; todo[at][2] = hi;
                    }
                    const unsigned long long in = __ballot(k < a.K && lo < m0 + BM);
                    if (lane == 0) { found = __popcll(all); more = in >> 63 != 0; }
                }
                __syncthreads();
                const int clients = found, on = more;
                for (int c0 = 0; c0 < clients; c0 += CLIENTS) {
                    const int n = min(CLIENTS, clients - c0);
                    for (int c = threadIdx.x; c < n * BN * 4; c += NT) {
                        const int q = c / (BN * 4), piece = c % 4, br = c / 4 % BN, col = n0 + br, r = r0 + piece * 8;
                        const int nr = col < a.Out ? max(0, min(8, a.R - r)) : 0;
                        const T* p = (const T*)a.lb + (nr ? todo[c0 + q][0] * a.lb_cs + (long)col * a.R + r : 0);
                        *reinterpret_cast<F*>(&(q < 2 ? xs1 : q < 4 ? ws0 : ws1)[slot_of(br, (q & 1) * 4 + piece)]) =
                            __builtin_bit_cast(F, load_raw<T, 8>(p, nr));
                    }
                    __syncthreads();
                    for (int q = 0; q < n; ++q) {
                        const T* bs = q < 2 ? xs1 : q < 4 ? ws0 : ws1;
                        const int lo = todo[c0 + q][1], hi = todo[c0 + q][2];
                        F b[RN];
#pragma unroll
                        for (int i = 0; i < RN; ++i) b[i] = *reinterpret_cast<const F*>(&bs[slot_of(wn + i * 16 + r16, (q & 1) * 4 + h)]);
#pragma unroll
                        for (int j = 0; j < RM; ++j) {
                            const int first = m0 + wm + j * 16, row = first + r16;
                            if (lo >= first + 16 || hi <= first) continue;
                            const bool mine = row >= lo && row < hi;
                            const int shift = shifts[row - m0];
                            const F uh = *reinterpret_cast<const F*>(&xs0[slot_of(row - m0, h)]);
                            const F ul = *reinterpret_cast<const F*>(&xs0[slot_of(row - m0, 4 + h)]);
#pragma unroll
                            for (int i = 0; i < RN; ++i) {
                                const f32x4 own = mma16(b[i], ul, mma16(b[i], uh, f32x4{0.f, 0.f, 0.f, 0.f}));
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[i][j][e] = mine ? acc[i][j][e] + __builtin_ldexpf(own[e], shift) : acc[i][j][e];
                            }
                        }
                    }
                    __syncthreads();
                }
                __syncthreads();
                if (!on) break;
            }
        }
        if (a.drop_out && a.drop.seeds) {         // the adapters' part alone is in the accumulators (and a part's clients are whole)
#pragma unroll
            for (int j = 0; j < RM; ++j) {
                const int row = m0 + wm + j * 16 + r16;
                const int k = row < a.T ? rows.client(row) : -1;
                if (k < 0) continue;
                const DropKey key(a.drop, k);
                const unsigned long long e0 = (unsigned long long)(row - rows.lo(k)) * a.Out;
#pragma unroll
                for (int i = 0; i < RN; ++i) {
                    const unsigned bits = keep_bits<4>(a.drop, key, e0 + n0 + wn + i * 16 + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = (bits >> e & 1u) ? acc[i][j][e] * a.drop.scale : 0.f;
                }
            }
        }
    }

    // rows behind the last: a copy of it, not stored
    const T *px[LX], *pw[LW];
#pragma unroll
    for (int i = 0; i < LX; ++i) {
        const int r = (wave * LX + i) * 8 + (lane >> 3);
        px[i] = (const T*)a.x + row_offset(min(m0 + r, a.T - 1), a.B, a.x_cs, a.x_rs) + ((lane & 7) ^ (r >> 1 & 7)) * 8;
    }
#pragma unroll
    for (int i = 0; i < LW; ++i) {
        const int r = (wave * LW + i) * 8 + (lane >> 3);
        pw[i] = (const T*)a.w + (long)min(n0 + r, a.Out - 1) * a.w_rs + ((lane & 7) ^ (r >> 1 & 7)) * 8;
    }
    auto fetch = [&](T* xs, T* ws, int t) {
#pragma unroll
        for (int i = 0; i < LX; ++i) to_lds16(px[i] + (long)t * STAGE, &xs[(wave * LX + i) * 8 * STAGE]);
#pragma unroll
        for (int i = 0; i < LW; ++i) to_lds16(pw[i] + (long)t * STAGE, &ws[(wave * LW + i) * 8 * STAGE]);
    };
    F xf[RM], wf[RN];
    auto read = [&](const T* xs, const T* ws, int kk) {
#pragma unroll
        for (int i = 0; i < RN; ++i) wf[i] = *reinterpret_cast<const F*>(&ws[slot_of(wn + i * 16 + r16, kk * 4 + h)]);
#pragma unroll
        for (int j = 0; j < RM; ++j) xf[j] = *reinterpret_cast<const F*>(&xs[slot_of(wm + j * 16 + r16, kk * 4 + h)]);
    };
    auto multiply = [&]() {
        if (APART) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < RM; ++j)
#pragma unroll
            for (int i = 0; i < RN; ++i) acc[i][j] = mma16(wf[i], xf[j], acc[i][j]);
        if (APART) __builtin_amdgcn_s_setprio(0);
    };
    const int stages = a.In / STAGE, t0 = (int)((long)stages * part / parts), t1 = (int)((long)stages * (part + 1) / parts);
    __syncthreads();                              // the adapters' tiles have been read
    if (t0 < t1) {
        auto next = [&](T* xn, T* wnext, int t) { fetch(xn, wnext, min(t, t1 - 1)); };      // (behind the last stage: that one again, unused)
        if constexpr (APART) {
            fetch(xs0, ws0, t0);
            wait_loads<>();
            bare_barrier();
            if (wave >= WAVES / 2) bare_barrier();
            // Stage t + 1 is loaded over what held t - 1: the half that is behind has read the last of that before the other
            // half's barrier in front of these loads. Both have their loads in before the first barrier of t + 1.
            auto step = [&](int t, const T* xs, const T* ws, T* xn, T* wnext) {
                read(xs, ws, 0);
                next(xn, wnext, t + 1);
                wait_lds();
                bare_barrier();
                multiply();
                bare_barrier();
                read(xs, ws, 1);
                wait_loads<>();
                wait_lds();
                bare_barrier();
                multiply();
                bare_barrier();
            };
            int t = t0;
            for (; t + 2 <= t1; t += 2) {
                step(t, xs0, ws0, xs1, ws1);
                step(t + 1, xs1, ws1, xs0, ws0);
            }
            if (t < t1) step(t, xs0, ws0, xs1, ws1);
            if (wave < WAVES / 2) bare_barrier();
        } else {
            // three stages under way: a 128 x 128 stage is multiplied in a fraction of what its loads take
            fetch(xs0, ws0, t0);
            next(xs1, ws1, t0 + 1);
            next(xs2, ws2, t0 + 2);
            auto step = [&](int t, const T* xs, const T* ws, T* xn, T* wnext) {
                wait_loads<2 * (LX + LW)>();
                wait_lds();
                bare_barrier();
                next(xn, wnext, t + 3);
                __builtin_amdgcn_sched_barrier(0);  // (left alone, the loads sink to the end of the products they hide behind)
                read(xs, ws, 0);
                multiply();
                read(xs, ws, 1);
                multiply();
            };
            int t = t0;
            for (; t + 4 <= t1; t += 4) {
                step(t, xs0, ws0, xs3, ws3);
                step(t + 1, xs1, ws1, xs0, ws0);
                step(t + 2, xs2, ws2, xs1, ws1);
                step(t + 3, xs3, ws3, xs2, ws2);
            }
            if (t < t1) step(t, xs0, ws0, xs3, ws3);
            if (t + 1 < t1) step(t + 1, xs1, ws1, xs0, ws0);
            if (t + 2 < t1) step(t + 2, xs2, ws2, xs1, ws1);
        }
        wait_loads<>();
    }
    if (a.In % STAGE && part == parts - 1) {      // the last columns, through registers
        const int k0 = stages * STAGE;
        __syncthreads();
        for (int c = threadIdx.x; c < BM * 8; c += NT) {
            const int r = c / 8, n = max(0, min(8, a.In - k0 - c % 8 * 8));
            const T* p = (const T*)a.x + row_offset(min(m0 + r, a.T - 1), a.B, a.x_cs, a.x_rs);
            *reinterpret_cast<F*>(&xs0[slot_of(r, c % 8)]) = __builtin_bit_cast(F, load_raw<T, 8>(n ? p + k0 + c % 8 * 8 : p, n));
        }
        for (int c = threadIdx.x; c < BN * 8; c += NT) {
            const int r = c / 8, n = max(0, min(8, a.In - k0 - c % 8 * 8));
            const T* p = (const T*)a.w + (long)min(n0 + r, a.Out - 1) * a.w_rs;
            *reinterpret_cast<F*>(&ws0[slot_of(r, c % 8)]) = __builtin_bit_cast(F, load_raw<T, 8>(n ? p + k0 + c % 8 * 8 : p, n));
        }
        __syncthreads();
        read(xs0, ws0, 0);
        multiply();
        read(xs0, ws0, 1);
        multiply();
    }

    // out through LDS, 16 bytes a lane and whole lines of a row: a wave owns 64 columns and a corner of the stages' memory
    static_assert(TN == 64, "columns of a wave");
    __syncthreads();
    char* corner = reinterpret_cast<char*>(WAVES == 8 ? (wave < 2 ? xs0 : wave < 4 ? xs1 : wave < 6 ? ws0 : ws1) : wave < 2 ? xs0 : ws0) +
                   (wave & 1) * (TM * 128);
    const int col0 = n0 + wn;
    if (base) {
        constexpr int RP = TM / 2 / 16;           // 16-row tiles per pass: fp32 rows are 256 bytes
#pragma unroll
        for (int j0 = 0; j0 < RM; j0 += RP) {
#pragma unroll
            for (int j = 0; j < RP; ++j)
#pragma unroll
                for (int i = 0; i < RN; ++i)
                    *reinterpret_cast<f32x4*>(corner + (j * 16 + r16) * 256 + ((i * 4 + h) ^ r16) * 16) = acc[i][j0 + j];
            wait_lds();
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r = 0; r < RP * 16; r += 4) {
                const int rr = r + (lane >> 4), row = m0 + wm + j0 * 16 + rr, col = col0 + r16 * 4;
                const f32x4 v = *reinterpret_cast<const f32x4*>(corner + rr * 256 + (r16 ^ (rr & 15)) * 16);
                if (row < a.T && col < a.Out)
                    store_raw<float, 4, false>(base + ((long)part * a.T + row) * a.Out + col, __builtin_bit_cast(Raw<float, 4>, v), min(4, a.Out - col));
            }
            wait_lds();
            __builtin_amdgcn_wave_barrier();
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < RN; ++i) {
        float bias[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = col0 + i * 16 + 4 * h + e;
            bias[e] = a.bias && col < a.Out ? (float)((const T*)a.bias)[col] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < RM; ++j) {
            const int rr = j * 16 + r16;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] + bias[e];
            *reinterpret_cast<Raw<T, 4>*>(corner + rr * 128 + ((i * 2 + (h >> 1)) ^ (rr & 7)) * 16 + (h & 1) * 8) = pack<T, 4>(v);
        }
    }
    wait_lds();
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < TM; r += 8) {
        const int rr = r + (lane >> 3), row = m0 + wm + rr, col = col0 + (lane & 7) * 8;
        const Raw<T, 8> v = *reinterpret_cast<const Raw<T, 8>*>(corner + rr * 128 + ((lane & 7) ^ (rr & 7)) * 16);
        if (row < a.T && col < a.Out) store_raw<T, 8>((T*)a.y + row_offset(row, a.B, a.y_cs, a.y_rs) + col, v, min(8, a.Out - col));
    }
}

// ------------------------------------------------------------------------------------------------ many fp32 or unaligned rows
// Rows of any alignment and length come in through registers. fp32 products from three bf16 terms per operand: 32 columns of the
// reduction are loaded, split and written as three planes into one of two LDS stages; six products of 16x16x32 follow. The
// splitting (about seven vector instructions an element) and the LDS traffic of a wave run beside the 96 matrix instructions of
// the other wave of its SIMD: the halves of the block are half a step apart, as above. 16-bit rows: one plane of 64 columns.
// Layout of a 32-column plane: a row is four 16-byte pieces; piece q of row r lies in slot q ^ (-(r / 4) & 3). LDS serves a 16-byte read
// in groups of lanes 0-3, 12-15, 20-23, 24-27 (and the like): with this order the four row blocks of a group sit in four slots
// (r / 4 & 3 itself: two of them meet, 36 % of the LDS cycles were conflicts).
__device__ __forceinline__ int split_slot(int row, int piece) { return row * 32 + (piece ^ (-(row >> 2) & 3)) * 8; }

template <int COLS>
__device__ __forceinline__ int staged_slot(int row, int piece) {
    if constexpr (COLS == 32) return split_slot(row, piece);
    else return slot_of(row, piece);
}

template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void staged_kernel(P2pflAdapter a, float* __restrict__ base, int parts, int tailed) {
    typedef typename Terms<T>::E E;
    typedef typename Frag<E>::type F;
    constexpr int NT = 64 * WM * WN, WAVES = WM * WN, NS = Terms<T>::N;
    constexpr int COLS = NS == 3 ? 32 : 64, KS = COLS / 32, PIECES = COLS / 8;      // of a stage; steps of 32 columns
    constexpr int UT = NS == 3 ? 3 : 2;           // terms of u
    constexpr bool APART = WAVES == 8;
    constexpr int TM = BM / WM, TN = BN / WN, RM = TM / 16, RN = TN / 16;
    constexpr int LX = BM * PIECES / NT, LW = BN * PIECES / NT;       // pieces of a thread per stage
    constexpr int XP = BM * COLS, WP = BN * COLS;                     // elements of a plane
    constexpr int UP = BM * 32, BP = BN * 32;                         // of a term of u and of B
    static_assert(TM == 64 && TN == 64 && LX * NT == BM * PIECES && LW * NT == BN * PIECES, "tile");
    static_assert(UT * UP <= NS * XP && NS * BP <= NS * WP && BM >= BN, "u and B in a stage");
    __shared__ __attribute__((aligned(16))) E pool[2][NS * (XP + WP)];
    int tm, tn;
    const int part = blockIdx.x % parts;
    tile_of(blockIdx.x / parts, (a.T + BM - 1) / BM, (a.Out + BN - 1) / BN, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r16 = lane & 15, h = lane >> 4;
    const int wm = wave / WN * TM, wn = wave % WN * TN;
    const Rows rows(a);
    f32x4 acc[RN][RM];
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
        for (int j = 0; j < RM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // rows behind the last: a copy of it, not stored
    const T *px[LX], *pw[LW];
#pragma unroll
    for (int i = 0; i < LX; ++i) {
        const int c = threadIdx.x + i * NT;
        px[i] = (const T*)a.x + row_offset(min(m0 + c / PIECES, a.T - 1), a.B, a.x_cs, a.x_rs) + c % PIECES * 8;
    }
#pragma unroll
    for (int i = 0; i < LW; ++i) {
        const int c = threadIdx.x + i * NT;
        pw[i] = (const T*)a.w + (long)min(n0 + c / PIECES, a.Out - 1) * a.w_rs + c % PIECES * 8;
    }
    const int stages = a.In / COLS, t0 = (int)((long)stages * part / parts), t1 = (int)((long)stages * (part + 1) / parts);
    Piece<T> xa[LX], wa[LW], xb[LX], wb[LW];      // two stages under way in registers
    auto fetch = [&](Piece<T> (&xv)[LX], Piece<T> (&wv)[LW], int t) {
        const long k0 = (long)min(t, t1 - 1) * COLS;                  // (behind the last stage: that one again, unused)
#pragma unroll
        for (int i = 0; i < LX; ++i) xv[i].load(px[i] + k0, 8);
#pragma unroll
        for (int i = 0; i < LW; ++i) wv[i].load(pw[i] + k0, 8);
    };
    if (t0 < t1) {                                // under way while the adapters are multiplied
        fetch(xa, wa, t0);
        fetch(xb, wb, t0 + 1);
    }

    // the adapters, 32 ranks at a time: u of the tile's rows, B_k of up to three clients per round (as in wide_kernel)
    if (tailed) {
        constexpr int CLIENTS = 3;
        __shared__ int todo[64][3], found, more, shifts[BM];
        const int k_first = rows.first_ending_after(m0);
        auto b_of = [&](int q) { return q == 0 ? &pool[0][NS * XP] : q == 1 ? &pool[1][NS * XP] : &pool[1][0]; };
        for (int r0 = 0; r0 < a.R; r0 += 32) {
            __syncthreads();
            for (int c = threadIdx.x; c < BM * 4; c += NT) {
                const int row = m0 + c / 4, r = r0 + c % 4 * 8;
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = row < a.T && r + j < a.R ? a.u[(long)row * a.R + r + j] : 0.f;
                const int shift = row_shift(v);
                if (c % 4 == 0) shifts[c / 4] = shift;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __builtin_ldexpf(v[j], -shift);
#pragma unroll
                for (int t = 0; t < UT; ++t) {    // each term is the rounding of what the others left
                    F f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) { f[j] = (E)v[j]; v[j] = __builtin_isinf(v[j]) ? 0.f : v[j] - (float)f[j]; }
                    *reinterpret_cast<F*>(&pool[0][t * UP + split_slot(c / 4, c % 4)]) = f;
                }
            }
            for (int kb = k_first; kb < a.K; kb += 64) {
                if (threadIdx.x < 64) {
                    const int k = kb + lane, lo = k < a.K ? rows.lo(k) : a.T, hi = k < a.K ? rows.hi(k) : a.T;
                    const bool here = lo < m0 + BM && hi > m0 && lo < hi && k < a.K && k % parts == part;
                    const unsigned long long all = __ballot(here);
                    if (here) {
                        const int at = __popcll(all & ((1ull << lane) - 1));
                        todo[at][0] = k; todo[at][1] = lo; todo[at][2] = hi;
                    }
                    const unsigned long long in = __ballot(k < a.K && lo < m0 + BM);
                    if (lane == 0) { found = __popcll(all); more = in >> 63 != 0; }
                }
                __syncthreads();
                const int clients = found, on = more;
                for (int c0 = 0; c0 < clients; c0 += CLIENTS) {
                    const int n = min(CLIENTS, clients - c0);
                    for (int c = threadIdx.x; c < n * BN * 4; c += NT) {
                        const int q = c / (BN * 4), piece = c % 4, br = c / 4 % BN, col = n0 + br, r = r0 + piece * 8;
                        const int nr = col < a.Out ? max(0, min(8, a.R - r)) : 0;
                        Piece<T> b;
                        b.load((const T*)a.lb + (nr ? todo[c0 + q][0] * a.lb_cs + (long)col * a.R + r : 0), nr);
                        b.template store<F>(b_of(q) + split_slot(br, piece), BP);
                    }
                    __syncthreads();
                    for (int q = 0; q < n; ++q) {
                        const E* bs = b_of(q);
                        const int lo = todo[c0 + q][1], hi = todo[c0 + q][2];
#pragma unroll
                        for (int j = 0; j < RM; ++j) {
                            const int first = m0 + wm + j * 16, row = first + r16;
                            if (lo >= first + 16 || hi <= first) continue;
                            const bool mine = row >= lo && row < hi;
                            const int shift = shifts[row - m0];
                            F u[UT];
#pragma unroll
                            for (int t = 0; t < UT; ++t) u[t] = *reinterpret_cast<const F*>(&pool[0][t * UP + split_slot(row - m0, h)]);
#pragma unroll
                            for (int i = 0; i < RN; ++i) {
                                f32x4 own = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                for (int w = 0; w < NS; ++w) {
                                    const F b = *reinterpret_cast<const F*>(bs + w * BP + split_slot(wn + i * 16 + r16, h));
#pragma unroll
                                    for (int t = 0; w + t < UT; ++t) own = mma16(b, u[t], own);
                                }
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[i][j][e] = mine ? acc[i][j][e] + __builtin_ldexpf(own[e], shift) : acc[i][j][e];
                            }
                        }
                    }
                    __syncthreads();
                }
                __syncthreads();
                if (!on) break;
            }
        }
        if (a.drop_out && a.drop.seeds) {         // the adapters' part alone is in the accumulators (and a part's clients are whole)
#pragma unroll
            for (int j = 0; j < RM; ++j) {
                const int row = m0 + wm + j * 16 + r16;
                const int k = row < a.T ? rows.client(row) : -1;
                if (k < 0) continue;
                const DropKey key(a.drop, k);
                const unsigned long long e0 = (unsigned long long)(row - rows.lo(k)) * a.Out;
#pragma unroll
                for (int i = 0; i < RN; ++i) {
                    const unsigned bits = keep_bits<4>(a.drop, key, e0 + n0 + wn + i * 16 + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = (bits >> e & 1u) ? acc[i][j][e] * a.drop.scale : 0.f;
                }
            }
        }
    }

    auto write = [&](E* buf, const Piece<T> (&xv)[LX], const Piece<T> (&wv)[LW]) {
#pragma unroll
        for (int i = 0; i < LX; ++i) {
            const int c = threadIdx.x + i * NT;
            xv[i].template store<F>(buf + staged_slot<COLS>(c / PIECES, c % PIECES), XP);
        }
#pragma unroll
        for (int i = 0; i < LW; ++i) {
            const int c = threadIdx.x + i * NT;
            wv[i].template store<F>(buf + NS * XP + staged_slot<COLS>(c / PIECES, c % PIECES), WP);
        }
    };
    F xf[KS][NS][RM], wf[KS][NS][RN];
    auto read = [&](const E* buf) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int t = 0; t < NS; ++t) {
#pragma unroll
                for (int j = 0; j < RM; ++j)
                    xf[s][t][j] = *reinterpret_cast<const F*>(buf + t * XP + staged_slot<COLS>(wm + j * 16 + r16, s * 4 + h));
#pragma unroll
                for (int i = 0; i < RN; ++i)
                    wf[s][t][i] = *reinterpret_cast<const F*>(buf + NS * XP + t * WP + staged_slot<COLS>(wn + i * 16 + r16, s * 4 + h));
            }
    };
    auto multiply = [&]() {
        if (APART) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int w = 0; w < NS; ++w)
#pragma unroll
                for (int t = 0; w + t < NS; ++t)
#pragma unroll
                    for (int j = 0; j < RM; ++j)
#pragma unroll
                        for (int i = 0; i < RN; ++i) acc[i][j] = mma16(wf[s][w][i], xf[s][t][j], acc[i][j]);
        if (APART) __builtin_amdgcn_s_setprio(0);
    };
    __syncthreads();                              // the adapters' tiles have been read
    if (t0 < t1) {
        write(pool[0], xa, wa);
        fetch(xa, wa, t0 + 2);
        __syncthreads();
        // Stage t + 1 is written over what held t - 1 and was read from there one barrier ago by the half that is behind; it is
        // read after the next barrier but one, when both halves have written.
        if (APART && wave >= WAVES / 2) bare_barrier();
        auto step = [&](int t, const E* buf, E* other, Piece<T> (&xv)[LX], Piece<T> (&wv)[LW]) {
            read(buf);
            write(other, xv, wv);
            fetch(xv, wv, t + 3);
            wait_lds();
            bare_barrier();
            multiply();
            if (APART) bare_barrier();
        };
        int t = t0;
        for (; t + 2 <= t1; t += 2) {
            step(t, pool[0], pool[1], xb, wb);
            step(t + 1, pool[1], pool[0], xa, wa);
        }
        if (t < t1) step(t, pool[0], pool[1], xb, wb);
        if (APART && wave < WAVES / 2) bare_barrier();
    }
    if (a.In % COLS && part == parts - 1) {                          // the last columns
        const int k0 = stages * COLS;
#pragma unroll
        for (int i = 0; i < LX; ++i) {
            const int n = max(0, min(8, a.In - k0 - (int)(threadIdx.x + i * NT) % PIECES * 8));
            xa[i].load(px[i] + (n ? k0 : 0), n);
        }
#pragma unroll
        for (int i = 0; i < LW; ++i) {
            const int n = max(0, min(8, a.In - k0 - (int)(threadIdx.x + i * NT) % PIECES * 8));
            wa[i].load(pw[i] + (n ? k0 : 0), n);
        }
        __syncthreads();
        write(pool[0], xa, wa);
        __syncthreads();
        read(pool[0]);
        multiply();
    }

    // out through LDS as fp32, four columns a lane
    __syncthreads();
    constexpr int RP = sizeof(pool) >= WAVES * 64 * 256 ? RM : RM / 2;      // 16-row tiles per pass
    static_assert(sizeof(pool) >= WAVES * RP * 16 * 256, "corners");
    char* corner = reinterpret_cast<char*>(&pool[0][0]) + wave * (RP * 16 * 256);
    const int col = n0 + wn + r16 * 4, n = min(4, a.Out - col);
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (!base && a.bias && n > 0) load_part<T, 4>((const T*)a.bias + col, n, bias);
#pragma unroll
    for (int j0 = 0; j0 < RM; j0 += RP) {
#pragma unroll
        for (int j = 0; j < RP; ++j)
#pragma unroll
            for (int i = 0; i < RN; ++i)
                *reinterpret_cast<f32x4*>(corner + (j * 16 + r16) * 256 + ((i * 4 + h) ^ r16) * 16) = acc[i][j0 + j];
        wait_lds();
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < RP * 16; r += 4) {
            const int rr = r + (lane >> 4), row = m0 + wm + j0 * 16 + rr;
            const f32x4 v = *reinterpret_cast<const f32x4*>(corner + rr * 256 + (r16 ^ (rr & 15)) * 16);
            if (row >= a.T || n <= 0) continue;
            const float o[4] = {v[0] + bias[0], v[1] + bias[1], v[2] + bias[2], v[3] + bias[3]};
            if (base) store_part<float, 4, false>(base + ((long)part * a.T + row) * a.Out + col, n, o);
            else store_part<T, 4>((T*)a.y + row_offset(row, a.B, a.y_cs, a.y_rs) + col, n, o);
        }
        wait_lds();
        __builtin_amdgcn_wave_barrier();
    }
}

// 16-byte loads need rows that start on 16 bytes.
inline bool aligned16(const P2pflAdapter& a) {
    return a.dtype != DT_F32 && ((size_t)a.x | (size_t)a.w) % 16 == 0 && (a.x_rs | a.x_cs | a.w_rs) % 8 == 0;
}

// Tile and parts of the reduction with the smallest estimate. A stage of 64 columns is bound by what a CU can bring into LDS,
// 38 bytes per ns in tiles of 256 x 256 and 31 in tiles of 128 x 128 (measured at 4096 columns: 1.7 and 1.06 us a stage), so the
// large tile wins wherever a split reduction fills the chip with it; splitting writes and reads fp32 parts (4 TB/s) and takes
// one more launch. Clients of fewer than sixteen rows on average leave their part to join_kernel: in a tile every one of them is
// a step of its own.
struct WidePlan { int tile, parts; bool rows_join; };

// Rows through registers: tiles of 256 x 128 (measured: 2.4 us a stage of 32 fp32 columns) or 128 x 128 (1.95).
WidePlan staged_plan(const P2pflAdapter& a) {
    const bool few = (long)a.T < 16L * a.K;
    const int cols = a.dtype == DT_F32 ? 32 : 64;
    WidePlan best{256, 1, few};
    double least = 1e30;
    for (int tile = 128; tile <= 256; tile += 128)
        for (int parts = 1; parts <= 8; parts *= 2) {
            if (parts > 1 && a.In / parts < 3 * cols) break;
            const long blocks = (long)((a.T + tile - 1) / tile) * ((a.Out + 127) / 128) * parts;
            const double stages = (a.In + cols - 1) / cols / (double)parts + 4;
            const double join = parts > 1 ? 6.0 + 8e-6 * parts / 4 * a.T * a.Out : 0.0;
            const double us = (double)((blocks + 255) / 256) * stages * (tile == 256 ? 2.4 : 1.95) + join;
            if (us < least) { least = us; best = {tile, parts, few}; }
        }
    return best;
}

WidePlan wide_plan(const P2pflAdapter& a) {
    const bool few = (long)a.T < 16L * a.K;
    WidePlan best{256, 1, few};
    double least = 1e30;
    for (int tile = 128; tile <= 256; tile += 128)
        for (int parts = 1; parts <= 8; parts *= 2) {
            if (parts > 1 && a.In / parts < 256) break;
            const long blocks = (long)((a.T + tile - 1) / tile) * ((a.Out + tile - 1) / tile) * parts;
            const double stages = (a.In + 63) / 64 / (double)parts + 3;
            const double join = parts > 1 ? 6.0 + 8e-6 * parts / 4 * a.T * a.Out : 0.0;
            const double us = (double)((blocks + 255) / 256) * stages * (tile == 256 ? 1.7 : 1.06) + join;
            if (us < least) { least = us; best = {tile, parts, few}; }
        }
    return best;
}

template <class T>
int shared_product(const P2pflAdapter& a, float* scratch, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (aligned16(a)) {
            const WidePlan p = wide_plan(a);
            const bool tailed = !p.rows_join;
            float* base = p.parts > 1 || !tailed ? scratch : nullptr;
            const int blocks = ((a.Out + p.tile - 1) / p.tile) * ((a.T + p.tile - 1) / p.tile) * p.parts;
            if (p.tile == 256) wide_kernel<T, 256, 256, 2, 4><<<blocks, 512, 0, s>>>(a, base, p.parts, tailed);
            else wide_kernel<T, 128, 128, 2, 2><<<blocks, 256, 0, s>>>(a, base, p.parts, tailed);
            if (!tailed) join<T>(a, nullptr, 0, base, p.parts, s);
            else if (base) add_parts<T>(a, base, p.parts, s);
            return (int)hipGetLastError();
        }
    }
    const WidePlan p = staged_plan(a);
    const bool tailed = !p.rows_join;
    float* base = p.parts > 1 || !tailed ? scratch : nullptr;
    const int blocks = ((a.Out + 127) / 128) * ((a.T + p.tile - 1) / p.tile) * p.parts;
    if (p.tile == 256) staged_kernel<T, 256, 128, 4, 2><<<blocks, 512, 0, s>>>(a, base, p.parts, tailed);
    else staged_kernel<T, 128, 128, 2, 2><<<blocks, 256, 0, s>>>(a, base, p.parts, tailed);
    if (!tailed) join<T>(a, nullptr, 0, base, p.parts, s);
    else if (base) add_parts<T>(a, base, p.parts, s);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ weight gradients
// out[k][wide][rank] or [k][rank][wide] = sum over the rows of client k of map[row][wide] * low[row][rank]: memory-bound (the
// map is read once per 32 ranks), so the products stay on fp32 MFMA whatever the map's type: u and v are not rounded.
// MFMA 16x16x4: lane l brings V consecutive columns of row l >> 4 of a step, instruction j multiplies column j of each lane.
// A block: 16 V columns x one chunk of a client's rows; its waves take every fourth step, four steps in flight each, and are
// added through LDS. Chunks of rows keep a client with many rows from being one block's work; they are joined in their order.
// Short chunks where there are few rows to fill the chip with, long ones where their fp32 parts would be the larger traffic.
__host__ __device__ inline int chunk_rows(int T) { return T <= 2048 ? 128 : T <= 8192 ? 256 : 512; }

struct WgradArgs {
    const void* map; long cs, rs;
    const float* low;
    float* out; long out_cs;
    int wide, ranks_first, drops;
};

struct Chunk {
    int k, r0, r1;
    int slot;                                     // of the client's chunks in scratch memory (-1: it has one, written in place)
};

// Chunk `id`, counted over the clients; every client has one at least (of no rows, if need be).
__device__ __forceinline__ bool find_chunk(const Rows& rows, int id, Chunk& c) {
    const int size = chunk_rows(rows.T);
    if (!rows.ptr) {
        const int per = max(1, (rows.B + size - 1) / size);
        c.k = id / per;
        if (c.k >= rows.K) return false;
        c.r0 = c.k * rows.B + id % per * size;
        c.r1 = min(c.r0 + size, (c.k + 1) * rows.B);
        c.slot = per > 1 ? id : -1;
        return true;
    }
    int before = 0, slots = 0;
    const int lane = threadIdx.x & 63;
    for (int k0 = 0; k0 < rows.K; k0 += 64) {
        const int kk = k0 + lane;
        const int n = kk < rows.K ? max(1, (rows.hi(kk) - rows.lo(kk) + size - 1) / size) : 0, m = n > 1 ? n : 0;
        int inc = n, minc = m;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int t = __shfl_up(inc, off, 64), u = __shfl_up(minc, off, 64);
            if (lane >= off) { inc += t; minc += u; }
        }
        const int total = __shfl(inc, 63, 64);
        if (id < before + total) {
            const int l = __ffsll((long long)__ballot(before + inc > id)) - 1;
            const int i = id - before - __shfl(inc - n, l, 64);
            c.k = k0 + l;
            c.r0 = rows.lo(c.k) + i * size;
            c.r1 = min(c.r0 + size, rows.hi(c.k));
            c.slot = __shfl(m, l, 64) ? slots + __shfl(minc - m, l, 64) + i : -1;
            return true;
        }
        before += total;
        slots += __shfl(minc, 63, 64);
    }
    return false;
}

// Chunks in scratch memory hold [R][In] of the first gradient, then [Out][R] of the second.
template <class T, int RT>
__global__ __launch_bounds__(256) void adapter_wgrad_kernel(P2pflAdapter a, WgradArgs ga, WgradArgs gb, int blocks_a, float* scratch, int slots,
                                                            int chunk0) {
    constexpr int V = 16 / sizeof(T), COLS = 16 * V, PITCH = COLS + 4, U = 4;
    __shared__ float sums[4][16 * RT][PITCH];
    const bool first = (int)blockIdx.x < blocks_a;
    const WgradArgs g = first ? ga : gb;
    const int tile = first ? blockIdx.x : blockIdx.x - blocks_a, rank0 = blockIdx.z * 16 * RT;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i16 = lane & 15, h = lane >> 4;
    const Rows rows(a);
    Chunk ch;
    if (!find_chunk(rows, chunk0 + blockIdx.y, ch) || ch.slot >= slots) return;      // (a row_ptr that decreases may count more of them)
    const int c = tile * COLS + i16 * V, n = max(0, min(V, g.wide - c));
    const bool drops = g.drops && a.drop.seeds;
    const DropKey key = drops ? DropKey(a.drop, ch.k) : DropKey();
    const int lo = rows.lo(ch.k);
    f32x4 acc[RT][V];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int r = ch.r0 + 4 * wave; r < ch.r1; r += 16 * U) {
        Raw<T, V> m[U];
        float low[U][RT];
#pragma unroll
        for (int s = 0; s < U; ++s) {
            const int row = r + 16 * s + h;
            const bool in = row < ch.r1;
            m[s] = load_raw<T, V>((const T*)g.map + (in && n ? row_offset(row, a.B, g.cs, g.rs) + c : 0), in ? n : 0);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const int rank = rank0 + 16 * t + i16;
                low[s][t] = in && rank < a.R ? g.low[(long)row * a.R + rank] : 0.f;
            }
        }
#pragma unroll
        for (int s = 0; s < U; ++s) {
            if (drops) keep_raw<T, V>(m[s], keep_bits<V>(a.drop, key, (unsigned long long)(r + 16 * s + h - lo) * g.wide + c));
            float mv[V];
            unpack<T, V>(m[s], mv);
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int v = 0; v < V; ++v) acc[t][v] = __builtin_amdgcn_mfma_f32_16x16x4f32(low[s][t], mv[v], acc[t][v], 0, 0, 0);
        }
    }
    // lane l: ranks 4 (l >> 4) + e, columns V (l & 15) .. + V - 1
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int v = 0; v < V; v += 4)
                *reinterpret_cast<f32x4*>(&sums[wave][16 * t + 4 * h + e][i16 * V + v]) =
                    f32x4{acc[t][v][e], acc[t][v + 1][e], acc[t][v + 2][e], acc[t][v + 3][e]};
    __syncthreads();
    const float f = drops ? a.drop.scale : 1.f;
    float* out = ch.slot < 0 ? g.out + ch.k * g.out_cs
                             : scratch + (long)ch.slot * a.R * ((ga.out ? ga.wide : 0) + (gb.out ? gb.wide : 0)) +
                                   (!first && ga.out ? (long)a.R * ga.wide : 0);
    for (int i = threadIdx.x; i < 16 * RT * COLS; i += 256) {
        const int q = g.ranks_first ? i / COLS : i % (16 * RT), w = g.ranks_first ? i % COLS : i / (16 * RT);
        const int rank = rank0 + q, col = tile * COLS + w;
        if (rank >= a.R || col >= g.wide) continue;
        const float t = (sums[0][q][w] + sums[1][q][w]) + (sums[2][q][w] + sums[3][q][w]);
        out[g.ranks_first ? (long)rank * g.wide + col : (long)col * a.R + rank] = t * f;
    }
}

// Adds the chunks of a client that has several.
__global__ __launch_bounds__(256) void adapter_wgrad_join_kernel(P2pflAdapter a, WgradArgs ga, WgradArgs gb, const float* scratch, int slots) {
    const Rows rows(a);
    const int k = blockIdx.y, lane = threadIdx.x & 63;
    const int size = chunk_rows(a.T);
    auto chunks = [&](int i) { return (rows.hi(i) - rows.lo(i) + size - 1) / size; };
    const int n = chunks(k);
    if (n <= 1) return;
    int slot = 0;
    if (rows.ptr)
        for (int i = lane; i < k; i += 64) { const int m = chunks(i); slot += m > 1 ? m : 0; }
    else slot = lane == 0 ? k * n : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) slot += __shfl_xor(slot, off, 64);
    const long na = ga.out ? (long)a.R * ga.wide : 0, both = na + (gb.out ? (long)a.R * gb.wide : 0);
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= both || slot + n > slots) return;
    const float* p = scratch + slot * both + i;
    float t = 0.f;
    int j = 0;
    for (; j + 4 <= n; j += 4, p += 4 * both) {
        const float v0 = p[0], v1 = p[both], v2 = p[2 * both], v3 = p[3 * both];
        t = (((t + v0) + v1) + v2) + v3;
    }
    for (; j < n; ++j, p += both) t += p[0];
    if (i < na) ga.out[k * ga.out_cs + i] = t;
    else gb.out[k * gb.out_cs + i - na] = t;
}

// Chunks that can be in scratch memory: those of clients with two or more.
inline long wgrad_slots(const P2pflAdapter& a) {
    const int size = chunk_rows(a.T);
    if (!a.row_ptr) return a.B > size ? (long)a.K * ((a.B + size - 1) / size) : 0;
    return a.T > size ? 2L * (a.T / size) : 0;
}

template <class T>
int weight_gradients(const P2pflAdapter& a, const WgradArgs& ga, const WgradArgs& gb, float* scratch, hipStream_t s) {
    constexpr int COLS = 16 * 16 / sizeof(T);
    const int blocks_a = ga.out ? (ga.wide + COLS - 1) / COLS : 0, blocks_b = gb.out ? (gb.wide + COLS - 1) / COLS : 0;
    const int size = chunk_rows(a.T), chunks = a.row_ptr ? a.T / size + a.K : a.K * max(1, (a.B + size - 1) / size);
    if (blocks_a + blocks_b == 0 || chunks == 0) return 0;
    const int slots = (int)wgrad_slots(a);
    for (int c0 = 0; c0 < chunks; c0 += 65535) {              // (the y dimension of a grid ends at 65535)
        const dim3 grid(blocks_a + blocks_b, min(65535, chunks - c0), a.R <= 16 ? 1 : (a.R + 31) / 32);
        if (a.R <= 16) adapter_wgrad_kernel<T, 1><<<grid, 256, 0, s>>>(a, ga, gb, blocks_a, scratch, slots, c0);
        else adapter_wgrad_kernel<T, 2><<<grid, 256, 0, s>>>(a, ga, gb, blocks_a, scratch, slots, c0);
    }
    if (slots) {
        const long both = (long)a.R * ((ga.out ? ga.wide : 0) + (gb.out ? gb.wide : 0));
        adapter_wgrad_join_kernel<<<dim3((unsigned)((both + 255) / 256), a.K), 256, 0, s>>>(a, ga, gb, scratch, slots);
    }
    return (int)hipGetLastError();
}

// The forward product; `scratch` of forward_scratch() floats: of either plan, for the data gradient's transposed W may be aligned
// where W is not.
inline long forward_scratch(const P2pflAdapter& a) {
    if (a.T <= SKINNY_ROWS) {
        const SkinnyParts p = skinny_parts(a);
        return (long)a.T * ((long)p.base * a.Out + (long)p.low * a.R);
    }
    long need = 0;
    for (const WidePlan& p : {staged_plan(a), wide_plan(a)})
        if (p.parts > 1 || p.rows_join) need = max(need, (long)p.parts * a.T * a.Out);
    return need;
}

template <class T>
int product(const P2pflAdapter& a, float* scratch, hipStream_t s) {
    if (a.T <= SKINNY_ROWS) return few_rows<T>(a, scratch, s);
    const int rc = shrink<T>(a, s);
    return rc ? rc : shared_product<T>(a, scratch, s);
}

}  // namespace

// What a type's translation unit offers to the entry points.
template <class T> int adapter_product(const P2pflAdapter& a, float* scratch, hipStream_t s);
template <class T> int adapter_weight_gradients(const P2pflAdapter& a, const float* v, float* dla, long dla_cs, float* dlb, long dlb_cs,
                                                float* scratch, hipStream_t s);

#ifdef ADAPTER_TYPE
template <> int adapter_product<ADAPTER_TYPE>(const P2pflAdapter& a, float* scratch, hipStream_t s) {
    return product<ADAPTER_TYPE>(a, scratch, s);
}
template <> int adapter_weight_gradients<ADAPTER_TYPE>(const P2pflAdapter& a, const float* v, float* dla, long dla_cs, float* dlb,
                                                       long dlb_cs, float* scratch, hipStream_t s) {
    const WgradArgs ga{a.x, a.x_cs, a.x_rs, v, dla, dla_cs, a.In, 1, 1};
    const WgradArgs gb{a.y, a.y_cs, a.y_rs, a.u, dlb, dlb_cs, a.Out, 0, 0};
    return weight_gradients<ADAPTER_TYPE>(a, ga, gb, scratch, s);
}
#endif
