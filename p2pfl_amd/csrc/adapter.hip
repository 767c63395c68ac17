// Entry points of the low-rank adapters (adapter.h): sizes of workspaces, the transpositions of the data gradient, the choice of
// the rows' type.
#include "adapter.h"

namespace {

// ------------------------------------------------------------------------------------------------ transposition
// [batch][rows][cols] -> [batch][cols][rows], 64 x 64 tiles through LDS; W, B and A of a data gradient in one launch.
template <class U>
struct Flip {
    const U* src; long s_cs, s_rs;
    U* dst; int batch, rows, cols;
    __host__ __device__ int tiles_r() const { return (rows + 63) / 64; }
    __host__ __device__ int tiles_c() const { return (cols + 63) / 64; }
    __host__ __device__ int tiles() const { return batch * tiles_r() * tiles_c(); }
};

template <class U>
__global__ __launch_bounds__(256) void transpose_kernel(Flip<U> w, Flip<U> b, Flip<U> a) {
    __shared__ U tile[64][64 + 4 / sizeof(U)];
    int id = blockIdx.x;
    const int nw = w.tiles(), nb = b.tiles();
    const Flip<U> f = id < nw ? w : id < nw + nb ? b : a;
    id -= id < nw ? 0 : id < nw + nb ? nw : nw + nb;
    const int c0 = id % f.tiles_c() * 64, r0 = id / f.tiles_c() % f.tiles_r() * 64, k = id / (f.tiles_c() * f.tiles_r());
    const U* src = f.src + k * f.s_cs;
    U* dst = f.dst + (long)k * f.rows * f.cols;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll 8
    for (int r = ty; r < 64; r += 4)
        if (r0 + r < f.rows && c0 + tx < f.cols) tile[r][tx] = src[(long)(r0 + r) * f.s_rs + c0 + tx];
    __syncthreads();
#pragma unroll 8
    for (int c = ty; c < 64; c += 4)
        if (c0 + c < f.cols && r0 + tx < f.rows) dst[(long)(c0 + c) * f.rows + r0 + tx] = tile[tx][c];
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

// W, A and B transposed, each rounded up to 16 bytes.
struct Transposed {
    long w, b, a;
    Transposed(const P2pflAdapter& p) {
        auto up = [&](long n) { return (floats_of(n, p.dtype) + 3) / 4 * 4; };
        w = up((long)p.In * p.Out); b = up((long)p.K * p.R * p.In); a = up((long)p.K * p.R * p.Out);
    }
};

}  // namespace

// Floats of scratch memory the two products need.
P2PFL_API long p2pfl_adapter_linear_scratch(const P2pflAdapter* a, int dgrad) {
    if (a->T <= 0) return 0;
    const Transposed t(*a);
    return forward_scratch(*a) + (dgrad ? t.w + t.b + t.a : 0);
}

P2PFL_API int p2pfl_adapter_linear_fwd(const P2pflAdapter* a, float* scratch, long scratch_len, void* stream) {
    if (a->T <= 0) return 0;
    if (scratch_len < p2pfl_adapter_linear_scratch(a, 0)) return -5;
    return by_type(a->dtype, [&](auto t) { return adapter_product<decltype(t)>(*a, scratch, (hipStream_t)stream); });
}

// As the forward pass with dy for x and the roles of A and B exchanged: `a` holds x = dy, In = the projection's outputs, Out =
// its inputs, w [In][Out] as stored, la = B [K][In][R], lb = A [K][R][Out].
P2PFL_API int p2pfl_adapter_linear_dgrad(const P2pflAdapter* a0, float* scratch, long scratch_len, void* stream) {
    P2pflAdapter a = *a0;
    if (a.T <= 0) return 0;
    if (scratch_len < p2pfl_adapter_linear_scratch(a0, 1)) return -5;
    hipStream_t s = (hipStream_t)stream;
    const Transposed len(a);
    float* wt = scratch;                                             // [Out][In]
    float* bt = wt + len.w;                                          // B transposed: [K][R][In]
    float* at = bt + len.b;                                          // A transposed: [K][Out][R]
    auto all = [&](auto u) {
        typedef decltype(u) U;
        const Flip<U> fw{(const U*)a.w, 0, a.w_rs, (U*)wt, 1, a.In, a.Out};
        const Flip<U> fb{(const U*)a.la, a.la_cs, a.R, (U*)bt, a.K, a.In, a.R};
        const Flip<U> fa{(const U*)a.lb, a.lb_cs, a.Out, (U*)at, a.K, a.R, a.Out};
        const long tiles = (long)fw.tiles() + fb.tiles() + fa.tiles();
        if (tiles * 256 > 0xffffffffL) return -3;
        transpose_kernel<U><<<(unsigned)tiles, 256, 0, s>>>(fw, fb, fa);
        return (int)hipGetLastError();
    };
    const int rc = a.dtype == DT_F32 ? all(0u) : all((unsigned short)0);
    if (rc) return rc;
    a.w = wt; a.w_rs = a.In;
    a.la = bt; a.la_cs = (long)a.R * a.In;
    a.lb = at; a.lb_cs = (long)a.R * a.Out;
    a.drop_out = 1;
    return by_type(a.dtype, [&](auto t) { return adapter_product<decltype(t)>(a, at + len.a, s); });
}

P2PFL_API long p2pfl_adapter_linear_wgrad_scratch(const P2pflAdapter* a) { return wgrad_slots(*a) * a->R * ((long)a->In + a->Out); }

// dA and dB (null: not wanted). `a` as in the forward pass, with y = dy and u; v beside it.
P2PFL_API int p2pfl_adapter_linear_wgrad(const P2pflAdapter* a, const float* v, float* dla, long dla_cs, float* dlb, long dlb_cs,
                                         float* scratch, long scratch_len, void* stream) {
    if (a->K <= 0) return 0;
    if (scratch_len < p2pfl_adapter_linear_wgrad_scratch(a)) return -5;
    return by_type(a->dtype, [&](auto t) {
        return adapter_weight_gradients<decltype(t)>(*a, v, dla, dla_cs, dlb, dlb_cs, scratch, (hipStream_t)stream);
    });
}
