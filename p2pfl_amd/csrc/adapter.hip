// Entry points of the low-rank adapters (adapter.h): sizes of workspaces, the transpositions of the data gradient, the choice of
// the rows' type.
#include "adapter.h"

namespace {

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
