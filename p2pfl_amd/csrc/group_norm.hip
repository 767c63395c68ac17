// Entry points of the group norm (group_norm.h): sizes of workspaces, the choice of the maps' type.
#include "group_norm.h"

namespace {

int pass_of(const P2pflGroupNorm& a, bool backwards, void* stream) {
    switch (a.dtype) {
        case DT_F32: return group_norm_pass<float>(a, backwards, (hipStream_t)stream);
        case DT_BF16: return group_norm_pass<__bf16>(a, backwards, (hipStream_t)stream);
        case DT_F16: return group_norm_pass<_Float16>(a, backwards, (hipStream_t)stream);
    }
    return -2;
}

}  // namespace


P2PFL_API int p2pfl_group_norm_fwd(const P2pflGroupNorm* a, void* stream) {
    if (a->K <= 0 || a->N <= 0 || a->S <= 0) return 0;
    return pass_of(*a, false, stream);
}

P2PFL_API int p2pfl_group_norm_bwd(const P2pflGroupNorm* a, void* stream) {
    if (a->K <= 0) return 0;
    if (a->N <= 0 || a->S <= 0) {                  // no elements: gradients of nothing are zero
        P2pflGroupNorm none = *a;
        none.N = 0;
        return param_grads(none, nullptr, (hipStream_t)stream);
    }
    return pass_of(*a, true, stream);
}

// Floats of scratch memory the two calls need (0: none).
P2PFL_API long p2pfl_group_norm_fwd_scratch(int K, int N, int S, int C, int G, int dtype) {
    P2pflGroupNorm a{};
    a.K = K; a.N = N; a.S = S; a.C = C; a.G = G; a.dtype = dtype;
    if (K <= 0 || N <= 0 || S <= 0) return 0;
    const Cut c = cut_of(a, vec_of(a), FWD);
    return c.chunks == 1 ? 0 : 2L * K * N * G * (c.chunks + 1);
}

P2PFL_API long p2pfl_group_norm_bwd_scratch(int K, int N, int S, int C, int G, int dtype) {
    P2pflGroupNorm a{};
    a.K = K; a.N = N; a.S = S; a.C = C; a.G = G; a.dtype = dtype;
    if (K <= 0 || N <= 0 || S <= 0) return 0;
    const Cut c = cut_of(a, BWD_VECTOR, backward_limits(a));
    return 2L * K * N * C * (c.chunks > 1 ? c.chunks + 1 : 1);
}
