"""Adapters at the limits that the calls state."""
import pytest
import torch

from test_adapter_linear import DEV, TYPES, U, make, make_drop, run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,p", [(60, 0.0), (700, 0.25)])
def test_as_many_clients_as_there_may_be(T, p, dtype):
    """65535 clients, few of them with rows: every client's gradients are written."""
    h = pytest.importorskip("p2pfl_amd.ops.hip")
    K, In, Out, R = h.ADAPTER_MAX_CLIENTS, 12, 20, 2
    owners = {3: (0, 5), 40000: (5, T // 2), 40001: (T // 2, T // 2 + 1), K - 1: (T // 2 + 1, T - 2)}
    ends = torch.zeros(K + 1, dtype=torch.int32)
    for k, (lo, hi) in owners.items():
        ends[k + 1:] = hi
    t = make(K, T, In, Out, R, TYPES[dtype], uniform=False, cuts=ends.tolist())
    drop = make_drop(p, K) if p else None
    o = run(t, 1.0, drop)
    x, dy = t["x"].double().cpu(), t["dy"].double().cpu()
    touched = torch.zeros(K, dtype=torch.bool)
    for k, (lo, hi) in owners.items():
        touched[k] = True
        m = 1.0
        if drop is not None:
            one = torch.ones(1, (hi - lo) * In, device=DEV)
            h.dropout(one, one, h.Drop(p, drop.seeds[k:k + 1], drop.step, drop.site))
            m = (one.view(-1, In) != 0).double().cpu() / (1 - p)
        a, b = t["la"][k].double().cpu(), t["lb"][k].double().cpu()
        u, v = (x[lo:hi] * m) @ a.t(), dy[lo:hi] @ b
        su, sv = (x[lo:hi] * m).abs() @ a.abs().t(), dy[lo:hi].abs() @ b.abs()
        for name, want, size in (("dla", v.t() @ (x[lo:hi] * m), sv.t() @ (x[lo:hi] * m).abs()), ("dlb", dy[lo:hi].t() @ u, dy[lo:hi].abs().t() @ su)):
            tol = ((T + In + Out) ** 0.5 + 16) * U * size + 1e-30          # (as in test_adapter_linear)
            assert ((o[name][k].double().cpu() - want).abs() <= tol).all(), (name, k)
    assert not o["dla"][~touched.to(DEV)].any() and not o["dlb"][~touched.to(DEV)].any()
    assert o["y"].isfinite().all() and (o["u"][T - 2:] == 0).all()


def test_arguments_without_dimensions_are_refused():
    from p2pfl_amd.ops import hip as h
    f = lambda *s: torch.zeros(*s)
    with pytest.raises(h.HipKernelError):
        h.adapter_linear_fwd(f(2, 3, 8), f(5, 8), f(()), f(2, 4, 8), f(2, 5, 4), f(2, 3, 5), f(2, 3, 4))
    for u, v in ((f(()), f(2, 3, 4)), (f(2, 3, 4), f(()))):
        with pytest.raises(h.HipKernelError):
            h.adapter_linear_wgrad(f(2, 3, 5), f(2, 3, 8), u, v, f(2, 4, 8), f(2, 5, 4))
    for x in (f(()), f(8)):
        with pytest.raises(h.HipKernelError):
            h.adapter_linear_fwd(x, f(5, 8), None, f(2, 4, 8), f(2, 5, 4), f(2, 3, 5), f(2, 3, 4))
        with pytest.raises(h.HipKernelError):
            h.adapter_linear_wgrad(f(2, 3, 5), x, f(2, 3, 4), f(2, 3, 4), f(2, 4, 8), f(2, 5, 4))
        with pytest.raises(h.HipKernelError):
            h.group_norm_fwd(x, None, None, x, 1)
    with pytest.raises(h.HipKernelError):
        h.dropout(f(()), f(()), h.Drop(0.1, torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64)))
