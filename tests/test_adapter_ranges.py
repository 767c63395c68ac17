"""Adapters whose intermediate rows u and v leave the range of the rows' type, by every way rows are multiplied: up to 64 rows, many
rows of few rows a client, many rows in tiles, of aligned and of any rows. Tolerances are those of test_adapter_linear: one
rounding of a result to its type, half a step of the type for u as an operand, fp32 sums."""
import pytest
import torch

from test_adapter_linear import DEV, TYPES, check, clients, make, make_drop, run

WAYS = [  # K, rows, In, Out
    (3, 40, 200, 136), (9, 96, 200, 136), (3, 300, 200, 136), (3, 300, 203, 131), (5, 2100, 328, 2120)]


def ragged(K, T):
    return [0] + [T * (i + 1) // K - i % 2 for i in range(K - 1)] + [T - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,T,In,Out", WAYS)
@pytest.mark.parametrize("fx,fa,fb", [(1.0, 1e5, 1e-4), (1.0, 1e-4, 3e4), (1e-3, 1e-4, 3e4)])
def test_rows_between_the_adapters_of_any_finite_size(K, T, In, Out, fx, fa, fb, dtype):
    """u (first) and v (second) around 2e5, beyond fp16; u around 2e-7 (third), below its smallest normal value. The sums over both
    adapters are of ordinary size again."""
    t = make(K, T, In, Out, 8, TYPES[dtype], uniform=False, cuts=ragged(K, T))
    for n, f in (("x", fx), ("la", fa), ("lb", fb)):
        t[n].copy_(t[n].float() * f)
    assert all(v.isfinite().all() for v in t.values())
    drop = make_drop(0.25, K)
    o = run(t, 2.0, drop)
    big = max(o["u"].abs().max().item(), o["v"].abs().max().item())
    assert big > 65520 and (fx == 1.0 or o["u"].abs().max() < 6.1e-5)
    check(t, o, 2.0, drop)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("K,T,In,Out", WAYS)
def test_rows_between_the_adapters_up_to_the_largest_float(K, T, In, Out, dtype):
    """u = 3.396e38: above the largest bf16, where a rounded term would be infinite."""
    t = make(K, T, In, Out, 4, TYPES[dtype], uniform=False, cuts=ragged(K, T))
    top = torch.finfo(torch.bfloat16).max
    row = torch.arange(T, device=DEV)
    t["x"].zero_()
    t["x"][row, row % In] = 1.0
    t["dy"].zero_()                                            # (their products with la would leave the range of every type)
    t["la"].fill_(top)
    t["lb"].fill_(2.0 ** -125)
    o = run(t, 1.002, None)
    assert (o["u"][:T - 1] > top).all() and o["u"].isfinite().all()
    check(t, o, 1.002, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,T,In,Out", WAYS)
def test_an_infinite_adapter_reaches_its_rows_alone(K, T, In, Out, dtype):
    t = make(K, T, In, Out, 8, TYPES[dtype], uniform=False, cuts=ragged(K, T))
    good = run(t, 1.0, None)
    t["la"][1, 3, 7] = float("inf")
    o = run(t, 1.0, None)
    lo, hi = clients(t)[1]
    other = torch.ones(T, dtype=torch.bool, device=DEV)
    other[lo:hi] = False
    assert torch.equal(o["y"][other], good["y"][other]) and torch.equal(o["dx"][other], good["dx"][other])
    x, b = t["x"][lo:hi, 7].float(), t["lb"][1, :, 3].float()
    sure = (x != 0)[:, None] & (b != 0)[None]
    assert sure.float().mean() > 0.9 and (o["u"][lo:hi, 3][x != 0].isinf()).all()
    got = o["y"][lo:hi].float()
    if dtype == "fp32" and T > 64 and T >= 16 * K:
        # in tiles b is three terms of either sign (or zero), and infinity times each is added up: infinite or NaN, never finite
        assert not got[sure].isfinite().any()
    else:
        want = torch.sign(x)[:, None] * torch.sign(b)[None] * float("inf")
        assert torch.equal(got[sure], want[sure])
