"""The large tiles of the adapters' products and long runs of rows, against the plain implementation in 64 bits of test_adapter_linear
(its tolerances). Each shape names what it is the smallest of: tiles of 256 x 256 take about T * Out above 4.2 million."""
import pytest
import torch

from test_adapter_linear import TYPES, check, clients, make, make_drop, run


def cuts_of(K, T):
    """Ragged clients, one of no rows, a few rows behind the last."""
    ends = [T * (i + 1) // K - (7 * i) % 5 for i in range(K)]
    if K > 3:
        ends[2] = ends[1]
    ends[-1] = T - 3
    return [0] + ends


TILES = [  # K, T, In, Out, R, p
    (5, 2100, 328, 2120, 8, 0.2),       # 256 x 256 whole: an odd number of stages, eight columns behind them; dgrad: 128 x 128 in four parts
    (7, 1200, 4104, 1096, 16, 0.0),     # 256 x 256 in eight parts, eight columns behind the last; dgrad: 256 x 256 whole, 17 stages
    (150, 3000, 520, 2056, 12, 0.1),    # thirteen clients in a tile: more than two rounds of six (fp32: four of three)
    (5, 2100, 331, 2121, 40, 0.2),      # rows of any alignment in 256 x 128, two rounds of ranks
    (17, 3000, 1544, 2056, 8, 0.0),     # dgrad in two parts of 256 x 256: clients shared out between them
    (2, 700, 72, 6200, 6, 0.5)]         # one stage


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,T,In,Out,R,p", TILES)
def test_large_tiles(K, T, In, Out, R, p, dtype):
    t = make(K, T, In, Out, R, TYPES[dtype], uniform=False, cuts=cuts_of(K, T))
    drop = make_drop(p, K) if p else None
    o, again = run(t, 0.5, drop), run(t, 0.5, drop)
    for n in o:
        assert torch.equal(o[n], again[n]), n
    check(t, o, 0.5, drop)


LONG = [  # K, T, In, Out, R, p
    (5, 6300, 264, 136, 16, 0.1),       # 32 rows a block of u, 16 ranks: a stage and eight columns
    (5, 6200, 1096, 72, 32, 0.0),       # 32 ranks, several stages
    (5, 6200, 520, 264, 50, 0.2),       # 64 ranks
    (4, 6150, 133, 67, 20, 0.1),        # rows of any alignment
    (3, 8300, 72, 88, 5, 0.3),          # weight gradients in chunks of 512 rows
    (3, 8300, 45, 37, 33, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,T,In,Out,R,p", LONG)
def test_long_runs_of_rows(K, T, In, Out, R, p, dtype):
    t = make(K, T, In, Out, R, TYPES[dtype], uniform=False, cuts=cuts_of(K, T))
    drop = make_drop(p, K) if p else None
    check(t, run(t, 1.5, drop), 1.5, drop)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,B,In,Out,R", [(4, 640, 200, 2056, 8), (2, 3200, 328, 712, 16)])
def test_large_tiles_of_equal_blocks(K, B, In, Out, R, dtype):
    t = make(K, K * B, In, Out, R, TYPES[dtype], uniform=True)
    drop = make_drop(0.1, K)
    o = run(t, 1.0, drop)
    check(t, o, 1.0, drop)
    flat = dict(t, x=t["x"].reshape(K * B, In), dy=t["dy"].reshape(K * B, Out),
                row_ptr=torch.arange(0, K * B + 1, B, dtype=torch.int32, device=t["x"].device))
    for n, v in run(flat, 1.0, drop).items():
        assert torch.equal(v.reshape(-1), o[n].reshape(-1)), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_bad_values_in_large_tiles_stay_in_their_rows(dtype):
    K, T, In, Out = 60, 2100, 328, 2120
    t = make(K, T, In, Out, 8, TYPES[dtype], uniform=False, cuts=cuts_of(K, T))
    good = run(t, 1.0, None)
    for k in (0, 17, K - 1):
        t["la"][k, 3, 5] = float("nan")
        t["lb"][k, 7, 2] = float("nan")
    o = run(t, 1.0, None)
    bad = torch.zeros(T, dtype=torch.bool, device=t["x"].device)
    for k in (0, 17, K - 1):
        lo, hi = clients(t)[k]
        bad[lo:hi] = True
    for n in ("y", "dx"):
        assert torch.equal(o[n][~bad], good[n][~bad])
        assert o[n][bad].isnan().all()
