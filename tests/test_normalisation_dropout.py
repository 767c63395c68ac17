"""Group norm with residual / activation / dropout and the counter-based dropout against plain implementations in 64 bits.

Tolerances: one rounding to the map's type is at most ``eps / 2`` of the value; the fp32 arithmetic before it is a chain of
fewer than 64 roundings of 2^-24 of the largest intermediate value; a sum of n terms errs by at most (additions a term goes
through) x 2^-24 x (sum of the magnitudes)."""
import math

import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def hip():
    from p2pfl_amd.ops import hip as h
    return h


# ------------------------------------------------------------------------------------------------ the generator
def philox(counter, key, rounds):
    """Philox4x32 in Python integers."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_oracle_generator_known_answers():
    """The published Random123 test vectors of philox4x32-10 (all zeros, all ones, digits of pi)."""
    assert philox([0] * 4, [0] * 2, 10) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert philox([0xffffffff] * 4, [0xffffffff] * 2, 10) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert philox([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0], 10) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def kept(seed, step, site, n, p, first=0):
    thr = round(p * 2 ** 32)
    out = []
    for q in range(first // 4, (first + n + 3) // 4):
        out += [w >= thr for w in philox([q & 0xFFFFFFFF, site, step & 0xFFFFFFFF, step >> 32],
                                         [seed & 0xFFFFFFFF, seed >> 32], 7)]
    return torch.tensor(out[first % 4:first % 4 + n])


def make_drop(p, K, site=3, step=5 + 2 ** 35, device=DEV):
    seeds = torch.tensor([0x1234567890ABCDEF + 977 * k for k in range(K)], dtype=torch.int64, device=device)
    return hip().Drop(p, seeds, torch.tensor([step], dtype=torch.int64, device=device), site)


def mask_of(drop, K, n):
    return torch.stack([kept(int(drop.seeds[k]), int(drop.step), drop.site, n, drop.p) for k in range(K)])


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,shape,p", [(1, (1,), 0.5), (3, (7,), 0.3), (2, (33, 5), 0.1), (50, (32, 8), 0.5), (1, (2049,), 0.9),
                                       (4, (1000,), 0.0), (2, (12,), 1.0)])
def test_dropout_mask_and_values(K, shape, p, dtype):
    n = math.prod(shape)
    slab = torch.randn(K, n + 13, device=DEV).to(TYPES[dtype])           # rows of odd stride: vectors of any alignment
    x, y = slab[:, 3:3 + n].unflatten(1, shape), torch.full((K, *shape), 9.0, device=DEV, dtype=TYPES[dtype])
    drop = make_drop(p, K)
    hip().dropout(x, y, drop)
    m = mask_of(drop, K, n).view(K, *shape)
    want = torch.where(m, x.cpu().double() / (1 - p if p < 1 else 1), 0.0)
    err = (y.cpu().double() - want).abs()
    # two fp32 roundings (the factor, the product), one to the type
    assert (err <= want.abs() * (torch.finfo(TYPES[dtype]).eps / 2 + 2.5 * U)).all()
    assert (y.cpu()[~m] == 0).all()


@pytest.mark.gpu
def test_dropout_rows_do_not_depend_on_their_neighbours_and_may_be_in_place():
    x = torch.randn(5, 4099, device=DEV)
    y = torch.empty_like(x)
    drop = make_drop(0.4, 5)
    hip().dropout(x, y, drop)
    for k in (0, 3, 4):
        one = x[k:k + 1].clone()
        hip().dropout(one, one, hip().Drop(0.4, drop.seeds[k:k + 1], drop.step, drop.site))
        assert torch.equal(one[0], y[k])
    other = torch.empty_like(x)
    hip().dropout(x, other, hip().Drop(0.4, drop.seeds, drop.step, drop.site + 1))
    assert not torch.equal(other, y)


@pytest.mark.gpu
def test_dropped_infinities_and_nans_are_zero():
    x = torch.full((2, 4096), float("nan"), device=DEV)
    x[1] = float("inf")
    y = torch.empty_like(x)
    drop = make_drop(0.5, 2)
    hip().dropout(x, y, drop)
    m = mask_of(drop, 2, 4096)
    assert (y.cpu()[~m] == 0).all() and y.cpu()[0][m[0]].isnan().all() and y.cpu()[1][m[1]].isinf().all()
    hip().dropout(x, y, make_drop(1.0, 2))
    assert (y == 0).all()


@pytest.mark.gpu
def test_dropout_element_offsets_beyond_32_bits():
    n = 2 ** 31 + 1029                                                   # bytes and elements of one client pass 2^31
    x = torch.ones(1, n, device=DEV, dtype=torch.bfloat16)
    hip().dropout(x, x, make_drop(0.5, 1))
    d = make_drop(0.5, 1)
    want = kept(int(d.seeds[0]), int(d.step), d.site, 1029, 0.5, first=2 ** 31)
    assert torch.equal(x[0, 2 ** 31:].cpu() != 0, want)
    assert torch.equal(x[0, :1024].cpu() != 0, kept(int(d.seeds[0]), int(d.step), d.site, 1024, 0.5))


@pytest.mark.gpu
def test_dropout_in_a_graph_follows_the_step():
    x = torch.randn(3, 1000, device=DEV)
    y, drop = torch.empty_like(x), make_drop(0.3, 3, step=0)
    hip().dropout(x, y, drop)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hip().dropout(x, y, drop)
        drop.step.add_(1)
    seen = []
    for i in range(4):
        eager = torch.empty_like(x)
        hip().dropout(x, eager, drop)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and int(drop.step) == i + 1
        assert all(not torch.equal(y, s) for s in seen)
        seen.append(y.clone())


# ------------------------------------------------------------------------------------------------ group norm
def gn_reference(x, w, b, G, act, res, mask, p, eps, dy=None, y_given=None):
    """fp64 on the CPU by the formulas: (y, mean, rstd, z) and, with dy, (dx, dw, db, dz) and the sums' magnitudes."""
    K, N, C = x.shape[0], x.shape[1], x.shape[-1]
    x = x.double().cpu().reshape(K, N, -1, C)
    S, c = x.shape[2], C // G
    w = torch.ones(K, C).double() if w is None else w.double().cpu()
    b = torch.zeros(K, C).double() if b is None else b.double().cpu()
    g = x.view(K, N, S, G, c)
    mean = g.mean(dim=(2, 4))
    var = (g - mean[:, :, None, :, None]).pow(2).mean(dim=(2, 4))
    rstd = (var + eps).rsqrt()
    xh = ((g - mean[:, :, None, :, None]) * rstd[:, :, None, :, None]).view(K, N, S, C)
    z = xh * w[:, None, None] + b[:, None, None]
    if res is not None:
        z = z + res.double().cpu().reshape(z.shape)
    f = torch.nn.functional
    y = {"none": lambda t: t, None: lambda t: t, "relu": f.relu, "silu": f.silu, "gelu": f.gelu}[act](z)
    k = torch.ones_like(z) if mask is None else mask.view(z.shape).double() / (1 - p)
    y = y * k
    if dy is None:
        return y, mean, rstd, z
    dz = dyk = dy.double().cpu().reshape(z.shape) * k
    if act == "relu":
        dz = dz * ((y_given.double().cpu().reshape(z.shape) if y_given is not None else z) > 0)
    elif act in ("silu", "gelu"):
        zz = z.clone().requires_grad_()
        dz = torch.autograd.grad({"silu": f.silu, "gelu": f.gelu}[act](zz), zz, dz)[0]
    t = (dz * w[:, None, None]).view(K, N, S, G, c)
    xg = xh.view(K, N, S, G, c)
    m1, m2 = t.mean(dim=(2, 4), keepdim=True), (t * xg).mean(dim=(2, 4), keepdim=True)
    dx = ((t - m1 - xg * m2) * rstd[:, :, None, :, None]).view(K, N, S, C)
    size = ((t.abs() + m1.abs() + (xg * m2).abs()) * rstd[:, :, None, :, None]).max()
    # magnitudes of the terms of dw and db. The gradient of an activation is at most 1.13, so a term is at most 1.13 |dy|
    # (|xhat|), and the roundings of x - mean shift xhat and z - and through act'', at most 1 / 2, act'(z) - by an absolute
    # U max|x| rstd: |dy| (1 + |xhat|) bounds what a relative error of a few U max|x| rstd applies to.
    return dx, (dz * xh).sum(dim=(1, 2)), dz.sum(dim=(1, 2)), dz, size, (dyk.abs() * (1 + xh.abs())).sum(dim=(1, 2)), dyk.abs().sum(dim=(1, 2))


def close(got, want, size):
    """One rounding to the type plus fp32 arithmetic on values up to ``size``."""
    tol = want.abs() * (torch.finfo(got.dtype).eps / 2) + 64 * U * float(size)
    tol = tol + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps       # (half a subnormal step of fp16)
    bad = (got.cpu().double().reshape(want.shape) - want).abs() - tol
    assert bad.max() <= 0, f"off by {bad.max():.3e} beyond the tolerance"


def slab_param(K, C, offset=0.0):
    return (torch.randn(K, C + 77, device=DEV) * 0.3 + offset)[:, 5:5 + C]


SHAPES = [  # K, N, positions, C, G
    (1, 1, (1,), 4, 2), (1, 1, (1,), 1, 1), (2, 3, (4, 4), 64, 32), (3, 2, (15, 15), 45, 9), (1, 2, (7,), 6, 6),
    (2, 1, (3, 5), 3, 1), (1, 3, (32, 32), 64, 8), (2, 2, (64, 64), 24, 3), (1, 1, (2, 2), 2048, 1), (1, 2, (9,), 4100, 4),
    (1, 1, (300, 5), 2048, 2), (4, 5, (2, 3, 2), 20, 4), (1, 2, (1000,), 8, 2), (2, 2, (129,), 130, 13)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,N,pos,C,G", SHAPES)
def test_group_norm_forward_and_backward(K, N, pos, C, G, dtype):
    h, dt = hip(), TYPES[dtype]
    for act, with_res, p in (("none", False, 0.0), ("relu", True, 0.0), ("silu", False, 0.25), ("gelu", True, 0.0), ("relu", False, 0.5)):
        x = (torch.randn(K, N, *pos, C, device=DEV) * 1.5 + 0.5).to(dt)
        res = torch.randn_like(x) if with_res else None
        w, b = slab_param(K, C, 1.0), slab_param(K, C)
        drop = make_drop(p, K) if p else None
        n = x[0].numel()
        mask = None
        if p:                            # (the mask itself is checked above: here it comes from the plain call)
            one = torch.empty(K, n, device=DEV)
            h.dropout(torch.ones(K, n, device=DEV), one, drop)
            mask = (one != 0).cpu()
        y, mean, rstd = torch.empty_like(x), torch.empty(K, N, G, device=DEV), torch.empty(K, N, G, device=DEV)
        h.group_norm_fwd(x, w, b, y, G, mean=mean, rstd=rstd, act=act, residual=res, drop=drop)
        ry, rmean, rrstd, z = gn_reference(x, w, b, G, act, res, mask, p, 1e-5)
        group = n // N // G
        size = max(float(z.abs().max()), float(ry.abs().max()), 1.0)
        # a group of few elements divides by a small deviation: xhat errs by the roundings of x relative to 1 / rstd
        size = size + float((x.abs().max() * rstd.max()).cpu()) * (1.0 if group < 4096 else 2.0)
        close(y, ry, size)
        assert ((mean.cpu().double() - rmean).abs() <= 64 * U * x.abs().max().item()).all()
        assert ((rstd.cpu().double() - rrstd).abs() <= rrstd * (64 * U) * (1 + (x.abs().max().item() * rrstd))).all()
        dy = torch.randn_like(x)
        dx, dres = torch.empty_like(x), torch.empty_like(x) if with_res else None
        dw, db = slab_param(K, C), slab_param(K, C)
        by_y = y if act == "relu" else None
        m64, r64 = rmean.float().to(DEV), rrstd.float().to(DEV)
        h.group_norm_bwd(dy, x, w, b, m64, r64, dx, dw, db, G, act=act, y=by_y, residual=None if by_y is not None else res,
                         dres=dres, drop=drop)
        rdx, rdw, rdb, rdz, gsize, aw, ab = gn_reference(x, w, b, G, act, res, mask, p, 1e-5, dy, by_y)
        amp = 1 + float((x.abs().max() * rstd.max()).cpu())              # xhat's own error, relative to its size
        close(dx, rdx, float(gsize) * amp)
        if with_res:
            close(dres, rdz, float(rdz.abs().max()) * amp)
        adds = 64 + N + math.prod(pos) / 128
        for got, want, mag in ((dw, rdw, aw), (db, rdb, ab)):
            assert ((got.cpu().double() - want).abs() <= U * mag * (adds + 64 * amp) + 1e-30).all()


@pytest.mark.gpu
def test_group_norm_gradient_against_differences():
    h = hip()
    K, N, S, C, G, e = 1, 2, 6, 8, 2, 1e-2
    x, w, b = torch.randn(K, N, S, C, device=DEV), torch.randn(K, C, device=DEV), torch.randn(K, C, device=DEV)
    dy = torch.randn_like(x)
    mean, rstd = torch.empty(K, N, G, device=DEV), torch.empty(K, N, G, device=DEV)

    def loss(x_, w_):
        y = torch.empty_like(x_)
        h.group_norm_fwd(x_, w_, b, y, G, mean=mean, rstd=rstd, act="silu")
        return (y.double() * dy.double()).sum().item()
    loss(x, w)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    h.group_norm_bwd(dy, x, w, b, mean, rstd, dx, dw, db, G, act="silu")
    for t, g in ((x, dx), (w, dw)):
        for i in range(0, t.numel(), 7):
            hi, lo = t.clone(), t.clone()
            hi.view(-1)[i] += e
            lo.view(-1)[i] -= e
            d = (loss(*((hi, w) if t is x else (x, hi))) - loss(*((lo, w) if t is x else (x, lo)))) / (2 * e)
            # central difference: e^2 / 6 of a third derivative of size ~100, and the fp32 values' 1e-6 / (2 e)
            assert abs(d - g.view(-1)[i].item()) < 2e-3 * max(1.0, abs(d)) + 3e-3


@pytest.mark.gpu
def test_group_norm_of_maps_far_from_zero():
    """mean = 1000 deviations: squares around the mean, not a difference of squares (which would lose every digit)."""
    x = torch.randn(1, 3, 32 * 32, 64, device=DEV) + 1000.0
    y = torch.empty_like(x)
    for S in (1024, 1024 * 3):                          # one slab, and chunks that are joined
        xx, yy = x.view(1, -1, S, 64), y.view(1, -1, S, 64)
        hip().group_norm_fwd(xx, None, None, yy, 8)
        ref = gn_reference(xx, None, None, 8, None, None, None, 0, 1e-5)[0]
        close(yy, ref, 1000.0 * 4)


@pytest.mark.gpu
@pytest.mark.parametrize("S", [9, 5000])
def test_group_norm_strided_maps_in_place_and_broadcast_gradients(S):
    h = hip()
    K, N, C, G = 3, 2, 16, 4
    big = torch.randn(N, S, K * C, device=DEV)                                  # clients side by side in the channels
    x = big.view(N, S, K, C).permute(2, 0, 1, 3)
    w, b = slab_param(K, C, 1.0), slab_param(K, C)
    y, mean, rstd = torch.empty(K, N, S, C, device=DEV), torch.empty(K, N, G, device=DEV), torch.empty(K, N, G, device=DEV)
    h.group_norm_fwd(x, w, b, y, G, mean=mean, rstd=rstd, act="gelu")
    packed = torch.empty_like(y)
    h.group_norm_fwd(x.contiguous(), w, b, packed, G, act="gelu")
    assert torch.equal(y, packed)
    dy = torch.randn(K, N, 1, C, device=DEV).expand(K, N, S, C)                 # the gradient of a mean over positions
    dx, dw, db = torch.empty_like(y), torch.empty(K, C, device=DEV), torch.empty(K, C, device=DEV)
    h.group_norm_bwd(dy, x, w, b, mean, rstd, dx, dw, db, G, act="gelu")
    dxp, dwp, dbp = dy.contiguous(), torch.empty(K, C, device=DEV), torch.empty(K, C, device=DEV)
    h.group_norm_bwd(dxp, x.contiguous(), w, b, mean, rstd, dxp, dwp, dbp, G, act="gelu")     # gradient in place
    assert torch.equal(dx, dxp) and torch.equal(dw, dwp) and torch.equal(db, dbp)
    before = big.clone()
    h.group_norm_fwd(x, w, b, x, G, act="gelu")                                 # the strided map in place
    assert torch.equal(x, y) and not torch.equal(before, big)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", ["relu", "silu"])
@pytest.mark.parametrize("S,C,G", [(9, 20, 4), (1024, 64, 8), (9000, 32, 4)])
def test_group_norm_results_in_the_place_of_their_inputs(S, C, G, act, dtype):
    h, dt = hip(), TYPES[dtype]
    K, N = 2, 3
    x, res, dy = (torch.randn(K, N, S, C, device=DEV).to(dt) for _ in range(3))
    w, b, drop = slab_param(K, C, 1.0), slab_param(K, C), make_drop(0.25, K)
    mean, rstd = (torch.empty(K, N, G, device=DEV) for _ in range(2))
    dw, db, dw2, db2 = (torch.empty(K, C, device=DEV) for _ in range(4))
    y, dx, dres = (torch.empty_like(x) for _ in range(3))
    h.group_norm_fwd(x, w, b, y, G, mean=mean, rstd=rstd, act=act, residual=res, drop=drop)
    for place in (x.clone(), res.clone()):
        first = torch.equal(place, x)
        h.group_norm_fwd(place if first else x, w, b, place, G, act=act, residual=res if first else place, drop=drop)
        assert torch.equal(place, y)
    kw = dict(act=act, drop=drop, **(dict(y=y) if act == "relu" else dict(residual=res)))
    h.group_norm_bwd(dy, x, w, b, mean, rstd, dx, dw, db, G, dres=dres, **kw)
    for swap in (False, True):
        px, pdy = x.clone(), dy.clone()
        h.group_norm_bwd(pdy, px, w, b, mean, rstd, px if swap else pdy, dw2, db2, G, dres=pdy if swap else px, **kw)
        assert torch.equal(px if swap else pdy, dx) and torch.equal(pdy if swap else px, dres)
        assert torch.equal(dw2, dw) and torch.equal(db2, db)


@pytest.mark.gpu
@pytest.mark.parametrize("S", [64, 6000])
def test_group_norm_bad_values_stay_in_their_group(S):
    h = hip()
    x = torch.randn(2, 2, S, 24, device=DEV)
    good = torch.empty_like(x)
    h.group_norm_fwd(x, None, None, good, 3, act="relu")
    x[1, 0, S // 2, 9] = float("nan")
    x[0, 1, S - 1, 23] = float("inf")
    y = torch.empty_like(x)
    h.group_norm_fwd(x, None, None, y, 3, act="relu")
    hit = torch.zeros(2, 2, 1, 24, dtype=torch.bool, device=DEV)
    hit[1, 0, :, 8:16] = True
    hit[0, 1, :, 16:] = True
    hit = hit.expand_as(y)
    assert y[hit].isnan().all() and torch.equal(y[~hit], good[~hit])


@pytest.mark.gpu
def test_group_norm_without_elements_and_repeats():
    h = hip()
    dw, db = torch.ones(2, 8, device=DEV), torch.ones(2, 8, device=DEV)
    x = torch.empty(2, 0, 4, 8, device=DEV)
    st = torch.empty(2, 0, 2, device=DEV)
    h.group_norm_fwd(x, None, None, x.clone(), 2, mean=st, rstd=st)
    h.group_norm_bwd(x, x, None, None, st, st, x.clone(), dw, db, 2)
    assert (dw == 0).all() and (db == 0).all()
    x, dy = torch.randn(3, 33, 700, 48, device=DEV), torch.randn(3, 33, 700, 48, device=DEV)
    w, b = slab_param(3, 48, 1.0), slab_param(3, 48)
    outs = []
    for _ in range(3):                                                          # every sum has a fixed order
        y, mean, rstd = torch.empty_like(x), torch.empty(3, 33, 6, device=DEV), torch.empty(3, 33, 6, device=DEV)
        h.group_norm_fwd(x, w, b, y, 6, mean=mean, rstd=rstd, act="silu")
        dx, dw, db = torch.empty_like(x), torch.empty(3, 48, device=DEV), torch.empty(3, 48, device=DEV)
        h.group_norm_bwd(dy, x, w, b, mean, rstd, dx, dw, db, 6, act="silu")
        outs.append((y, mean, rstd, dx, dw, db))
    for o in outs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(o, outs[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("S", [16, 6000])
def test_group_norm_in_graphs_that_run_beside_each_other(S):
    """Two captured graphs own their workspaces: replayed on two streams they do not disturb each other."""
    h = hip()
    sets = []
    for i in range(2):
        x, dy = torch.randn(2, 8, S, 32, device=DEV), torch.randn(2, 8, S, 32, device=DEV)
        t = {"x": x, "dy": dy, "w": slab_param(2, 32, 1.0), "b": slab_param(2, 32), "y": torch.empty_like(x),
             "m": torch.empty(2, 8, 4, device=DEV), "r": torch.empty(2, 8, 4, device=DEV), "dx": torch.empty_like(x),
             "dw": torch.empty(2, 32, device=DEV), "db": torch.empty(2, 32, device=DEV)}

        def step(t=t):
            h.group_norm_fwd(t["x"], t["w"], t["b"], t["y"], 4, mean=t["m"], rstd=t["r"], act="silu")
            h.group_norm_bwd(t["dy"], t["x"], t["w"], t["b"], t["m"], t["r"], t["dx"], t["dw"], t["db"], 4, act="silu")
        step()
        torch.cuda.synchronize()
        want = {k: t[k].clone() for k in ("y", "dx", "dw", "db")}
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        sets.append((t, want, g, torch.cuda.Stream()))
    for _ in range(3):
        for t, _, _, _ in sets:
            for k in ("y", "dx", "dw", "db"):
                t[k].zero_()
        torch.cuda.synchronize()
        for _, _, g, st in sets:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for t, want, _, _ in sets:
            assert all(torch.equal(t[k], v) for k, v in want.items())


# ------------------------------------------------------------------------------------------------ refusals (no GPU needed)
@pytest.mark.gpu
@pytest.mark.parametrize("K,N,S,C,G", [(2, 3, 16, 64, 8), (1, 1, 6000, 64, 2), (2, 2, 5000, 45, 9)])
def test_group_norm_with_its_own_workspace_on_another_stream(K, N, S, C, G):
    h = hip()
    for dt in TYPES.values():
        x, dy = torch.randn(K, N, S, C, device=DEV).to(dt), torch.randn(K, N, S, C, device=DEV).to(dt)
        w, b = slab_param(K, C, 1.0), slab_param(K, C)
        new = lambda: (torch.empty_like(x), torch.empty(K, N, G, device=DEV), torch.empty(K, N, G, device=DEV), torch.empty_like(x),
                       torch.empty(K, C, device=DEV), torch.empty(K, C, device=DEV))

        def both(y, mean, rstd, dx, dw, db, fs=None, bs=None):
            h.group_norm_fwd(x, w, b, y, G, mean=mean, rstd=rstd, act="silu", scratch=fs)
            h.group_norm_bwd(dy, x, w, b, mean, rstd, dx, dw, db, G, act="silu", scratch=bs)

        want = new()
        both(*want)
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            fs, bs = (h.group_norm_scratch(K, N, S, C, G, dt, x.device, back) for back in (False, True))
            for _ in range(3):
                for buf in (fs, bs):
                    if buf is not None:
                        buf.fill_(float("nan"))
                got = new()
                both(*got, fs, bs)
                assert all(torch.equal(p, q) for p, q in zip(got, want))
        with pytest.raises(h.HipKernelError, match="workspace"):
            h.group_norm_bwd(dy, x, w, b, *want[1:], G, act="silu", scratch=bs[:-1])


def test_dropout_refusals():
    h = hip()
    s, t = torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int64)
    for bad in (lambda: h.Drop(-0.1, s, t), lambda: h.Drop(1.1, s, t), lambda: h.Drop(float("nan"), s, t),
                lambda: h.Drop(0.1, s.int(), t), lambda: h.Drop(0.1, s, torch.zeros(2, dtype=torch.int64)),
                lambda: h.Drop(0.1, s, t, -1), lambda: h.Drop(0.1, s, t, 2 ** 32)):
        with pytest.raises(h.HipKernelError):
            bad()
    d, x = h.Drop(0.1, s, t), torch.zeros(2, 8)
    for a, b in ((x.double(), x.double()), (x, x.half()), (x, torch.zeros(2, 9)), (torch.zeros(3, 8), torch.zeros(3, 8)),
                 (torch.zeros(8, 2).t(), x), (x, torch.zeros(1, 8).expand(2, 8)),
                 (torch.zeros(2, 1).expand(2, 2 ** 34 + 1),) * 2,
                 (x, x)):                                       # (the last one: nothing wrong but the device)
        with pytest.raises(h.HipKernelError):
            h.dropout(a, b, d)


def test_group_norm_refusals():
    h = hip()
    x, w = torch.zeros(2, 3, 4, 6), torch.zeros(2, 6)
    st = torch.zeros(2, 3, 2)
    ok = dict(w=w, b=w, y=x.clone(), groups=2)

    def fwd(x=x, **kw):
        a = {**ok, **kw}
        h.group_norm_fwd(x, a.pop("w"), a.pop("b"), a.pop("y"), a.pop("groups"), **a)
    for kw in (dict(groups=4), dict(groups=0), dict(act="tanh"), dict(w=torch.zeros(2, 5)), dict(w=w.half()),
               dict(y=x.half()), dict(y=torch.zeros(2, 3, 4, 1).expand(2, 3, 4, 6)), dict(x=torch.zeros(2, 6)),
               dict(x=torch.zeros(2, 3, 6, 4).transpose(2, 3)), dict(residual=torch.zeros(2, 3, 4, 5)), dict(x=x.double()),
               dict(mean=torch.zeros(2, 3, 3)), dict(rstd=st.double()),
               dict(drop=h.Drop(0.1, torch.zeros(3, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))),
               dict(x=torch.zeros(1, 1, 1, 2049), w=None, b=None, y=torch.zeros(1, 1, 1, 2049), groups=1), dict()):
        with pytest.raises(h.HipKernelError):
            fwd(**kw)
    for kw in (dict(mean=None), dict(dw=torch.zeros(2, 5)), dict(dx=torch.zeros(2, 3, 4, 5)), dict(dres=x.half()),
               dict(dw=torch.zeros(1, 6).expand(2, 6)), dict()):
        a = dict(mean=st, rstd=st, dx=x.clone(), dw=w.clone(), db=w.clone()) | kw
        with pytest.raises(h.HipKernelError):
            h.group_norm_bwd(x, x, w, w, a["mean"], a["rstd"], a["dx"], a["dw"], a["db"], 2, dres=a.get("dres"))
