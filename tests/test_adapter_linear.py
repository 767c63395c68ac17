"""Low-rank adapters of many clients beside one shared projection against a plain implementation in 64 bits.

Tolerances: a result is rounded once to its type (``eps / 2`` of the value). Before it stands a sum of n products in fp32,
which errs by at most n 2^-24 of the sum of the products' magnitudes; a blocked sum of random terms stays under
4 sqrt(n) 2^-24 of the root of their squares' sum times sqrt(n) - the bound used is (sqrt(n) + 16) 2^-24 of the magnitudes'
sum. In 16 bits u (v) is rounded once as an operand of the adapters' part: eps / 2 of that part's magnitudes."""
import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def hip():
    from p2pfl_amd.ops import hip as h
    return h


def make(K, T, In, Out, R, dt, *, uniform, bias=True, cuts=None, seed_slab=True):
    g = lambda *s, f=1.0: (torch.randn(*s, device=DEV) * f).to(dt)
    lead = (K, T // K) if uniform else (T,)
    t = {"x": g(*lead, In), "dy": g(*lead, Out), "w": g(Out, In, f=In ** -0.5), "b": g(Out) if bias else None,
         "la": g(K, R * In + 24, f=In ** -0.5)[:, 8:8 + R * In].unflatten(1, (R, In)),         # slab views
         "lb": g(K, R * Out + 24, f=R ** -0.5)[:, 8:8 + R * Out].unflatten(1, (Out, R)), "row_ptr": None}
    if not uniform:
        t["row_ptr"] = torch.tensor(cuts, dtype=torch.int32, device=DEV)
    return t


def run(t, scale, drop):
    h = hip()
    K, R, In = t["la"].shape
    Out = t["w"].shape[0]
    lead = t["x"].shape[:-1]
    dt = t["x"].dtype
    o = {"y": torch.full((*lead, Out), 7.0, device=DEV, dtype=dt), "u": torch.full((*lead, R), 7.0, device=DEV),
         "dx": torch.full((*lead, In), 7.0, device=DEV, dtype=dt), "v": torch.full((*lead, R), 7.0, device=DEV),
         "dla": torch.full((K, R, In), 7.0, device=DEV), "dlb": torch.full((K, Out, R), 7.0, device=DEV)}
    kw = dict(row_ptr=t["row_ptr"], drop=drop)
    h.adapter_linear_fwd(t["x"], t["w"], t["b"], t["la"], t["lb"], o["y"], o["u"], scale=scale, **kw)
    h.adapter_linear_dgrad(t["dy"], t["w"], t["la"], t["lb"], o["dx"], o["v"], scale=scale, **kw)
    h.adapter_linear_wgrad(t["dy"], t["x"], o["u"], o["v"], o["dla"], o["dlb"], **kw)
    return o


def clients(t):
    K = t["la"].shape[0]
    if t["row_ptr"] is None:
        B = t["x"].shape[1]
        return [(k * B, (k + 1) * B) for k in range(K)]
    p = t["row_ptr"].tolist()
    return list(zip(p, p[1:]))


def masks(t, drop):
    """Factors 0 or 1 / (1 - p) of every client's own rows, from the plain dropout call."""
    In, out = t["x"].shape[-1], []
    for k, (lo, hi) in enumerate(clients(t)):
        if drop is None or hi <= lo:
            out.append(1.0)
            continue
        one = torch.ones(1, (hi - lo) * In, device=DEV)
        hip().dropout(one, one, hip().Drop(drop.p, drop.seeds[k:k + 1], drop.step, drop.site))
        out.append((one.view(-1, In) != 0).double().cpu() / (1 - drop.p))
    return out


def reference(t, scale, m):
    """fp64 results, the magnitudes' sums of the shared and of the adapters' parts, and of the products' factors."""
    d = {k: v.double().cpu().reshape(-1, v.shape[-1]) if k in ("x", "dy") else v.double().cpu()
         for k, v in t.items() if v is not None and k != "row_ptr"}
    (K, R, In), Out, T = d["la"].shape, d["w"].shape[0], d["x"].shape[0]
    z = torch.zeros
    r = {"y": d["x"] @ d["w"].t() + d.get("b", 0.0), "u": z(T, R).double(), "dx": d["dy"] @ d["w"], "v": z(T, R).double(),
         "dla": z(K, R, In).double(), "dlb": z(K, Out, R).double()}
    s = {"y": d["x"].abs() @ d["w"].abs().t(), "u": z(T, R).double(), "dx": d["dy"].abs() @ d["w"].abs(), "v": z(T, R).double(),
         "dla": z(K, R, In).double(), "dlb": z(K, Out, R).double()}
    low = {"y": z(T, Out).double(), "dx": z(T, In).double()}
    for k, (lo, hi) in enumerate(clients(t)):
        a, b, xd, dy = d["la"][k], d["lb"][k], d["x"][lo:hi] * m[k], d["dy"][lo:hi]
        r["u"][lo:hi], r["v"][lo:hi] = scale * xd @ a.t(), scale * dy @ b
        s["u"][lo:hi], s["v"][lo:hi] = scale * xd.abs() @ a.abs().t(), scale * dy.abs() @ b.abs()
        r["y"][lo:hi] += r["u"][lo:hi] @ b.t()
        r["dx"][lo:hi] += (r["v"][lo:hi] @ a) * m[k]
        low["y"][lo:hi] = s["u"][lo:hi] @ b.abs().t()
        low["dx"][lo:hi] = (s["v"][lo:hi] @ a.abs()) * m[k]
        r["dla"][k], r["dlb"][k] = r["v"][lo:hi].t() @ xd, dy.t() @ r["u"][lo:hi]
        s["dla"][k], s["dlb"][k] = s["v"][lo:hi].t() @ xd.abs(), dy.abs().t() @ s["u"][lo:hi]
    return r, s, low


def check(t, o, scale, drop):
    r, s, low = reference(t, scale, masks(t, drop))
    (K, R, In), Out, T = t["la"].shape, t["w"].shape[0], r["y"].shape[0]
    half = torch.finfo(t["x"].dtype).eps / 2
    terms = {"y": In + R, "dx": Out + R, "u": In, "v": Out, "dla": T + Out, "dlb": T + In}
    for name, got in o.items():
        want = r[name]
        got = got.cpu().double().reshape(want.shape)
        tol = (terms[name] ** 0.5 + 16) * U * (s[name] + low.get(name, 0.0)) + 1e-30
        if name in low:
            tol = tol + half * want.abs() + (half * 1.01 * low[name] if half > U else 0) + torch.finfo(t["x"].dtype).tiny * half
        bad = (got - want).abs() - tol
        assert bad.max() <= 0, f"{name}: off by {bad.max():.3e} beyond the tolerance"


def make_drop(p, K, device=DEV):
    return hip().Drop(p, torch.tensor([11 + 10 ** 9 * k for k in range(K)], dtype=torch.int64, device=device),
                      torch.tensor([3], dtype=torch.int64, device=device), 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,B,In,Out,R,p", [(1, 1, 1, 1, 1, 0.0), (3, 1, 64, 48, 4, 0.0), (2, 7, 33, 65, 5, 0.3), (5, 32, 784, 256, 8, 0.1),
                                            (1, 300, 129, 257, 16, 0.5), (20, 9, 100, 30, 33, 0.0), (2, 130, 512, 384, 64, 0.25),
                                            (3, 17, 2048, 10, 12, 0.1), (1, 16, 96, 512, 130, 0.2), (64, 1, 1024, 1024, 16, 0.0), (2, 1100, 40, 72, 6, 0.2),
                                            (4, 200, 1056, 520, 16, 0.0)])
def test_equal_blocks_of_rows(K, B, In, Out, R, p, dtype):
    t = make(K, K * B, In, Out, R, TYPES[dtype], uniform=True)
    drop = make_drop(p, K) if p else None
    check(t, run(t, 1.5, drop), 1.5, drop)


RAGGED = [  # T, cuts, In, Out, R, p
    (1, [0, 0, 1], 40, 24, 3, 0.0), (1, [0, 0, 0], 40, 24, 3, 0.0), (200, [0, 5, 5, 130, 131, 193], 96, 160, 8, 0.2),
    (333, [0, 0, 333, 333], 77, 51, 7, 0.5), (400, [0] + [i * 3 + 3 for i in range(129)], 128, 136, 16, 0.1),
    (64, list(range(0, 61)), 512, 256, 16, 0.0), (129, [3, 3, 128], 256, 128, 40, 0.1), (5, [0, 2, 4, 5], 4096, 64, 16, 0.0),
    (33, [0, 16, 33], 1000, 1000, 4, 0.3), (2900, [0, 600, 700, 700, 2850], 72, 56, 20, 0.1),
    (1200, [100, 1200], 264, 130, 40, 0.0), (700, [0] + sorted([3 * i % 701 for i in range(99)]) + [690], 64, 48, 8, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T,cuts,In,Out,R,p", RAGGED)
def test_ragged_and_empty_clients_and_rows_without_one(T, cuts, In, Out, R, p, dtype):
    K = len(cuts) - 1
    t = make(K, T, In, Out, R, TYPES[dtype], uniform=False, cuts=cuts, bias=False)
    drop = make_drop(p, K) if p else None
    o = run(t, 0.5, drop)
    check(t, o, 0.5, drop)
    owned = torch.zeros(T, dtype=torch.bool)
    for k, (lo, hi) in enumerate(clients(t)):
        owned[lo:hi] = True
        if hi == lo:
            assert (o["dla"][k] == 0).all() and (o["dlb"][k] == 0).all()
    assert (o["u"].cpu()[~owned] == 0).all() and (o["v"].cpu()[~owned] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_strided_rows_and_only_one_gradient(dtype):
    h, dt = hip(), TYPES[dtype]
    T, In, Out, R, K = 70, 48, 56, 6, 3
    t = make(K, T, In, Out, R, dt, uniform=False, cuts=[0, 20, 20, 66])
    want = run(t, 1.0, None)
    wide = torch.randn(T, In + 11, device=DEV).to(dt)
    wide[:, 5:5 + In] = t["x"]
    ww = torch.randn(Out, In + 3, device=DEV).to(dt)
    ww[:, 1:1 + In] = t["w"]
    yy = torch.full((T, Out + 9), 3.0, device=DEV, dtype=dt)
    u = torch.empty(T, R, device=DEV)
    h.adapter_linear_fwd(wide[:, 5:5 + In], ww[:, 1:1 + In], t["b"], t["la"], t["lb"], yy[:, 4:4 + Out], u, row_ptr=t["row_ptr"])
    check(t, {"y": yy[:, 4:4 + Out], "u": u}, 1.0, None)                 # (unaligned rows take another kernel's order of sums)
    assert (yy[:, :4] == 3).all() and (yy[:, 4 + Out:] == 3).all()
    dla, dlb = torch.empty_like(want["dla"]), torch.empty_like(want["dlb"])
    h.adapter_linear_wgrad(t["dy"], t["x"], want["u"], want["v"], dla, None, row_ptr=t["row_ptr"])
    h.adapter_linear_wgrad(t["dy"], t["x"], want["u"], want["v"], None, dlb, row_ptr=t["row_ptr"])
    assert torch.equal(dla, want["dla"]) and torch.equal(dlb, want["dlb"])


@pytest.mark.gpu
def test_equal_blocks_and_row_ptr_agree_and_repeat():
    K, B, In, Out, R = 6, 20, 160, 96, 8
    t = make(K, K * B, In, Out, R, torch.bfloat16, uniform=True)
    drop = make_drop(0.2, K)
    a, again = run(t, 1.0, drop), run(t, 1.0, drop)
    flat = dict(t, x=t["x"].reshape(K * B, In), dy=t["dy"].reshape(K * B, Out),
                row_ptr=torch.arange(0, K * B + 1, B, dtype=torch.int32, device=DEV))
    b = run(flat, 1.0, drop)
    for n in a:
        assert torch.equal(a[n], again[n])
        assert torch.equal(a[n].reshape(-1), b[n].reshape(-1))


@pytest.mark.gpu
def test_bad_values_of_one_client_stay_in_its_rows():
    K, B, In, Out, R = 4, 40, 64, 64, 8
    t = make(K, K * B, In, Out, R, torch.float32, uniform=True)
    good = run(t, 1.0, None)
    t["la"][2, 3, 5] = float("nan")
    t["lb"][1, 7, 2] = float("inf")
    o = run(t, 1.0, None)
    for n in ("y", "dx"):
        assert torch.equal(o[n][[0, 3]], good[n][[0, 3]])
    assert o["y"][2].isnan().all() and not o["y"][1, :, :7].isnan().any()


@pytest.mark.gpu
def test_captured_training_pass_follows_row_ptr_and_step():
    T, In, Out, R, K = 150, 96, 80, 8, 5
    t = make(K, T, In, Out, R, torch.bfloat16, uniform=False, cuts=[0, 10, 60, 60, 100, 149])
    drop = make_drop(0.3, K)
    h = hip()
    bufs = {"y": torch.empty(T, Out, device=DEV, dtype=torch.bfloat16), "u": torch.empty(T, R, device=DEV),
            "dx": torch.empty(T, In, device=DEV, dtype=torch.bfloat16), "v": torch.empty(T, R, device=DEV),
            "dla": torch.empty(K, R, In, device=DEV), "dlb": torch.empty(K, Out, R, device=DEV)}

    def step():
        kw = dict(row_ptr=t["row_ptr"], drop=drop)
        h.adapter_linear_fwd(t["x"], t["w"], t["b"], t["la"], t["lb"], bufs["y"], bufs["u"], **kw)
        h.adapter_linear_dgrad(t["dy"], t["w"], t["la"], t["lb"], bufs["dx"], bufs["v"], **kw)
        h.adapter_linear_wgrad(t["dy"], t["x"], bufs["u"], bufs["v"], bufs["dla"], bufs["dlb"], **kw)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for cuts in ([0, 10, 60, 60, 100, 149], [0, 0, 0, 150, 150, 150], [5, 6, 7, 8, 9, 10]):
        t["row_ptr"].copy_(torch.tensor(cuts, dtype=torch.int32))
        drop.step.add_(1)
        want = run(t, 1.0, drop)
        for v in bufs.values():
            v.zero_()
        g.replay()
        torch.cuda.synchronize()
        for n, v in want.items():
            assert torch.equal(bufs[n], v), n


@pytest.mark.gpu
def test_gradients_against_differences():
    K, B, In, Out, R, e = 2, 3, 12, 10, 3, 1e-2
    t = make(K, K * B, In, Out, R, torch.float32, uniform=True)
    drop = make_drop(0.25, K)
    o = run(t, 2.0, drop)

    def loss(**kw):
        return (run({**t, **kw}, 2.0, drop)["y"].double() * t["dy"].double()).sum().item()
    for name, grad in (("x", "dx"), ("la", "dla"), ("lb", "dlb")):
        for i in range(0, t[name].numel(), 5):
            hi, lo = t[name].clone().contiguous(), t[name].clone().contiguous()
            hi.view(-1)[i] += e
            lo.view(-1)[i] -= e
            d = (loss(**{name: hi}) - loss(**{name: lo})) / (2 * e)
            # y is bilinear: the difference is exact but for 60 values' fp32 roundings (2^-24 of ~10 each) over 2 e
            assert abs(d - o[grad].reshape(-1)[i].item()) < 4e-3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,B,In,Out,R", [(3, 1, 256, 192, 4), (2, 65, 129, 70, 5), (5, 40, 784, 256, 8), (2, 600, 512, 640, 16)])
@pytest.mark.parametrize("ragged", [False, True])
def test_own_workspaces_on_another_stream(K, B, In, Out, R, dtype, ragged):
    h, dt = hip(), TYPES[dtype]
    T = K * B
    cuts = [0] + [max(0, T - 1)] * (K - 1) + [T]
    t = make(K, T, In, Out, R, dt, uniform=not ragged, cuts=cuts)
    drop = make_drop(0.25, K)
    want = run(t, 0.5, drop)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        bufs = {w: h.adapter_linear_scratch(w, t["dy"] if w == "dgrad" else t["x"], K, In, Out, R, t["row_ptr"])
                for w in ("fwd", "dgrad", "wgrad")}
        got = {n: torch.full_like(v, 3.0) for n, v in want.items()}
        for _ in range(3):               # (the same buffers again: whatever a call left there does not matter)
            for buf in bufs.values():
                if buf is not None:
                    buf.fill_(float("nan"))
            kw = dict(row_ptr=t["row_ptr"], drop=drop)
            h.adapter_linear_fwd(t["x"], t["w"], t["b"], t["la"], t["lb"], got["y"], got["u"], scale=0.5, scratch=bufs["fwd"], **kw)
            h.adapter_linear_dgrad(t["dy"], t["w"], t["la"], t["lb"], got["dx"], got["v"], scale=0.5, scratch=bufs["dgrad"], **kw)
            h.adapter_linear_wgrad(t["dy"], t["x"], got["u"], got["v"], got["dla"], got["dlb"], scratch=bufs["wgrad"], **kw)
            for n in want:
                assert torch.equal(got[n], want[n]), n
    if bufs["dgrad"] is not None:
        for bad in (bufs["dgrad"][:0], bufs["dgrad"].double(), bufs["dgrad"].cpu()):
            with pytest.raises(h.HipKernelError, match="workspace"):
                h.adapter_linear_dgrad(t["dy"], t["w"], t["la"], t["lb"], got["dx"], got["v"], scratch=bad, row_ptr=t["row_ptr"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_without_rows_or_clients_and_rows_that_repeat(dtype):
    h, dt = hip(), TYPES[dtype]
    t = make(3, 0, 40, 24, 4, dt, uniform=True)
    o = run(t, 1.0, make_drop(0.5, 3))
    assert not o["dla"].any() and not o["dlb"].any() and o["y"].shape == (3, 0, 24)
    t = make(2, 0, 40, 24, 4, dt, uniform=False, cuts=[0, 0, 0])
    o = run(t, 1.0, None)
    assert not o["dla"].any() and not o["dlb"].any()
    for T in (3, 90):                    # no client at all: the shared projection alone
        t = make(0, T, 40, 24, 4, dt, uniform=False, cuts=[0])
        o = run(t, 1.0, None)
        check(t, {n: v for n, v in o.items() if v.numel()}, 1.0, None)
    for T in (5, 200):                   # one row for all (stride 0)
        t = make(2, T, 64, 48, 4, dt, uniform=False, cuts=[0, T // 2, T])
        t["x"], t["dy"] = t["x"][:1].expand(T, 64), t["dy"][:1].expand(T, 48)
        drop = make_drop(0.5, 2)
        check(t, run(t, 1.0, drop), 1.0, drop)


def test_refusals():
    h = hip()
    f = lambda *s: torch.zeros(*s)
    ok = dict(x=f(2, 3, 8), w=f(5, 8), b=f(5), la=f(2, 4, 8), lb=f(2, 5, 4), y=f(2, 3, 5), u=f(2, 3, 4))
    ptr = torch.zeros(3, dtype=torch.int32)
    drop3 = h.Drop(0.1, torch.zeros(3, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))

    def fwd(kw):
        a = {**ok, **kw}
        pos = [a.pop(n) for n in ("x", "w", "b", "la", "lb", "y", "u")]
        h.adapter_linear_fwd(*pos, **a)
    for kw in (dict(x=f(3, 3, 8)), dict(x=f(2, 3, 7)), dict(x=f(6, 8)), dict(row_ptr=ptr), dict(w=f(8, 5)), dict(w=f(8, 5).t()),
               dict(b=f(4)), dict(b=f(10)[::2]), dict(la=f(2, 8, 4).transpose(1, 2)), dict(lb=f(2, 4, 5)), dict(lb=f(3, 5, 4)),
               dict(y=f(2, 3, 6)), dict(y=f(1, 3, 5).expand(2, 3, 5)), dict(u=f(2, 3, 5)), dict(u=f(2, 3, 4).half()), dict(la=f(2, 4, 8).half()),
               dict(x=f(2, 3, 8).double()), dict(la=f(2, 0, 8), lb=f(2, 5, 0), u=f(2, 3, 0)), dict(drop=drop3),
               dict(la=f(1, 1, 1).expand(2, 1025, 8)), dict()):
        with pytest.raises(h.HipKernelError):
            fwd(kw)
    rag = dict(x=f(6, 8), y=f(6, 5), u=f(6, 4))
    for p in (ptr.long(), ptr[:2], torch.zeros(6, dtype=torch.int32)[::2], ptr):
        with pytest.raises(h.HipKernelError):
            fwd({**rag, "row_ptr": p})
    with pytest.raises(h.HipKernelError):
        h.adapter_linear_dgrad(f(2, 3, 5), f(5, 8), f(2, 4, 8), f(2, 5, 4), f(2, 3, 9), f(2, 3, 4))
    for dla, dlb in ((None, None), (f(2, 4, 9), None), (None, f(2, 5, 3)), (f(1, 4, 8).expand(2, 4, 8), None), (f(2, 4, 8), f(2, 5, 4))):
        with pytest.raises(h.HipKernelError):
            h.adapter_linear_wgrad(f(2, 3, 5), f(2, 3, 8), f(2, 3, 4), f(2, 3, 4), dla, dlb)


def test_results_in_place_are_refused():
    h = hip()
    f = lambda *s: torch.zeros(*s)
    x, w, la, lb, u = f(2, 3, 8), f(8, 8), f(2, 4, 8), f(2, 8, 4), f(2, 3, 4)
    for call in (lambda: h.adapter_linear_fwd(x, w, None, la, lb, x, u), lambda: h.adapter_linear_dgrad(x, w, la, lb, x, u)):
        with pytest.raises(h.HipKernelError, match="take the place"):
            call()
