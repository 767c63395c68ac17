"""Timed cases of the client-batched training and serving operators: group normalisation with an activation over
channels-last maps, counter-based dropout, and low-rank adapters of many clients beside one shared projection.

``run`` computes a case in its plain form (elementary torch operations in fp32) or, with ``own`` set, through
:mod:`p2pfl_amd.ops.hip`. Tensors lead with the client dimension K; affine parameters are views of a ``[K, P]`` slab.

The dropout mask is a function of (client seed, step, site, element index) alone: element ``e`` of a client takes word
``e % 4`` of the 7-round Philox4x32 block with counter ``(e // 4, site, step low, step high)`` and key ``(seed low, seed
high)`` (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) and is dropped where that word
is below ``round(p 2^32)``. A dropped element is zero whatever it held."""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
MASK32 = 0xFFFFFFFF


def listed():
    return [
        # one sample through the last residual stage of the CIFAR-10 ResNet9 (4 x 4 x 512): a call that is all latency
        {"name": "gn-one-sample", "op": "gn", "pass": "fwd", "K": 1, "N": 1, "S": 16, "C": 512, "G": 32, "act": "relu",
         "res": True, "p": 0.0, "dtype": "fp32"},
        # the backward pass of ten ResNet9 nodes, batch 32, after the first convolution (32 x 32 x 64)
        {"name": "gn-resnet9-backward", "op": "gn", "pass": "bwd", "K": 10, "N": 32, "S": 1024, "C": 64, "G": 32,
         "act": "relu", "res": True, "p": 0.0, "dtype": "fp32"},
        # fifty nodes in half precision with dropout behind the activation: the largest maps
        {"name": "gn-dropout-50-nodes", "op": "gn", "pass": "fwd", "K": 50, "N": 32, "S": 1024, "C": 64, "G": 16,
         "act": "silu", "res": False, "p": 0.1, "dtype": "bf16"},
        # odd maps (15 x 15), channel groups of five, forward and backward: nothing is a multiple of a vector
        {"name": "gn-odd-train", "op": "gn", "pass": "train", "K": 3, "N": 37, "S": 225, "C": 45, "G": 9,
         "act": "gelu", "res": True, "p": 0.0, "dtype": "fp16"},
        # the hidden layer of fifty SYSCALL MLPs, batch 32
        {"name": "dropout-syscall", "op": "dropout", "K": 50, "n": 32 * 256, "p": 0.5, "dtype": "fp32"},
        # the first maps of a hundred ResNet9 nodes (32 samples of 32 x 32 x 64): a pure stream
        {"name": "dropout-100-nodes", "op": "dropout", "K": 100, "n": 32 * 1024 * 64, "p": 0.1, "dtype": "bf16"},
        # one request's next token: the shared weights are read for one row
        {"name": "adapter-one-token", "op": "adapter", "pass": "fwd", "K": 8, "T": 1, "In": 4096, "Out": 4096, "R": 16,
         "uniform": False, "free": 0, "p": 0.0, "dtype": "bf16"},
        # next tokens of 64 requests over 48 adapters, some without one
        {"name": "adapter-64-tokens", "op": "adapter", "pass": "fwd", "K": 48, "T": 64, "In": 4096, "Out": 4096, "R": 16,
         "uniform": False, "free": 5, "p": 0.0, "dtype": "bf16"},
        # fifty nodes adapt the first layer of one MNIST MLP (784 -> 256), batch 32
        {"name": "adapter-mlp-train", "op": "adapter", "pass": "train", "K": 50, "T": 1600, "In": 784, "Out": 256, "R": 8,
         "uniform": True, "free": 0, "p": 0.1, "dtype": "fp32"},
        # a hundred nodes adapt the dense layer of one MNIST CNN (3136 -> 2048), batch 32
        {"name": "adapter-cnn-train", "op": "adapter", "pass": "train", "K": 100, "T": 3200, "In": 3136, "Out": 2048,
         "R": 16, "uniform": True, "free": 0, "p": 0.1, "dtype": "fp32"},
        # prompts of 24 requests, ragged lengths
        {"name": "adapter-prompts", "op": "adapter", "pass": "fwd", "K": 24, "T": 8192, "In": 4096, "Out": 4096, "R": 32,
         "uniform": False, "free": 100, "p": 0.0, "dtype": "bf16"},
        # odd sizes everywhere: unaligned rows, a rank of five, ragged and empty clients
        {"name": "adapter-odd-train", "op": "adapter", "pass": "train", "K": 13, "T": 1999, "In": 1001, "Out": 333, "R": 5,
         "uniform": False, "free": 7, "p": 0.25, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gn", "gn", "dropout", "adapter", "adapter"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "gn":
        while True:
            G = rng.choice([1, 2, 3, 4, 8, 16, 32])
            C = G * _log(rng, 1, 64)
            K, N, S = _log(rng, 1, 50), _log(rng, 1, 64), _log(rng, 1, 4096)
            if C <= 1024 and 4096 <= K * N * S * C <= 30_000_000 and S * (C // G) >= 4:
                break
        act = rng.choice(["none", "relu", "silu", "gelu"])
        # relu's gradient jumps at zero, so its backward pass is timed from a given result, not from one of its own
        pas = rng.choice(["fwd", "bwd"] if act == "relu" else ["fwd", "bwd", "train"])
        return {"op": "gn", "pass": pas, "K": K, "N": N, "S": S, "C": C, "G": G, "act": act,
                "res": rng.random() < 0.5, "p": rng.choice([0.0, 0.0, 0.1, 0.3]), "dtype": dtype}
    if op == "dropout":
        while True:
            K, n = _log(rng, 1, 200), _log(rng, 64, 4_000_000)
            if 4096 <= K * n <= 120_000_000:
                break
        return {"op": "dropout", "K": K, "n": n, "p": rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]), "dtype": dtype}
    while True:
        K, In, Out, R = _log(rng, 1, 100), _log(rng, 64, 4096), _log(rng, 8, 4096), rng.choice([1, 4, 5, 8, 16, 32, 64])
        if rng.random() < 0.7:
            In, Out = max(64, In // 32 * 32), max(16, Out // 16 * 16)
        uniform = rng.random() < 0.4
        T = K * _log(rng, 1, 64) if uniform else _log(rng, 1, 8192)
        if T * In * Out <= 20_000_000_000 and K * R <= 2048 and T * K * R <= 20_000_000:
            break
    pas = rng.choice(["fwd", "fwd", "train"])
    return {"op": "adapter", "pass": pas, "K": K, "T": T, "In": In, "Out": Out, "R": R, "uniform": uniform,
            "free": 0 if uniform else min(T // 2, rng.choice([0, 0, 3, 17])),
            "p": rng.choice([0.0, 0.1, 0.25]) if pas == "train" else 0.0, "dtype": dtype}


# ----------------------------------------------------------------------------- inputs
def _normal(shape, gen, dtype=torch.float32, scale=1.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return t.mul_(scale).to(dtype)


def _seeds(K, seed):
    rng = random.Random(seed ^ 0x5EED)
    seeds = torch.tensor([rng.getrandbits(63) for _ in range(K)], dtype=torch.int64, device="cuda")
    step = torch.tensor([rng.getrandbits(20)], dtype=torch.int64, device="cuda")
    return seeds, step, 1 + rng.getrandbits(8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = {"case": case, "act": case.get("act"), "p": case["p"]}
    st["seeds"], st["step"], st["site"] = _seeds(case["K"], seed)
    if case["op"] == "dropout":
        st["x"] = _normal((case["K"], case["n"]), gen, dt)
        st["y"] = torch.empty_like(st["x"])
        return st
    if case["op"] == "gn":
        K, N, S, C, G = (case[k] for k in "KNSCG")
        slab = _normal((K, 2 * C + 192), gen, scale=0.2)
        slab[:, 64:64 + C] += 1.0
        st["w"], st["b"] = slab[:, 64:64 + C], slab[:, 64 + C:64 + 2 * C]
        x = _normal((K, N, S, C), gen)
        x *= _normal((K, 1, 1, C), gen, scale=0.3) + 1.0
        x += _normal((K, 1, 1, C), gen, scale=0.5) + 0.25
        st["x"] = x.to(dt)
        st["res"] = _normal((K, N, S, C), gen, dt) if case["res"] else None
        st["y"] = torch.empty_like(st["x"])
        st["mean"] = torch.empty(K, N, G, device="cuda")
        st["rstd"] = torch.empty(K, N, G, device="cuda")
        if case["pass"] != "fwd":
            st["dy"] = _normal((K, N, S, C), gen, dt)
            st["dx"] = torch.empty_like(st["x"])
            st["dres"] = torch.empty_like(st["x"]) if case["res"] else None
            st["dw"], st["db"] = torch.empty(K, C, device="cuda"), torch.empty(K, C, device="cuda")
        if case["pass"] == "bwd":                 # what the forward pass left
            y, mean, rstd = _gn_fwd(st)
            st["y"].copy_(y)
            st["mean"].copy_(mean)
            st["rstd"].copy_(rstd)
        return st
    K, T, In, Out, R = (case[k] for k in ("K", "T", "In", "Out", "R"))
    st["scale"] = 2.0
    st["w"] = _normal((Out, In), gen, dt, In ** -0.5)
    st["b"] = _normal((Out,), gen, dt, 0.1)
    st["la"] = _normal((K, R, In), gen, dt, In ** -0.5)
    st["lb"] = _normal((K, Out, R), gen, dt, 0.5 * R ** -0.5)
    lead = (K, T // K) if case["uniform"] else (T,)
    st["x"] = _normal((*lead, In), gen, dt)
    st["row_ptr"] = None
    if not case["uniform"]:                       # rows of a client are consecutive; the last `free` rows have no adapter
        rng = random.Random(seed ^ 0xC0DE)
        cuts = sorted(rng.randint(0, T - case["free"]) for _ in range(K - 1))
        st["row_ptr"] = torch.tensor([0, *cuts, T - case["free"]], dtype=torch.int32, device="cuda")
    st["y"] = torch.empty(*lead, Out, device="cuda", dtype=dt)
    st["u"] = torch.empty(*lead, R, device="cuda")
    if case["pass"] == "train":
        st["dy"] = _normal((*lead, Out), gen, dt)
        st["dx"] = torch.empty_like(st["x"])
        st["v"] = torch.empty_like(st["u"])
        st["dla"] = torch.empty(K, R, In, device="cuda")
        st["dlb"] = torch.empty(K, Out, R, device="cuda")
    return st


# ----------------------------------------------------------------------------- plain forms
def _mulhilo(a, m):
    """(high, low) 32-bit halves of a * m for int64 tensors holding 32-bit values (the product wraps, its bits do not)."""
    q = a * m
    return (q >> 32) & MASK32, q & MASK32


def _philox(c0, c1, c2, c3, k0, k1):
    """Seven rounds of Philox4x32 on int64 tensors holding 32-bit values."""
    for r in range(7):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return torch.stack([c0, c1, c2, c3], dim=-1)


def _kept(st, n):
    """[K, n] truth values: which of the first n elements of each client stay."""
    q = torch.arange((n + 3) // 4, device="cuda").unsqueeze(0)
    k0, k1 = (st["seeds"] & MASK32).unsqueeze(1), ((st["seeds"] >> 32) & MASK32).unsqueeze(1)
    site = torch.full_like(q, st["site"])
    words = _philox(q, site, (st["step"] & MASK32).expand_as(q), ((st["step"] >> 32) & MASK32).expand_as(q), k0, k1)
    return words.flatten(1)[:, :n] >= round(st["p"] * 2 ** 32)


def _drop(st, x, kept):
    return torch.where(kept, x * (1.0 / (1.0 - st["p"])), torch.zeros((), device="cuda"))


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    return z


def _dact(z, act, y):
    if act == "relu":                             # by the output, as the call has it
        return (y > 0).float()
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    return torch.ones_like(z)


def _gn_z(st, mean, rstd):
    """(normalised map, value before the activation), both [K, N, S, C] in fp32."""
    K, N, S, C = st["x"].shape
    x = st["x"].float().view(K, N, S, -1, C // mean.shape[2])
    xh = ((x - mean[:, :, None, :, None]) * rstd[:, :, None, :, None]).view(K, N, S, C)
    z = xh * st["w"][:, None, None, :] + st["b"][:, None, None, :]
    return xh, z if st["res"] is None else z + st["res"].float()


def _gn_fwd(st):
    K, N, S, C = st["x"].shape
    x = st["x"].float().view(K, N, S, st["mean"].shape[2], -1)
    mean = x.mean(dim=(2, 4))
    var = (x - mean[:, :, None, :, None]).square().mean(dim=(2, 4))
    rstd = 1.0 / torch.sqrt(var + EPS)
    y = _act(_gn_z(st, mean, rstd)[1], st["act"])
    if st["p"] > 0:
        y = _drop(st, y, _kept(st, N * S * C).view_as(y))
    return y.to(st["x"].dtype), mean, rstd


def _gn_bwd(st, y, mean, rstd):
    K, N, S, C = st["x"].shape
    G = mean.shape[2]
    xh, z = _gn_z(st, mean, rstd)
    dz = st["dy"].float()
    if st["p"] > 0:
        dz = _drop(st, dz, _kept(st, N * S * C).view_as(dz))
    dz = dz * _dact(z, st["act"], y)
    dw, db = (dz * xh).sum(dim=(1, 2)), dz.sum(dim=(1, 2))
    t = (dz * st["w"][:, None, None, :]).view(K, N, S, G, -1)
    xg = xh.view(K, N, S, G, -1)
    m1, m2 = t.mean(dim=(2, 4), keepdim=True), (t * xg).mean(dim=(2, 4), keepdim=True)
    dx = ((t - m1 - xg * m2) * rstd[:, :, None, :, None]).view(K, N, S, C).to(st["x"].dtype)
    return dx, dw, db, None if st["res"] is None else dz.to(st["x"].dtype)


def _clients(st):
    """[T, K] truth values: which client a row belongs to; [T]: its row within that client."""
    T = st["case"]["T"]
    t = torch.arange(T, device="cuda")
    ptr = st["row_ptr"] if st["row_ptr"] is not None else torch.arange(st["case"]["K"] + 1, device="cuda") * st["x"].shape[1]
    lo, hi = ptr[:-1].long(), ptr[1:].long()
    of = (t[:, None] >= lo) & (t[:, None] < hi)
    return of, t - (of * lo).sum(1)


def _adapter_kept(st, of, local):
    """[T, In] truth values; element (row of the client, column) has index row * In + column. Every row's own counters."""
    T, In = st["case"]["T"], st["case"]["In"]
    e = (local[:, None] * In + torch.arange(In, device="cuda"))
    seed = (of * st["seeds"]).sum(1, keepdim=True)
    q = torch.div(e, 4, rounding_mode="floor")
    words = _philox(q, torch.full_like(q, st["site"]), (st["step"] & MASK32).expand_as(q),
                    ((st["step"] >> 32) & MASK32).expand_as(q), seed & MASK32, (seed >> 32) & MASK32)
    return torch.gather(words, 2, (e % 4).unsqueeze(2)).squeeze(2) >= round(st["p"] * 2 ** 32)


def _adapter_plain(st):
    case = st["case"]
    K, T, In, Out, R = (case[k] for k in ("K", "T", "In", "Out", "R"))
    x, w = st["x"].float().view(T, In), st["w"].float()
    la, lb = st["la"].float(), st["lb"].float()
    of, local = _clients(st)
    xd = x
    if st["p"] > 0:
        kept = _adapter_kept(st, of, local)
        xd = _drop(st, x, kept)
    if case["uniform"]:
        per = lambda t: t.view(K, T // K, t.shape[-1])
        u = torch.bmm(per(xd), la.transpose(1, 2)).view(T, R) * st["scale"]
        low = torch.bmm(per(u), lb.transpose(1, 2)).view(T, Out)
    else:
        wide = (xd @ la.view(K * R, In).t()).view(T, K, R) * of[:, :, None] * st["scale"]
        u = wide.sum(1)
        low = wide.view(T, K * R) @ lb.transpose(1, 2).reshape(K * R, Out)
    y = x @ w.t() + st["b"].float() + low
    lead = st["x"].shape[:-1]
    out = {"y": y.view(*lead, Out).to(st["x"].dtype), "u": u.view(*lead, R)}
    if case["pass"] == "fwd":
        return out
    dy = st["dy"].float().view(T, Out)
    if case["uniform"]:
        v = torch.bmm(per(dy), lb).view(T, R) * st["scale"]
        low = torch.bmm(per(v), la).view(T, In)
        dla = torch.bmm(per(v).transpose(1, 2), per(xd))
        dlb = torch.bmm(per(dy).transpose(1, 2), per(u))
    else:
        wv = (dy @ lb.transpose(1, 2).reshape(K * R, Out).t()).view(T, K, R) * of[:, :, None] * st["scale"]
        v = wv.sum(1)
        low = wv.view(T, K * R) @ la.view(K * R, In)
        dla = (wv.view(T, K * R).t() @ xd).view(K, R, In)
        dlb = (wide.view(T, K * R).t() @ dy).view(K, R, Out).transpose(1, 2).contiguous()
    if st["p"] > 0:
        low = _drop(st, low, kept)
    dx = dy @ w + low
    return out | {"dx": dx.view(*lead, In).to(st["x"].dtype), "dla": dla, "dlb": dlb}


# ----------------------------------------------------------------------------- one pass
def _run_own(st):
    from p2pfl_amd.ops import hip
    case = st["case"]
    drop = hip.Drop(st["p"], st["seeds"], st["step"], st["site"]) if st["p"] > 0 else None
    if case["op"] == "dropout":
        hip.dropout(st["x"], st["y"], drop)
        return {"y": st["y"]}
    if case["op"] == "gn":
        G, act = case["G"], case["act"]
        out = {}
        if case["pass"] != "bwd":
            hip.group_norm_fwd(st["x"], st["w"], st["b"], st["y"], G, mean=st["mean"], rstd=st["rstd"], eps=EPS, act=act,
                               residual=st["res"], drop=drop)
            out |= {"y": st["y"], "mean": st["mean"], "rstd": st["rstd"]}
        if case["pass"] != "fwd":
            hip.group_norm_bwd(st["dy"], st["x"], st["w"], st["b"], st["mean"], st["rstd"], st["dx"], st["dw"], st["db"], G,
                               act=act, y=st["y"] if act == "relu" else None, residual=st["res"], dres=st["dres"], drop=drop)
            out |= {"dx": st["dx"], "dw": st["dw"], "db": st["db"], "dres": st["dres"]}
        return out
    kw = {"scale": st["scale"], "row_ptr": st["row_ptr"]}
    hip.adapter_linear_fwd(st["x"], st["w"], st["b"], st["la"], st["lb"], st["y"], st["u"], drop=drop, **kw)
    out = {"y": st["y"], "u": st["u"]}
    if case["pass"] == "train":
        hip.adapter_linear_dgrad(st["dy"], st["w"], st["la"], st["lb"], st["dx"], st["v"], drop=drop, **kw)
        hip.adapter_linear_wgrad(st["dy"], st["x"], st["u"], st["v"], st["dla"], st["dlb"], row_ptr=st["row_ptr"], drop=drop)
        out |= {"dx": st["dx"], "dla": st["dla"], "dlb": st["dlb"]}
    return out


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    if case["op"] == "dropout":
        return {"y": _drop(st, st["x"].float(), _kept(st, case["n"])).to(st["x"].dtype)}
    if case["op"] == "adapter":
        return _adapter_plain(st)
    out, y, mean, rstd = {}, st["y"], st["mean"], st["rstd"]
    if case["pass"] != "bwd":
        y, mean, rstd = _gn_fwd(st)
        out |= {"y": y, "mean": mean, "rstd": rstd}
    if case["pass"] != "fwd":
        out |= dict(zip(("dx", "dw", "db", "dres"), _gn_bwd(st, y, mean, rstd)))
    return out


def work(case):
    z = SIZE[case["dtype"]]
    if case["op"] == "dropout":
        n = case["K"] * case["n"]
        return {"bytes": 2 * n * z, "flops": n}
    if case["op"] == "gn":
        n = case["K"] * case["N"] * case["S"] * case["C"]
        r = int(case["res"])
        # forward: map (+ residual) in, result out; backward: gradient and map in, gradient out (+ the residual and its
        # gradient; relu goes by the result)
        fwd = n * z * (2 + r)
        bwd = n * z * (3 + (r + 1 if case["act"] == "relu" else 2 * r) if case["act"] != "none" else 3 + r)
        flops = {"fwd": 10 * n, "bwd": 20 * n, "train": 30 * n}[case["pass"]]
        small = 8 * case["K"] * case["C"]
        # of a training pass: map, residual and incoming gradient in, result and gradients out
        train = n * z * (4 + 2 * r)
        return {"bytes": {"fwd": fwd, "bwd": bwd, "train": train}[case["pass"]] + small, "flops": flops}
    K, T, In, Out, R = (case[k] for k in ("K", "T", "In", "Out", "R"))
    used = min(K, T)
    low = used * R * (In + Out)
    nbytes = z * (T * (In + Out) + In * Out + Out + low) + 4 * T * R
    flops = 2 * T * (In * Out + R * (In + Out))
    if case["pass"] == "train":
        nbytes += z * T * (In + Out) + 4 * K * R * (In + Out)
        flops += 2 * T * (In * Out + 2 * R * (In + Out))
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------------------- the definition in 64 bits
def _word_stream(key, step, site, first, count):
    """Words of the counter blocks [first, first + count) of one client, as the definition has them, [count, 4]."""
    lo32 = 2 ** 32 - 1
    ctr = torch.arange(first, first + count, device="cuda", dtype=torch.int64)
    x = [ctr & lo32, torch.full_like(ctr, site), torch.full_like(ctr, step & lo32), torch.full_like(ctr, step >> 32)]
    key = [key & lo32, key >> 32]

    def product(a, m):                            # 32 x 32 -> (low, high) through 16-bit halves: nothing wraps
        al, ah, ml, mh = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
        mid = ah * ml + ((al * ml) >> 16)
        mid2 = al * mh + (mid & 0xFFFF)
        return ((mid2 & 0xFFFF) << 16) | ((al * ml) & 0xFFFF), ah * mh + (mid >> 16) + (mid2 >> 16)

    for _ in range(7):
        lo_a, hi_a = product(x[0], 0xD2511F53)
        lo_b, hi_b = product(x[2], 0xCD9E8D57)
        x = [hi_b ^ x[1] ^ key[0], lo_b, hi_a ^ x[3] ^ key[1], lo_a]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return torch.stack(x, 1)


def _weight_of(st, k, n):
    """fp64 factors 0 or 1 / (1 - p) of the first n elements of client k."""
    words = _word_stream(int(st["seeds"][k]), int(st["step"]), st["site"], 0, -(-n // 4)).reshape(-1)[:n]
    return (words >= round(st["p"] * 2 ** 32)).double() / (1.0 - st["p"])


def _exact_act(z, act):
    f = torch.nn.functional
    return {"none": lambda t: t, "relu": f.relu, "silu": f.silu, "gelu": f.gelu}[act](z)


def _exact_gn(st, case):
    K, N, S, C, G = (case[k] for k in "KNSCG")
    parts = []
    for k in range(K):                            # one client after another: fp64 maps of all would not fit beside the rest
        x = st["x"][k].double().requires_grad_(case["pass"] != "fwd")
        w, b = st["w"][k].double().requires_grad_(), st["b"][k].double().requires_grad_()
        res = None if st["res"] is None else st["res"][k].double().requires_grad_(case["pass"] != "fwd")
        with torch.set_grad_enabled(case["pass"] != "fwd"):
            g = x.reshape(N, S, G, C // G).movedim(2, 1).reshape(N, G, -1)
            var, mean = torch.var_mean(g, dim=2, correction=0, keepdim=True)
            rstd = (var + EPS).rsqrt()
            hat = ((g - mean) * rstd).reshape(N, G, S, C // G).movedim(1, 2).reshape(N, S, C)
            z = torch.addcmul(b, hat, w)
            z = z if res is None else z + res
            m = _weight_of(st, k, N * S * C).view(N, S, C) if case["p"] > 0 else 1.0
            if case["pass"] == "bwd" and case["act"] == "relu":     # by the given output
                y = torch.where(st["y"][k] > 0, z, torch.zeros_like(z)) * m
            else:
                y = _exact_act(z, case["act"]) * m
        got = {}
        if case["pass"] != "bwd":
            got |= {"y": y.detach(), "mean": mean.detach().view(N, G), "rstd": rstd.detach().view(N, G)}
        if case["pass"] != "fwd":
            want = [x, w, b] + ([] if res is None else [res])
            grads = torch.autograd.grad(y, want, st["dy"][k].double())
            got |= dict(zip(("dx", "dw", "db", "dres"), list(grads) + [None] * (4 - len(want))))
        parts.append(got)
    return {n: None if v is None else torch.stack([q[n] for q in parts]) for n, v in parts[0].items()}


def _exact_adapter(st, case):
    K, T, In, Out, R = (case[k] for k in ("K", "T", "In", "Out", "R"))
    s = st["scale"]
    x, w = st["x"].double().reshape(T, In), st["w"].double()
    ptr = st["row_ptr"].tolist() if st["row_ptr"] is not None else [k * (T // K) for k in range(K + 1)]
    train = case["pass"] == "train"
    y = torch.addmm(st["b"].double(), x, w.t())
    u = torch.zeros(T, R, device="cuda", dtype=torch.float64)
    if train:
        dy = st["dy"].double().reshape(T, Out)
        dx = dy @ w
        dla, dlb = torch.zeros(K, R, In, device="cuda").double(), torch.zeros(K, Out, R, device="cuda").double()
    for k, (lo, hi) in enumerate(zip(ptr, ptr[1:])):
        if hi <= lo:
            continue
        a, b = st["la"][k].double(), st["lb"][k].double()
        m = _weight_of(st, k, (hi - lo) * In).view(-1, In) if case["p"] > 0 else None
        xd = x[lo:hi] if m is None else x[lo:hi] * m
        u[lo:hi] = xd @ a.t() * s
        y[lo:hi] += u[lo:hi] @ b.t()
        if train:
            v = dy[lo:hi] @ b * s
            dx[lo:hi] += v @ a if m is None else (v @ a) * m
            dla[k], dlb[k] = v.t() @ xd, dy[lo:hi].t() @ u[lo:hi]
    lead = st["x"].shape[:-1]
    out = {"y": y.view(*lead, Out), "u": u.view(*lead, R)}
    return out | {"dx": dx.view(*lead, In), "dla": dla, "dlb": dlb} if train else out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "dropout":
        n = case["n"]
        return {"y": torch.stack([st["x"][k].double() * _weight_of(st, k, n) for k in range(case["K"])])}
    if case["op"] == "adapter":
        return _exact_adapter(st, case)
    return _exact_gn(st, case)
