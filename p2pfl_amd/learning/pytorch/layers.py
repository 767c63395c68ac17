"""Layers for models of a federation, on the client-batched kernels of :mod:`p2pfl_amd.ops.hip`.

* :class:`GroupNormAct` - group normalisation with residual, activation and dropout. It keeps nothing between steps: unlike
  BatchNorm's running statistics, which do not average well over nodes with different data, there is only the affine pair to
  federate.
* :class:`CounterDropout` - dropout whose mask is a function of (node seed, step, element): nothing is stored for the backward
  pass, and a hipGraph replay draws new masks.
* :class:`AdapterLinear` - a frozen projection shared by all co-resident nodes with a low-rank adapter per node; only the
  adapter is trained, exchanged and averaged. :func:`adapt` puts adapters on every linear layer of a model.

Under ``torch.func.vmap`` - how :class:`~p2pfl_amd.runtime.module_engine.ModuleEngine` steps all co-resident nodes at once - one
kernel call covers the nodes. On the CPU the layers compute the same functions with stock operations, the dropout masks
included. A client's mask goes by its own seed where seeds are vmapped (the engine's are: by the node, :func:`place_dropouts`),
by the layer's seed and the client's place otherwise. On the GPU vmapped clients share one step: leave it out of a vmapped state;
and gradients are autograd's (``backward()``, ``torch.autograd.grad``) of a function, vmapped or not: ``torch.func.grad`` and its
like are refused there.
"""
from __future__ import annotations

import hashlib
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ...ops import hip

_ACT = {"none": lambda z: z, None: lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}
_GOLDEN = 0x9E3779B97F4A7C15 - 2 ** 64          # seeds of the nodes of a shard: seed + node * this, modulo 2^64


# ----------------------------------------------------------------------------- the generator on any device
def _mulhilo(a, m: int):
    q = a * m                                    # (wraps modulo 2^64: its bits are the product's)
    return (q >> 32) & 0xFFFFFFFF, q & 0xFFFFFFFF


def keep_mask(seeds: torch.Tensor, step: torch.Tensor, site: int, n: int, p: float) -> torch.Tensor:
    """[K, n] truth values: which elements of each client :func:`p2pfl_amd.ops.hip.dropout` keeps, in stock operations. ``step`` [1],
    or one for each of the K."""
    k0, k1 = (seeds & 0xFFFFFFFF).unsqueeze(1), ((seeds >> 32) & 0xFFFFFFFF).unsqueeze(1)
    c0 = torch.arange((n + 3) // 4, device=seeds.device).expand(seeds.numel(), -1)
    c1, c2, c3 = torch.full_like(c0, site), (step & 0xFFFFFFFF).unsqueeze(1).expand_as(c0), (step >> 32 & 0xFFFFFFFF).unsqueeze(1).expand_as(c0)
    for _ in range(7):
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([c0, c1, c2, c3], dim=-1).flatten(1)[:, :n] >= (2 ** 32 if p >= 1.0 else min(round(p * 2 ** 32), 2 ** 32 - 1))


def _drop(p: float, seed, step, site: int, K: int):
    """The call's :class:`hip.Drop` for K clients that share a base seed, or None."""
    if p == 0.0:
        return None
    return hip.Drop(p, _seeds(seed, K), step, site)


def _seeds(seed, K: int):
    """[K] seeds: given, or by the place behind one seed."""
    return seed if seed.numel() == K else seed + torch.arange(K, device=seed.device) * _GOLDEN


def _clients(B: int, t, dim: Optional[int]):
    """The physical tensor of a vmapped [1, ...] argument as [B, ...] clients."""
    if t is None:
        return None
    t = t.movedim(dim, 0) if dim is not None else t.unsqueeze(0).expand(B, *t.shape)
    return t.flatten(0, 1)


def _untransformed(*tensors) -> None:
    if any(t is not None and torch._C._functorch.is_functorch_wrapped_tensor(t) for t in tensors):
        raise NotImplementedError("gradients of these layers on the GPU are autograd's: backward() or torch.autograd.grad of a function, "
                                  "vmapped or not, instead of torch.func.grad")


def _vmapped(B: int, seed, step, dims, steps: bool = False):
    """Seed and step of a vmapped dropout as the physical clients have them."""
    if dims[0] is not None or seed.numel() > 1:
        seed = _clients(B, seed, dims[0])
    if dims[1] is not None:
        if not steps:
            raise hip.HipKernelError("dropout: vmapped clients share one step: leave it out of the vmapped state")
        step = _clients(B, step, dims[1])
    return seed, step


class _Mask(torch.autograd.Function):
    """:func:`keep_mask` of x [K, ...]."""

    @staticmethod
    def forward(x, seed, step, p, site):
        return keep_mask(_seeds(seed, x.shape[0]), step, site, x[0].numel(), p).view(x.shape)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.mark_non_differentiable(output)

    @staticmethod
    def backward(ctx, _):
        return None, None, None, None, None

    @staticmethod
    def vmap(info, in_dims, x, seed, step, *rest):
        B = info.batch_size
        keep = _Mask.apply(_clients(B, x, in_dims[0]), *_vmapped(B, seed, step, in_dims[1:3], True), *rest)
        return keep.unflatten(0, (B, -1)), 0


class _GroupNorm(torch.autograd.Function):
    """x and residual [K, N, ..., C]; w, b [K, C]."""

    @staticmethod
    def forward(x, w, b, residual, seed, step, groups, eps, act, p, site):
        K, N = x.shape[:2]
        x = _channels_last(x)
        residual = None if residual is None else _channels_last(residual)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean, rstd = (torch.empty(K, N, groups, device=x.device) for _ in range(2))
        hip.group_norm_fwd(x, _rows(w), _rows(b), y, groups, mean=mean, rstd=rstd, eps=eps, act=act, residual=residual,
                           drop=_drop(p, seed, step, site, K))
        return y, mean, rstd

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, w, b, residual, seed, step, ctx.groups, _, ctx.act, ctx.p, ctx.site = inputs
        y, mean, rstd = output
        ctx.mark_non_differentiable(mean, rstd)
        by_y = ctx.act == "relu"                  # (its gradient goes by the result)
        ctx.has_res = residual is not None
        ctx.save_for_backward(x, w, b, y if by_y else None, None if by_y else residual, mean, rstd, seed, step)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _mean, _rstd):
        x, w, b, y, residual, mean, rstd, seed, step = ctx.saved_tensors
        _untransformed(dy, x, w, b, residual)
        K = x.shape[0]
        x, dy = _channels_last(x), _channels_last(dy)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dres = torch.empty_like(dx) if ctx.has_res else None
        dw, db = torch.empty(w.shape, device=x.device), torch.empty(b.shape, device=x.device)
        hip.group_norm_bwd(dy, x, _rows(w), _rows(b), mean, rstd, dx, dw, db, ctx.groups, act=ctx.act, y=y,
                           residual=None if residual is None else _channels_last(residual), dres=dres,
                           drop=_drop(ctx.p, seed, step, ctx.site, K))
        return dx, dw, db, dres, None, None, None, None, None, None, None

    @staticmethod
    def vmap(info, in_dims, x, w, b, residual, seed, step, *rest):
        B = info.batch_size
        out = _GroupNorm.apply(*(_clients(B, t, d) for t, d in zip((x, w, b, residual), in_dims)),
                               *_vmapped(B, seed, step, in_dims[4:6]), *rest)
        return tuple(t.unflatten(0, (B, -1)) for t in out), (0, 0, 0)


class _Dropout(torch.autograd.Function):
    """x [K, ...]."""

    @staticmethod
    def forward(x, seed, step, p, site):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        hip.dropout(x.contiguous(), y, _drop(p, seed, step, site, x.shape[0]))
        return y

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, seed, step, ctx.p, ctx.site = inputs
        ctx.save_for_backward(seed, step)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        seed, step = ctx.saved_tensors
        _untransformed(dy, seed, step)
        return _Dropout.forward(dy, seed, step, ctx.p, ctx.site), None, None, None, None

    @staticmethod
    def vmap(info, in_dims, x, seed, step, *rest):
        B = info.batch_size
        y = _Dropout.apply(_clients(B, x, in_dims[0]), *_vmapped(B, seed, step, in_dims[1:3]), *rest)
        return y.unflatten(0, (B, -1)), 0


class _Adapter(torch.autograd.Function):
    """x [K, B, In]; w [Out, In] and b [Out] shared and frozen; la [K, R, In], lb [K, Out, R]."""

    @staticmethod
    def forward(x, w, b, la, lb, seed, step, scale, p, site):
        K, B, _ = x.shape
        y = torch.empty(K, B, w.shape[0], dtype=x.dtype, device=x.device)
        u = torch.empty(K, B, la.shape[1], device=x.device)
        hip.adapter_linear_fwd(x.contiguous(), w, b, _rows(la), _rows(lb), y, u, scale=scale, drop=_drop(p, seed, step, site, K))
        return y, u

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, w, _, la, lb, seed, step, ctx.scale, ctx.p, ctx.site = inputs
        ctx.mark_non_differentiable(output[1])
        ctx.save_for_backward(x, w, la, lb, output[1], seed, step)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _u):
        x, w, la, lb, u, seed, step = ctx.saved_tensors
        _untransformed(dy, x, la, lb)
        drop = _drop(ctx.p, seed, step, ctx.site, x.shape[0])
        x, dy = x.contiguous(), dy.contiguous()
        dx, v = torch.empty_like(x), torch.empty_like(u)
        dla, dlb = torch.empty(la.shape, device=x.device), torch.empty(lb.shape, device=x.device)
        hip.adapter_linear_dgrad(dy, w, _rows(la), _rows(lb), dx, v, scale=ctx.scale, drop=drop)
        hip.adapter_linear_wgrad(dy, x, u, v, dla, dlb, drop=drop)
        return dx, None, None, dla.to(la.dtype), dlb.to(lb.dtype), None, None, None, None, None

    @staticmethod
    def vmap(info, in_dims, x, w, b, la, lb, seed, step, *rest):
        if in_dims[1] is not None or in_dims[2] is not None:
            raise NotImplementedError("AdapterLinear: the projection is shared by the vmapped clients")
        B = info.batch_size
        x, la, lb = (_clients(B, t, d) for t, d in ((x, in_dims[0]), (la, in_dims[3]), (lb, in_dims[4])))
        out = _Adapter.apply(x, w, b, la, lb, *_vmapped(B, seed, step, in_dims[5:7]), *rest)
        return tuple(t.unflatten(0, (B, -1)) for t in out), (0, 0)


def _rows(t):
    """A [K, ...] parameter with packed rows (a slab view already is)."""
    return t if t.is_contiguous() or t[0].is_contiguous() else t.contiguous()


def _channels_last(t):
    """A map [K, N, ..., C] with dense channels and evenly spaced positions."""
    if t.is_contiguous():
        return t
    span = None
    for size, stride in zip(reversed(t.shape[2:-1]), reversed(t.stride()[2:-1])):
        if size > 1 and span is not None and stride != span:
            return t.contiguous()
        span = stride * size if size > 1 else span
    return t if t.stride(-1) == 1 else t.contiguous()


class _Counted(nn.Module):
    """Seed and step of a dropout. They live beside the model, not in it: no payload or checkpoint entry. ``seed`` None: from
    torch's generator. Every training pass moves the step on: activation checkpointing, which runs a pass twice, would see two
    masks (the backward pass here stores none, so there is nothing to save by it). A copy of a layer draws the masks of the original
    (:func:`place_dropouts` gives the models of nodes their own), and a resumed run those of the first steps again."""

    _sites = 0

    def __init__(self, p: float, seed: Optional[int] = None, device=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability {p} outside [0, 1]")
        self.p = float(p)
        self.site = _Counted._sites = (_Counted._sites + 1) % 2 ** 32
        if seed is None:
            seed = int(torch.randint(2 ** 62, (1,)))
        self.register_buffer("seed", torch.tensor([seed], dtype=torch.int64, device=device), persistent=False)
        self.register_buffer("step", torch.zeros(1, dtype=torch.int64, device=device), persistent=False)

    def _draw(self):
        """(probability, step) of this pass; the counter moves on for the next. A pass without dropout has no step: it would hold on
        to a counter that a later pass changes."""
        if not self.training or self.p == 0.0:
            return 0.0, None
        with torch.no_grad():
            used = self.step.clone()              # (the backward pass draws the same mask again)
            self.step.add_(1)
        return self.p, used

    def _stock(self, x, p: float, step):
        if p == 0.0:
            return x
        keep = _Mask.apply(x.detach().unsqueeze(0), self.seed, step, p, self.site).squeeze(0)
        return torch.where(keep, x * (1.0 / (1.0 - p) if p < 1.0 else 0.0), torch.zeros((), dtype=x.dtype, device=x.device))


def place_dropouts(models, first: int = 0):
    """Gives the dropouts of the models of nodes ``first``, ``first + 1``, ... seeds that go by the node and sites that go by the place in
    the model: a node's masks are the same whichever nodes share its card. Seeds start from the first model's, which has to be
    the same on all cards. Returns, for each dropout of the model, its name and the [K, 1] seeds and steps whose rows the models'
    layers hold from now on."""
    table = []
    for site, layers in enumerate(zip(*([(n, m) for n, m in model.named_modules() if isinstance(m, _Counted)] for model in models))):
        name, m0 = layers[0]
        seeds = m0.seed + torch.arange(first, first + len(models), device=m0.seed.device) * _GOLDEN
        seeds, steps = seeds.unsqueeze(1), torch.zeros(len(models), 1, dtype=torch.int64, device=seeds.device)
        for k, (_, m) in enumerate(layers):
            m.site, m.seed, m.step = site, seeds[k], steps[k]
        table.append((name, seeds, steps))
    return table


class CounterDropout(_Counted):
    """Dropout (p) of any tensor while training."""

    def __init__(self, p: float = 0.5, seed: Optional[int] = None):
        super().__init__(p, seed)

    def forward(self, x):
        p, step = self._draw()
        if p == 0.0:
            return x
        if not x.is_cuda:
            return self._stock(x, p, step)
        return _Dropout.apply(x.unsqueeze(0), self.seed, step, p, self.site).squeeze(0)

    def extra_repr(self):
        return f"p={self.p}"


class GroupNormAct(_Counted):
    """``drop(act(group_norm(x) + residual))`` of maps [N, C, ...]; channels-last memory is taken and returned as it is."""

    def __init__(self, groups: int, channels: int, act: Optional[str] = None, eps: float = 1e-5, p: float = 0.0,
                 seed: Optional[int] = None):
        super().__init__(p, 0 if p == 0.0 and seed is None else seed)
        if channels % groups:
            raise ValueError(f"{channels} channels do not divide into {groups} groups")
        if act not in hip.ACTIVATIONS:
            raise ValueError(f"unknown activation {act!r}")
        self.groups, self.eps, self.act = groups, eps, act
        self.weight, self.bias = nn.Parameter(torch.ones(channels)), nn.Parameter(torch.zeros(channels))

    def forward(self, x, residual=None):
        p, step = self._draw()
        if not x.is_cuda:
            y = F.group_norm(x, self.groups, self.weight, self.bias, self.eps)
            y = _ACT[self.act](y if residual is None else y + residual)
            return y if p == 0.0 else self._stock(y.movedim(1, -1), p, step).movedim(-1, 1)
        last = lambda t: None if t is None else t.movedim(1, -1).unsqueeze(0)
        y = _GroupNorm.apply(last(x), self.weight.float().unsqueeze(0), self.bias.float().unsqueeze(0),
                             last(residual if residual is None else residual.to(x.dtype)), self.seed, step, self.groups, self.eps,
                             self.act, p, self.site)[0]
        return y.squeeze(0).movedim(-1, 1)

    def extra_repr(self):
        return f"{self.groups}, {self.weight.shape[0]}, act={self.act}, p={self.p}"


class AdapterLinear(_Counted):
    """``x W^T + b + (alpha / rank) drop(x) A^T B^T`` with W, b frozen. W and b are shared, not copied and no part of the state: the
    nodes of a shard read ONE projection, and a payload holds A and B alone. B starts at zero (the adapter changes nothing)."""

    frozen_buffers = ("weight", "bias")           # buffers that are neither trained nor state

    def __init__(self, base: nn.Linear, rank: int = 8, alpha: float = 16.0, p: float = 0.0, seed: Optional[int] = None):
        if rank < 1:
            raise ValueError(f"an adapter of rank {rank}")
        device = base.weight.device
        super().__init__(p, 0 if p == 0.0 and seed is None else seed, device)
        self.register_buffer("weight", base.weight.detach(), persistent=False)
        self.register_buffer("bias", None if base.bias is None else base.bias.detach(), persistent=False)
        self.scale = alpha / rank
        self.train(base.training)
        self.a = nn.Parameter(torch.empty(rank, base.in_features, device=device))
        self.b = nn.Parameter(torch.zeros(base.out_features, rank, device=device))
        nn.init.kaiming_uniform_(self.a, a=5 ** 0.5)

    def forward(self, x):
        p, step = self._draw()
        w, b = self.weight.to(x.dtype), None if self.bias is None else self.bias.to(x.dtype)
        la, lb = self.a.to(x.dtype), self.b.to(x.dtype)
        if not x.is_cuda:
            return F.linear(x, w, b) + self.scale * F.linear(F.linear(self._stock(x, p, step), la), lb)
        y = _Adapter.apply(x.reshape(1, -1, x.shape[-1]), w, b, la.unsqueeze(0), lb.unsqueeze(0), self.seed, step, self.scale, p,
                           self.site)[0]
        return y.reshape(*x.shape[:-1], w.shape[0])

    def extra_repr(self):
        return f"{self.a.shape[1]} -> {self.b.shape[0]}, rank {self.a.shape[0]}, p={self.p}"


def adapt(model: nn.Module, rank: int = 8, alpha: float = 16.0, p: float = 0.0) -> nn.Module:
    """Freezes ``model`` and replaces its linear layers by :class:`AdapterLinear` in place; what is left to train, and of its
    parameters to exchange and to keep in a checkpoint, are the adapters: its other parameters become buffers beside the state, like
    the projections. (Statistics that a layer keeps, BatchNorm's, stay in the state.) Weights are loaded before, not after. A layer
    that stands in several places keeps one adapter for all of them."""
    linears = [m for m in model.modules() if type(m) is nn.Linear]
    if not linears:
        raise ValueError("no linear layer to put an adapter on")
    for q in model.parameters():
        q.requires_grad_(False)
    made = {m: AdapterLinear(m, rank, alpha, p) for m in linears}
    for m in list(model.modules()):
        for name, child in m._modules.items():
            if child in made:
                setattr(m, name, made[child])
    model = made.get(model, model)
    own = set(made.values())
    for m in model.modules():
        if m not in own:
            _freeze(m)
    return model


def _freeze(m: nn.Module) -> None:
    """Makes the module's own parameters buffers that are no part of its state."""
    names = [n for n, q in m._parameters.items() if q is not None]
    for name in names:
        m.register_buffer(name, m._parameters.pop(name).detach(), persistent=False)
    if names:
        m.frozen_buffers = (*getattr(m, "frozen_buffers", ()), *names)


def share_frozen(first: nn.Module, other: nn.Module) -> None:
    """Makes the frozen buffers of ``other`` those of ``first``, a model of the same structure: adapters that are averaged have to
    stand beside the same weights, and nodes of one GPU need one copy of them."""
    layers = dict(first.named_modules())
    for name, m in other.named_modules():
        for b in getattr(m, "frozen_buffers", ()):
            mine, theirs = m._buffers[b], layers[name]._buffers[b] if name in layers else None
            if (mine is None) != (theirs is None) or mine is not None and mine.shape != theirs.shape:
                raise ValueError(f"the frozen {name}.{b} of two nodes' models differ: {None if mine is None else tuple(mine.shape)} "
                                 f"and {None if theirs is None else tuple(theirs.shape)}")
            m._buffers[b] = theirs


def frozen_digest(model: nn.Module) -> Optional[str]:
    """A fingerprint of the frozen buffers of a model (None: it has none), the same wherever they are kept."""
    h, some = hashlib.sha256(), False
    for name, m in model.named_modules():
        for b in getattr(m, "frozen_buffers", ()):
            t = m._buffers[b]
            if t is not None:
                t = t.detach().cpu().contiguous()
                h.update(f"{name}.{b} {t.dtype} {tuple(t.shape)};".encode())
                h.update(t.reshape(-1).view(torch.uint8).numpy().tobytes())
                some = True
    return h.hexdigest() if some else None
