"""ctypes bindings of ``libp2pfl_hip.so`` (the gfx950 kernels under ``p2pfl_amd/csrc``).

Every wrapper takes torch tensors whose *leading* dimension is the client dimension; the
client stride is ``t.stride(0)``, so views into the ``[clients, P]`` slabs
(``slab[:, off:off+n].unflatten(1, shape)``) are passed without copies. Kernels are enqueued
on the current torch HIP stream, so they compose with torch ops and can be captured into a
hipGraph with ``torch.cuda.graph``.

The library is mandatory on a GPU box: if it is missing, calls raise instead of silently
falling back to eager PyTorch.
"""
from __future__ import annotations

import ctypes
import functools
import struct
import threading
from ctypes import c_float, c_int, c_long, c_void_p
from typing import Optional

import torch

from .build import HIP_LIB

_lib = None


class HipKernelError(RuntimeError):
    pass


def load():
    """Load (once) and return the kernel library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not HIP_LIB.exists():
            raise HipKernelError(
                f"{HIP_LIB} is missing: run `python -m p2pfl_amd.ops.build` (or __graft_entry__.build()) first")
        _lib = ctypes.CDLL(str(HIP_LIB))
        for name in dir(_Sig):
            if name.startswith("p2pfl_"):
                fn = getattr(_lib, name)
                fn.argtypes = getattr(_Sig, name)
                fn.restype = c_long if name.endswith("_scratch") else c_int
    return _lib


def available() -> bool:
    return HIP_LIB.exists() and torch.cuda.is_available()


P, L, I, F = c_void_p, c_long, c_int, c_float

# Precision policy of the matrix products (see csrc/common.h). The reference trains 32-bit
# (fedstellar/learning/pytorch/lightninglearner.py:182-193), so the default is "fp32": fp32 storage, fp32 accumulation,
# fp32 operands on v_mfma_f32_32x32x2_f32 (exact fp32 fma chains) everywhere except the stage-2 convolutions (the
# matrix-core-bound kernels of a step), which form every fp32 product from three bf16 terms per operand - an EXACT
# decomposition (3 x 8 significand bits), six bf16 MFMAs with fp32 accumulation, dropped cross terms <= 2^-24 of the
# product: the same accuracy against a float64 oracle as the fp32 MFMA kernels at 2.7x fewer matrix-core cycles.
# "fp32-mfma" runs those convolutions on v_mfma_f32_32x32x2_f32 too (nothing but fp32 instructions anywhere);
# "bf16" rounds all operands to bf16 with fp32 accumulation (16x the matrix-core rate; a labelled fast mode).
# Every product wrapper takes ``prec`` (name or None = default).
PRECISIONS = {"bf16": 0, "fp32-mfma": 1, "fp32": 2}
SPLIT_TERMS = 3
_default_prec = "fp32"


def set_default_precision(name: str) -> None:
    global _default_prec
    if name not in PRECISIONS:
        raise ValueError(f"unknown precision {name!r}: expected one of {sorted(PRECISIONS)}")
    _default_prec = name


def default_precision() -> str:
    return _default_prec


_PRODUCT_OPS = frozenset((
    "linear_fwd", "linear_dgrad", "linear_wgrad", "linear_wgrad_adam", "linear_wgrad_adam_dgrad", "linear_wgrad_sgdm",
    "conv1_fwd", "conv1_wgrad", "conv1_wgrad_scratch",
    "conv2_prep_alloc", "conv2_prep", "conv2_fwd", "conv2_wgrad_scratch", "conv2_wgrad_scratch_opt", "conv2_wgrad",
    "conv2_dgrad"))


class _Bound:
    """This module with ``prec`` pre-set on every matrix-product wrapper (what an engine holds)."""

    def __init__(self, prec: str):
        _prec(prec)
        self.precision = prec
        self._cache = {}

    def __getattr__(self, name):
        import functools
        import sys
        fn = self._cache.get(name)
        if fn is None:
            fn = getattr(sys.modules[__name__], name)
            if name in _PRODUCT_OPS:
                fn = functools.partial(fn, prec=self.precision)
            self._cache[name] = fn
        return fn


def bound(prec=None) -> "_Bound":
    return _Bound(_default_prec if prec is None else prec)


def _prec(prec) -> int:
    if prec is None:
        prec = _default_prec
    try:
        return PRECISIONS[prec]
    except KeyError:
        raise ValueError(f"unknown precision {prec!r}: expected one of {sorted(PRECISIONS)}") from None


class _Sig:
    p2pfl_linear_fwd = [P, L, P, L, P, L, P, L, I, I, I, I, I, P, L, P, L, I, P]
    p2pfl_linear_fwd_scratch = [I, I, I, I]
    p2pfl_linear_dgrad = [P, L, P, L, P, L, P, L, I, I, I, I, P, L, I, P]
    p2pfl_linear_dgrad_scratch = [I, I, I, I]
    p2pfl_linear_wgrad = [P, L, P, L, P, L, P, L, I, I, I, I, P, L, I, P]
    p2pfl_linear_wgrad_adam = [P, L, P, L, P, P, P, L, P, P, P, L, I, I, I, I, F, F, F, F, F, I, P, I, P, L, I, P]
    p2pfl_linear_wgrad_adam_dgrad = [P, L, P, L, P, P, P, L, P, P, P, L, P, L, I, I, I, I, F, F, F, F, F, I, P, I, P, L, I, P]
    p2pfl_linear_wgrad_sgdm = [P, L, P, L, P, P, L, P, P, L, I, I, I, I, F, F, F, I, P, L, I, P]
    p2pfl_conv1_fwd = [P, L, P, L, P, L, P, L, P, L, P, L, I, I, I, I, I, P]
    p2pfl_conv1_wgrad = [P, L, P, L, P, L, P, L, P, L, P, L, P, L, I, I, I, I, I, P, P]
    p2pfl_conv1_wgrad_scratch = [I, I, I, I]
    p2pfl_conv2_wgrad_opt = [P, L, P, L, P, L, P, L, P, L, P, L, I, I, I, I, I, I, I, P, P]
    p2pfl_linear_head = [P, L, P, L, P, L, P, L, P, L, P, L, P, L, P, L, P, L, P, P, P, P, P, L, I, I, I, I, I, P, P, L, P]
    p2pfl_linear_head_scratch = [I, I, I, I]
    p2pfl_linear_head_accepts = [I, I, I]
    p2pfl_linear_wgrad_adam_dgrad_accepts = [I, I, I, I]
    p2pfl_conv2_prep = [P, L, P, L, I, I, I, I, I, P]
    p2pfl_conv2_fwd = [P, L, P, L, P, L, P, L, P, L, I, I, I, I, I, I, I, P]
    p2pfl_conv2_wgrad = [P, L, P, L, P, L, P, L, P, L, P, L, I, I, I, I, I, I, I, P]
    p2pfl_conv2_wgrad_scratch = [I, I, I, I]
    p2pfl_conv2_dgrad = [P, L, P, L, P, L, P, L, I, I, I, I, I, I, I, P]
    p2pfl_softmax_ce = [P, L, P, L, P, L, P, L, P, P, P, P, P, L, I, I, I, P]
    p2pfl_mse_input = [P, L, P, L, P, L, P, L, P, P, P, L, I, I, I, P]
    p2pfl_zero_rows = [P, L, I, I, P]
    p2pfl_adam_step = [P, P, P, P, L, L, L, I, F, F, F, F, F, I, P, P]
    p2pfl_adam_step2 = [P, P, P, P, L, L, L, L, I, F, F, F, F, F, I, P, P]
    p2pfl_sgdm_step = [P, P, P, L, L, L, I, F, F, F, P]
    p2pfl_fedavg = [P, L, I, P, L, P, L, P, P, P, P, P, I, L, P]
    p2pfl_fedavg_inplace = [P, L, I, P, L, I, P, P, P, P, P, I, L, P]
    p2pfl_fedavg_inplace_chunk = [I]
    p2pfl_aes128_ecb = [P, P, P, L, I, P]
    p2pfl_dropout = [P, L, P, L, L, I, I, P, P]
    p2pfl_adapter_linear_fwd = [P, P, L, P]
    p2pfl_adapter_linear_dgrad = [P, P, L, P]
    p2pfl_adapter_linear_scratch = [P, I]
    p2pfl_adapter_linear_wgrad = [P, P, P, L, P, L, P, L, P]
    p2pfl_adapter_linear_wgrad_scratch = [P]
    p2pfl_group_norm_fwd = [P, P]
    p2pfl_group_norm_bwd = [P, P]
    p2pfl_group_norm_fwd_scratch = [I, I, I, I, I, I]
    p2pfl_group_norm_bwd_scratch = [I, I, I, I, I, I]


class OptStruct(ctypes.Structure):
    """``P2pflOpt`` of csrc/opt_epi.h: the optimizer step a gradient-producing kernel applies in its epilogue."""
    _fields_ = [("kind", c_int), ("t", c_int),
                ("pw", c_void_p), ("mw", c_void_p), ("vw", c_void_p),
                ("pb", c_void_p), ("mb", c_void_p), ("vb", c_void_p),
                ("cs", c_long),
                ("lr", c_float), ("beta1", c_float), ("beta2", c_float), ("eps", c_float),
                ("weight_decay", c_float), ("momentum", c_float),
                ("bc", c_void_p)]


def fold_opt(kind: str, w, mw, vw, b, mb, vb, *, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, momentum=0.9,
             t: int = 1, bc=None) -> OptStruct:
    """Optimizer epilogue for one layer: ``w/mw/vw`` [K,...] and ``b/mb/vb`` [K,Out] are views of the parameter /
    moment slabs (``vw``/``vb`` None for SGD-momentum) that share ONE row stride. ``kind``: "adam" | "sgd"."""
    cs = w.stride(0)
    views = [w, mw, b, mb] + ([vw, vb] if kind == "adam" else [])
    for v in views:
        _t(v)
        if v.shape[0] > 1 and v.stride(0) != cs:        # (one client: the stride of a size-1 dimension means nothing)
            raise HipKernelError("optimizer epilogue: all parameter / moment views must share one row stride")
    ptr = lambda v: None if v is None else v.data_ptr()
    return OptStruct(1 if kind == "adam" else 2, int(t), ptr(w), ptr(mw), ptr(vw) if kind == "adam" else None,
                     ptr(b), ptr(mb), ptr(vb) if kind == "adam" else None, cs, lr, beta1, beta2, eps, weight_decay,
                     momentum, None if bc is None else _t(bc).data_ptr())


def _optp(opt):
    return None if opt is None else ctypes.byref(opt)


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _chk(code: int, what: str) -> None:
    if code != 0:
        raise HipKernelError(f"{what} failed with code {code}")


def _t(t: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    if not t.is_cuda:
        raise HipKernelError("HIP kernels need tensors on the GPU")
    if t.dtype != dtype:
        raise HipKernelError(f"expected {dtype}, got {t.dtype}")
    # all dims but the first must be densely packed
    exp = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != exp:
            raise HipKernelError(f"inner dimensions must be contiguous, got shape {tuple(t.shape)} stride {t.stride()}")
        exp *= size
    return t


def _pc(t: Optional[torch.Tensor], dtype=torch.float32):
    """(pointer, client stride in elements) of a [K, ...] tensor; (None, 0) for None."""
    if t is None:
        return None, 0
    _t(t, dtype)
    return t.data_ptr(), (t.stride(0) if t.dim() > 0 else 0)


# ----------------------------------------------------------------------------- linear
_fwd_scratch = {}


def linear_fwd_scratch(K: int, B: int, In: int, Out: int, device) -> Optional[torch.Tensor]:
    """Scratch buffer :func:`linear_fwd` wants for this problem (None: none) - skinny heads with few clients split
    their reduction over several blocks whose partial tiles go through it."""
    need = int(load().p2pfl_linear_fwd_scratch(K, B, In, Out))
    return torch.empty(need, dtype=torch.float32, device=device) if need else None


def linear_fwd(x, w, b, y, relu: bool, sidx=None, scratch: Optional[torch.Tensor] = None, prec=None) -> None:
    """y[k] = act(x[k] @ w[k].T + b[k]);  x [K,B,In], w [K,Out,In], b [K,Out], y [K,B,Out].

    ``sidx`` [K,B] int32: x is the whole data set [K,n,In] and row r of the product is x[k, sidx[k, r]] (the
    mini-batch gather of a first dense layer happens in the operand loader). ``scratch``: buffer from
    :func:`linear_fwd_scratch` owned by the caller; without it one per (device, stream, thread) is kept here."""
    K, B, Out = y.shape
    In = x.shape[2]
    assert w.shape == (K, Out, In) and b.shape == (K, Out) and (sidx is not None or x.shape[1] == B)
    (xp, xs), (wp, ws), (bp, bs), (yp, ys), (sp, ss) = _pc(x), _pc(w), _pc(b), _pc(y), _pc(sidx, torch.int32)
    assert sidx is None or sidx.shape == (K, B)
    lib = load()
    stream = _stream()
    need = int(lib.p2pfl_linear_fwd_scratch(K, B, In, Out))
    cp = 0
    if need:
        if scratch is not None and scratch.numel() >= need:
            buf = _t(scratch)
        else:
            key = (y.device, int(stream or 0), threading.get_ident())
            buf = _fwd_scratch.get(key)
            if buf is None or buf.numel() < need:
                buf = _fwd_scratch[key] = torch.empty(need, dtype=torch.float32, device=y.device)
        cp = buf.data_ptr()
    _chk(lib.p2pfl_linear_fwd(xp, xs, wp, ws, bp, bs, yp, ys, K, B, In, Out, int(relu), sp, ss, cp, need,
                              _prec(prec), stream), "linear_fwd")


def linear_dgrad_scratch(K: int, B: int, In: int, Out: int, device) -> Optional[torch.Tensor]:
    """Scratch buffer :func:`linear_dgrad` wants for this problem (None: none) - shards with too few tiles to fill the
    chip split the reduction over several workgroups whose partial tiles go through it."""
    need = int(load().p2pfl_linear_dgrad_scratch(K, B, In, Out))
    return torch.empty(need, dtype=torch.float32, device=device) if need else None


def linear_dgrad(dy, w, act, dx, scratch: Optional[torch.Tensor] = None, prec=None) -> None:
    """dx[k] = (dy[k] @ w[k]) * (act[k] > 0)   (act None: no mask). ``scratch``: buffer from
    :func:`linear_dgrad_scratch` owned by the caller; without it one per (device, stream, thread) is kept here."""
    K, B, Out = dy.shape
    In = w.shape[2]
    assert w.shape == (K, Out, In) and dx.shape == (K, B, In)
    (dp, ds), (wp, ws), (ap, as_), (xp, xs) = _pc(dy), _pc(w), _pc(act), _pc(dx)
    lib = load()
    stream = _stream()
    need = int(lib.p2pfl_linear_dgrad_scratch(K, B, In, Out))
    cp = 0
    if need:
        if scratch is not None and scratch.numel() >= need:
            buf = _t(scratch)
        else:
            key = (dx.device, int(stream or 0), threading.get_ident(), "dgrad")
            buf = _fwd_scratch.get(key)
            if buf is None or buf.numel() < need:
                buf = _fwd_scratch[key] = torch.empty(need, dtype=torch.float32, device=dx.device)
        cp = buf.data_ptr()
    _chk(lib.p2pfl_linear_dgrad(dp, ds, wp, ws, ap, as_, xp, xs, K, B, In, Out, cp, need, _prec(prec), stream),
         "linear_dgrad")


def linear_wgrad(dy, x, dw, db, sidx=None, prec=None) -> None:
    """dw[k] = dy[k].T @ x[k];  db[k] = dy[k].sum(0).   (``sidx``: batch rows gathered from x, see linear_fwd)"""
    K, B, Out = dy.shape
    In = x.shape[2]
    assert dw.shape == (K, Out, In) and db.shape == (K, Out) and (sidx is None or sidx.shape == (K, B))
    (dp, ds), (xp, xs), (wp, ws), (bp, bs), (sp, ss) = _pc(dy), _pc(x), _pc(dw), _pc(db), _pc(sidx, torch.int32)
    _chk(load().p2pfl_linear_wgrad(dp, ds, xp, xs, wp, ws, bp, bs, K, B, In, Out, sp, ss, _prec(prec), _stream()),
         "linear_wgrad")


def linear_wgrad_adam(dy, x, w, mw, vw, b, mb, vb, *, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0,
                      t: int, bc=None, fresh: bool = False, sidx=None, prec=None) -> None:
    """Fused ``dw = dy.T @ x`` + Adam update of (w, b) and their moments; the gradient is never
    written to memory. w/mw/vw are [K,Out,In] slab views with one common row stride, b/mb/vb [K,Out].
    ``fresh``: first step of a new optimizer - the moments count as zero and are not read (only written)."""
    K, B, Out = dy.shape
    In = x.shape[2]
    assert w.shape == (K, Out, In) and b.shape == (K, Out)
    assert w.stride(0) == mw.stride(0) == vw.stride(0) and b.stride(0) == mb.stride(0) == vb.stride(0)
    (dp, ds), (xp, xs), (sp, ss) = _pc(dy), _pc(x), _pc(sidx, torch.int32)
    _chk(load().p2pfl_linear_wgrad_adam(dp, ds, xp, xs, _t(w).data_ptr(), _t(mw).data_ptr(), _t(vw).data_ptr(),
                                        w.stride(0), _t(b).data_ptr(), _t(mb).data_ptr(), _t(vb).data_ptr(),
                                        b.stride(0), K, B, In, Out, lr, beta1, beta2, eps, weight_decay, t,
                                        None if bc is None else _t(bc).data_ptr(), int(fresh), sp, ss, _prec(prec),
                                        _stream()), "linear_wgrad_adam")


def linear_wgrad_adam_dgrad(dy, x, w, mw, vw, b, mb, vb, dx, *, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0,
                            t: int, bc=None, fresh: bool = False, sidx=None, prec=None) -> bool:
    """:func:`linear_wgrad_adam` that also writes the layer's data gradient ``dx = dy @ w`` ([K,B,In], no mask) from
    the weights it reads anyway - one pass over the weights less than ``linear_dgrad`` + ``linear_wgrad_adam``.
    fp32 policies only. Returns False (nothing launched) when the shape is not covered: run the two kernels then."""
    K, B, Out = dy.shape
    In = x.shape[2]
    assert w.shape == (K, Out, In) and b.shape == (K, Out) and dx.shape == (K, B, In)
    assert w.stride(0) == mw.stride(0) == vw.stride(0) and b.stride(0) == mb.stride(0) == vb.stride(0)
    if _prec(prec) == PRECISIONS["bf16"]:
        return False
    (dp, ds), (xp, xs), (sp, ss), (gp, gs) = _pc(dy), _pc(x), _pc(sidx, torch.int32), _pc(dx)
    rc = load().p2pfl_linear_wgrad_adam_dgrad(dp, ds, xp, xs, _t(w).data_ptr(), _t(mw).data_ptr(), _t(vw).data_ptr(),
                                              w.stride(0), _t(b).data_ptr(), _t(mb).data_ptr(), _t(vb).data_ptr(),
                                              b.stride(0), gp, gs, K, B, In, Out, lr, beta1, beta2, eps, weight_decay, t,
                                              None if bc is None else _t(bc).data_ptr(), int(fresh), sp, ss,
                                              _prec(prec), _stream())
    if rc == -4:
        return False
    _chk(rc, "linear_wgrad_adam_dgrad")
    return True


def linear_wgrad_sgdm(dy, x, w, mw, b, mb, *, lr, momentum=0.9, weight_decay=0.0, fresh: bool = False,
                      sidx=None, prec=None) -> None:
    """Fused ``dw = dy.T @ x`` + SGD-momentum update of (w, b) and their momentum buffers (same layout rules
    as :func:`linear_wgrad_adam`)."""
    K, B, Out = dy.shape
    In = x.shape[2]
    assert w.shape == (K, Out, In) and b.shape == (K, Out)
    assert w.stride(0) == mw.stride(0) and b.stride(0) == mb.stride(0)
    (dp, ds), (xp, xs), (sp, ss) = _pc(dy), _pc(x), _pc(sidx, torch.int32)
    _chk(load().p2pfl_linear_wgrad_sgdm(dp, ds, xp, xs, _t(w).data_ptr(), _t(mw).data_ptr(), w.stride(0),
                                        _t(b).data_ptr(), _t(mb).data_ptr(), b.stride(0), K, B, In, Out, lr,
                                        momentum, weight_decay, int(fresh), sp, ss, _prec(prec), _stream()),
         "linear_wgrad_sgdm")


# ----------------------------------------------------------------------------- conv
def conv1_fwd(data, sidx, w, bias, a1, code, ks: int, prec=None) -> None:
    """Stage-1 conv(1->F, ks x ks, same) + ReLU + 2x2 maxpool.

    data [K,n,784] fp32, sidx [K,B] int32 or None, w [K,F,ks*ks], bias [K,F],
    a1 [K,B,F,196] fp32 out, code [K,B,F,196] uint8 out.
    """
    K, B, Fm = a1.shape[0], a1.shape[1], a1.shape[2]
    (dp, ds), (sp, ss), (wp, ws), (bp, bs), (ap, as_) = _pc(data), _pc(sidx, torch.int32), _pc(w), _pc(bias), _pc(a1)
    cp, cs = _pc(code, torch.uint8)
    _chk(load().p2pfl_conv1_fwd(dp, ds, sp, ss, wp, ws, bp, bs, ap, as_, cp, cs, K, B, Fm, ks, _prec(prec), _stream()),
         "conv1_fwd")


_c1_scratch = {}


def conv1_wgrad_scratch(K: int, B: int, ks: int, device, prec=None) -> torch.Tensor:
    """Scratch buffer of :func:`conv1_wgrad` (per-wave partial tiles) for this problem size."""
    need = int(load().p2pfl_conv1_wgrad_scratch(K, B, ks, _prec(prec)))
    return torch.empty(max(need, 1), dtype=torch.float32, device=device)


def conv1_wgrad(g, code, data, sidx, dw, db, ks: int, scratch: Optional[torch.Tensor] = None, opt: Optional[OptStruct] = None,
                prec=None) -> None:
    """Stage-1 weight / bias gradient: per-wave partial tiles go through ``scratch`` and a finishing pass adds them up
    in a fixed order (no atomics: bitwise reproducible), then stores dw / db - or, with ``opt`` (:func:`fold_opt`),
    applies the layer's optimizer step instead (dw / db may then be None)."""
    K, B, Fm = g.shape[0], g.shape[1], g.shape[2]
    (gp, gs), (dp, ds), (sp, ss), (wp, ws), (bp, bs) = _pc(g), _pc(data), _pc(sidx, torch.int32), _pc(dw), _pc(db)
    cp, cs = _pc(code, torch.uint8)
    lib = load()
    need = int(lib.p2pfl_conv1_wgrad_scratch(K, B, ks, _prec(prec)))
    if scratch is not None and scratch.numel() >= need:
        buf = _t(scratch)
    else:
        key = (g.device, int(_stream() or 0), threading.get_ident())
        buf = _c1_scratch.get(key)
        if buf is None or buf.numel() < need:
            buf = _c1_scratch[key] = torch.empty(need, dtype=torch.float32, device=g.device)
    _chk(lib.p2pfl_conv1_wgrad(gp, gs, cp, cs, dp, ds, sp, ss, wp, ws, bp, bs, buf.data_ptr(), buf.numel(), K, B, Fm, ks,
                               _prec(prec), _optp(opt), _stream()), "conv1_wgrad")


def _prep_dtype(prec):
    return torch.float32 if _prec(prec) == PRECISIONS["fp32-mfma"] else torch.bfloat16


def _prep_terms(prec) -> int:
    return SPLIT_TERMS if _prec(prec) == PRECISIONS["fp32"] else 1


def conv2_prep_alloc(K: int, ks: int, device, prec=None) -> torch.Tensor:
    """Workspace of :func:`conv2_prep`: per client a tap-major copy (fp32 or bf16, by ``prec``) of the stage-2
    weights for the forward pass followed by the mirrored, transposed copy for the data gradient."""
    return torch.empty(K, _prep_terms(prec) * 2 * ks * ks * 64 * 32, dtype=_prep_dtype(prec), device=device)


def conv2_prep(w, wprep, ks: int, prec=None) -> None:
    """w [K,Cout=64,Cin*ks*ks] fp32 -> wprep (see conv2_prep_alloc). Run once per weight update."""
    K, Cout = w.shape[0], w.shape[1]
    Cin = w.shape[2] // (ks * ks)
    (wp, ws), (pp, ps) = _pc(w), _pc(wprep, _prep_dtype(prec))
    _chk(load().p2pfl_conv2_prep(wp, ws, pp, ps, K, Cin, Cout, ks, _prec(prec), _stream()), "conv2_prep")


def conv2_fwd(a1, w, bias, a2, code, ks: int, wprep=None, prec=None, coresident: bool = False) -> None:
    """Stage-2 conv(Cin->Cout, ks x ks, same) + ReLU + 2x2 maxpool on the matrix cores.
    ``coresident`` (fp32 only): the small-footprint kernel variant that fits on a CU beside the fused wgrad+Adam
    kernel - what the two-stream training step launches on its side stream.

    a1 [K,B,Cin,196], w [K,Cout,Cin*ks*ks], bias [K,Cout], a2 [K,B,Cout,49], code uint8 like a2.
    ``wprep``: workspace already filled by :func:`conv2_prep` for these weights (else made here).
    """
    K, B, Cin = a1.shape[0], a1.shape[1], a1.shape[2]
    Cout = w.shape[1]
    if wprep is None:
        wprep = conv2_prep_alloc(K, ks, a1.device, prec)
        conv2_prep(w, wprep, ks, prec)
    (ap, as_), (pp, ps), (bp, bs), (op, os_) = _pc(a1), _pc(wprep, _prep_dtype(prec)), _pc(bias), _pc(a2)
    cp, cs = _pc(code, torch.uint8)
    _chk(load().p2pfl_conv2_fwd(ap, as_, pp, ps, bp, bs, op, os_, cp, cs, K, B, Cin, Cout, ks, _prec(prec),
                                int(coresident), _stream()), "conv2_fwd")


_wgrad_scratch = {}


def conv2_wgrad_scratch(K: int, B: int, ks: int, device, prec=None) -> Optional[torch.Tensor]:
    """Scratch buffer :func:`conv2_wgrad` wants for this problem size (None: it needs none). With few clients
    the batch is split over more blocks and their partial sums go through this buffer."""
    need = int(load().p2pfl_conv2_wgrad_scratch(K, B, ks, _prec(prec)))
    return torch.empty(need, dtype=torch.float32, device=device) if need else None


def conv2_wgrad_scratch_opt(K: int, B: int, ks: int, device, prec=None) -> torch.Tensor:
    """Scratch of :func:`conv2_wgrad` with an optimizer epilogue: the partial-sum pass is then always taken."""
    need = max(int(load().p2pfl_conv2_wgrad_scratch(K, B, ks, _prec(prec))), K * (ks * ks * 64 * 32 + 64))
    return torch.empty(need, dtype=torch.float32, device=device)


def conv2_wgrad(g, code, a1, dw, db, ks: int, scratch: Optional[torch.Tensor] = None, prec=None,
                coresident: bool = False, opt: Optional[OptStruct] = None) -> None:
    """Stage-2 weight/bias gradient: dw [K,Cout,Cin*ks*ks], db [K,Cout] (overwritten) - or, with ``opt``
    (:func:`fold_opt`), the layer's optimizer step applied by the reduction pass (dw / db may then be None).

    ``scratch``: buffer from :func:`conv2_wgrad_scratch` owned by the caller (one call in flight per buffer);
    without it a module-level buffer per (device, stream, thread) is used."""
    K, B, Cout = g.shape[0], g.shape[1], g.shape[2]
    Cin = a1.shape[2]
    (gp, gs), (ap, as_), (wp, ws), (bp, bs) = _pc(g), _pc(a1), _pc(dw), _pc(db)
    cp, cs = _pc(code, torch.uint8)
    lib = load()
    stream = _stream()
    need = int(lib.p2pfl_conv2_wgrad_scratch(K, B, ks, _prec(prec)))
    if opt is not None:
        need = max(need, K * (ks * ks * Cout * Cin + Cout))
    sp = 0
    if need:
        if scratch is not None and scratch.numel() >= need:
            buf = _t(scratch)
        else:
            key = (g.device, int(stream or 0), threading.get_ident(), _prec(prec))
            buf = _wgrad_scratch.get(key)
            if buf is None or buf.numel() < need:
                buf = _wgrad_scratch[key] = torch.empty(need, dtype=torch.float32, device=g.device)
        sp = buf.data_ptr()
        need = buf.numel()
    _chk(lib.p2pfl_conv2_wgrad_opt(gp, gs, cp, cs, ap, as_, wp, ws, bp, bs, sp, need, K, B, Cin, Cout, ks, _prec(prec),
                                   int(coresident), _optp(opt), stream), "conv2_wgrad")


def conv2_dgrad(g, code, w, da1, ks: int, wprep=None, prec=None, coresident: bool = False) -> None:
    K, B, Cout = g.shape[0], g.shape[1], g.shape[2]
    Cin = da1.shape[2]
    if wprep is None:
        wprep = conv2_prep_alloc(K, ks, g.device, prec)
        conv2_prep(w, wprep, ks, prec)
    (gp, gs), (pp, ps), (dp, ds) = _pc(g), _pc(wprep, _prep_dtype(prec)), _pc(da1)
    cp, cs = _pc(code, torch.uint8)
    _chk(load().p2pfl_conv2_dgrad(gp, gs, cp, cs, pp, ps, dp, ds, K, B, Cin, Cout, ks, _prec(prec), int(coresident),
                                  _stream()), "conv2_dgrad")


# ----------------------------------------------------------------------------- loss / misc
def softmax_ce(logits, labels, sidx, dlogits, loss_sum, correct, count, confusion=None, n_valid=None) -> None:
    """Fused softmax-CE fwd/bwd + metric counters. logits [K,B,C]; labels [K,n] int32."""
    K, B, C = logits.shape
    (lp, ls), (yp, ys), (sp, ss), (dp, ds) = _pc(logits), _pc(labels, torch.int32), _pc(sidx, torch.int32), _pc(dlogits)
    nvp, nvs = _pc(n_valid, torch.int32)
    _chk(load().p2pfl_softmax_ce(lp, ls, yp, ys, sp, ss, dp, ds, _t(loss_sum).data_ptr(),
                                 _t(correct, torch.int32).data_ptr(), _t(count, torch.int32).data_ptr(),
                                 None if confusion is None else _t(confusion, torch.int32).data_ptr(),
                                 nvp, nvs, K, B, C, _stream()), "softmax_ce")


def linear_wgrad_adam_dgrad_accepts(K: int, B: int, In: int, Out: int) -> bool:
    """Would :func:`linear_wgrad_adam_dgrad` take K clients of this layer (its chip-filling rule, csrc/linear.hip)?"""
    return bool(load().p2pfl_linear_wgrad_adam_dgrad_accepts(K, B, In, Out))


def linear_head_accepts(B: int, In: int, C: int) -> bool:
    return bool(load().p2pfl_linear_head_accepts(B, In, C))


def linear_head_scratch(K: int, B: int, In: int, C: int, device) -> Optional[torch.Tensor]:
    """Scratch buffer with which :func:`linear_head` takes its two-kernel form over (client, column slice) grids (wide
    heads: In >= 1024); None: the one-kernel form covers this shape."""
    need = int(load().p2pfl_linear_head_scratch(K, B, In, C))
    return torch.empty(need, dtype=torch.float32, device=device) if need else None


def linear_head(x, w, b, labels, sidx, loss_sum, correct, count, confusion=None, n_valid=None, *, dx=None, dw=None,
                db=None, logits=None, relu_mask: bool = False, opt: Optional[OptStruct] = None,
                scratch: Optional[torch.Tensor] = None) -> None:
    """The classification head of a training step (csrc/head.hip): logits = x w^T + b, softmax cross-entropy + metric
    counters, ``dx = (dlogits w) * [x > 0 if relu_mask]``, and either the gradients ``dw`` / ``db`` or - with ``opt``
    (:func:`fold_opt` over these very ``w`` / ``b`` views) - the optimizer step in place. One kernel per client, or
    - with ``scratch`` from :func:`linear_head_scratch` - two kernels over column slices of the clients.
    x [K,B,In] (B <= 32), w [K,C,In] (C <= 16), b [K,C], labels [K,n] int32, dx [K,B,In] or None."""
    K, B, In = x.shape
    C = w.shape[1]
    assert w.shape == (K, C, In) and b.shape == (K, C)
    assert dx is None or dx.shape == (K, B, In)
    (xp, xs), (wp, ws), (bp, bs), (gp, gs) = _pc(x), _pc(w), _pc(b), _pc(dx)
    (dwp, dws), (dbp, dbs), (lp, ls) = _pc(dw), _pc(db), _pc(logits)
    (yp, ys), (sp, ss), (nvp, nvs) = _pc(labels, torch.int32), _pc(sidx, torch.int32), _pc(n_valid, torch.int32)
    _chk(load().p2pfl_linear_head(xp, xs, wp, ws, bp, bs, gp, gs, dwp, dws, dbp, dbs, lp, ls, yp, ys, sp, ss,
                                  _t(loss_sum).data_ptr(), _t(correct, torch.int32).data_ptr(),
                                  _t(count, torch.int32).data_ptr(),
                                  None if confusion is None else _t(confusion, torch.int32).data_ptr(),
                                  nvp, nvs, K, B, In, C, int(relu_mask), _optp(opt),
                                  None if scratch is None else scratch.data_ptr(),
                                  0 if scratch is None else scratch.numel(), _stream()), "linear_head")


def mse_input(out, data, sidx, dout, loss_sum, count, n_valid=None) -> None:
    """Reconstruction loss fwd/bwd of the auto-encoders: MSE between ``out`` [K,B,D] and the batch's INPUT rows, gathered
    from ``data`` [K,n,D] with ``sidx`` [K,B] (None: rows 0..B-1). ``dout`` None: evaluation. ``loss_sum`` += mean loss
    of the batch x its samples, ``count`` += samples."""
    K, B, D = out.shape
    if data.shape[2] != D or data.stride(1) != D:
        raise HipKernelError(f"mse_input: data rows of {data.shape[2]} (stride {data.stride(1)}) for outputs of {D}")
    (op, os_), (xp, xs), (sp, ss), (dp, ds) = _pc(out), _pc(data), _pc(sidx, torch.int32), _pc(dout)
    nvp, nvs = _pc(n_valid, torch.int32)
    _chk(load().p2pfl_mse_input(op, os_, xp, xs, sp, ss, dp, ds, _t(loss_sum).data_ptr(),
                                _t(count, torch.int32).data_ptr(), nvp, nvs, K, B, D, _stream()), "mse_input")


def zero_rows(t) -> None:
    """Zero a [K, ...] (possibly slab-strided) view."""
    K = t.shape[0]
    n = t[0].numel()
    p, s = _pc(t)
    _chk(load().p2pfl_zero_rows(p, s, n, K, _stream()), "zero_rows")


# ----------------------------------------------------------------------------- optimizers
def adam_step(p, g, m, v, *, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, t: int, bc=None) -> None:
    """One Adam step over [K, P] slabs; p / m / v share one row stride, the gradient slab may have its own.

    ``bc``: optional device tensor [2] = (1/(1-beta1^t), 1/sqrt(1-beta2^t)) read by the kernel at
    run time instead of the host-computed scalars (lets a captured graph be replayed for any t)."""
    K, n = p.shape
    cs = p.stride(0)
    assert m.stride(0) == cs and v.stride(0) == cs and g.shape == p.shape and g.stride(1) == 1
    _chk(load().p2pfl_adam_step(_t(p).data_ptr(), _t(g).data_ptr(), _t(m).data_ptr(), _t(v).data_ptr(), cs, g.stride(0), n, K,
                                lr, beta1, beta2, eps, weight_decay, t,
                                None if bc is None else _t(bc).data_ptr(), _stream()), "adam_step")


def adam_step_ranges(p, g, m, v, ranges, *, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, t: int,
                     bc=None) -> None:
    """Adam step over the column ranges ``[(a0, b0), (a1, b1)]`` (a0 < b0 <= a1 < b1) of [K, P] slabs in ONE launch."""
    (a0, b0), (a1, b1) = ranges
    assert 0 <= a0 < b0 <= a1 < b1 <= p.shape[1]
    cs = p.stride(0)
    assert g.stride(0) == cs and m.stride(0) == cs and v.stride(0) == cs and g.shape == p.shape
    _chk(load().p2pfl_adam_step2(_t(p[:, a0:]).data_ptr(), _t(g[:, a0:]).data_ptr(), _t(m[:, a0:]).data_ptr(),
                                 _t(v[:, a0:]).data_ptr(), cs, b0 - a0, a1 - b0, b1 - a1, p.shape[0], lr, beta1, beta2,
                                 eps, weight_decay, t, None if bc is None else _t(bc).data_ptr(), _stream()),
         "adam_step_ranges")


def sgdm_step(p, g, buf, *, lr, momentum=0.9, weight_decay=0.0) -> None:
    K, n = p.shape
    cs = p.stride(0)
    assert buf.stride(0) == cs and g.shape == p.shape and g.stride(1) == 1
    _chk(load().p2pfl_sgdm_step(_t(p).data_ptr(), _t(g).data_ptr(), _t(buf).data_ptr(), cs, g.stride(0), n, K, lr, momentum,
                                weight_decay, _stream()), "sgdm_step")


# ----------------------------------------------------------------------------- FedAvg
def fedavg(local, remote, out, src_ptr, src_row, src_w, dst_ptr, dst_row) -> None:
    """Grouped weighted row reduce (see csrc/fedavg.hip). `remote` may be None."""
    n_local, n = local.shape
    G = src_ptr.numel() - 1
    rp, rs = (remote.data_ptr(), remote.stride(0)) if remote is not None and remote.numel() else (local.data_ptr(), local.stride(0))
    _chk(load().p2pfl_fedavg(_t(local).data_ptr(), local.stride(0), n_local, rp, rs, _t(out).data_ptr(),
                             out.stride(0), _t(src_ptr, torch.int32).data_ptr(),
                             _t(src_row, torch.int32).data_ptr(), _t(src_w).data_ptr(),
                             _t(dst_ptr, torch.int32).data_ptr(), _t(dst_row, torch.int32).data_ptr(), G, n,
                             _stream()), "fedavg")


def fedavg_inplace(slab, remote, src_ptr, src_row, src_w, dst_ptr, dst_row) -> bool:
    """:func:`fedavg` with ``out`` = ``slab`` itself: every source row (slab rows, then ``remote`` rows) is read once,
    whatever the number of groups using it, and the destinations are overwritten in place (csrc/fedavg.hip).
    False (nothing ran): too many rows for the kernel's LDS pool - reduce into a second slab with :func:`fedavg`."""
    n_local, n = slab.shape
    n_remote = int(remote.shape[0]) if remote is not None and remote.numel() else 0
    lib = load()
    if int(lib.p2pfl_fedavg_inplace_chunk(n_local + n_remote)) == 0:
        return False
    rp, rs = (remote.data_ptr(), remote.stride(0)) if n_remote else (None, 0)
    G = src_ptr.numel() - 1
    _chk(lib.p2pfl_fedavg_inplace(_t(slab).data_ptr(), slab.stride(0), n_local, rp, rs, n_remote,
                                  _t(src_ptr, torch.int32).data_ptr(), _t(src_row, torch.int32).data_ptr(),
                                  _t(src_w).data_ptr(), _t(dst_ptr, torch.int32).data_ptr(),
                                  _t(dst_row, torch.int32).data_ptr(), G, n, _stream()), "fedavg_inplace")
    return True


def aes128_ecb(src, dst, round_keys, decrypt: bool) -> None:
    """AES-128-ECB over a flat uint8 buffer (length % 16 == 0) with expanded round keys [176] uint8."""
    n = src.numel()
    assert n % 16 == 0 and dst.numel() == n and round_keys.numel() == 176
    _chk(load().p2pfl_aes128_ecb(_t(src, torch.uint8).data_ptr(), _t(dst, torch.uint8).data_ptr(),
                                 _t(round_keys, torch.uint8).data_ptr(), n // 16, int(decrypt), _stream()),
         "aes128_ecb")


# ----------------------------------------------------------------------------- typed maps
# The normalisation, dropout and adapter kernels take fp32, bf16 and fp16 maps (one type per call); sums are fp32.
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _launch(fn, what: str, device, *args) -> None:
    """Launch on the current stream of ``device``, whichever device is current."""
    idx = device.index
    if idx == torch._C._cuda_getDevice():
        code = fn(*args, torch._C._cuda_getCurrentRawStream(idx))
        if code:
            _chk(code, what)
        return
    with torch.cuda.device(device):
        _chk(fn(*args, torch._C._cuda_getCurrentRawStream(idx)), what)


def _typed(t: torch.Tensor, what: str, like: Optional[torch.Tensor] = None) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise HipKernelError(f"{what}: expected fp32, bf16 or fp16, got {t.dtype}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise HipKernelError(f"{what}: expected {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    return code


def _gpu(t: torch.Tensor):
    """The kernel library, for a call whose arguments have been checked."""
    if not t.is_cuda:
        raise HipKernelError("HIP kernels need tensors on the GPU")
    return load()


def _packed(t: torch.Tensor, what: str, out: bool = False) -> torch.Tensor:
    """``t`` [K, ...] with packed inner dimensions; ``out``: one that is written, whose clients may not share memory."""
    if t.numel() == 0:
        return t                                 # (the strides of an empty tensor say nothing)
    exp = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != exp:
            raise HipKernelError(f"{what}: inner dimensions must be contiguous, got shape {tuple(t.shape)} stride {t.stride()}")
        exp *= size
    if out and t.dim() and t.shape[0] > 1 and t.stride(0) < exp:
        raise HipKernelError(f"{what}: clients share memory, got shape {tuple(t.shape)} stride {t.stride()}")
    return t


def _same(t: torch.Tensor, what: str, shape: tuple, dtype, device, out: bool = False, name: str = "") -> torch.Tensor:
    """``t`` checked to be of this shape and type on this device, with packed inner dimensions."""
    if t.shape != shape:
        raise HipKernelError(f"{what} {name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise HipKernelError(f"{what} {name}: expected a tensor on {device}, got {t.device}")
    if t.dtype != dtype:
        raise HipKernelError(f"{what} {name}: expected {dtype}, got {t.dtype}")
    return t if t.is_contiguous() else _packed(t, f"{what} {name}", out)


def _scratch(need: int, scratch: Optional[torch.Tensor], device, what: str):
    """(pointer, floats, owner) of a workspace: the caller's, or one of the caching allocator that belongs to this call
    alone (in a captured graph: to that graph)."""
    if need <= 0:
        return None, 0, None
    if scratch is None:
        scratch = torch.empty(need, dtype=torch.float32, device=device)
    elif scratch.numel() < need or scratch.dtype != torch.float32 or scratch.device != device or not scratch.is_contiguous():
        raise HipKernelError(f"{what}: the workspace has to be {need} contiguous fp32 values on {device}")
    return scratch.data_ptr(), scratch.numel(), scratch


# ----------------------------------------------------------------------------- dropout
# ``P2pflDrop`` of csrc/philox.h: seeds, step, site, threshold, all, scale. (Argument structures of these calls are packed in one
# go: field by field through ctypes took longer than the smallest kernels.)
_DROP = "qqIIif"
_NO_DROP = (0, 0, 0, 0, 0, 1.0)


class Drop:
    """A dropout without a stored mask: whether element ``e`` of client ``k`` stays is a function of ``(seeds[k], step,
    site, e)`` alone (csrc/philox.h), so the backward pass draws the same mask again and a node's masks do not depend on
    the nodes beside it.

    ``p`` in [0, 1]: probability of a zero; kept elements are scaled by ``1 / (1 - p)``. ``seeds`` [K] int64 and ``step``
    [1] int64 live on the GPU and are read when the kernel runs: a captured graph draws new masks once ``step`` has been
    advanced. ``site`` in [0, 2^32) tells the dropouts of one step apart."""

    def __init__(self, p: float, seeds: torch.Tensor, step: torch.Tensor, site: int = 0):
        p, site = float(p), int(site)
        if not 0.0 <= p <= 1.0:
            raise HipKernelError(f"dropout probability {p} outside [0, 1]")
        if not 0 <= site < 2 ** 32:
            raise HipKernelError(f"dropout site {site} outside [0, 2^32)")
        for t, what in ((seeds, "seeds"), (step, "step")):
            if t.dtype != torch.int64 or t.dim() != 1 or not t.is_contiguous():
                raise HipKernelError(f"dropout {what}: expected a contiguous 1-D int64 tensor")
        if step.numel() != 1 or step.device != seeds.device:
            raise HipKernelError("dropout step: expected one value on the device of the seeds")
        self.p, self.seeds, self.step, self.site = p, seeds, step, site
        thr = min(int(round(p * 2 ** 32)), 2 ** 32 - 1)
        self._fields = (seeds.data_ptr(), step.data_ptr(), site, thr, int(p >= 1.0), 0.0 if p >= 1.0 else 1.0 / (1.0 - p))

    def _for(self, K: int, device, n: int) -> tuple:
        if self.seeds.numel() != K or self.seeds.device != device:
            raise HipKernelError(f"dropout: expected {K} seeds on {device}, got {self.seeds.numel()} on {self.seeds.device}")
        if n >= 2 ** 34:
            raise HipKernelError(f"dropout: {n} elements of one client exceed the generator's 2^34")
        return self._fields


def dropout(x, y, drop: Drop) -> None:
    """y[k] = keep ? x[k] / (1 - p) : 0 over [K, ...] maps (``y`` may be ``x``). The backward pass is the same call on the
    gradient. A dropped element is zero whatever it held. fp32 / bf16 / fp16, rounded once."""
    code = _typed(x, "dropout x")
    _typed(y, "dropout y", x)
    if x.dim() < 1 or y.shape != x.shape:
        raise HipKernelError(f"dropout: x {tuple(x.shape)} and y {tuple(y.shape)} have to be of one shape [K, ...]")
    K = x.shape[0]
    n = x.numel() // K if K else 0
    fields = struct.pack(_DROP, *drop._for(K, x.device, n))
    _packed(x, "dropout x"), _packed(y, "dropout y", True)
    lib = _gpu(x)
    if n:
        _launch(lib.p2pfl_dropout, "dropout", x.device, x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), n, K, code,
                fields)


# ----------------------------------------------------------------------------- group norm
ACTIVATIONS = {"none": 0, None: 0, "relu": 1, "silu": 2, "gelu": 3}
GROUP_NORM_MAX_CHANNELS = 2048        # channels of one group


# ``P2pflGroupNorm`` of csrc/group_norm.hip: six maps (pointer, client, sample and position stride), w, b, mean, rstd, dw, db,
# scratch, drop, sizes, eps.
_GROUP_NORM = struct.Struct("24q" "4q" "2q" "4q" "2q" + _DROP + "7if")
_NO_MAP = (0, 0, 0, 0)


def _gn_map(t: Optional[torch.Tensor], what: str, name: str, x: torch.Tensor, out: bool = False) -> tuple:
    """Strides of a channels-last map [K, N, ..., C]: any client, sample and position stride, dense channels."""
    if t is None:
        return _NO_MAP
    if t is not x:
        if t.dtype != x.dtype or t.device != x.device:
            raise HipKernelError(f"{what} {name}: expected {x.dtype} on {x.device}, got {t.dtype} on {t.device}")
        if t.shape != x.shape:
            raise HipKernelError(f"{what} {name}: expected shape {tuple(x.shape)}, got {tuple(t.shape)}")
    if t.is_contiguous():
        shape = t.shape
        C = shape[-1]
        row = t.numel() // shape[0] if shape[0] else 0
        return t.data_ptr(), row, row // shape[1] if shape[1] else 0, C
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise HipKernelError(f"{what} {name}: channels have to be dense and last, got shape {tuple(t.shape)} stride {t.stride()}")
    ss = span = None
    for size, stride in zip(reversed(t.shape[2:-1]), reversed(t.stride()[2:-1])):
        if size == 1:
            continue
        if span is not None and stride != span:
            raise HipKernelError(f"{what} {name}: positions have to be evenly spaced, got shape {tuple(t.shape)} stride {t.stride()}")
        ss = stride if ss is None else ss
        span = stride * size
    if out and any(size > 1 and stride == 0 for size, stride in zip(t.shape, t.stride())):
        raise HipKernelError(f"{what} {name}: elements share memory, got shape {tuple(t.shape)} stride {t.stride()}")
    return t.data_ptr(), t.stride(0), t.stride(1), ss or 0


def _gn_param(t, what: str, name: str, shape, device, out: bool = False) -> tuple:
    if t is None:
        return 0, 0
    return _same(t, what, shape, torch.float32, device, out, name).data_ptr(), t.stride(0)


def _gn_stat(t, what: str, name: str, shape, device, required: bool) -> int:
    if t is None:
        if required:
            raise HipKernelError(f"{what}: needs the forward pass's {name}")
        return 0
    if t.shape != shape or t.dtype != torch.float32 or t.device != device or not t.is_contiguous():
        raise HipKernelError(f"{what} {name}: expected contiguous fp32 {tuple(shape)} on {device}")
    return t.data_ptr()


def _gn_sizes(what: str, x, groups, act, drop):
    """(K, N, S, C, G, activation, type), the dropout's fields."""
    if x.dim() < 3:
        raise HipKernelError(f"{what}: expected a channels-last map [K, N, ..., C], got {tuple(x.shape)}")
    code = _typed(x, f"{what} x")
    if act not in ACTIVATIONS:
        raise HipKernelError(f"{what}: unknown activation {act!r}: expected one of none, relu, silu, gelu")
    shape = x.shape
    K, N, C, n = shape[0], shape[1], shape[-1], x.numel()
    S = n // (K * N * C) if n else 0
    groups = int(groups)
    if groups < 1 or C % groups:
        raise HipKernelError(f"{what}: {C} channels do not divide into {groups} groups")
    if C // groups > GROUP_NORM_MAX_CHANNELS:
        raise HipKernelError(f"{what}: groups of {C // groups} channels exceed {GROUP_NORM_MAX_CHANNELS}")
    if max(K, N, S) > 2 ** 30:
        raise HipKernelError(f"{what}: {tuple(shape)} is too large")
    return (K, N, S, C, groups, ACTIVATIONS[act], code), \
        _NO_DROP if drop is None or drop.p == 0.0 else drop._for(K, x.device, N * S * C)


@functools.lru_cache(maxsize=1024)
def _gn_scratch(backward: bool, K: int, N: int, S: int, C: int, G: int, code: int) -> int:
    lib = load()
    return int((lib.p2pfl_group_norm_bwd_scratch if backward else lib.p2pfl_group_norm_fwd_scratch)(K, N, S, C, G, code))


def group_norm_scratch(K: int, N: int, S: int, C: int, groups: int, dtype, device, backward: bool = False) -> Optional[torch.Tensor]:
    """Workspace :func:`group_norm_fwd` (or ``_bwd``) wants for maps [K, N, S, C] (None: none). A call without one takes
    its own from the caching allocator; a kept one serves one call at a time."""
    need = _gn_scratch(backward, K, N, S, C, groups, _DTYPES[dtype])
    return torch.empty(need, dtype=torch.float32, device=device) if need else None


def group_norm_fwd(x, w, b, y, groups: int, *, mean=None, rstd=None, eps: float = 1e-5, act=None, residual=None,
                   drop: Optional[Drop] = None, scratch: Optional[torch.Tensor] = None) -> None:
    """y = drop(act(group_norm(x) * w + b + residual)) over channels-last maps [K, N, ..., C] of K clients.

    Statistics are over the positions and the C / groups channels of a group, in fp32; ``w`` / ``b`` [K, C] fp32 (slab
    views, or None); ``mean`` / ``rstd`` [K, N, groups] fp32 out, for the backward pass. ``act``: none, relu, silu, gelu
    (the erf form). ``drop``: element ``((n S) + s) C + c`` of a client, the same mask as :func:`dropout` over ``y[k]``.
    Maps are fp32, bf16 or fp16 of one type, with any client, sample and position stride; ``y`` may be ``x`` or
    ``residual``, but may not overlap them otherwise."""
    what, dev = "group_norm_fwd", x.device
    sizes, drop_fields = _gn_sizes(what, x, groups, act, drop)
    K, N, _, C, G, _, code = sizes
    maps = _gn_map(x, what, "x", x) + _gn_map(y, what, "y", x, True) + _gn_map(residual, what, "residual", x)
    params = _gn_param(w, what, "w", (K, C), dev) + _gn_param(b, what, "b", (K, C), dev)
    stats = _gn_stat(mean, what, "mean", (K, N, G), dev, False), _gn_stat(rstd, what, "rstd", (K, N, G), dev, False)
    lib = _gpu(x)
    if x.numel() == 0:
        return
    p, n, keep = _scratch(_gn_scratch(False, *sizes[:5], code), scratch, dev, what)
    _launch(lib.p2pfl_group_norm_fwd, what, dev,
            _GROUP_NORM.pack(*maps, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, *params, *stats, 0, 0, 0, 0, p or 0, n, *drop_fields, *sizes, eps))


def group_norm_bwd(dy, x, w, b, mean, rstd, dx, dw, db, groups: int, *, act=None, y=None, residual=None, dres=None,
                   drop: Optional[Drop] = None, scratch: Optional[torch.Tensor] = None) -> None:
    """Gradients of :func:`group_norm_fwd`: ``dx`` and ``dres`` (the residual's, or None) like ``x``, ``dw`` / ``db``
    [K, C] fp32 (or None), added up in a fixed order.

    silu and gelu recompute the value before the activation from ``x`` and ``residual`` (the forward pass's). relu goes by
    the forward pass's result ``y`` where it is given - ``residual`` is not read then - and recomputes otherwise. Outputs
    may be ``dy`` or ``x`` themselves, but may not overlap the inputs otherwise."""
    what, dev = "group_norm_bwd", x.device
    sizes, drop_fields = _gn_sizes(what, x, groups, act, drop)
    K, N, _, C, G, _, code = sizes
    maps = _gn_map(x, what, "x", x) + _gn_map(y, what, "y", x) + _gn_map(residual, what, "residual", x) \
        + _gn_map(dy, what, "dy", x) + _gn_map(dx, what, "dx", x, True) + _gn_map(dres, what, "dres", x, True)
    params = _gn_param(w, what, "w", (K, C), dev) + _gn_param(b, what, "b", (K, C), dev)
    stats = _gn_stat(mean, what, "mean", (K, N, G), dev, True), _gn_stat(rstd, what, "rstd", (K, N, G), dev, True)
    grads = _gn_param(dw, what, "dw", (K, C), dev, True) + _gn_param(db, what, "db", (K, C), dev, True)
    lib = _gpu(x)
    if K == 0 or C == 0:
        return
    p, n, keep = _scratch(_gn_scratch(True, *sizes[:5], code), scratch, dev, what)
    _launch(lib.p2pfl_group_norm_bwd, what, dev,
            _GROUP_NORM.pack(*maps, *params, *stats, *grads, p or 0, n, *drop_fields, *sizes, 0.0))


# ----------------------------------------------------------------------------- adapters
ADAPTER_MAX_RANK, ADAPTER_MAX_FEATURES, ADAPTER_MAX_ROWS, ADAPTER_MAX_CLIENTS = 1024, 2 ** 20, 2 ** 22, 2 ** 16 - 1


# ``P2pflAdapter`` of csrc/adapter.hip: x, its client and row stride; w, its row stride; bias; la, lb and their client strides; u; y,
# its client and row stride; row_ptr; drop; drop_out, K, T, B, In, Out, R, type; scale.
_ADAPTER = struct.Struct("15q" + _DROP + "8if")


def _adapter_rows(what: str, t, name: str, lead, width: int, dtype, device, out: bool = False):
    """(pointer, client stride, row stride) of the rows [K, B, width] or [T, width]."""
    _same(t, what, (*lead, width), dtype, device, out, name)
    if t.dim() == 2:
        return t.data_ptr(), 0, t.stride(0)
    return t.data_ptr(), t.stride(0), width


def _adapter_sizes(what: str, x, K: int, R: int, In: int, Out: int, row_ptr, drop, drop_width: int):
    """(leading dimensions, row_ptr, the dropout's fields, (K, T, B, In, Out, R, type)) of a call over the rows of ``x`` (its last
    dimension aside), checked."""
    code = _typed(x, what)
    lead = tuple(x.shape[:-1])
    if x.dim() == 3 and row_ptr is None:
        if lead[0] != K:
            raise HipKernelError(f"{what}: rows of {lead[0]} clients for the adapters of {K}")
    elif x.dim() != 2 or row_ptr is None:
        raise HipKernelError(f"{what}: expected rows [K, B, features], or [T, features] with row_ptr, got {tuple(x.shape)}")
    if row_ptr is not None:
        if row_ptr.dtype != torch.int32 or tuple(row_ptr.shape) != (K + 1,) or not row_ptr.is_contiguous() \
                or row_ptr.device != x.device:
            raise HipKernelError(f"{what} row_ptr: expected {K + 1} contiguous int32 values on {x.device}")
    T = lead[0] if x.dim() == 2 else lead[0] * lead[1]
    if not 1 <= R <= ADAPTER_MAX_RANK or min(In, Out) < 1 or max(In, Out) > ADAPTER_MAX_FEATURES \
            or T > ADAPTER_MAX_ROWS or K > ADAPTER_MAX_CLIENTS or T * max(In, Out) > 2 ** 37:
        raise HipKernelError(f"{what}: {T} rows of {K} clients, {In} -> {Out} features, rank {R}: outside the kernel's limits "
                             f"({ADAPTER_MAX_ROWS} rows, {ADAPTER_MAX_CLIENTS} clients, {ADAPTER_MAX_FEATURES} features, "
                             f"ranks 1 to {ADAPTER_MAX_RANK})")
    rows_of_one = lead[1] if x.dim() == 3 else T
    return lead, 0 if row_ptr is None else row_ptr.data_ptr(), \
        _NO_DROP if drop is None or drop.p == 0.0 else drop._for(K, x.device, rows_of_one * drop_width), \
        (K, T, lead[1] if x.dim() == 3 else 0, In, Out, R, code)


def adapter_linear_fwd(x, w, b, la, lb, y, u, *, scale: float = 1.0, row_ptr=None, drop: Optional[Drop] = None,
                       scratch: Optional[torch.Tensor] = None) -> None:
    """y = x w^T + b + u lb[k]^T with u = scale drop(x) la[k]^T: the adapters of K clients beside ONE shared projection.

    x [K,B,In] and y [K,B,Out] (client k's rows are x[k]), or x [T,In] and y [T,Out] with ``row_ptr`` [K+1] int32 on the GPU:
    client k has the rows ``row_ptr[k]`` .. ``row_ptr[k + 1] - 1`` (none, if they are equal; it never decreases); rows
    outside all of them get the shared projection alone. w [Out,In], b [Out] or None, la [K,R,In], lb [K,Out,R], all of the
    rows' type (fp32, bf16 or fp16); u [K,B,R] / [T,R] fp32 out, for the gradients (zero for rows without a client).
    ``drop``: dropout of the adapters' input, element ``row In + column`` of client k's own rows: the mask of
    :func:`dropout` over x[k]. ``y`` and ``u`` may not overlap the inputs. ``scratch``: a buffer from
    :func:`adapter_linear_scratch`, one call in flight; without it the call takes its own.

    Beside more than 64 rows fp32 operands are sums of bf16 terms: elements of x, w and lb above 3.389e38, and infinities (an infinite
    lb in 16 bits too), give results that are infinite or NaN where a plain product might still have a number or an infinity."""
    what = "adapter_linear_fwd"
    if la.dim() != 3 or w.dim() != 2:
        raise HipKernelError(f"{what}: expected w [Out, In] and la [K, R, In], got {tuple(w.shape)} and {tuple(la.shape)}")
    (Out, In), (K, R) = w.shape, la.shape[:2]
    lead, ptr, drop_fields, sizes = _adapter_sizes(what, x, K, R, In, Out, row_ptr, drop, In)
    dt, dev = x.dtype, x.device
    if b is not None and (b.dim() != 1 or Out > 1 and b.stride(0) != 1):
        raise HipKernelError(f"{what} b: expected a contiguous tensor")
    fields = _ADAPTER.pack(
        *_adapter_rows(what, x, "x", lead, In, dt, dev), _same(w, what, (Out, In), dt, dev, name="w").data_ptr(), w.stride(0),
        0 if b is None else _same(b, what, (Out,), dt, dev, name="b").data_ptr(),
        _same(la, what, (K, R, In), dt, dev, name="la").data_ptr(), la.stride(0),
        _same(lb, what, (K, Out, R), dt, dev, name="lb").data_ptr(), lb.stride(0), _adapter_low(what, u, "u", lead, R, dev),
        *_adapter_rows(what, y, "y", lead, Out, dt, dev, True), ptr, *drop_fields, 0, *sizes, scale)
    _adapter_apart(what, x, y)
    lib = _gpu(x)
    p, n, keep = _scratch(lib.p2pfl_adapter_linear_scratch(fields, 0), scratch, dev, what)
    _launch(lib.p2pfl_adapter_linear_fwd, what, dev, fields, p, n)


def _adapter_apart(what: str, rows, result) -> None:
    """Blocks read whole rows while others write theirs."""
    if result.data_ptr() == rows.data_ptr() and rows.numel():
        raise HipKernelError(f"{what}: the result cannot take the place of the rows")


def _adapter_low(what, t, name, lead, R, device) -> int:
    _same(t, what, (*lead, R), torch.float32, device, name=name)
    if not t.is_contiguous():
        raise HipKernelError(f"{what} {name}: expected a contiguous tensor")
    return t.data_ptr()


def adapter_linear_dgrad(dy, w, la, lb, dx, v, *, scale: float = 1.0, row_ptr=None, drop: Optional[Drop] = None,
                         scratch: Optional[torch.Tensor] = None) -> None:
    """dx = dy w + drop'(v la[k]) with v = scale dy lb[k], the data gradient of :func:`adapter_linear_fwd` (same shapes, same
    ``scale``, ``row_ptr`` and ``drop``). v [K,B,R] / [T,R] fp32 out, for :func:`adapter_linear_wgrad`. ``dx`` and ``v``
    may not overlap the inputs. ``scratch``: a buffer from :func:`adapter_linear_scratch`, one call in flight; without it the call
    takes its own."""
    what = "adapter_linear_dgrad"
    if la.dim() != 3 or w.dim() != 2:
        raise HipKernelError(f"{what}: expected w [Out, In] and la [K, R, In], got {tuple(w.shape)} and {tuple(la.shape)}")
    (Out, In), (K, R) = w.shape, la.shape[:2]
    lead, ptr, drop_fields, sizes = _adapter_sizes(what, dy, K, R, Out, In, row_ptr, drop, In)
    dt, dev = dy.dtype, dy.device
    fields = _ADAPTER.pack(
        *_adapter_rows(what, dy, "dy", lead, Out, dt, dev), _same(w, what, (Out, In), dt, dev, name="w").data_ptr(), w.stride(0), 0,
        _same(lb, what, (K, Out, R), dt, dev, name="lb").data_ptr(), lb.stride(0),
        _same(la, what, (K, R, In), dt, dev, name="la").data_ptr(), la.stride(0), _adapter_low(what, v, "v", lead, R, dev),
        *_adapter_rows(what, dx, "dx", lead, In, dt, dev, True), ptr, *drop_fields, 0, *sizes, scale)
    _adapter_apart(what, dy, dx)
    lib = _gpu(dy)
    p, n, keep = _scratch(lib.p2pfl_adapter_linear_scratch(fields, 1), scratch, dev, what)
    _launch(lib.p2pfl_adapter_linear_dgrad, what, dev, fields, p, n)


def adapter_linear_scratch(which: str, x, K: int, In: int, Out: int, R: int, row_ptr=None) -> Optional[torch.Tensor]:
    """Workspace of :func:`adapter_linear_fwd` ("fwd"), ``_dgrad`` ("dgrad") or ``_wgrad`` ("wgrad") for rows like ``x`` (its last
    dimension aside) of K clients, an In -> Out projection and rank R; None: none."""
    if which not in ("fwd", "dgrad", "wgrad"):
        raise HipKernelError(f"adapter_linear_scratch: unknown call {which!r}")
    a, b = (Out, In) if which == "dgrad" else (In, Out)
    _, ptr, drop_fields, sizes = _adapter_sizes("adapter_linear_scratch", x, K, R, a, b, row_ptr, None, In)
    need = 0
    for aligned in (0, 1):                   # (rows of any alignment: two plans)
        fields = _ADAPTER.pack(*(aligned,) * 14, ptr, *drop_fields, 0, *sizes, 1.0)
        need = max(need, load().p2pfl_adapter_linear_wgrad_scratch(fields) if which == "wgrad" else
                   load().p2pfl_adapter_linear_scratch(fields, int(which == "dgrad")))
    return torch.empty(need, dtype=torch.float32, device=x.device) if need else None


def adapter_linear_wgrad(dy, x, u, v, dla, dlb, *, row_ptr=None, drop: Optional[Drop] = None,
                         scratch: Optional[torch.Tensor] = None) -> None:
    """dla[k] = v^T drop(x) [K,R,In] and dlb[k] = dy^T u [K,Out,R] over client k's rows, fp32 (one of them may be None);
    ``u`` from :func:`adapter_linear_fwd` and ``v`` from :func:`adapter_linear_dgrad`. Clients without rows get zeros. The
    sums have a fixed order; u and v are not rounded, whatever the rows' type. ``scratch``: a buffer from
    :func:`adapter_linear_scratch`, one call in flight; without it the call takes its own."""
    what = "adapter_linear_wgrad"
    some = dla if dla is not None else dlb
    if some is None or some.dim() != 3 or x.dim() < 2 or dy.dim() < 2 or u.dim() < 2:
        raise HipKernelError(f"{what}: expected rows, u and v, and dla [K, R, In] and / or dlb [K, Out, R]")
    K, R, In, Out = some.shape[0], u.shape[-1], x.shape[-1], dy.shape[-1]
    lead, ptr, drop_fields, sizes = _adapter_sizes(what, x, K, R, In, Out, row_ptr, drop, In)
    dt, dev = x.dtype, x.device
    fields = _ADAPTER.pack(*_adapter_rows(what, x, "x", lead, In, dt, dev), 0, 0, 0, 0, 0, 0, 0,
                           _adapter_low(what, u, "u", lead, R, dev), *_adapter_rows(what, dy, "dy", lead, Out, dt, dev), ptr,
                           *drop_fields, 0, *sizes, 1.0)
    vp = _adapter_low(what, v, "v", lead, R, dev)
    ap = bp = None
    acs = bcs = 0
    if dla is not None:
        ap, acs = _same(dla, what, (K, R, In), torch.float32, dev, True, "dla").data_ptr(), dla.stride(0)
    if dlb is not None:
        bp, bcs = _same(dlb, what, (K, Out, R), torch.float32, dev, True, "dlb").data_ptr(), dlb.stride(0)
    lib = _gpu(x)
    p, n, keep = _scratch(lib.p2pfl_adapter_linear_wgrad_scratch(fields), scratch, dev, what)
    _launch(lib.p2pfl_adapter_linear_wgrad, what, dev, fields, vp, ap, acs, bp, bcs, p, n)
