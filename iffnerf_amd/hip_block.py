"""The feed-forward half of a transformer block with its gradients, on libiffnerf_hip: ``layer_norm``, ``gated_mlp``, ``dropout``.

What fine-tuning the image backbone runs per block -- ``x + dropout(gated_mlp(layer_norm(x)))`` -- as differentiable functions of GPU
tensors (the training loop of the reference, pose_estimation/train.py:97-119, back-propagates through the identification module and with
it through pose_estimation/backbone.py:12-14).  ``hip_vit.train_natively`` installs them on a backbone module.  fp32, bf16 and fp16;
arithmetic and sums are fp32, a result is rounded once; every gradient is the same bits on every run.  Calls run on the current stream of
the tensors' device, allocate through torch (so they can be captured into a hipGraph; take the gradients of a captured step with
``torch.autograd.grad``) and raise ``RuntimeError`` for what they do not serve, CPU tensors and tensors with a forward-mode tangent among
it.  First derivatives only.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check


# A small call is bound by the host: what a backward pass runs on autograd's own thread costs three times what it costs in a loop (torch's
# current_device there 2.5 us, the binding under it 0.3), so the backward passes look nothing up that the forward pass knew
# (forward + backward of 8 x 64 values: dropout 66 us, 72 with those lookups; norm with parameters 96, 106; torch's own product 41).
_TYPES = _lib.TYPES
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _run(name: str, x: torch.Tensor, *args) -> None:
    """Entry point ``name`` with ``args`` on the current stream of x's device."""
    i, fn = x.get_device(), getattr(_lib._lib or _lib.lib(), name)
    if i == _current_device():
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc:
        check(rc, name)


@functools.lru_cache(maxsize=1024)
def _bytes(name: str, *sizes) -> int:
    """What the size query ``name`` of the library answers (a function of the sizes alone)."""
    return int(getattr(_lib.lib(), name)(*sizes))


def _no_tangents(*tensors: Optional[torch.Tensor]) -> None:
    """Inside a forward-mode level: the kernels would drop a tangent."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("layer_norm, gated_mlp and dropout have no forward-mode derivative: a tensor with a tangent cannot be an argument")


def _first_derivative(backward):
    """``once_differentiable``, entered only where a second derivative could be asked for (autograd runs backward in grad mode then)."""
    guarded = once_differentiable(backward)

    def run(ctx, dy):
        if forward_ad._current_level >= 0:
            _no_tangents(dy)
        return guarded(ctx, dy) if torch.is_grad_enabled() else backward(ctx, dy)
    return run


def _serves(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor (got {type(t).__name__})")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on the GPU (got device {t.device}); libiffnerf_hip has no CPU path")
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{name} must be fp32, bf16 or fp16 (got {t.dtype})")


def _beside(t: torch.Tensor, x: torch.Tensor, name: str, shape, *types) -> torch.Tensor:
    """A parameter next to x: its device, one of ``types``, exactly ``shape``; contiguous."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor (got {type(t).__name__})")
    if t.device != x.device:
        raise RuntimeError(f"{name} is on {t.device}, the input on {x.device}")
    if t.dtype not in types:
        raise RuntimeError(f"{name} is {t.dtype}; with an input of {x.dtype} it must be {' or '.join(str(k) for k in types)}")
    if t.shape != shape:
        raise RuntimeError(f"{name} must have shape {tuple(shape)} (got {tuple(t.shape)})")
    return t.contiguous()


def _trains(*tensors: Optional[torch.Tensor]) -> bool:
    if forward_ad._current_level >= 0:
        _no_tangents(*tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _saved(t: torch.Tensor, shape, dtype: torch.dtype, device: int, name: str) -> torch.Tensor:
    """A saved tensor as the backward pass is handed it, any strides.  A hook on saved tensors (``save_on_cpu``, compression) may have put a
    copy in its place: its values are what was saved, its strides need not be, and another shape, type or device is not read."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device:
        raise RuntimeError(f"{name}: what was saved for the backward pass came back as {tuple(t.shape)} {t.dtype} on {t.device}; saved was "
                           f"{tuple(shape)} {dtype} on GPU {device}")
    return t


def _workspace(nbytes: int, x: torch.Tensor) -> torch.Tensor:
    return x.new_empty((max(nbytes, 16),), dtype=torch.uint8)


# ---------------------------------------------------------------------------------------------------- layer norm
def _rows(x: torch.Tensor):
    """x [..., D] as rows (i, j) at i s0 + j s1: (tensor, n0, n1, s0, s1).  A contiguous tensor, a slice of its second-last axis (the
    patch tokens behind a class token) and anything else with at most two row strides is read in place; the rest is copied."""
    D = x.shape[-1]
    if x.is_contiguous():
        return x, 1, x.numel() // D, 0, D
    if D == 1 or x.stride(-1) == 1:
        dims = []                                              # (size, stride), outermost first, adjacent axes merged
        for n, s in zip(x.shape[:-1], x.stride()[:-1]):
            if n == 1:
                continue
            if dims and dims[-1][1] == n * s:
                dims[-1] = (dims[-1][0] * n, s)
            else:
                dims.append((n, s))
        if len(dims) <= 2:
            (n0, s0), (n1, s1) = ([(1, 0)] * (2 - len(dims)) + dims) if x.numel() else ((0, 0), (0, 0))
            return x, n0, n1, s0, s1
    return x.contiguous(), 1, x.numel() // D, 0, D


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows = _rows(x)
        y, stats, par = _layer_norm(x, rows, weight, bias, eps, True)
        ctx.save_for_backward(rows[0], weight, stats)
        ctx.how = (rows[0].stride(), rows[1:], x.shape[-1], _TYPES[x.dtype], par)
        return y

    @staticmethod
    @_first_derivative
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        strides, rows, D, ty, par = ctx.how
        dev = dy.get_device()
        if _saved(x, dy.shape, dy.dtype, dev, "layer_norm").stride() != strides:
            x, *rows = _rows(x)
        n0, n1, s0, s1 = rows
        stats = _saved(stats, (n0 * n1, 2), torch.float32, dev, "layer_norm").contiguous()
        if weight is not None:
            weight = _saved(weight, (D,), par, dev, "layer_norm").contiguous()
        dy = dy.contiguous()
        dx = torch.empty_like(dy) if need_x else None
        dw = x.new_empty((D,), dtype=par) if need_w else None
        db = x.new_empty((D,), dtype=par) if need_b else None
        nbytes, ws = 0, None
        if need_w or need_b:
            nbytes = _bytes("iff_layer_norm_backward_workspace", n0 * n1, D)
            ws = _workspace(nbytes, x)
        _run("iff_layer_norm_backward", x, x.data_ptr(), ty, n0, n1, s0, s1, D, _ptr(weight), _TYPES[par], stats.data_ptr(), dy.data_ptr(),
             _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes)
        return dx, dw, db, None


def _layer_norm(x, rows, weight, bias, eps, keep):
    xr, n0, n1, s0, s1 = rows
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = x.new_empty((n0 * n1, 2), dtype=torch.float32) if keep else None
    par = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
    _run("iff_layer_norm_forward", x, xr.data_ptr(), _TYPES[x.dtype], n0, n1, s0, s1, x.shape[-1], _ptr(weight), _ptr(bias), _TYPES[par],
         eps, y.data_ptr(), _ptr(stats))
    return y, stats, par


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """Layer norm over the last axis of ``x`` [..., D] (any D >= 1): ``(x - mean) / sqrt(var + eps) * weight + bias``, in x's type and
    shape, contiguous.  ``weight`` / ``bias`` [D]: fp32 or x's type, both the same.  Differentiable in all three.  Rows are read in place
    where at most two strides describe them (``tokens[:, 1:]``); other layouts are copied first.  The default ``eps`` is the backbone's."""
    _serves(x, "layer_norm: x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"layer_norm: x must have a last axis of at least one value (got shape {tuple(x.shape)})")
    if not eps >= 0.0:
        raise RuntimeError(f"layer_norm: eps must not be negative (got {eps})")
    if weight is not None:
        weight = _beside(weight, x, "layer_norm: weight", x.shape[-1:], torch.float32, x.dtype)
    if bias is not None:
        bias = _beside(bias, x, "layer_norm: bias", x.shape[-1:], *((torch.float32, x.dtype) if weight is None else (weight.dtype,)))
    if _trains(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _layer_norm(x, _rows(x), weight, bias, float(eps), False)[0]


# ---------------------------------------------------------------------------------------------------- gated feed-forward
def _mlp_forward(x, w12, b12, w3, b3, act, keep):
    M, D = x.shape
    O, H = w3.shape
    ty = _TYPES[x.dtype]
    y = x.new_empty((M, O))
    kept_bytes = _bytes("iff_gated_mlp_kept_bytes", ty, M, D, H, O) if keep else 0
    kept = x.new_empty((kept_bytes,), dtype=torch.uint8) if keep else None
    nbytes = _bytes("iff_gated_mlp_forward_workspace", ty, M, D, H, O)
    ws = _workspace(nbytes, x)
    _run("iff_gated_mlp_forward", x, x.data_ptr(), ty, M, D, H, O, w12.data_ptr(), _ptr(b12), w3.data_ptr(), _ptr(b3), act, y.data_ptr(),
         _ptr(kept), kept_bytes, ws.data_ptr(), nbytes)
    return y, kept, (ty, M, D, H, O)


class _GatedMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w12, b12, w3, b3, act):
        y, kept, ctx.sizes = _mlp_forward(x, w12, b12, w3, b3, act, True)
        ctx.save_for_backward(x, w12, w3, kept)
        return y

    @staticmethod
    @_first_derivative
    def backward(ctx, dy):
        x, w12, w3, kept = ctx.saved_tensors
        sizes = ctx.sizes
        ty, M, D, H, O = sizes
        dt, dev = dy.dtype, dy.get_device()
        x = _saved(x, (M, D), dt, dev, "gated_mlp").contiguous()
        w12 = _saved(w12, (2 * H, D), dt, dev, "gated_mlp").contiguous()
        w3 = _saved(w3, (O, H), dt, dev, "gated_mlp").contiguous()
        kept = _saved(kept, (_bytes("iff_gated_mlp_kept_bytes", *sizes),), torch.uint8, dev, "gated_mlp").contiguous()
        dy, need = dy.contiguous(), ctx.needs_input_grad
        dx = x.new_empty((M, D)) if need[0] else None
        dw12 = x.new_empty((2 * H, D)) if need[1] else None
        db12 = x.new_empty((2 * H,)) if need[2] else None
        dw3 = x.new_empty((O, H)) if need[3] else None
        db3 = x.new_empty((O,)) if need[4] else None
        nbytes = _bytes("iff_gated_mlp_backward_workspace", *sizes)
        ws = _workspace(nbytes, x)
        _run("iff_gated_mlp_backward", x, x.data_ptr(), ty, M, D, H, O, w12.data_ptr(), w3.data_ptr(), kept.data_ptr(),
             dy.data_ptr(), _ptr(dx), _ptr(dw12), _ptr(db12), _ptr(dw3), _ptr(db3), ws.data_ptr(), nbytes)
        return dx, dw12, db12, dw3, db3, None


def gated_mlp(x: torch.Tensor, w12: torch.Tensor, b12: Optional[torch.Tensor], w3: torch.Tensor, b3: Optional[torch.Tensor],
              activation: str = "silu") -> torch.Tensor:
    """Gated feed-forward block: ``[g | u] = x @ w12.T + b12``, ``(act(g) * u) @ w3.T + b3``.  ``x`` [..., D], ``w12`` [2 H, D] (gate rows
    first -- the ``w12`` / ``w3`` layout of DINOv2's gated feed-forward), ``w3`` [O, H], biases [2 H] / [O] or None; one type and device.
    ``activation``: "silu" or "gelu" (exact).  Differentiable in all five.  The hidden activation is rounded to the type once (up to 8
    rows it has twice the type's precision); what the backward pass keeps next to it is fp32.  fp32 operands are multiplied as three bf16
    pieces each, in fp32's accuracy."""
    _serves(x, "gated_mlp: x")
    if activation not in _lib.ACTIVATIONS:
        raise RuntimeError(f"gated_mlp: activation must be one of {sorted(_lib.ACTIVATIONS)} (got {activation!r})")
    if x.dim() < 1 or not isinstance(w3, torch.Tensor) or w3.dim() != 2 or x.shape[-1] < 1 or min(w3.shape) < 1:
        raise RuntimeError("gated_mlp: x [..., D], w12 [2 H, D], w3 [O, H] with no empty width expected")
    D, (O, H) = x.shape[-1], w3.shape
    w12 = _beside(w12, x, "gated_mlp: w12", (2 * H, D), x.dtype)
    w3 = _beside(w3, x, "gated_mlp: w3", (O, H), x.dtype)
    b12 = None if b12 is None else _beside(b12, x, "gated_mlp: b12", (2 * H,), x.dtype)
    b3 = None if b3 is None else _beside(b3, x, "gated_mlp: b3", (O,), x.dtype)
    x2 = x.reshape(-1, D).contiguous()
    act = _lib.ACTIVATIONS[activation]
    if _trains(x2, w12, b12, w3, b3):
        y = _GatedMlp.apply(x2, w12, b12, w3, b3, act)
    else:
        y = _mlp_forward(x2, w12, b12, w3, b3, act, False)[0]
    return y.reshape(*x.shape[:-1], O)


# ---------------------------------------------------------------------------------------------------- dropout
def _dropout(x, residual, threshold, seed, seed_dev, offset):
    y = torch.empty_like(x)
    _run("iff_dropout", x, x.data_ptr(), _TYPES[x.dtype], x.numel(), _ptr(residual), threshold, seed, _ptr(seed_dev), offset, y.data_ptr())
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed, seed_dev, offset):
        ctx.save_for_backward(seed_dev)           # (a seed tensor that changes before the backward pass is noticed by its version)
        ctx.how = (threshold, seed, offset)
        ctx.seed_shape = None if seed_dev is None else seed_dev.shape
        return _dropout(x, residual, threshold, seed, seed_dev, offset)

    @staticmethod
    @_first_derivative
    def backward(ctx, dy):
        threshold, seed, offset = ctx.how
        need, (seed_dev,) = ctx.needs_input_grad, ctx.saved_tensors
        if seed_dev is not None:
            seed_dev = _saved(seed_dev, ctx.seed_shape, torch.int64, dy.get_device(), "dropout")
        dx = _dropout(dy.contiguous(), None, threshold, seed, seed_dev, offset) if need[0] else None
        return dx, dy if need[1] else None, None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], offset: int = 0, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + x * keep / (1 - p)`` without a stored mask: ``keep`` is a function of (seed, offset, index) -- 16 bits of Philox 4x32-10
    per value, so ``p`` is taken to the nearest 2^-16 -- and the backward pass computes it again.  ``seed``: 0 <= int < 2^64, or an int64
    tensor of one value on x's device, read when the kernel runs (a captured step draws a new one per replay by refilling it);
    ``offset``: 0 <= int < 2^64, another stream of the same seed.  Two calls with equal (seed, offset) drop the same positions.  A dropped
    value never reaches the result, not even as a NaN.  ``residual``: x's shape, type and device."""
    _serves(x, "dropout: x")
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"dropout: p must be between 0 and 1 (got {p})")
    seed_dev = None
    if isinstance(seed, torch.Tensor):
        if seed.device != x.device or seed.dtype != torch.int64 or seed.numel() != 1:
            raise RuntimeError(f"dropout: a seed tensor must be one int64 on {x.device} (got {tuple(seed.shape)} {seed.dtype} on {seed.device})")
        seed_dev, seed = seed.contiguous(), 0
    for name, v in (("seed", seed), ("offset", offset)):
        if not isinstance(v, int) or not 0 <= v < 2 ** 64:
            raise RuntimeError(f"dropout: {name} must be an integer of 0 .. 2^64 - 1 (got {v!r})")
    if residual is not None:
        residual = _beside(residual, x, "dropout: residual", x.shape, x.dtype)
    threshold = int(math.floor(p * 65536 + 0.5))
    x = x.contiguous()
    if _trains(x, residual):
        return _Dropout.apply(x, residual, threshold, seed, seed_dev, offset)
    return _dropout(x, residual, threshold, seed, seed_dev, offset)
