"""The join of a block with the residual stream and the norms on either side of it, as one kernel
forward and one backward (``csrc/gb_residual_norm.cu``):

    v      = norm(update) * post_weight + post_bias      # or update itself
    stream = residual + scale * gate * v
    normed = norm(stream) * weight + bias                # or None

``kind="rms"`` divides by the root mean square, ``kind="layer"`` centres first.  ``normed`` is the
norm of the stream as it is returned (rounded to its type).  ``models/llama.py`` and
``models/gpt2.py`` join their blocks with it, with residual scales, gates and sandwich norms where
the configuration asks for them.

On the GPU: streams of float32, bfloat16 or float16 up to 8192 wide; statistics, sums and parameter
gradients are held in float32 and added in a fixed order; the autograd node is C++
(``csrc_torch/gb_ops.cpp``).  On the CPU the same formulas run as plain torch operations.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from gpubridge_b200.ops import _build_ops

MAX_WIDTH = 8192
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_KINDS = ("rms", "layer")


class Joined(NamedTuple):
    stream: torch.Tensor
    normed: torch.Tensor | None


def _norm(x, weight, bias, layer, eps):
    centred = x - x.mean(-1, keepdim=True) if layer else x
    y = centred * (centred.square().mean(-1, keepdim=True) + eps).rsqrt() * weight
    return y if bias is None else y + bias


def _plain(residual, update, weight, bias, post_weight, post_bias, gate, scale, eps, layer, out_dtype):
    """The formulas in torch operations (CPU runs); differentiable as they stand."""
    wide = torch.float64 if residual.dtype == torch.float64 else torch.float32

    def up(t):
        return None if t is None else t.to(wide)

    v = up(update)
    if post_weight is not None:
        v = _norm(v, up(post_weight), up(post_bias), layer, eps)
    if gate is not None:
        v = v * up(gate)
    stream = (up(residual) + scale * v).to(residual.dtype)
    if weight is None:
        return Joined(stream, None)
    return Joined(stream, _norm(up(stream), up(weight), up(bias), layer, eps).to(out_dtype))


def _check(residual, update, weight, bias, post_weight, post_bias, gate, kind, out_dtype) -> None:
    if kind not in _KINDS:
        raise ValueError(f"kind must be rms or layer, got {kind!r}")
    if residual.dim() < 1 or residual.shape[-1] == 0:
        raise ValueError(f"residual needs a last dimension to norm over, got shape {tuple(residual.shape)}")
    if update.shape != residual.shape:
        raise ValueError(f"update has shape {tuple(update.shape)}, residual {tuple(residual.shape)}")
    d = residual.shape[-1]
    for name, p in (("weight", weight), ("bias", bias), ("post_weight", post_weight), ("post_bias", post_bias)):
        if p is not None and p.shape != (d,):
            raise ValueError(f"{name} has shape {tuple(p.shape)}, the last dimension is {d}")
    if bias is not None and weight is None or post_bias is not None and post_weight is None:
        raise ValueError("a bias needs the weight of its norm")
    if gate is not None:
        each = (residual.shape[0], *(1,) * (residual.dim() - 2), d)
        if gate.shape != (d,) and (residual.dim() < 2 or gate.shape != each):
            raise ValueError(f"gate is [{d}] or {list(each)} (a gate for each sequence), got {list(gate.shape)}")
    for name, p in (("update", update), ("weight", weight), ("bias", bias), ("post_weight", post_weight),
                    ("post_bias", post_bias), ("gate", gate)):
        if p is not None and p.device != residual.device:
            raise ValueError(f"{name} is on {p.device}, residual on {residual.device}")
    if not out_dtype.is_floating_point:
        raise ValueError(f"out_dtype must be a floating type, got {out_dtype}")
    if residual.device.type != "cuda":
        return
    if d > MAX_WIDTH:
        raise ValueError(f"rows of up to {MAX_WIDTH} values on the GPU, got {d}")
    for name, dtype in (("residual", residual.dtype), ("out_dtype", out_dtype),
                        *((n, p.dtype) for n, p in (("weight", weight), ("bias", bias), ("post_weight", post_weight),
                                                    ("post_bias", post_bias), ("gate", gate)) if p is not None)):
        if dtype not in _FLOATS:
            raise ValueError(f"{name} is float32, bfloat16 or float16 on the GPU, got {dtype}")
    if residual.dtype != torch.float32 and out_dtype != residual.dtype:
        raise ValueError(f"a stream of {residual.dtype} has its norm in the same type, got {out_dtype}")
    raise ValueError("the operands are ordinary strided tensors: no sparse ones and no subclass such as DTensor")


def residual_norm(residual: torch.Tensor, update: torch.Tensor, weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, *, post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  scale: float = 1.0, eps: float = 1e-5, kind: str = "rms",
                  out_dtype: torch.dtype | None = None) -> Joined:
    """``(stream, normed)`` as in the module docstring; ``normed`` is None without ``weight``.

    Args:
        residual, update: same shape ``[..., d]``; the stream has ``residual``'s type.
        weight, bias: of the norm that follows; bias also with ``kind="rms"``.
        post_weight, post_bias: of a norm of the update before it joins.
        gate: a factor for each channel, ``[d]``, or for each channel of each entry of the first
            dimension, ``[batch, 1, ..., d]``.
        scale: a number that multiplies the update.
        out_dtype: type of ``normed``: the autocast type for a float32 stream under autocast (what
            the next Linear would cast to), else ``residual``'s.

    Differentiable in every tensor, once.  Types on the GPU: stream, update and ``normed`` are all
    float32, all bfloat16 or all float16, or a float32 stream with update and ``normed`` in one of
    the others.  A float32 update of a float32 stream keeps its precision, whatever ``normed``'s type;
    any other update is converted to ``normed``'s.
    """
    if residual.is_cuda:
        got = _build_ops.load().residual_norm(residual, update, weight, bias, post_weight, post_bias, gate, scale, eps,
                                              kind, out_dtype)
        if got is not None:
            return Joined(*got)
    if out_dtype is None:
        out_dtype = residual.dtype
        if residual.dtype == torch.float32 and torch.is_autocast_enabled(residual.device.type):
            out_dtype = torch.get_autocast_dtype(residual.device.type)
    _check(residual, update, weight, bias, post_weight, post_bias, gate, kind, out_dtype)
    return _plain(residual, update, weight, bias, post_weight, post_bias, gate, float(scale), float(eps),
                  kind == "layer", out_dtype)
