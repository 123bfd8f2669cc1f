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
gradients are held in float32 and added in a fixed order.  On the CPU the same formulas run as plain
torch operations.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from gpubridge_b200.ops import _lib

launches = 0
MAX_WIDTH = 8192
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KINDS = ("rms", "layer")


class Joined(NamedTuple):
    stream: torch.Tensor
    normed: torch.Tensor | None


def _declare(lib):
    if getattr(lib, "_residual_norm_declared", False):
        return lib
    vp, i, f, lg = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong
    lib.gb_residual_norm_fwd.argtypes = [i, i, i, i, vp, lg, vp, lg, vp, vp, vp, vp, vp, vp, vp, i, vp, i,
                                         lg, lg, i, i, f, f, vp]
    lib.gb_residual_norm_workers.argtypes = [lg, i, i, ctypes.POINTER(i), ctypes.POINTER(i)]
    lib.gb_residual_norm_workers.restype = None
    lib.gb_residual_norm_bwd.argtypes = [i, i, i, i, vp, vp, vp, vp, lg, vp, vp, vp, vp, vp, i, vp, i, vp, vp,
                                         vp, vp, vp, vp, vp, vp, vp, lg, lg, i, i, f, vp]
    lib._residual_norm_declared = True
    return lib


def _rows(t: torch.Tensor, d: int) -> torch.Tensor:
    """``t`` as [rows, d] whose rows are dense (a view where the strides allow it)."""
    t = t.reshape(-1, d)
    return t if d == 1 or t.stride(1) == 1 else t.contiguous()


def _aligned(d: int, *tensors: torch.Tensor | None) -> bool:
    """Whether every row begins on a boundary of eight values, so that vectors may be moved."""
    for t in tensors:
        if t is None:
            continue
        step = 8 * t.element_size()
        if t.data_ptr() % step or (t.shape[0] > 1 and t.stride(0) % 8):
            return False
    return d % 8 == 0


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, update, weight, bias, post_weight, post_bias, gate, scale, eps, layer, out_dtype):
        global launches
        ctx.set_materialize_grads(False)
        d = residual.shape[-1]
        r2, u2 = _rows(residual, d), _rows(update, d)
        rows = r2.shape[0]
        device = residual.device
        stream = torch.empty(residual.shape, dtype=residual.dtype, device=device)
        normed = None if weight is None else torch.empty(residual.shape, dtype=out_dtype, device=device)
        groups = 1 if gate is None or gate.dim() == 1 else gate.shape[0]
        needs = any(ctx.needs_input_grad)
        stats = torch.empty((rows, 4), dtype=torch.float32, device=device) if needs else None
        param = next((p for p in (weight, post_weight) if p is not None), None)
        code = 0 if param is None else _CODES[param.dtype]
        gate_code = 0 if gate is None else _CODES[gate.dtype]
        types = (_CODES[residual.dtype], _CODES[update.dtype], _CODES[out_dtype])
        if rows:
            vec = 8 if _aligned(d, r2, u2) else 1
            with torch.cuda.device(device):
                _lib.check(_declare(_lib.lib()).gb_residual_norm_fwd(
                    *types, vec, r2.data_ptr(), r2.stride(0), u2.data_ptr(), u2.stride(0), stream.data_ptr(),
                    _ptr(normed), _ptr(stats), _ptr(weight), _ptr(bias), _ptr(post_weight), _ptr(post_bias),
                    code, _ptr(gate), gate_code, rows, rows // groups, d, layer, scale, eps,
                    _lib.stream_ptr(device)), "gb_residual_norm_fwd")
            launches += 1
        ctx.save_for_backward(update, stream, stats, weight, bias, post_weight, post_bias, gate)
        ctx.rest = (types, code, gate_code, groups, scale, layer)
        if normed is None:
            return stream
        return stream, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, d_stream, d_normed=None):
        global launches
        update, stream, stats, weight, bias, post_weight, post_bias, gate = ctx.saved_tensors
        types, code, gate_code, groups, scale, layer = ctx.rest
        nothing = (None,) * 11
        if d_stream is None and d_normed is None:
            return nothing
        d = stream.shape[-1]
        u2 = _rows(update, d)
        rows, device = u2.shape[0], stream.device
        given = [None if g is None else g.contiguous() for g in (d_stream, d_normed)]
        if d_normed is None:                       # the following norm took no part
            weight = bias = None
        d_residual = torch.empty(stream.shape, dtype=stream.dtype, device=device) if ctx.needs_input_grad[0] else None
        d_update = torch.empty(update.shape, dtype=update.dtype, device=device)
        outs = [None if p is None else torch.empty_like(p) for p in (weight, bias, post_weight, post_bias)]
        d_gate = None if gate is None else torch.empty_like(gate)
        if rows:
            vec = 8 if _aligned(d, u2, *(None if g is None else g.view(-1, d) for g in given)) else 1
            lib = _declare(_lib.lib())
            blocks, owners = ctypes.c_int(), ctypes.c_int()
            lib.gb_residual_norm_workers(rows, d, vec, blocks, owners)
            sums = [t for t in outs if t is not None]
            part = torch.empty(blocks.value * len(sums) * d, dtype=torch.float32, device=device)
            gate_part = (None if gate is None else
                         torch.empty((owners.value + groups - 1) * d, dtype=torch.float32, device=device))
            slots = [t.data_ptr() for t in sums] + [None] * (4 - len(sums))
            with torch.cuda.device(device):
                _lib.check(lib.gb_residual_norm_bwd(
                    *types, vec, _ptr(given[0]), _ptr(given[1]), stream.data_ptr(), u2.data_ptr(), u2.stride(0),
                    stats.data_ptr(), _ptr(weight), _ptr(bias), _ptr(post_weight), _ptr(post_bias), code,
                    _ptr(gate), gate_code, _ptr(d_residual), d_update.data_ptr(), _ptr(part), _ptr(gate_part),
                    *slots, _ptr(d_gate), rows, rows // groups, d, layer, scale,
                    _lib.stream_ptr(device)), "gb_residual_norm_bwd")
            launches += 2
        else:
            for t in (*outs, d_gate):
                if t is not None:
                    t.zero_()
        return (d_residual, d_update, *outs, d_gate, None, None, None, None)


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
    the others; an update of another type is converted to ``normed``'s.
    """
    if out_dtype is None:
        out_dtype = residual.dtype
        kind_of = residual.device.type
        if residual.dtype == torch.float32 and torch.is_autocast_enabled(kind_of):
            out_dtype = torch.get_autocast_dtype(kind_of)
    _check(residual, update, weight, bias, post_weight, post_bias, gate, kind, out_dtype)
    scale, eps, layer = float(scale), float(eps), int(kind == "layer")
    if residual.device.type != "cuda":
        return _plain(residual, update, weight, bias, post_weight, post_bias, gate, scale, eps, layer, out_dtype)
    d = residual.shape[-1]
    if d > MAX_WIDTH:
        raise ValueError(f"rows of up to {MAX_WIDTH} values, got {d}")
    for name, dtype in (("residual", residual.dtype), ("out_dtype", out_dtype)):
        if dtype not in _CODES:
            raise ValueError(f"{name} is float32, bfloat16 or float16 on the GPU, got {dtype}")
    if residual.dtype != torch.float32 and out_dtype != residual.dtype:
        raise ValueError(f"a stream of {residual.dtype} has its norm in the same type, got {out_dtype}")
    if update.dtype != out_dtype:
        update = update.to(out_dtype)
    first = next((p for p in (weight, post_weight) if p is not None), None)
    params = []
    for p in (weight, bias, post_weight, post_bias):
        if p is not None:
            if p.dtype not in _CODES:
                raise ValueError(f"parameters are float32, bfloat16 or float16 on the GPU, got {p.dtype}")
            p = p.to(first.dtype).contiguous()
        params.append(p)
    if gate is not None:
        if gate.dtype not in _CODES:
            raise ValueError(f"gate is float32, bfloat16 or float16 on the GPU, got {gate.dtype}")
        gate = gate.contiguous()
    got = _ResidualNorm.apply(residual, update, *params, gate, scale, eps, layer, out_dtype)
    return Joined(got, None) if weight is None else Joined(*got)
