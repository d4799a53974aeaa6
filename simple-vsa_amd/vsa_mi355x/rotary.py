"""Rotary positions of video tokens on MI355X: a latent grid's table and the
rotation of q and k by it, before the attention.

A pair of channels at angle a becomes (x1 cos a - x2 sin a, x2 cos a + x1 sin a);
the angle is the token's position along an axis of the grid times the pair's
frequency.  Both are HIP kernels (``vsa_rotary_table``, ``vsa_rotary``); the
rotation is differentiable to any order (its gradient is the opposite rotation).
Nothing here runs on the CPU: a CPU tensor or a missing kernel library raises.
"""

from __future__ import annotations

import functools
import math
import operator
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from .launch import on_device

ROTARY_METHODS = ("linear", "ntk", "yarn")
MAX_ROTARY_CHANNELS = 256
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


# ---------------------------------------------------------------------------
# Table
# ---------------------------------------------------------------------------

def _three(x, name, kind=float) -> Tuple:
    x = tuple(x) if isinstance(x, (tuple, list)) else (x,) * 3
    if len(x) != 3:
        raise ValueError(f"{name} must have three entries (T, H, W)")
    return tuple(kind(v) for v in x)


@functools.lru_cache(maxsize=64)
def _axes(shape, channels, theta, start, factor, method, original):
    """(the axes' structs, tokens, pairs) of checked arguments."""
    if min(shape) <= 0:
        raise ValueError("dit_seq_shape must be positive")
    if math.prod(shape) >= 1 << 31:
        raise ValueError("a rotary table holds fewer than 2^31 tokens")
    if min(channels) < 0 or any(c % 2 for c in channels) or not \
            0 < sum(channels) <= MAX_ROTARY_CHANNELS:
        raise ValueError("axis_channels must be even, and together in "
                         f"[2, {MAX_ROTARY_CHANNELS}]")
    if not (theta > 0 and math.isfinite(theta)):
        raise ValueError("theta must be positive and finite")
    if not all(f > 0 and math.isfinite(f) for f in factor):
        raise ValueError("factor must be positive and finite")
    if not all(abs(x) <= 2.0 ** 52 for x in start):
        raise ValueError("start must lie within 2^52")
    if method not in ROTARY_METHODS:
        raise ValueError(f"method must be one of {ROTARY_METHODS}")
    if method == "yarn":
        if original is None:
            raise ValueError("the yarn method needs original_shape, the trained (T, H, W)")
        if not all(x > 0 and math.isfinite(x) for x in original):
            raise ValueError("original_shape must be positive")
    else:
        original = (0.0,) * 3
    kind = ROTARY_METHODS.index(method)
    axes = _lib.ROTARY_AXES.pack(*(x for i in range(3) for x in (
        shape[i], channels[i], kind, 0, start[i], theta, factor[i], original[i])))
    return axes, math.prod(shape), sum(channels) // 2


def build_rotary_table(dit_seq_shape: Tuple[int, int, int], axis_channels: Tuple[int, int, int],
                       theta: float = 10000.0, *, start=(0, 0, 0),
                       factor: Union[float, Tuple[float, float, float]] = 1.0,
                       method: str = "linear", original_shape=None,
                       device: torch.device | str = "cuda") -> Tuple[Tensor, Tensor]:
    """``(cos, sin)``, fp32 ``[T*H*W, sum(axis_channels) / 2]``, of the raster-order
    tokens of a ``(T, H, W)`` grid: pair i of an axis with d channels turns by
    ``(start + index) * theta ** (-2 i / d)``.  A plain sequence is ``(S, 1, 1)``
    with ``(channels, 0, 0)``.

    ``method`` scales the axes for grids longer than a model was trained on, by
    ``factor`` (one number or one an axis): "linear" divides the positions,
    "ntk" takes ``theta * factor ** (d / (d - 2))``, "yarn" keeps the frequencies
    that turn 32 times or more in ``original_shape`` (the trained sizes), divides
    those that turn once or less, a ramp between, and multiplies cos and sin by
    ``0.1 ln(factor) + 1``.  Angles are made in 64 bits."""
    axes, tokens, pairs = _axes(
        _three(dit_seq_shape, "dit_seq_shape", operator.index),
        _three(axis_channels, "axis_channels", operator.index),
        float(theta), _three(start, "start"), _three(factor, "factor"), method,
        None if original_shape is None else _three(original_shape, "original_shape"))
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("the MI355X implementation requires a GPU device")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    cos = torch.empty((tokens, pairs), dtype=torch.float32, device=device)
    sin = torch.empty_like(cos)
    with on_device(device):
        _lib.call("vsa_rotary_table", axes, cos.data_ptr(), sin.data_ptr(),
                  torch._C._cuda_getCurrentRawStream(device.index))
    return cos, sin


# ---------------------------------------------------------------------------
# Rotation
# ---------------------------------------------------------------------------

def token_order(x: Tensor) -> bool:
    """True for a [B, H, S, D] tensor whose heads lie closer together than its
    tokens (a per-head view of token-major memory)."""
    return x.shape[1] > 1 and x.shape[2] > 1 and x.stride(1) < x.stride(2)


def empty_in_order(x: Tensor) -> Tensor:
    """An uninitialised tensor of x's shape, dense, in x's order of heads and tokens."""
    if x.is_contiguous():
        return torch.empty_like(x)
    b, h, s, d = x.shape
    if token_order(x):
        return torch.empty((b, s, h, d), dtype=x.dtype, device=x.device).transpose(1, 2)
    return torch.empty((b, h, s, d), dtype=x.dtype, device=x.device)


def _strides(shape, stride) -> Tuple[int, int, int]:
    """Strides of batch, head and token for the C ABI; 0 for a dimension of one."""
    (b, h, s, _), (sb, sh, ss, _) = shape, stride
    return (sb if b > 1 else 0, sh if h > 1 else 0, ss if s > 1 else 0)


@functools.lru_cache(maxsize=256)
def _rest_of(q, qs, qo, k, ks, ko, table, positions, wide, interleaved, inverse, dtype) -> bytes:
    """The struct behind its pointers, from shapes and strides alone."""
    b, h, s, d = q
    rows, pairs = table
    return _lib.ROTARY_OP.pack(
        0, 0, 0, 0, 0, 0, 0, *_strides(q, qs), *_strides(k or q, ks), *_strides(q, qo),
        *_strides(k or q, ko), s if positions == 2 else 0, b, s, rows, h, k[1] if k else 0, d,
        2 * pairs, interleaved, inverse, wide, dtype)[_lib.ROTARY_POINTERS.size:]


def _rotate(q, k, cos, sin, positions, interleaved, inverse):
    """One launch: (q turned, k turned); k may be None."""
    q_out = empty_in_order(q)
    if q.stride(3) != 1:
        q = q.contiguous()
    k_out = None
    kk, ko = q, q_out
    if k is not None:
        k_out = ko = empty_in_order(k)
        kk = k if k.stride(3) == 1 else k.contiguous()
    rest = _rest_of(q.shape, q.stride(), q_out.stride(), None if k is None else kk.shape, kk.stride(),
                    ko.stride(), cos.shape, 0 if positions is None else positions.dim(),
                    positions is not None and positions.dtype is torch.int64, interleaved, inverse,
                    _lib.DTYPE_CODES[q.dtype])
    pointers = _lib.ROTARY_POINTERS.pack(
        q.data_ptr(), kk.data_ptr(), q_out.data_ptr(), ko.data_ptr(), cos.data_ptr(),
        sin.data_ptr(), 0 if positions is None else positions.data_ptr())
    dev = q.device
    with on_device(dev):
        _lib.call("vsa_rotary", pointers + rest, torch._C._cuda_getCurrentRawStream(dev.index))
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """Its gradient is itself, turned the other way."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(cos, sin, positions)
        ctx.options = interleaved, inverse
        return _rotate(q, k, cos, sin, positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        cos, sin, positions = ctx.saved_tensors
        interleaved, inverse = ctx.options
        if not ctx.needs_input_grad[0]:
            gq = None
        if not ctx.needs_input_grad[1]:
            gk = None
        # through autograd again only where a second derivative may be wanted
        turn = _Rotary.apply if torch.is_grad_enabled() else _rotate
        if gq is None:
            if gk is not None:
                gk = turn(gk, None, cos, sin, positions, interleaved, not inverse)[0]
        else:
            gq, gk = turn(gq, gk, cos, sin, positions, interleaved, not inverse)
        return gq, gk, None, None, None, None, None


def _check_rotary(q, k, cos, sin, positions) -> None:
    if q.ndim != 4 or (k is not None and k.ndim != 4):
        raise ValueError("q and k must have shape [batch, heads, seq_len, dim]")
    b, _, s, d = q.shape
    if k is not None:
        if k.shape[0] != b or k.shape[2] != s or k.shape[3] != d:
            raise ValueError("q and k must share batch, sequence length and head dimension")
        if k.dtype != q.dtype:
            raise ValueError("q and k must have the same dtype")
    if q.dtype not in _DTYPES:
        raise ValueError("the MI355X kernels support float16, bfloat16 and float32")
    if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or \
            sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32 tensors of one shape [positions, channels / 2]")
    if not 2 <= 2 * cos.shape[1] <= d:
        raise ValueError(f"the table turns {2 * cos.shape[1]} channels of a head of {d}")
    if d > 256:
        raise ValueError("the MI355X kernels support head_dim <= 256")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("cos and sin get no gradient: detach them")
    if positions is None:
        if cos.shape[0] < s:
            raise ValueError(f"the table has {cos.shape[0]} positions for {s} tokens")
    else:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be int32 or int64")
        if tuple(positions.shape) not in ((s,), (b, s)):
            raise ValueError("positions must have shape [seq_len] or [batch, seq_len]")
        if cos.shape[0] == 0:
            raise ValueError("the table has no positions")
    if not q.is_cuda:
        raise ValueError("the MI355X implementation requires GPU tensors")
    dev = q.device
    if not (cos.device == dev and sin.device == dev and (k is None or k.device == dev)
            and (positions is None or positions.device == dev)):
        raise ValueError("q, k, the table and the positions must be on the same GPU device")


def mi355x_rotary(q: Tensor, k: Optional[Tensor], cos: Tensor, sin: Tensor,
                  positions: Optional[Tensor] = None, *, interleaved: bool = False,
                  inverse: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """``(q, k)`` turned by their positions: ``[batch, heads, seq_len, dim]`` (their
    head counts may differ; ``k`` may be None), the first ``2 * cos.shape[1]``
    channels of each head, in pairs ``(i, i + n/2)`` or, with ``interleaved``,
    ``(2i, 2i + 1)``; the other channels are copied.  ``inverse`` turns back.

    Token s takes row s of the table ``cos``, ``sin`` (``build_rotary_table``), or
    row ``positions[s]`` / ``positions[b, s]``; a negative position copies the
    token (a padding slot of ``slot_rows``), one past the table gives NaN.

    Per-head views of token-major memory and slices of a packed projection are
    read in place; the results are dense, in the order of heads and tokens of
    the input.  Differentiable in q and k to any order."""
    _check_rotary(q, k, cos, sin, positions)
    cos, sin = cos.contiguous(), sin.contiguous()
    if positions is not None:
        positions = positions.contiguous()
    interleaved, inverse = bool(interleaved), bool(inverse)
    if k is not None and k.shape[1] == 0:
        return mi355x_rotary(q, None, cos, sin, positions, interleaved=interleaved,
                             inverse=inverse)[0], k * 1
    if q.numel() == 0:
        if k is not None and k.numel():
            return q * 1, mi355x_rotary(k, None, cos, sin, positions, interleaved=interleaved,
                                        inverse=inverse)[0]
        return q * 1, None if k is None else k * 1
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, cos, sin, positions, interleaved, inverse)
    return _rotate(q, k, cos, sin, positions, interleaved, inverse)
