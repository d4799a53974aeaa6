"""Cross attention of video tokens to an encoder's states on MI355X: queries of
one length, keys and values of another, each sample with its own valid keys.

    out = softmax(sm_scale * q k^T over the sample's valid keys) v

The forward and the backward are one call each into the C ABI
(``vsa_cross_fwd`` / ``vsa_cross_bwd``), on torch's current stream, with a
workspace from torch's allocator.  Nothing here runs on the CPU: a CPU tensor or
a missing kernel library raises.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .launch import _ptr, _workspace, on_device
from .mi355x import KERNEL_DTYPES, _i32
from .rotary import empty_in_order, token_order

MAX_HEAD_DIM = 256
MAX_TOKENS = (1 << 31) - 256
MAX_SCALE = 2.0 ** 127   # times log2(e) it stays finite in fp32


def _far(stride: int, element_size: int) -> bool:
    """Whether a tile's rows lie out of reach of a 32-bit offset."""
    return stride > (1 << 30) // (64 * element_size)


def _rows16(x: Tensor) -> Tensor:
    """x itself where the kernels read its rows in place (channels next to each
    other, every row 16-byte aligned, a tile's rows within reach), else a dense
    copy in x's order of heads and tokens."""
    if x.is_contiguous():
        return x if x.data_ptr() % 16 == 0 else x.clone()
    es = x.element_size()
    if x.stride(3) == 1 and x.data_ptr() % 16 == 0:
        b, h, s = _strides(x.shape, x.stride())
        if (b | h | s) * es % 16 == 0 and x.shape[3] <= s and not _far(s, es):
            return x
    if token_order(x) and not _far(x.shape[1] * x.shape[3], es):
        return x.transpose(1, 2).clone(memory_format=torch.contiguous_format).transpose(1, 2)
    return x.clone(memory_format=torch.contiguous_format)


def _strides(shape, stride):
    """Strides of batch, head and token for the C ABI: 0 for a dimension of one, those
    of a row where there is one token."""
    (b, h, s, d), (sb, sh, ss, _) = shape, stride
    return sb if b > 1 else 0, sh if h > 1 else 0, ss if s > 1 else d


def _three(x: Tensor) -> bytes:
    return _lib.STRIDES.pack(*_strides(x.shape, x.stride()))


def _dense(shape, stride) -> bytes:
    """The strides of ``empty_in_order``'s result."""
    b, h, s, d = shape
    if h > 1 and s > 1 and stride[1] < stride[2]:
        return _lib.STRIDES.pack(*_strides(shape, (s * h * d, d, h * d, 1)))
    return _lib.STRIDES.pack(*_strides(shape, (h * s * d, s * d, d, 1)))


class _Plan(NamedTuple):
    """What a call takes from its sizes alone: the struct behind its pointers, the
    strides of the results, bytes of scratch."""
    rest: bytes
    q: bytes
    k: bytes
    v: bytes
    forward: int
    backward: int


@functools.lru_cache(maxsize=256)
def _plan_of(q, qs, k, ks, vs, lens, mask, dtype, scale, device) -> _Plan:
    """``device`` is the current one: the splits follow its number of CUs."""
    (b, h, sq, d), (_, hk, skv, _) = q, k
    rest = _lib.CROSS.pack(0, 0, 0, 0, 0, *_strides(q, qs), *_strides(k, ks), *_strides(k, vs), mask or 0, sq,
                           skv, b, h, hk, d, dtype, scale)[_lib.CROSS_POINTERS.size:]
    n = (ctypes.c_int64 * 2)()
    at = ctypes.addressof(n)
    # a pointer's presence is all that is read
    _lib.call("vsa_cross_sizes", _lib.CROSS_POINTERS.pack(256, 256, 256, 256 * lens, 256 * (mask is not None))
              + rest, at, at + 8)
    return _Plan(rest, _dense(q, qs), _dense(k, ks), _dense(k, vs), *n)


def _plan(q, k, v, lens, mask, scale) -> _Plan:
    return _plan_of(q.shape, q.stride(), k.shape, k.stride(), v.stride(), lens is not None,
                    None if mask is None else mask.stride(0), _lib.DTYPE_CODES[q.dtype], scale,
                    q.device.index)


def _pointers(q, k, v, lens, mask) -> bytes:
    return _lib.CROSS_POINTERS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if lens is None else lens.data_ptr(),
        0 if mask is None else mask.data_ptr())


def _lens(kv_lens: Optional[Tensor], skv: int, device) -> Optional[Tensor]:
    """kv_lens as the kernels read it; 64-bit ones are clamped before they lose bits."""
    if kv_lens is None:
        return None
    return _i32(kv_lens.clamp(0, skv) if kv_lens.dtype is torch.int64 else kv_lens, device)


def _forward(q, k, v, lens, mask, scale, keep):
    """(out, lo, lse); the last two only where the backward needs them (``keep``)."""
    dev = q.device
    with on_device(dev):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        out = empty_in_order(q)
        lo = lse = None
        if keep:
            lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev)
            if q.dtype != torch.float32:
                lo = torch.empty(q.shape, dtype=torch.uint8, device=dev)
        plan = _plan(q, k, v, lens, mask, scale)
        scratch = _workspace(plan.forward, dev)
        _lib.call("vsa_cross_fwd", _pointers(q, k, v, lens, mask) + plan.rest, out.data_ptr(),
                  plan.q, _ptr(lo), _ptr(lse), _ptr(scratch),
                  torch._C._cuda_getCurrentRawStream(dev.index))
    return out, lo, lse


def _backward(q, k, v, lens, mask, scale, out, lo, lse, dout):
    dev = q.device
    with on_device(dev):
        # (the saved ones too: a saved-tensor hook may give back other addresses)
        q, k, v, out, dout = (_rows16(x) for x in (q, k, v, out, dout))
        dq, dk, dv = (empty_in_order(x) for x in (q, k, v))
        lo = lo if lo is None else _rows16(lo.contiguous())
        plan = _plan(q, k, v, lens, mask, scale)
        scratch = _workspace(plan.backward, dev)
        _lib.call("vsa_cross_bwd", _pointers(q, k, v, lens, mask) + plan.rest, out.data_ptr(),
                  _three(out), _ptr(lo), dout.data_ptr(), _three(dout), lse.data_ptr(),
                  dq.data_ptr(), plan.q, dk.data_ptr(), plan.k, dv.data_ptr(), plan.v,
                  _ptr(scratch), torch._C._cuda_getCurrentRawStream(dev.index))
    return dq, dk, dv


class _Cross(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lens, mask, scale):
        out, lo, lse = _forward(q, k, v, lens, mask, scale, True)
        ctx.save_for_backward(q, k, v, lens, mask, out, lo, lse)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, lens, mask, out, lo, lse = ctx.saved_tensors
        return (*_backward(q, k, v, lens, mask, ctx.scale, out, lo, lse, dout), None, None, None)


def _check(q, k, v, kv_lens, key_mask, sm_scale) -> None:
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q, k, and v must have shape [batch, heads, seq_len, dim]")
    b, h, sq, d = q.shape
    if k.shape[0] != b or v.shape[0] != b:
        raise ValueError("q, k, and v must share the batch dimension")
    if v.shape[1] != k.shape[1] or v.shape[2] != k.shape[2]:
        raise ValueError("k and v must have the same heads and sequence length")
    if k.shape[3] != d or v.shape[3] != d:
        raise ValueError("q, k, and v must have the same head dimension")
    if (h and not k.shape[1]) or (k.shape[1] and h % k.shape[1]):
        raise ValueError(f"the {h} heads of q must be a multiple of the {k.shape[1]} of k and v")
    if not q.dtype == k.dtype == v.dtype:
        raise ValueError("q, k, and v must have the same dtype")
    if q.dtype not in KERNEL_DTYPES:
        raise ValueError("the MI355X kernels support float16, bfloat16 and float32")
    if not 1 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"the MI355X kernels support head_dim <= {MAX_HEAD_DIM}")
    if kv_lens is not None:
        if tuple(kv_lens.shape) != (b,):
            raise ValueError("kv_lens must have shape [batch]")
        if kv_lens.dtype not in (torch.int32, torch.int64):
            raise ValueError("kv_lens must be int32 or int64")
    if key_mask is not None:
        if tuple(key_mask.shape) != (b, k.shape[2]):
            raise ValueError("key_mask must have shape [batch, kv seq_len]")
        if key_mask.dtype != torch.bool:
            raise ValueError("key_mask must be bool (True: the key is attended to)")
    if sm_scale is not None and not abs(sm_scale) <= MAX_SCALE:
        raise ValueError("sm_scale must be finite, and lie within 2^127")
    if b > 65535 or h > 65535 or k.shape[2] > MAX_TOKENS or \
            (h and sq > MAX_TOKENS // (h // k.shape[1])):
        raise ValueError("the MI355X kernels support at most 65535 samples and heads, and fewer "
                         "than 2^31 query rows of a key head and keys")
    if not q.is_cuda:
        raise ValueError("the MI355X implementation requires GPU tensors")
    dev = q.device
    if not (k.device == dev and v.device == dev and (kv_lens is None or kv_lens.device == dev)
            and (key_mask is None or key_mask.device == dev)):
        raise ValueError("q, k, v, kv_lens and key_mask must be on the same GPU device")


def mi355x_cross_attention(q: Tensor, k: Tensor, v: Tensor, kv_lens: Optional[Tensor] = None,
                           key_mask: Optional[Tensor] = None, *,
                           sm_scale: Optional[float] = None) -> Tensor:
    """Attention of ``q`` ``[batch, heads, seq_len, dim]`` to an encoder's ``k``, ``v``
    ``[batch, kv_heads, kv_len, dim]`` (``heads`` a multiple of ``kv_heads``; any
    lengths), over the keys below ``kv_lens[b]`` (clamped to ``[0, kv_len]``) whose
    ``key_mask[b]`` is True.  A sample without a valid key gets zeros; what lies
    behind a masked key (NaN included) has no influence.  ``sm_scale`` defaults to
    ``1/sqrt(dim)``.

    Per-head views of token-major memory, slices of a packed projection and
    expanded (broadcast) tensors are read in place where their rows start 16-byte
    aligned; the result is dense, in q's order of heads and tokens.
    Differentiable once in q, k and v."""
    _check(q, k, v, kv_lens, key_mask, sm_scale)
    d = q.shape[3]
    if q.numel() == 0 or k.numel() == 0:
        # nothing to attend with or to: zeros, in the graph of every input
        rest = sum(x[..., :0].sum() for x in (q, k, v))
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device) + rest
    scale = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(d)
    lens = _lens(kv_lens, k.shape[2], q.device)
    mask = key_mask
    if mask is not None and mask.stride(1) != 1 and mask.shape[1] > 1:
        mask = mask.contiguous()
    if d % 8:   # rows of whole 16-byte pieces; zero channels change no product
        q, k, v = (torch.nn.functional.pad(x, (0, 8 - d % 8)) for x in (q, k, v))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        q, k, v = (_rows16(x) for x in (q, k, v))   # kept for the backward as they are read
        out = _Cross.apply(q, k, v, lens, mask, scale)
    else:
        out = _forward(q, k, v, lens, mask, scale, False)[0]
    return out[..., :d] if d % 8 else out
