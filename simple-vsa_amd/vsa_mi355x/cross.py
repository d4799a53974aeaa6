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
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .launch import _ptr, _workspace, on_device
from .mi355x import KERNEL_DTYPES, _i32
from .rotary import empty_in_order, strides

MAX_HEAD_DIM = 256
MAX_TOKENS = (1 << 31) - 256
MAX_SCALE = 2.0 ** 127   # times log2(e) it stays finite in fp32


def _rows16(x: Tensor) -> Tensor:
    """x itself where the kernels read its rows in place (channels next to each
    other, every row 16-byte aligned, a tile's rows within reach of a 32-bit
    offset), else a dense copy."""
    if x.is_contiguous():
        return x if x.data_ptr() % 16 == 0 else x.clone()
    es = x.element_size()
    if x.stride(3) == 1 and x.data_ptr() % 16 == 0:
        b, h, s = _strides(x)
        if (b | h | s) * es % 16 == 0 and x.shape[3] <= s <= (1 << 30) // (64 * es):
            return x
    return x.clone(memory_format=torch.contiguous_format)


def _strides(x: Tensor):
    """Strides for the C ABI; those of a row where there is one token."""
    b, h, s = strides(x)
    return b, h, s if x.shape[2] > 1 else x.shape[3]


def _pack(q, k, v, lens, mask, scale) -> bytes:
    b, h, sq, d = q.shape
    return _lib.CROSS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if lens is None else lens.data_ptr(),
        0 if mask is None else mask.data_ptr(), *_strides(q), *_strides(k), *_strides(v),
        0 if mask is None else mask.stride(0), sq, k.shape[2], b, h, k.shape[1], d,
        _lib.DTYPE_CODES[q.dtype], scale)


def _lens(kv_lens: Optional[Tensor], skv: int, device) -> Optional[Tensor]:
    """kv_lens as the kernels read it; 64-bit ones are clamped before they lose bits."""
    if kv_lens is None:
        return None
    return _i32(kv_lens.clamp(0, skv) if kv_lens.dtype is torch.int64 else kv_lens, device)


def _three(x: Tensor) -> bytes:
    return _lib.STRIDES.pack(*_strides(x))


@functools.lru_cache(maxsize=256)
def _sizes(b, h, hk, sq, skv, d, lens, masked, dtype, device):
    """Bytes of (forward scratch, backward scratch) on ``device``, the current one
    (the splits follow its number of CUs)."""
    # a pointer's presence is all that is read
    c = _lib.CROSS.pack(256, 256, 256, 256 if lens else 0, 256 if masked else 0, *(0, 0, 256) * 3, 0, sq, skv, b, h,
                        hk, d, dtype, 1.0)
    n = (ctypes.c_int64 * 2)()
    at = ctypes.addressof(n)
    _lib.call("vsa_cross_sizes", c, at, at + 8)
    return tuple(n)


def _scratch(q, k, lens, mask, which: int) -> Optional[Tensor]:
    b, h, sq, d = q.shape
    return _workspace(_sizes(b, h, k.shape[1], sq, k.shape[2], d, lens is not None,
                             mask is not None, _lib.DTYPE_CODES[q.dtype], q.device.index)[which],
                      q.device)


def _forward(q, k, v, lens, mask, scale, keep):
    """(out, lo, lse); the last two only where the backward needs them (``keep``)."""
    dev = q.device
    with on_device(dev):
        out = empty_in_order(q)
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        lo = lse = None
        if keep:
            lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev)
            if q.dtype != torch.float32:
                lo = torch.empty(q.shape, dtype=torch.uint8, device=dev)
        scratch = _scratch(q, k, lens, mask, 0)
        _lib.call("vsa_cross_fwd", _pack(q, k, v, lens, mask, scale), out.data_ptr(), _three(out),
                  _ptr(lo), _ptr(lse), _ptr(scratch),
                  torch._C._cuda_getCurrentRawStream(dev.index))
    return out, lo, lse


def _backward(q, k, v, lens, mask, scale, out, lo, lse, dout):
    dev = q.device
    with on_device(dev):
        dq, dk, dv = (empty_in_order(x) for x in (q, k, v))
        # (the saved ones too: a saved-tensor hook may give back other addresses)
        q, k, v, out, dout = (_rows16(x) for x in (q, k, v, out, dout))
        lo = lo if lo is None else _rows16(lo.contiguous())
        scratch = _scratch(q, k, lens, mask, 1)
        _lib.call("vsa_cross_bwd", _pack(q, k, v, lens, mask, scale), out.data_ptr(), _three(out),
                  _ptr(lo), dout.data_ptr(), _three(dout), lse.data_ptr(), dq.data_ptr(),
                  _three(dq), dk.data_ptr(), _three(dk), dv.data_ptr(), _three(dv), _ptr(scratch),
                  torch._C._cuda_getCurrentRawStream(dev.index))
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
