"""What the cross attention refuses, before anything reaches a GPU."""

import ctypes

import pytest
import torch

from vsa_mi355x import _lib, mi355x_cross_attention


def _args(**kw):
    a = dict(q=torch.zeros(2, 4, 5, 64), k=torch.zeros(2, 2, 7, 64), v=torch.zeros(2, 2, 7, 64),
             kv_lens=None, key_mask=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(q=torch.zeros(4, 5, 64)), "batch, heads"),
    (dict(q=torch.zeros(3, 4, 5, 64)), "batch"),
    (dict(v=torch.zeros(2, 1, 7, 64)), "same heads"),
    (dict(v=torch.zeros(2, 2, 6, 64)), "sequence length"),
    (dict(q=torch.zeros(2, 4, 5, 32)), "head dimension"),
    (dict(q=torch.zeros(2, 3, 5, 64)), "multiple"),
    (dict(k=torch.zeros(2, 0, 7, 64), v=torch.zeros(2, 0, 7, 64)), "multiple"),
    (dict(k=torch.zeros(2, 2, 7, 64).half()), "same dtype"),
    (dict(q=torch.zeros(2, 4, 5, 64).double(), k=torch.zeros(2, 2, 7, 64).double(),
          v=torch.zeros(2, 2, 7, 64).double()), "float16"),
    (dict(q=torch.zeros(2, 4, 5, 264), k=torch.zeros(2, 2, 7, 264),
          v=torch.zeros(2, 2, 7, 264)), "256"),
    (dict(kv_lens=torch.zeros(3, dtype=torch.int32)), "kv_lens"),
    (dict(kv_lens=torch.zeros(2)), "int32"),
    (dict(key_mask=torch.ones(2, 8, dtype=torch.bool)), "key_mask"),
    (dict(key_mask=torch.ones(2, 7)), "bool"),
    (dict(sm_scale=float("nan")), "finite"),
    (dict(sm_scale=float("inf")), "finite"),
    ({}, "GPU"),
])
def test_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        mi355x_cross_attention(**_args(**kw))


_P, _I64, _I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32


class Cross(ctypes.Structure):
    """``struct vsa_cross`` of the header."""
    _fields_ = ([(n, _P) for n in ("q", "k", "v", "kv_lens", "key_mask")]
                + [(n, _I64 * 3) for n in ("q_stride", "k_stride", "v_stride")]
                + [(n, _I64) for n in ("mask_stride", "sq", "skv")]
                + [(n, _I32) for n in ("batch", "heads", "kv_heads", "head_dim", "dtype")]
                + [("scale", ctypes.c_float)])


def test_packed_struct_has_the_headers_size():
    assert _lib.CROSS.size == ctypes.sizeof(Cross)


def test_entry_points_refuse_without_a_launch():
    lib = _lib.load()
    buf = torch.zeros(256)
    p = (buf.data_ptr() + 255) // 256 * 256
    st = (ctypes.c_int64 * 3)(64, 64, 64)
    n = (ctypes.c_int64 * 2)()
    at = ctypes.addressof(n)
    s3 = ctypes.addressof(st)

    def struct(**kw):
        c = Cross()
        c.q = c.k = c.v = p
        c.q_stride[:] = c.k_stride[:] = c.v_stride[:] = [64, 64, 64]
        c.sq, c.skv, c.batch, c.heads, c.kv_heads, c.head_dim = 4, 6, 2, 4, 2, 64
        c.scale = 0.125
        for name, x in kw.items():
            if name.endswith("stride") and name != "mask_stride":
                getattr(c, name)[:] = x
            else:
                setattr(c, name, x)
        return c

    def sizes(**kw):
        c = struct(**kw)
        return lib.vsa_cross_sizes(ctypes.addressof(c), at, at + 8)

    assert sizes() == 0 and n[0] >= 0 and n[1] > 0
    assert sizes(q=None) == -1 and sizes(dtype=9) == -3
    for kw in (dict(batch=0), dict(heads=3), dict(kv_heads=0), dict(head_dim=60),
               dict(head_dim=264), dict(sq=0), dict(skv=0), dict(skv=1 << 31), dict(sq=1 << 31),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(batch=65536),
               dict(v_stride=[64, 64, 32])):
        assert sizes(**kw) == -2, kw
    assert sizes(k=p + 8) == -7 and sizes(v_stride=[64, 4, 64]) == -7
    assert sizes(q_stride=[-64, 64, 64]) == -7 and sizes(k_stride=[64, 64, 1 << 30]) == -7
    assert sizes(kv_lens=p + 2) == -7
    c = struct()
    assert lib.vsa_cross_fwd(ctypes.addressof(c), None, s3, None, None, None, None) == -1
    assert lib.vsa_cross_fwd(ctypes.addressof(c), p + 2, s3, None, None, None, None) == -7
    c = struct(key_mask=p)
    assert lib.vsa_cross_fwd(ctypes.addressof(c), p, s3, None, None, None, None) == -1   # no scratch
    c = struct()
    bwd = [ctypes.addressof(c), p, s3, None, p, s3, p, p, s3, p, s3, p, s3, p, None]
    for i in (1, 2, 4, 6, 7, 9, 11, 13):
        bad = list(bwd)
        bad[i] = None
        assert lib.vsa_cross_bwd(*bad) == -1, i
    bwd[9] = p + 4
    assert lib.vsa_cross_bwd(*bwd) == -7


def test_workspaces_are_bounded():
    """The parts of a split never exceed what one row of workgroups can fill: the
    forward's scratch at a few queries on a long context, and the backward's at a
    long video on a prompt."""
    lib = _lib.load()
    n = (ctypes.c_int64 * 2)()
    at = ctypes.addressof(n)
    for b, h, sq, skv, d in ((1, 12, 64, 40960, 128), (8, 12, 1, 512, 128),
                             (1, 40, 40960, 512, 128), (1, 1, 1, 1 << 20, 64)):
        c = Cross()
        c.q = c.k = c.v = 256
        c.q_stride[:] = c.k_stride[:] = c.v_stride[:] = [256, 256, 256]
        c.sq, c.skv, c.batch, c.heads, c.kv_heads, c.head_dim, c.scale = sq, skv, b, h, h, d, 1.0
        assert lib.vsa_cross_sizes(ctypes.addressof(c), at, at + 8) == 0
        assert n[0] <= 1 << 28 and n[1] <= 1 << 30, (n[0], n[1])


@pytest.mark.parametrize("scale", [1e39, -1e39, 3e38, -3e38])
def test_scales_that_fp32_cannot_hold_in_base_two_are_refused(scale):
    with pytest.raises(ValueError, match="finite"):
        mi355x_cross_attention(**_args(sm_scale=scale))
    c = Cross()
    c.q = c.k = c.v = 256
    c.q_stride[:] = c.k_stride[:] = c.v_stride[:] = [64, 64, 64]
    c.sq, c.skv, c.batch, c.heads, c.kv_heads, c.head_dim = 4, 6, 2, 4, 2, 64
    n = (ctypes.c_int64 * 2)()
    at = ctypes.addressof(n)
    for c.scale, rc in ((scale, -2), (2.0 ** 127, 0), (-2.0 ** 127, 0)):
        assert _lib.load().vsa_cross_sizes(ctypes.addressof(c), at, at + 8) == rc


def test_lengths_of_64_bits_are_clamped_before_they_lose_bits():
    from vsa_mi355x.cross import _lens
    lens = torch.tensor([(1 << 32) + 3, -(1 << 32) + 3, 1 << 31, 5, -1])
    assert _lens(lens, 7, lens.device).tolist() == [7, 0, 7, 5, 0]
    assert _lens(lens, 7, lens.device).dtype == torch.int32
    assert _lens(None, 7, lens.device) is None


def test_the_outputs_rest_and_gradients_are_aligned():
    """The rest of the output is read eight bytes at a time; rows on 16 bytes."""
    lib = _lib.load()
    buf = torch.zeros(256)
    p = (buf.data_ptr() + 255) // 256 * 256
    st = (ctypes.c_int64 * 3)(64, 64, 64)
    s3 = ctypes.addressof(st)
    c = Cross()
    c.q = c.k = c.v = p
    c.q_stride[:] = c.k_stride[:] = c.v_stride[:] = [64, 64, 64]
    c.sq, c.skv, c.batch, c.heads, c.kv_heads, c.head_dim, c.scale = 4, 6, 2, 4, 2, 64, 0.125
    at = ctypes.addressof(c)
    assert lib.vsa_cross_fwd(at, p, s3, p + 4, None, p, None) == -7
    assert lib.vsa_cross_fwd(at, p, s3, None, p + 2, p, None) == -7
    assert lib.vsa_cross_fwd(at, p, s3, None, None, p + 128, None) == -7
    good = [at, p, s3, p, p, s3, p, p, s3, p, s3, p, s3, p, None]
    for i, off in ((1, 8), (3, 4), (4, 8), (6, 2), (7, 8), (9, 8), (11, 8), (13, 128)):
        bad = list(good)
        bad[i] = p + off
        assert lib.vsa_cross_bwd(*bad) == -7, i
