"""What the rotary operators refuse, before anything reaches a GPU."""

import ctypes

import pytest
import torch

from vsa_mi355x import _lib, build_rotary_table, mi355x_rotary, mi355x_vsa_tiled


@pytest.mark.parametrize("args,kw,text", [
    (((2, 3), (4, 4, 4)), {}, "dit_seq_shape"),
    (((2, 0, 3), (4, 4, 4)), {}, "positive"),
    (((1 << 12, 1 << 12, 1 << 12), (4, 4, 4)), {}, "2\\^31"),
    (((2, 2, 2), (4, 3, 4)), {}, "even"),
    (((2, 2, 2), (0, 0, 0)), {}, "axis_channels"),
    (((2, 2, 2), (128, 128, 2)), {}, "256"),
    (((2, 2, 2), (4, 4, -4)), {}, "axis_channels"),
    (((2, 2, 2), (4, 4, 4), 0.0), {}, "theta"),
    (((2, 2, 2), (4, 4, 4)), dict(factor=0.0), "factor"),
    (((2, 2, 2), (4, 4, 4)), dict(factor=float("nan")), "factor"),
    (((2, 2, 2), (4, 4, 4)), dict(start=(float("inf"), 0, 0)), "start"),
    (((2, 2, 2), (4, 4, 4)), dict(method="dynamic"), "method"),
    (((2, 2, 2), (4, 4, 4)), dict(method="yarn", factor=2.0), "original_shape"),
    (((2, 2, 2), (4, 4, 4)), dict(method="yarn", original_shape=(0, 1, 1)), "original_shape"),
    (((2, 2, 2), (4, 4, 4)), dict(device="cpu"), "GPU"),
])
def test_table_refusals(args, kw, text):
    with pytest.raises(ValueError, match=text):
        build_rotary_table(*args, **kw)


@pytest.mark.parametrize("args", [((2, 2.5, 2), (4, 4, 4)), ((2, 2, 2), (4, 4.0, 4))])
def test_table_sizes_are_integers(args):
    with pytest.raises(TypeError):
        build_rotary_table(*args)


def _args(**kw):
    a = dict(q=torch.zeros(2, 3, 5, 16), k=torch.zeros(2, 1, 5, 16), cos=torch.zeros(5, 8),
             sin=torch.zeros(5, 8), positions=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(q=torch.zeros(3, 5, 16)), "batch, heads"),
    (dict(k=torch.zeros(2, 1, 6, 16)), "share"),
    (dict(k=torch.zeros(2, 1, 5, 16, dtype=torch.float16)), "same dtype"),
    (dict(q=torch.zeros(2, 3, 5, 16).double(), k=None), "float16"),
    (dict(cos=torch.zeros(5, 8).half()), "float32"),
    (dict(sin=torch.zeros(5, 7)), "one shape"),
    (dict(cos=torch.zeros(5, 9), sin=torch.zeros(5, 9)), "channels"),
    (dict(cos=torch.zeros(5, 0), sin=torch.zeros(5, 0)), "channels"),
    (dict(cos=torch.zeros(4, 8), sin=torch.zeros(4, 8)), "4 positions"),
    (dict(cos=torch.zeros(5, 8, requires_grad=True)), "gradient"),
    (dict(positions=torch.zeros(5)), "int32"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), "positions"),
    (dict(positions=torch.zeros(1, 5, dtype=torch.int32)), "positions"),
    (dict(q=torch.zeros(1, 1, 5, 264), k=None), "256"),
    ({}, "GPU"),
])
def test_rotation_refusals(kw, text):
    with pytest.raises(ValueError, match=text):
        mi355x_rotary(**_args(**kw))


def test_tiled_op_checks_its_table():
    q = torch.zeros(1, 2, 8, 64)
    with pytest.raises(ValueError):
        mi355x_vsa_tiled(q, q, q, (2, 2, 2), 1, rotary=(torch.zeros(7, 32), torch.zeros(7, 32)))


_P, _I64, _I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32


class Axis(ctypes.Structure):
    """``struct vsa_rotary_axis`` of the header."""
    _fields_ = ([(n, _I32) for n in ("positions", "channels", "method", "reserved")]
                + [(n, ctypes.c_double) for n in ("start", "theta", "factor", "original")])


class Op(ctypes.Structure):
    """``struct vsa_rotary_op`` of the header."""
    _fields_ = ([(n, _P) for n in ("q", "k", "q_out", "k_out", "cos", "sin", "positions")]
                + [(n, _I64 * 3) for n in ("q_stride", "k_stride", "q_out_stride",
                                           "k_out_stride")]
                + [(n, _I64) for n in ("positions_stride", "batch", "tokens", "rows")]
                + [(n, _I32) for n in ("q_heads", "k_heads", "head_dim", "channels",
                                       "interleaved", "inverse", "positions64", "dtype")])


def test_packed_structs_have_the_headers_size():
    assert _lib.ROTARY_AXES.size == ctypes.sizeof(Axis * 3)
    assert _lib.ROTARY_OP.size == ctypes.sizeof(Op)


def test_entry_points_refuse_without_a_launch():
    lib = _lib.load()
    buf = torch.zeros(64)
    p = (buf.data_ptr() + 15) // 16 * 16
    axes = (Axis * 3)(*(Axis(2, 4, 0, 0, 0.0, 1e4, 1.0, 0.0)
                    for _ in range(3)))
    at = ctypes.addressof(axes)
    assert lib.vsa_rotary_table(None, p, p, None) == -1
    assert lib.vsa_rotary_table(at, p + 2, p, None) == -7
    for name, bad in (("positions", 0), ("channels", 3), ("channels", 300), ("theta", 0.0),
                      ("factor", -1.0), ("method", 3), ("start", float("nan"))):
        old = getattr(axes[1], name)
        setattr(axes[1], name, bad)
        assert lib.vsa_rotary_table(at, p, p, None) == -2, name
        setattr(axes[1], name, old)
    axes[0].method = 2
    assert lib.vsa_rotary_table(at, p, p, None) == -2    # yarn without the trained length

    def op(**kw):
        o = Op()
        for n in ("q", "k", "q_out", "k_out", "cos", "sin"):
            setattr(o, n, p)
        o.batch = o.tokens = o.rows = o.q_heads = o.k_heads = 1
        o.head_dim, o.channels = 8, 8
        for n, x in kw.items():
            setattr(o, n, x)
        return lib.vsa_rotary(ctypes.addressof(o), None)

    assert lib.vsa_rotary(None, None) == -1
    assert op(q=None) == -1 and op(k=None) == -1
    assert op(dtype=7) == -3
    for kw in (dict(channels=7), dict(channels=10), dict(head_dim=264), dict(tokens=0),
               dict(rows=0), dict(tokens=2), dict(q_heads=0), dict(batch=0)):
        assert op(**kw) == -2, kw
    assert op(q=p + 1) == -7 and op(cos=p + 2) == -7 and op(positions=p + 2) == -7
