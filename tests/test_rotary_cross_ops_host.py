"""The custom ops of the rotary positions and the cross attention: registered, and
their fake implementations have the kernels' shapes and orders (no GPU needed)."""

import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vsa_mi355x import ops  # noqa: F401  (registers the ops)


def _t(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, device="cuda", dtype=dtype)


def test_ops_are_registered():
    for name in ("rotary", "cross_fwd", "cross_bwd"):
        assert hasattr(torch.ops.vsa_mi355x, name), name


def test_rotary_fake():
    with FakeTensorMode():
        q = _t(2, 40, 3, 64).transpose(1, 2)           # token-major
        k = _t(2, 40, 2, 1, 64)[:, :, :, 0].transpose(1, 2)
        cos = _t(40, 32, dtype=torch.float32)
        a, b = torch.ops.vsa_mi355x.rotary(q, k, cos, cos, None, False, False)
        assert a.shape == q.shape and a.stride() == q.stride()
        assert b.shape == k.shape and b.stride() == k.stride()
        a, b = torch.ops.vsa_mi355x.rotary(q, None, cos, cos, None, True, True)
        assert b.numel() == 0


def test_cross_fake():
    with FakeTensorMode():
        q = _t(2, 4, 9, 64)
        kv = _t(2, 7, 2, 2, 64)                         # [B, S, 2, H, D]
        k, v = (kv[:, :, i].transpose(1, 2) for i in range(2))
        out, lo, lse = torch.ops.vsa_mi355x.cross_fwd(q, k, v, None, None, 0.125, True)
        assert out.shape == lo.shape == q.shape and lse.shape == (2, 4, 9)
        assert lse.dtype == torch.float32
        dq, dk, dv = torch.ops.vsa_mi355x.cross_bwd(out, q, k, v, None, None, out, lo, lse, 0.125)
        assert dq.shape == q.shape and dk.shape == k.shape
        assert dk.transpose(1, 2).is_contiguous() and dv.transpose(1, 2).is_contiguous()
        _, lo, lse = torch.ops.vsa_mi355x.cross_fwd(q, k, v, None, None, 0.125, False)
        assert lo.numel() == lse.numel() == 0
