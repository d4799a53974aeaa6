"""GPU: rotary positions and cross attention as custom ops: the eager functions'
values and gradients bit for bit, accepted by ``opcheck``, and a block compiled
with ``fullgraph=True`` that equals the eager one."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from vsa_mi355x import _lib
    _lib.load()
    yield


def _randn(*shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


@pytest.mark.parametrize("layout", ["head", "token"])
def test_ops_equal_the_eager_functions(layout):
    import vsa_mi355x as V
    from vsa_mi355x import ops
    cos, sin = V.build_rotary_table((40, 1, 1), (48, 0, 0), device=DEV)
    pos = torch.arange(40, device=DEV).flip(0)
    t = (lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)) if layout == "token" else \
        (lambda x: x)
    q, gq = (t(_randn(2, 4, 40, 64, seed=i)) for i in (1, 2))
    k, v = (t(_randn(2, 2, 40, 64, seed=i)) for i in (3, 4))
    lens = torch.tensor([40, 7], device=DEV)
    mask = torch.rand(2, 40, generator=torch.Generator().manual_seed(5)).to(DEV) < 0.7

    def run(m):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        a, b = m.mi355x_rotary(leaves[0], leaves[1], cos, sin, pos, interleaved=True)
        out = m.mi355x_cross_attention(a, b, leaves[2], lens, mask, sm_scale=0.2)
        one, none = m.mi355x_rotary(out, None, cos, sin, inverse=True)
        assert none is None
        return [out.detach(), one.detach(), *torch.autograd.grad(one, leaves, gq)]

    for a, b in zip(run(ops), run(V)):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(ops.mi355x_cross_attention(q, k, v), V.mi355x_cross_attention(q, k, v))


def test_odd_head_dim_and_empty():
    import vsa_mi355x as V
    from vsa_mi355x import ops
    q, k, v = (_randn(1, 2, 9, 20, seed=i) for i in range(3))
    assert torch.equal(ops.mi355x_cross_attention(q, k, v), V.mi355x_cross_attention(q, k, v))
    assert not ops.mi355x_cross_attention(q, k[:, :, :0], v[:, :, :0]).any()


def test_opcheck():
    import vsa_mi355x as V
    from vsa_mi355x import ops  # noqa: F401
    cos, sin = V.build_rotary_table((24, 1, 1), (64, 0, 0), device=DEV)
    q = _randn(1, 4, 24, 64, seed=1).requires_grad_()
    k = _randn(1, 2, 24, 64, seed=2).requires_grad_()
    v = _randn(1, 2, 24, 64, seed=3).requires_grad_()
    torch.library.opcheck(torch.ops.vsa_mi355x.rotary, (q, k, cos, sin, None, False, False))
    lens = torch.tensor([20], dtype=torch.int32, device=DEV)
    torch.library.opcheck(torch.ops.vsa_mi355x.cross_fwd, (q, k, v, lens, None, 0.125, True))


def test_a_block_compiles_whole():
    import vsa_mi355x as V
    from vsa_mi355x import ops
    cos, sin = V.build_rotary_table((64, 1, 1), (64, 0, 0), device=DEV)
    q, k, v = (_randn(1, 2, 64, 64, seed=i) for i in range(3))
    ek, ev = (_randn(1, 2, 50, 64, seed=i) for i in (7, 8))
    vbs = torch.full((1,), 64, dtype=torch.int32, device=DEV)

    def block(m, q, k, v):
        q, k = m.mi355x_rotary(q, k, cos, sin)
        x = m.mi355x_vsa(q, k, v, vbs, vbs, 1, (1, 1, 64))
        return m.mi355x_cross_attention(x, ek, ev)

    compiled = torch.compile(lambda *x: block(ops, *x), fullgraph=True, backend="aot_eager")
    leaves = [[x.clone().requires_grad_() for x in (q, k, v)] for _ in range(2)]
    a, b = compiled(*leaves[0]), block(V, *leaves[1])
    assert torch.equal(a, b)
    g = _randn(1, 2, 64, 64, seed=9)
    for x, y in zip(torch.autograd.grad(a, leaves[0], g), torch.autograd.grad(b, leaves[1], g)):
        assert torch.equal(x, y)
