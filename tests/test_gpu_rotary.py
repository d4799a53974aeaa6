"""GPU: rotary tables and the rotation of q and k against 64-bit formulas.

Tolerances: the angle is a product of two 64-bit numbers, off by 2^-52 of itself
for each of the few operations behind it (8 of them are allowed), and a table's
entry is rounded once to fp32 (2^-24).  The rotation's two products and their
sum round in fp32 (3 * 2^-24 of |x1| + |x2|) and the result once to its type
(half an eps; half the smallest subnormal below that)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def _gpu_only():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from vsa_mi355x import _lib
    _lib.load()
    yield


def _table64(shape, channels, theta, start, factor, method, original):
    """(cos, sin, largest angle) in 64 bits, axis by axis."""
    cos, sin, most = [], [], 0.0
    T, H, W = shape
    token = torch.arange(T * H * W)
    for a, d in enumerate(channels):
        index = (token // (H * W), token // W % H, token % W)[a].double() + start[a]
        for i in range(d // 2):
            f, m = theta ** (-2.0 * i / d), 1.0
            if method == "linear":
                f /= factor[a]
            elif method == "ntk" and d > 2:
                f = (theta * factor[a] ** (d / (d - 2.0))) ** (-2.0 * i / d)
            elif method == "yarn":
                keep = min(1.0, max(0.0, (original[a] * f / (2 * math.pi) - 1) / 31))
                f, m = f * keep + f / factor[a] * (1 - keep), 0.1 * math.log(factor[a]) + 1
            angle = index * f
            cos.append(angle.cos() * m)
            sin.append(angle.sin() * m)
            most = max(most, angle.abs().max().item() * m)
    return torch.stack(cos, 1), torch.stack(sin, 1), most


@pytest.mark.parametrize("shape,channels,kw", [
    ((1, 1, 1), (2, 0, 0), {}),
    ((5, 7, 9), (44, 42, 42), {}),
    ((3, 4, 33), (0, 32, 34), dict(factor=(1.0, 2.0, 3.0))),
    ((21, 30, 52), (16, 56, 56), dict(start=(3, 0.5, -7), method="ntk", factor=4.0)),
    ((1000, 1, 1), (128, 0, 0), dict(start=(3000000, 0, 0))),
    ((513, 1, 1), (256, 0, 0), dict(method="yarn", factor=16.0, original_shape=(4096, 1, 1))),
    ((2, 1, 40), (2, 0, 6), dict(method="ntk", factor=2.0, theta=500.0)),
])
def test_table_against_64_bits(shape, channels, kw):
    from vsa_mi355x import build_rotary_table
    cos, sin = build_rotary_table(shape, channels, device=DEV, **kw)
    three = lambda x: x if isinstance(x, tuple) else (x,) * 3   # noqa: E731
    c, s, most = _table64(shape, channels, kw.get("theta", 10000.0), three(kw.get("start", 0)),
                          three(kw.get("factor", 1.0)), kw.get("method", "linear"),
                          kw.get("original_shape"))
    for got, ref in ((cos, c), (sin, s)):
        assert got.dtype == torch.float32 and got.shape == ref.shape
        tol = ref.abs() * 2.0 ** -24 + 8 * 2.0 ** -52 * max(most, 1.0)
        assert ((got.cpu().double() - ref).abs() <= tol).all()


def _turn64(x, cos, sin, positions, interleaved, sign=1.0):
    """The rotation in 64 bits and the size of its terms, |x1| + |x2|."""
    b, h, s, d = x.shape
    y, size = x.double().clone(), x.double().abs()
    n = cos.shape[1]
    p = torch.arange(s).expand(b, s) if positions is None else positions.long().expand(b, s)
    on = (p >= 0)[..., None]
    c = torch.where(on, cos.double()[p.clamp(min=0)], 1.0)[:, None]
    w = torch.where(on, sin.double()[p.clamp(min=0)], 0.0)[:, None] * sign
    i = torch.arange(n)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    a, e = x.double()[..., one], x.double()[..., two]
    y[..., one], y[..., two] = a * c - e * w, e * c + a * w
    size[..., one] = size[..., two] = a.abs() + e.abs()
    return y, size


def _near(got, ref, size):
    t = got.dtype
    u = torch.finfo(t).eps / 2
    tiny = torch.finfo(t).tiny * u
    tol = ref.abs() * u + tiny + size * 3 * 2.0 ** -24
    assert ((got.cpu().double() - ref).abs() <= tol).all()


def _memory(x, layout):
    """x on the GPU in a memory layout."""
    if layout == "head":
        return x.to(DEV)
    if layout == "token":
        return x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    if layout == "packed":    # the middle of a [B, S, 3, H, D] projection
        b, h, s, d = x.shape
        buf = torch.full((b, s, 3, h, d), 7.0, dtype=x.dtype, device=DEV)
        buf[:, :, 1] = x.transpose(1, 2).to(DEV)
        return buf[:, :, 1].transpose(1, 2)
    assert layout == "odd"    # rows that start on 2 bytes of 16, channels two apart
    b, h, s, d = x.shape
    buf = torch.full((b, h, s, 2 * d + 3), 7.0, dtype=x.dtype, device=DEV)[..., 1:2 * d + 1:2]
    buf.copy_(x)
    return buf


CASES = [
    # dtype, B, Hq, Hk, S, D, channels, interleaved, layout, positions
    ("bf16", 1, 2, 2, 1, 128, 128, False, "head", None),
    ("bf16", 2, 3, 1, 70, 128, 128, True, "token", None),
    ("fp16", 2, 5, 5, 33, 80, 60, True, "packed", "sample"),
    ("fp16", 2, 5, 5, 33, 80, 60, False, "packed", "sample"),
    ("fp32", 1, 4, 2, 129, 64, 64, False, "token", "shared"),
    ("fp32", 3, 1, 1, 17, 72, 48, True, "head", "long"),
    ("bf16", 1, 9, 7, 40, 96, 2, True, "head", None),
    ("bf16", 1, 1, 1, 40, 7, 6, False, "odd", None),
    ("bf16", 2, 2, 2, 9, 7, 4, True, "odd", "sample"),
    ("fp16", 1, 24, 24, 300, 256, 256, False, "token", None),
    ("fp32", 1, 2, 2, 65, 256, 200, True, "odd", None),
    ("bf16", 2, 40, 40, 1030, 128, 64, False, "token", "sample"),
]


@pytest.mark.parametrize("dtype,b,hq,hk,s,d,n,inter,layout,where", CASES)
def test_rotation_and_gradient_against_64_bits(dtype, b, hq, hk, s, d, n, inter, layout, where):
    from vsa_mi355x import mi355x_rotary
    g = torch.Generator().manual_seed(hq * 1000 + s)
    dt = DTYPES[dtype]
    q, k, gq, gk = (torch.randn(b, h, s, d, generator=g).to(dt) for h in (hq, hk, hq, hk))
    angle = torch.rand(s + 5, n // 2, generator=g).double() * 6.3
    cos, sin = angle.cos().float(), angle.sin().float()
    pos = None
    if where is not None:
        pos = torch.randint(-1, s + 5, (s,) if where == "shared" else (b, s), generator=g)
        pos = pos.to(torch.int64 if where == "long" else torch.int32)
    ql, kl = (_memory(x, layout).requires_grad_() for x in (q, k))
    qo, ko = mi355x_rotary(ql, kl, cos.to(DEV), sin.to(DEV), None if pos is None else pos.to(DEV),
                           interleaved=inter)
    dq, dk = torch.autograd.grad((qo, ko), (ql, kl), (_memory(gq, layout), _memory(gk, layout)))
    for got, x, sign in ((qo, q, 1.0), (ko, k, 1.0), (dq, gq, -1.0), (dk, gk, -1.0)):
        assert got.shape == x.shape and got.dtype == dt
        _near(got.detach(), *_turn64(x, cos, sin, pos, inter, sign))
    with torch.no_grad():
        again = mi355x_rotary(ql, kl, cos.to(DEV), sin.to(DEV),
                              None if pos is None else pos.to(DEV), interleaved=inter)
    assert torch.equal(again[0], qo) and torch.equal(again[1], ko)
    if layout != "head":
        assert qo.stride(3) == 1


def test_one_tensor_no_heads_no_tokens_and_the_way_back():
    from vsa_mi355x import build_rotary_table, mi355x_rotary
    cos, sin = build_rotary_table((4, 3, 2), (8, 4, 4), device=DEV)
    q = torch.randn(2, 3, 24, 20, device=DEV)
    a, none = mi355x_rotary(q, None, cos, sin)
    assert none is None
    b, k = mi355x_rotary(q, q[:, :0], cos, sin)
    assert torch.equal(a, b) and k.shape == (2, 0, 24, 20)
    back, _ = mi355x_rotary(a, None, cos, sin, inverse=True)
    assert (back - q).abs().max() <= 8 * 2.0 ** -24 * q.abs().max() * 2
    e, f = mi355x_rotary(q[:, :, :0], q[:, :1, :0], cos, sin)
    assert e.shape == (2, 3, 0, 20) and f.shape == (2, 1, 0, 20)


def test_positions_past_the_table_give_nan_and_negative_ones_copy():
    from vsa_mi355x import build_rotary_table, mi355x_rotary
    cos, sin = build_rotary_table((4, 1, 1), (16, 0, 0), device=DEV)
    q = torch.randn(1, 2, 4, 24, device=DEV)
    pos = torch.tensor([3, 4, -1, -2 ** 31], dtype=torch.int32, device=DEV)
    y, _ = mi355x_rotary(q, None, cos, sin, pos)
    assert y[:, :, 0].isfinite().all() and y[:, :, 1, :16].isnan().all()
    assert torch.equal(y[:, :, 1, 16:], q[:, :, 1, 16:])
    assert torch.equal(y[:, :, 2:], q[:, :, 2:])


def test_second_derivative_and_one_gradient_alone():
    from vsa_mi355x import build_rotary_table, mi355x_rotary
    cos, sin = build_rotary_table((9, 1, 1), (32, 0, 0), device=DEV)
    q = torch.randn(1, 2, 9, 32, device=DEV, requires_grad=True)
    k = torch.randn(1, 1, 9, 32, device=DEV)
    y, z = mi355x_rotary(q, k, cos, sin)
    (g,) = torch.autograd.grad(y.pow(2).sum(), q, create_graph=True)
    # the rotation keeps |q|, so the gradient of |q'|^2 is 2 q and that of its sum is 2
    assert (g - 2 * q).abs().max() <= 32 * 2.0 ** -24 * q.abs().max()
    (gg,) = torch.autograd.grad(g.sum(), q)
    assert (gg - 2).abs().max() <= 64 * 2.0 ** -24
    assert z.requires_grad and y.requires_grad
    k.requires_grad_()
    _, z = mi355x_rotary(q.detach(), k, cos, sin)
    (gk,) = torch.autograd.grad(z.sum(), k)
    ref, size = _turn64(torch.ones(1, 1, 9, 32), cos.cpu(), sin.cpu(), None, False, -1.0)
    _near(gk, ref, size)


def test_table_and_rotation_in_a_graph_and_on_another_stream():
    from vsa_mi355x import build_rotary_table, mi355x_rotary
    q = torch.randn(2, 4, 50, 64, device=DEV, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    with torch.no_grad():
        cos, sin = build_rotary_table((5, 10, 1), (32, 32, 0), start=(7, 0, 0), device=DEV)
        want = mi355x_rotary(q, q, cos, sin)[1]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = mi355x_rotary(q, q, *build_rotary_table((5, 10, 1), (32, 32, 0),
                                                          start=(7, 0, 0), device=DEV))[1]
        side.synchronize()
        assert torch.equal(got, want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c2, s2 = build_rotary_table((5, 10, 1), (32, 32, 0), start=(7, 0, 0), device=DEV)
            out = mi355x_rotary(q, q, c2, s2)[1]
        for i in range(4):
            q.copy_(torch.randn(q.shape, device=DEV))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(c2, cos)
            assert torch.equal(out, mi355x_rotary(q, q, cos, sin)[1]), i


def test_offsets_past_32_bits():
    """The last head of a projection output of more than 2^31 elements."""
    from vsa_mi355x import build_rotary_table, mi355x_rotary
    s, h, d = 66000, 260, 128
    buf = torch.empty((1, s, h, d), dtype=torch.bfloat16, device=DEV)
    assert buf.numel() > 1 << 31
    x = torch.randn(1, s, 2, d, device=DEV).to(torch.bfloat16)
    buf[:, :, -2:] = x
    cos, sin = build_rotary_table((s, 1, 1), (d, 0, 0), device=DEV)
    got, _ = mi355x_rotary(buf[:, :, -2:].transpose(1, 2), None, cos, sin)
    want, _ = mi355x_rotary(x.transpose(1, 2), None, cos, sin)
    assert torch.equal(got, want)


@pytest.mark.parametrize("token_major,inter,tile,dtype,gate", [
    (False, False, (4, 4, 4), torch.bfloat16, "full"), (True, True, (4, 8, 8), torch.float16, None),
    (True, False, (4, 4, 4), torch.bfloat16, "token"), (False, True, (2, 8, 8), torch.float32, None),
    (True, False, (4, 8, 8), torch.float32, "full")])
def test_tiled_op_with_rotary_equals_rotating_first(token_major, inter, tile, dtype, gate):
    from vsa_mi355x import build_rotary_table, mi355x_rotary, mi355x_vsa_tiled
    shape, h, d = (5, 12, 20), 3, 64
    s = math.prod(shape)
    g = torch.Generator().manual_seed(5)
    dims = (2, s, h, d) if token_major else (2, h, s, d)
    q, k, v, do = (torch.randn(dims, generator=g).to(dtype).to(DEV) for _ in range(4))
    gt = None
    if gate is not None:
        gt = torch.rand((*dims[:3], d if gate == "full" else 1), generator=g).to(dtype).to(DEV)
    cos, sin = build_rotary_table(shape, (16, 24, 16), device=DEV)

    def run(fused):
        leaves = [x.clone().requires_grad_() for x in (q, k, v, *([gt] if gate else []))]
        a, b, c, *w = leaves
        if fused:
            out = mi355x_vsa_tiled(a, b, c, shape, 4, tile, w[0] if w else None, token_major,
                                   rotary=(cos, sin), rotary_interleaved=inter)
        else:
            t = (lambda x: x.transpose(1, 2)) if token_major else (lambda x: x)
            a, b = (t(x) for x in mi355x_rotary(t(a), t(b), cos, sin, interleaved=inter))
            out = mi355x_vsa_tiled(a, b, c, shape, 4, tile, w[0] if w else None, token_major)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    for x, y in zip(run(True), run(False)):
        assert torch.equal(x, y)
    with torch.no_grad():
        out = mi355x_vsa_tiled(q, k, v, shape, 4, tile, gt, token_major, rotary=(cos, sin),
                               rotary_interleaved=inter)
    assert torch.equal(out, run(True)[0])
