"""GPU: cross attention and its gradients against 64-bit formulas, with the bounds
of ``cross_reference``; masks, layouts, streams, graphs and far offsets."""

import pytest
import torch

from cross_reference import reference

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


def _memory(x, layout):
    """x ([B, H, S, D]) in a memory layout, on the GPU."""
    b, h, s, d = x.shape
    if layout == "head":
        return x.to(DEV)
    if layout == "token":
        return x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    if layout == "packed":
        buf = torch.full((b, s, 3, h, d), 7.0, dtype=x.dtype, device=DEV)
        buf[:, :, 1] = x.transpose(1, 2).to(DEV)
        return buf[:, :, 1].transpose(1, 2)
    assert layout == "odd"   # rows that do not start on 16 bytes
    buf = torch.full((b, h, s, d + 3), 7.0, dtype=x.dtype, device=DEV)[..., 1:d + 1]
    buf.copy_(x)
    return buf


def _inputs(dtype, b, h, hk, sq, n, d, seed):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    return [torch.randn(b, x, s, d, generator=g).to(dt)
            for x, s in ((h, sq), (hk, n), (hk, n), (h, sq))]


def _masks(kind, b, n, seed):
    """(kv_lens, key_mask) on the GPU, or None."""
    g = torch.Generator().manual_seed(seed)
    lens = mask = None
    if "lens" in kind:
        lens = torch.randint(1, n + 1, (b,), generator=g, dtype=torch.int32)
    if "over" in kind:       # lengths outside [0, n] are clamped
        lens = torch.tensor([n + 100, -5, 1][:b], dtype=torch.int64)
    if "holes" in kind:
        mask = torch.rand(b, n, generator=g) < 0.6
        mask[:, n - 1] = True
    if "left" in kind:       # padding in front
        mask = torch.arange(n).expand(b, n) >= n // 2
    if "empty" in kind:
        if lens is None and mask is None:
            lens = torch.full((b,), n, dtype=torch.int32)
        if lens is not None:
            lens[0] = 0
        else:
            mask[0] = False
    return tuple(x if x is None else x.to(DEV) for x in (lens, mask))


def _check(names, got, ref, tol):
    for name, x, r, t in zip(names, got, ref, tol):
        assert x.shape == r.shape, name
        x = x.detach().double()
        assert x.isfinite().all(), name
        over = ((x - r).abs() - t).max().item()
        worst = ((x - r).abs() / t.clamp(min=1e-300)).max().item()
        print(f"{name}: {worst:.3f} of its bound", flush=True)
        assert over <= 0, (name, worst)


NAMES = ["out", "dq", "dk", "dv"]
CASES = [
    # dtype, B, H, Hk, Sq, Skv, D, layout, masks
    ("bf16", 1, 1, 1, 1, 1, 64, "head", ""),
    ("bf16", 2, 3, 3, 1, 77, 128, "token", "lens"),
    ("bf16", 3, 4, 2, 5, 33, 64, "packed", "over"),
    ("bf16", 2, 2, 2, 130, 257, 128, "token", "holes"),
    ("bf16", 1, 2, 1, 300, 64, 128, "head", "left"),
    ("bf16", 2, 2, 2, 64, 512, 128, "head", "lens holes empty"),
    ("bf16", 1, 12, 3, 1, 2000, 128, "packed", ""),
    ("bf16", 1, 2, 2, 40, 3001, 64, "token", "holes"),
    ("bf16", 1, 2, 2, 3001, 40, 64, "token", ""),
    ("bf16", 2, 2, 2, 129, 129, 256, "head", "lens"),
    ("bf16", 1, 2, 1, 33, 500, 256, "token", "holes"),
    ("bf16", 2, 3, 1, 100, 65, 80, "packed", "empty"),
    ("bf16", 1, 2, 2, 70, 90, 40, "odd", "lens"),
    ("bf16", 1, 1, 1, 65, 66, 1, "head", ""),
    ("bf16", 1, 2, 2, 31, 95, 100, "token", "holes"),
    ("fp16", 2, 2, 2, 200, 226, 64, "token", "holes"),
    ("fp16", 1, 8, 2, 9, 70, 96, "head", "left empty"),
    ("fp16", 1, 2, 2, 1025, 513, 128, "packed", ""),
    ("fp16", 1, 1, 1, 64, 64, 200, "odd", "lens"),
    ("fp32", 1, 1, 1, 1, 1, 8, "head", ""),
    ("fp32", 2, 4, 2, 1, 700, 64, "token", "lens"),
    ("fp32", 2, 4, 2, 150, 333, 80, "packed", "lens empty"),
    ("fp32", 1, 2, 2, 257, 129, 128, "token", "holes"),
    ("fp32", 1, 1, 1, 130, 131, 256, "head", "holes"),
    ("fp32", 1, 2, 1, 40, 900, 256, "odd", ""),
]


@pytest.mark.parametrize("dtype,b,h,hk,sq,n,d,layout,kind", CASES)
def test_forward_and_gradients_against_64_bits(dtype, b, h, hk, sq, n, d, layout, kind):
    from vsa_mi355x import mi355x_cross_attention
    print(f"case {dtype} b={b} h={h}/{hk} sq={sq} skv={n} d={d} {layout} {kind}", flush=True)
    host = _inputs(dtype, b, h, hk, sq, n, d, seed=sq * 7 + n)
    lens, mask = _masks(kind, b, n, seed=n)
    q, k, v, do = (_memory(x, layout) for x in host)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = mi355x_cross_attention(*leaves, lens, mask)
    grads = torch.autograd.grad(out, leaves, do)
    ref, tol = reference(*(x.to(DEV) for x in host), lens, mask)
    _check(NAMES, [out, *grads], ref, tol)
    with torch.no_grad():
        assert torch.equal(mi355x_cross_attention(*leaves, lens, mask), out)
    again = torch.autograd.grad(mi355x_cross_attention(*leaves, lens, mask), leaves, do)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3, 1.5])
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp32", 128)])
def test_scales(dtype, d, scale):
    from vsa_mi355x import mi355x_cross_attention
    host = _inputs(dtype, 1, 2, 2, 70, 100, d, seed=3)
    lens = torch.tensor([90], device=DEV)
    leaves = [x.to(DEV).requires_grad_() for x in host[:3]]
    out = mi355x_cross_attention(*leaves, lens, sm_scale=scale)
    grads = torch.autograd.grad(out, leaves, host[3].to(DEV))
    ref, tol = reference(*(x.to(DEV) for x in host), lens, scale=scale)
    _check(NAMES, [out, *grads], ref, tol)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "lowest"])
@pytest.mark.parametrize("dtype,sq,n,d", [("bf16", 40, 300, 128), ("fp16", 3, 70, 64),
                                          ("fp32", 140, 100, 80), ("bf16", 200, 64, 256)])
def test_nothing_behind_a_mask_has_influence(dtype, sq, n, d, bad):
    """Keys and values that are not valid hold what breaks a sum; the results are
    those of zeros there, bit for bit, and their gradients zero."""
    from vsa_mi355x import mi355x_cross_attention
    b, h = 3, 2
    host = _inputs(dtype, b, h, h, sq, n, d, seed=11)
    lens = torch.tensor([n - 3, n, 0], dtype=torch.int32, device=DEV)
    _, mask = _masks("holes", b, n, seed=2)
    ok = mask & (torch.arange(n, device=DEV) < lens[:, None])
    if bad == "lowest":
        bad = torch.finfo(DTYPES[dtype]).min

    def run(fill):
        q, k, v, do = (x.to(DEV) for x in host)
        k, v = (torch.where(ok[:, None, :, None], x, torch.full_like(x, fill)) for x in (k, v))
        leaves = [x.requires_grad_() for x in (q, k, v)]
        out = mi355x_cross_attention(*leaves, lens, mask)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    got, want = run(bad), run(0.0)
    for x, y in zip(got, want):
        assert x.isfinite().all()
        assert torch.equal(x, y)
    assert not got[0][2].any() and not got[1][2].any()
    for x in got[2:]:
        assert not x[~ok[:, None].expand(b, h, n)].any()


def test_scores_far_from_zero():
    """Rows whose scores reach +-2000 and keys of one large value: the largest score
    of a row is taken off before the exponential."""
    from vsa_mi355x import mi355x_cross_attention
    q, k, v, do = _inputs("fp32", 1, 2, 2, 40, 200, 64, seed=4)
    q, k = q * 40, k * 8
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v)]
    out = mi355x_cross_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, do.to(DEV))
    ref, tol = reference(*(x.to(DEV) for x in (q, k, v, do)))
    _check(NAMES, [out, *grads], ref, tol)


def test_broadcast_states_and_one_gradient_alone():
    """One prompt for every sample: an expanded batch is read in place, and its
    gradient is the sum over the samples."""
    from vsa_mi355x import mi355x_cross_attention
    q, k, v, do = _inputs("fp32", 4, 2, 2, 33, 70, 64, seed=8)
    q, do = q.to(DEV), do.to(DEV)
    k1, v1 = (x[:1].to(DEV).requires_grad_() for x in (k, v))
    out = mi355x_cross_attention(q, k1.expand(4, -1, -1, -1), v1.expand(4, -1, -1, -1))
    dk, dv = torch.autograd.grad(out, (k1, v1), do)
    ref, tol = reference(q, k1.detach().expand(4, -1, -1, -1), v1.detach().expand(4, -1, -1, -1),
                         do)
    # the sum over four samples rounds three times in fp32
    _check(NAMES, [out, dk, dv], [ref[0], ref[2].sum(0, True), ref[3].sum(0, True)],
           [tol[0], *(t.sum(0, True) + 4 * 2.0 ** -24 * r.abs().sum(0, True)
                      for t, r in zip(tol[2:], ref[2:]))])


def test_gradients_against_differences():
    """(f(x + t d) - f(x - t d)) / 2t of f = sum(out * w), w one element of each
    sample and head (a bound on a sum of all would say nothing), on the kernels,
    against the kernels' gradients.  The difference of the kernels' outputs is off by the
    outputs' bounds over t, the quotient by what the same quotient in 64 bits is
    off its derivative."""
    from vsa_mi355x import mi355x_cross_attention
    host = _inputs("fp32", 2, 4, 2, 21, 45, 64, seed=21)
    lens, mask = _masks("lens holes", 2, 45, seed=5)
    q, k, v, w = (x.to(DEV) for x in host)
    w = torch.zeros_like(w)
    w[:, :, 13, 7] = 1.0
    leaves = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(mi355x_cross_attention(*leaves, lens, mask), leaves, w)
    t = 2.0 ** -2
    for i, name in enumerate("qkv"):
        g = torch.Generator().manual_seed(i)
        d = torch.randint(-1, 2, leaves[i].shape, generator=g).to(DEV).float()
        ends, ends64, off = [], [], 0.0
        for sign in (1, -1):
            x = [y.detach() for y in (q, k, v)]
            x[i] = x[i] + sign * t * d      # exact enough: both sides take the same values
            ends.append((mi355x_cross_attention(*x, lens, mask).double() * w.double()).sum())
            (r,), (b,) = reference(*x, None, lens, mask)
            ends64.append((r * w.double()).sum())
            off += (b * w.double().abs()).sum().item()
        ref, tol = reference(q.detach(), k.detach(), v.detach(), w, lens, mask)
        want = (ref[1 + i] * d.double()).sum().item()
        quotient = ((ends[0] - ends[1]) / (2 * t)).item()
        cut = abs(((ends64[0] - ends64[1]) / (2 * t)).item() - want)
        got = (grads[i].double() * d.double()).sum().item()
        bound = off / (2 * t) + cut + (tol[1 + i] * d.double().abs()).sum().item()
        print(f"{name}: gradient {got:.6f} difference {quotient:.6f} bound {bound:.2g}", flush=True)
        assert abs(got - quotient) <= bound
        assert bound < 0.05 * (ref[1 + i] * d.double()).abs().sum().item()


def test_empty_dimensions():
    from vsa_mi355x import mi355x_cross_attention
    for b, h, sq, n in ((0, 2, 3, 4), (2, 0, 3, 4), (2, 2, 0, 4), (2, 2, 3, 0)):
        q = torch.randn(b, h, sq, 64, device=DEV, requires_grad=True)
        k = torch.randn(b, h, n, 64, device=DEV, requires_grad=True)
        out = mi355x_cross_attention(q, k, k)
        assert out.shape == q.shape and not out.any()
        gq, gk = torch.autograd.grad(out.sum(), (q, k))
        assert not gq.any() and not gk.any() and gk.shape == k.shape


def test_second_derivative_is_refused():
    from vsa_mi355x import mi355x_cross_attention
    q = torch.randn(1, 1, 4, 64, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(mi355x_cross_attention(q, q, q).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)


def test_layouts_of_results_and_padding_rows_left_alone():
    from vsa_mi355x import mi355x_cross_attention
    host = _inputs("bf16", 2, 3, 3, 50, 60, 64, seed=9)
    q, k, v = (_memory(x, "packed").requires_grad_() for x in host[:3])
    before = [x._base.clone() if x._base is not None else x.detach().clone() for x in (q, k, v)]
    out = mi355x_cross_attention(q, k, v)
    assert out.transpose(1, 2).is_contiguous()
    gq, gk, gv = torch.autograd.grad(out, (q, k, v), host[3].to(DEV))
    assert gq.shape == q.shape and gk.shape == k.shape
    for x, y in zip((q, k, v), before):
        assert torch.equal(x._base if x._base is not None else x.detach(), y)


def test_another_stream_and_two_calls_at_once():
    """Two streams at once: each call has a workspace of its own."""
    from vsa_mi355x import mi355x_cross_attention
    sets = [[x.to(DEV) for x in _inputs("bf16", 1, 4, 4, 1, 4000, 128, seed=s)] for s in (1, 2)]
    want = [mi355x_cross_attention(*s[:3]) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(mi355x_cross_attention(*sets[i][:3]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_step_in_a_graph_replayed():
    """Forward and backward captured once, replayed on new values; the key mask and
    the lengths are read at each replay."""
    from vsa_mi355x import mi355x_cross_attention
    b, h, sq, n, d = 2, 3, 65, 300, 64
    host = _inputs("bf16", b, h, h, sq, n, d, seed=6)
    q, k, v, do = (x.to(DEV) for x in host)
    lens = torch.tensor([n, 10], dtype=torch.int32, device=DEV)
    mask = torch.ones(b, n, dtype=torch.bool, device=DEV)
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def step():
        out = mi355x_cross_attention(*leaves, lens, mask)
        return [out, *torch.autograd.grad(out, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        g = torch.Generator().manual_seed(100 + i)
        with torch.no_grad():
            for x in (q, k, v, do):
                x.copy_(torch.randn(x.shape, generator=g))
        lens.copy_(torch.tensor([n - 70 * i, 5 * i]))
        mask.copy_(torch.rand(b, n, generator=g) < 0.8)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, step()):
            assert torch.equal(x, y), i


def test_offsets_past_32_bits():
    """Keys and values that are the last heads of a projection output of more than
    2^31 elements, and queries of another."""
    from vsa_mi355x import mi355x_cross_attention
    s, h, d = 66000, 260, 128
    buf = torch.empty((1, s, h, d), dtype=torch.bfloat16, device=DEV)
    assert buf.numel() > 1 << 31
    x = torch.randn(1, s, 2, d, device=DEV).to(torch.bfloat16)
    buf[:, :, -2:] = x
    far, near = buf[:, :, -2:].transpose(1, 2), x.transpose(1, 2)
    q = torch.randn(1, 2, 3, d, device=DEV).to(torch.bfloat16)
    assert torch.equal(mi355x_cross_attention(q, far, far), mi355x_cross_attention(q, near, near))
    few = near[:, :, :50].contiguous()
    got = mi355x_cross_attention(far, few, few)
    assert torch.equal(got, mi355x_cross_attention(near, few, few))


def test_a_blocks_attention_together():
    """The attention of a video model's block: the grid's table, q and k turned, the
    sparse attention on raster tokens, and its output's attention to a prompt, with
    the gradients of all; every key block is routed, so that nothing hangs on a tie.
    Against the same in fp32 by autograd on the CPU.  Each of the three 16-bit
    stages rounds inputs, weights and results by 2^-8 at most, so a norm of the
    difference may reach about 10 of them; a wrong term is off by its whole size."""
    import math

    from oracle import vsa_oracle as O
    from vsa_mi355x import (build_rotary_table, build_vsa_metadata, mi355x_cross_attention,
                            mi355x_rotary, mi355x_vsa_tiled)
    shape, tile, h, d, n = (4, 8, 12), (4, 4, 4), 2, 64, 77
    s, nb = math.prod(shape), 6
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(1, s, h, d, generator=g).to(torch.bfloat16) for _ in range(4))
    ek, ev = (torch.randn(1, h, n, d, generator=g).to(torch.bfloat16) for _ in range(2))
    lens = torch.tensor([50], dtype=torch.int32)
    cos, sin = build_rotary_table(shape, (16, 24, 24), device=DEV)
    leaves = [x.to(DEV).requires_grad_() for x in (q, k, v, ek, ev)]
    a = mi355x_vsa_tiled(*leaves[:3], shape, nb, tile, token_major=True, rotary=(cos, sin))
    out = mi355x_cross_attention(a.transpose(1, 2), *leaves[3:], lens.to(DEV))
    grads = torch.autograd.grad(out, leaves, do.transpose(1, 2).to(DEV))

    meta = build_vsa_metadata(shape, tile, device=DEV)
    tpi, npi = meta["tile_partition_indices"].cpu(), meta["non_pad_index"].cpu()
    vbs = meta["variable_block_sizes"].cpu()
    host = [x.float().requires_grad_() for x in (q, k, v, ek, ev)]
    c, w = cos.cpu()[None, None], sin.cpu()[None, None]

    def turn(x):
        x1, x2 = x[..., :d // 2], x[..., d // 2:]
        return torch.cat((x1 * c - x2 * w, x2 * c + x1 * w), -1)

    qt, kt, vt = (x.transpose(1, 2) for x in host[:3])
    qt, kt = turn(qt), turn(kt)
    tl = [torch.zeros(1, h, nb * 64, d).index_copy(2, npi, x[:, :, tpi]) for x in (qt, kt, vt)]
    o = O.torch_vsa(*tl, vbs, vbs, nb, tile)
    back = torch.empty(s, dtype=torch.long)
    back[tpi] = npi
    o = o[:, :, back]
    p = torch.softmax(o @ host[3][:, :, :50].transpose(2, 3) * d ** -0.5, -1)
    ref = p @ host[4][:, :, :50]
    want = torch.autograd.grad(ref, host, do.transpose(1, 2).float())
    for x, y in zip([out, *grads], [ref, *want]):
        x = x.detach().float().cpu()
        rel = ((x - y).norm() / y.norm()).item()
        print(f"relative difference {rel:.2e}", flush=True)
        assert rel <= 10 * 2.0 ** -8
    # and the pieces: the tiled op's rotary is mi355x_rotary's, bit for bit
    with torch.no_grad():
        qr, kr = mi355x_rotary(*(x.transpose(1, 2) for x in leaves[:2]), cos, sin)
        again = mi355x_vsa_tiled(qr.transpose(1, 2), kr.transpose(1, 2), leaves[2], shape, nb, tile,
                                 token_major=True)
    assert torch.equal(a, again)


@pytest.mark.parametrize("how", ["one", "lens", "mask", "both"])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 40), ("fp32", 64), ("bf16", 256)])
def test_a_single_valid_key_has_no_gradient_of_q_and_k(dtype, d, how):
    """Its weight is 1 whatever the scores: the output is its value, dv the sum of the
    outputs' gradients, dq and dk exactly zero.  The other sample is an ordinary one."""
    from vsa_mi355x import mi355x_cross_attention
    n = 1 if how == "one" else 200
    host = _inputs(dtype, 2, 4, 2, 37, n, d, seed=41)
    lens = mask = None
    at = 0
    if how in ("lens", "both"):
        lens = torch.tensor([n if how == "both" else 1, 150], dtype=torch.int32)
    if how in ("mask", "both"):
        at = 170
        mask = torch.zeros(2, n, dtype=torch.bool)
        mask[0, at] = True
        mask[1, ::3] = True
    lens, mask = (None if x is None else x.to(DEV) for x in (lens, mask))
    leaves = [x.to(DEV).requires_grad_() for x in host[:3]]
    out = mi355x_cross_attention(*leaves, lens, mask)
    grads = torch.autograd.grad(out, leaves, host[3].to(DEV))
    ref, tol = reference(*(x.to(DEV) for x in host), lens, mask)
    _check(NAMES, [out, *grads], ref, tol)
    if dtype != "fp32":   # (there the weight and its inverse round: within the bound above)
        one = leaves[2][0, :, at:at + 1].repeat_interleave(2, 0)
        assert torch.equal(out[0], one.expand_as(out[0]))
    for x in grads[:2]:
        assert not x[0].any() and (how == "one" or x[1].any())


@pytest.mark.parametrize("n,d", [(3, 40), (60, 128), (100, 64)])
def test_few_keys_take_no_more_rounding_than_their_results(n, d):
    """dk of a prompt of a few keys is off by little more than its own rounding: dS
    enters the product with its rounding's rest."""
    from vsa_mi355x import mi355x_cross_attention
    host = _inputs("bf16", 3, 8, 4, 691, n, d, seed=43)
    leaves = [x.to(DEV).requires_grad_() for x in host[:3]]
    grads = torch.autograd.grad(mi355x_cross_attention(*leaves), leaves, host[3].to(DEV))
    ref, _ = reference(*(x.to(DEV) for x in host))
    for name, x, y in zip(NAMES[1:], grads, ref[1:]):
        # the rest is itself rounded, 2^-16 of dS, and the fp32 sums are off by less:
        # 1/256 of the result's own rounding, which 1.15 leaves room for (dS rounded
        # once would make it sqrt(2)); P enters dv rounded once
        if name != "dv":
            own = (y.to(torch.bfloat16).double() - y).norm()
            assert (x.double() - y).norm() <= 1.15 * own, name


@pytest.mark.parametrize("dtype,n,d", [("bf16", 2000, 128), ("fp16", 1500, 64), ("bf16", 900, 256),
                                       ("fp16", 1000, 40)])
def test_spread_weights_lose_no_more_than_the_results_rounding(dtype, n, d):
    """Where the weights spread over many keys, dS is far smaller than dP and delta:
    dq stays within its own rounding, with delta from the output and its rest."""
    from vsa_mi355x import mi355x_cross_attention
    host = _inputs(dtype, 1, 2, 2, 300, n, d, seed=47)
    host[3] *= 8   # (clear of fp16's subnormals: dS is about 1e-2)
    leaves = [x.to(DEV).requires_grad_() for x in host[:3]]
    dq, = torch.autograd.grad(mi355x_cross_attention(*leaves), leaves[:1], host[3].to(DEV))
    ref, _ = reference(*(x.to(DEV) for x in host))
    # a rest is off by 1/508 of the output's unit in the last place: delta by less than
    # 2^-15 of sum |dO O|, dS by as much of P delta, against 2^-9 of dq in its rounding
    own = (ref[1].to(DTYPES[dtype]).double() - ref[1]).norm()
    assert (dq.double() - ref[1]).norm() <= 1.15 * own


@pytest.mark.parametrize("d", [64, 60])
def test_copied_views_keep_their_order_with_and_without_gradients(d):
    """Token-major views whose rows do not start on 16 bytes are copied; the result
    and the gradients are dense in the order of the view all the same."""
    from vsa_mi355x import mi355x_cross_attention
    b, h, sq, n = 2, 3, 33, 20
    host = _inputs("bf16", b, h, h, sq, n, d, seed=53)

    def odd(x):   # token-major, 2 bytes off
        buf = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)
        view = buf[1:].view(x.shape[0], x.shape[2], x.shape[1], d).transpose(1, 2)
        view.copy_(x)
        return view
    q, k, v, do = (odd(x) for x in host)
    want = torch.empty(b, sq, h, d).transpose(1, 2).stride()
    with torch.no_grad():
        plain = mi355x_cross_attention(q, k, v)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = mi355x_cross_attention(*leaves)
    if d % 8 == 0:
        assert plain.stride() == out.stride() == want
    assert torch.equal(plain, out) and plain.stride() == out.stride()
    grads = torch.autograd.grad(out, leaves, do)
    ref, tol = reference(*(x.to(DEV) for x in host))
    _check(NAMES, [out, *grads], ref, tol)
