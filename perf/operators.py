"""Cases of the operators around the sparse attention of a video model's block: the
rotary positions of its latent grid, and its cross attention to an encoder's states.

With ``own`` false, ``run`` computes an operator in its plain form (torch operations
in 32 bits; angles in 64), with ``own`` true by the package's entry points.

A case's keys:

* ``op``: "table", "rotary" or "cross"; ``train``: the gradients are computed too;
* ``dtype``; ``B``; ``H`` query heads, ``Hk`` key heads; ``Sq``, ``Skv`` tokens (rotary: Sq for
  both); ``D``;
* ``layout``: "head" for [B, H, S, D] memory, "token" for per-head views of [B, S, H, D]
  memory, "packed" for slices of one [B, S, Hq + 2 Hk, D] projection (rotary; of
  [B, S, 2 Hk, D] for a cross attention's k and v, whose q is as in "token");
* table: ``grid`` "TxHxW", ``axes`` channels of each axis "t,h,w", ``start`` first position
  of the first axis, ``method``, ``factor`` and ``original`` (its long-context scaling);
* rotary: ``rot`` channels that turn, ``interleaved``, ``indexed`` (each sample has positions of
  its own, -1 where a token is padding);
* cross: ``lens`` "full" or "ragged" (sample b of B has (b + 1) / B of the keys), ``empty``
  (the first sample has none), ``holes`` (a key mask that drops an eighth of the keys).
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEFAULTS = dict(op="cross", train=False, dtype="bf16", B=1, H=1, Hk=0, Sq=1, Skv=0, D=128,
                layout="head", grid="", axes="", start=0, method="linear", factor=1.0, original=0,
                rot=0, interleaved=False, indexed=False, lens="full", empty=False, holes=False)
THETA = 10000.0
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "simple-vsa_amd")


def _package():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import vsa_mi355x
    return vsa_mi355x


def _case(name=None, **kw):
    c = dict(DEFAULTS, **kw)
    c["Hk"] = c["Hk"] or c["H"]
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # a latent grid's table, made once a resolution
        _case("table_grid", op="table", grid="21x30x52", axes="44,42,42"),
        # positions far into a long sequence, scaled beyond the trained length
        _case("table_far", op="table", grid="92160x1x1", axes="128,0,0", start=1000000,
              method="yarn", factor=16.0, original=65536),
        # one new token of each sample, where a call's own cost counts
        _case("rotary_token", op="rotary", B=4, H=12, Sq=1, rot=128, indexed=True),
        # a training step of a 12-head model at 16k tokens, views of the projections' output
        _case("rotary_train", op="rotary", train=True, H=12, Sq=16384, rot=128, interleaved=True,
              layout="token"),
        # the headline benchmark's tokens: 40 heads, 41k of them
        _case("rotary_video", op="rotary", H=40, Sq=40960, rot=128),
        # slices of one packed projection, part of an uncommon head, samples padded to the longest
        _case("rotary_packed_odd", op="rotary", dtype="fp16", B=2, H=10, Sq=8191, D=80, rot=60,
              interleaved=True, layout="packed", indexed=True),
        # a single query token of each sample on its prompt
        _case("cross_token", B=8, H=12, Sq=1, Skv=512, lens="ragged"),
        # a few latent queries that read a whole video
        _case("cross_few_long", H=12, Sq=64, Skv=40960),
        # the headline benchmark's tokens on a prompt of 512, at inference
        _case("cross_video", H=40, Sq=40960, Skv=512, layout="token"),
        # a training step at 16k tokens, prompts of two lengths, k and v of one projection
        _case("cross_train", train=True, B=2, H=12, Sq=16384, Skv=512, layout="packed",
              lens="ragged"),
        # small heads, half precision, a prompt with dropped tokens
        _case("cross_train_d64", train=True, dtype="fp16", H=24, Sq=40960, Skv=226, D=64,
              holes=True),
        # 32 bits, shared key heads, odd sizes, a sample without a prompt
        _case("cross_train_fp32", train=True, dtype="fp32", B=2, H=10, Hk=5, Sq=3001, Skv=333,
              D=80, lens="ragged", empty=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["table", "rotary", "rotary", "cross", "cross", "cross"])
    if op == "table":
        if rng.random() < 0.5:
            grid = "%dx%dx%d" % (rng.randint(1, 33), rng.randint(2, 60), rng.randint(2, 60))
            axes = rng.choice(["44,42,42", "16,56,56", "22,20,22", "0,32,32"])
            return _case(op=op, grid=grid, axes=axes, method=rng.choice(["linear", "ntk"]),
                         factor=rng.choice([1.0, 2.0, 4.0]))
        return _case(op=op, grid="%dx1x1" % _log_int(rng, 1, 92160),
                     axes="%d,0,0" % rng.choice([128, 64, 60, 256]),
                     start=_log_int(rng, 1, 4000000), method=rng.choice(["linear", "ntk", "yarn"]),
                     factor=rng.choice([1.0, 3.0, 16.0]), original=rng.choice([4096, 16384]))
    d = rng.choice([64, 128, 128, 128, 256, 80, 96, 40])
    hk = rng.choice([1, 2, 3, 5, 8, 12, 24])
    h = hk * rng.choice([1, 1, 1, 2, 4])
    kw = dict(op=op, train=rng.random() < 0.6, dtype=rng.choice(["bf16"] * 4 + ["fp16", "fp32"]),
              B=rng.choice([1, 1, 2, 3, 8]), H=h, Hk=hk, D=d,
              layout=rng.choice(["head", "token", "packed"]))
    if op == "rotary":
        kw.update(Sq=_log_int(rng, 1, 92160), rot=rng.choice([d, d, d // 2, d - 4]),
                  interleaved=rng.random() < 0.5, indexed=rng.random() < 0.3)
    else:
        kw.update(Sq=_log_int(rng, 1, 92160), Skv=_log_int(rng, 1, 40960),
                  lens=rng.choice(["full", "ragged"]), holes=rng.random() < 0.3)
        kw["empty"] = kw["B"] > 1 and rng.random() < 0.2
    return _case(**kw)


def _cost(case):
    """Seconds of the plain form, about: its 32-bit products, and the passes over its scores
    and its tokens."""
    w = work(case)
    scores = case["B"] * case["H"] * case["Sq"] * case["Skv"] if case["op"] == "cross" else 0
    return w["flops"] / 8e13 + (w["bytes"] + 16 * scores) / 2e12


def _scores(case):
    return case["B"] * case["H"] * case["Sq"] * case["Skv"]


def draw(rng):
    most = max(_cost(c) for c in listed())
    widest = max(_scores(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most and _scores(case) <= widest and work(case)["bytes"] <= 2e9:
            return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _triple(text, sep="x"):
    return tuple(int(x) for x in text.split(sep))


def _lens(case):
    """Keys of each sample."""
    b, n = case["B"], case["Skv"]
    lens = [n] * b if case["lens"] == "full" else [max(1, n * (i + 1) // b) for i in range(b)]
    return [0] + lens[1:] if case["empty"] else lens


def _in_memory(x, layout):
    """[B, H, S, D] values in the case's memory order."""
    return x if layout == "head" else x.transpose(1, 2).contiguous().transpose(1, 2)


def _split(x, layout, heads):
    """Tensors of `heads` heads each out of [B, sum(heads), S, D] values: slices of one
    [B, S, sum(heads), D] projection, or tensors of their own."""
    if layout == "packed":
        return _in_memory(x, "token").split(heads, dim=1)
    return [_in_memory(y.contiguous(), layout) for y in x.split(heads, dim=1)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    if c["op"] == "table":
        # another seed is another window of a longer video
        at = seed % 1009
        return dict(case=c, grid=_triple(c["grid"]), axes=_triple(c["axes"], ","),
                    start=(c["start"] + at, at, at), device=dev)
    b, h, hk, s, d = c["B"], c["H"], c["Hk"], c["Sq"], c["D"]
    if c["op"] == "rotary":
        q, k = _split(rand(b, h + 2 * hk, s, d).to(dt), c["layout"], [h, hk, hk])[:2]
        pairs = c["rot"] // 2
        f = THETA ** (-torch.arange(pairs, device=dev, dtype=torch.float64) / pairs)
        angle = (torch.arange(s, device=dev, dtype=torch.float64) + seed % 1009)[:, None] * f
        positions = None
        if c["indexed"]:   # a window of the table for each sample, padding behind its tokens
            first = torch.randint(0, s, (b, 1), generator=gen, device=dev)
            positions = (first + torch.arange(s, device=dev)) % s
            if s > 1:
                last = s - torch.arange(b, device=dev)[:, None] * s // (2 * b)
                positions = torch.where(torch.arange(s, device=dev) < last, positions, -1)
            positions = positions.to(torch.int32)
        st = dict(case=c, q=q, k=k, cos=angle.cos().float(), sin=angle.sin().float(),
                  positions=positions)
        if c["train"]:
            st["dq"], st["dk"] = (_in_memory(rand(*x.shape).to(dt), c["layout"]) for x in (q, k))
            st["q"], st["k"] = q.detach().requires_grad_(), k.detach().requires_grad_()
        return st
    n = c["Skv"]
    # keys of a prompt lean to one side, as an encoder's states do
    q = _in_memory((rand(b, h, s, d) + 0.3 * rand(b, h, 1, d)).to(dt), c["layout"])
    kv = rand(b, 2 * hk, n, d) + 0.3 * rand(b, 2 * hk, 1, d)
    k, v = _split(kv.to(dt), c["layout"], [hk, hk])
    lens = mask = None
    if c["lens"] != "full" or c["empty"]:
        lens = torch.tensor(_lens(c), dtype=torch.int32, device=dev)
    if c["holes"]:
        mask = torch.rand((b, n), generator=gen, device=dev) >= 0.125
    st = dict(case=c, q=q, k=k, v=v, lens=lens, mask=mask, scale=1.0 / math.sqrt(d))
    if c["train"]:
        st["do"] = _in_memory(rand(b, h, s, d).to(dt), c["layout"])
        for x in ("q", "k", "v"):
            st[x] = st[x].detach().requires_grad_()
    return st


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _plain_axis(case, axis, device):
    """Frequencies of an axis (64 bits) and the factor of its cosines and sines."""
    d = _triple(case["axes"], ",")[axis]
    pairs, s = d // 2, case["factor"]
    theta = THETA * s ** (d / (d - 2)) if case["method"] == "ntk" and d > 2 else THETA
    f = theta ** (-torch.arange(pairs, device=device, dtype=torch.float64) / max(pairs, 1))
    if case["method"] == "linear":
        return f / s, 1.0
    if case["method"] == "yarn":
        keep = ((case["original"] * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        return f * (keep + (1 - keep) / s), 0.1 * math.log(s) + 1
    return f, 1.0


def _plain_table(state):
    c, grid, dev = state["case"], state["grid"], state["device"]
    parts = []
    for axis in range(3):
        f, m = _plain_axis(c, axis, dev)
        pos = torch.arange(grid[axis], device=dev, dtype=torch.float64) + state["start"][axis]
        shape = [1, 1, 1, f.numel()]
        shape[axis] = grid[axis]
        angle = (pos[:, None] * f).view(shape).expand(*grid, f.numel())
        angle = angle.reshape(math.prod(grid), f.numel())
        parts.append((angle.cos() * m, angle.sin() * m))
    return [torch.cat(x, dim=1).float() for x in zip(*parts)]


def _plain_turn(x, cos, sin, positions, rot, interleaved, sign):
    y = x.detach().float()
    if positions is None:
        co, si = cos[:x.shape[2]], sin[:x.shape[2]]
    else:
        on = (positions >= 0)[..., None]
        at = positions.clamp(min=0).long()
        co, si = torch.where(on, cos[at], 1.0), torch.where(on, sin[at], 0.0)
        co, si = co[:, None], si[:, None]
    si = si * sign
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack((a * co - b * si, b * co + a * si), dim=-1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat((a * co - b * si, b * co + a * si), dim=-1)
    return torch.cat((turned, y[..., rot:]), dim=-1).to(x.dtype)


def _plain_rotary(st):
    c = st["case"]
    rest = (st["cos"], st["sin"], st["positions"], c["rot"], c["interleaved"])
    out = [_plain_turn(st[x], *rest, 1.0) for x in ("q", "k")]
    if c["train"]:
        out += [_plain_turn(st[x], *rest, -1.0) for x in ("dq", "dk")]
    return out


def _valid(st):
    """[B, 1, 1, Skv]: the keys that a sample's queries see."""
    n, dev = st["k"].shape[2], st["k"].device
    ok = torch.ones((st["k"].shape[0], n), dtype=torch.bool, device=dev)
    if st["lens"] is not None:
        ok = ok & (torch.arange(n, device=dev) < st["lens"][:, None])
    if st["mask"] is not None:
        ok = ok & st["mask"]
    return ok[:, None, None]


def _plain_cross(st):
    c, dt = st["case"], st["q"].dtype
    group = c["H"] // c["Hk"]
    q = st["q"].detach().float()
    k, v = (st[x].detach().float().repeat_interleave(group, dim=1) for x in ("k", "v"))
    ok = _valid(st)
    s = torch.matmul(q, k.transpose(-2, -1)) * st["scale"]
    s = torch.where(ok, s, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    del s
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, v)
    if not c["train"]:
        return out.to(dt)
    do = st["do"].float()
    dv = torch.matmul(p.transpose(-2, -1), do)
    ds = torch.matmul(do, v.transpose(-2, -1))
    ds = p * (ds - (do * out).sum(dim=-1, keepdim=True)) * st["scale"]
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-2, -1), q)
    dk, dv = (x.view(c["B"], c["Hk"], group, c["Skv"], c["D"]).sum(2) for x in (dk, dv))
    return [x.to(dt) for x in (out, dq, dk, dv)]


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _own_run(st):
    vsa, c = _package(), st["case"]
    if c["op"] == "table":
        original = (c["original"],) * 3 if c["method"] == "yarn" else None
        return list(vsa.build_rotary_table(st["grid"], st["axes"], THETA, start=st["start"],
                                           method=c["method"], factor=c["factor"],
                                           original_shape=original, device=st["device"]))
    if c["op"] == "rotary":
        q, k = vsa.mi355x_rotary(st["q"], st["k"], st["cos"], st["sin"], st["positions"],
                                 interleaved=c["interleaved"])
        if not c["train"]:
            return [q, k]
        grads = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
        return [q.detach(), k.detach(), *grads]
    out = vsa.mi355x_cross_attention(st["q"], st["k"], st["v"], st["lens"], st["mask"])
    if not c["train"]:
        return out
    grads = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["do"])
    return [out.detach(), *grads]


def run(state):
    if own:
        return _own_run(state)
    return {"table": _plain_table, "rotary": _plain_rotary,
            "cross": _plain_cross}[state["case"]["op"]](state)


def work(case):
    c = case
    if c["op"] == "table":
        n = math.prod(_triple(c["grid"])) * (sum(_triple(c["axes"], ",")) // 2)
        return {"bytes": 8 * n, "flops": 0}
    e = DTYPES[c["dtype"]].itemsize
    passes = 2 if c["train"] else 1
    if c["op"] == "rotary":
        rows = c["B"] * (c["H"] + c["Hk"]) * c["Sq"]
        table = 4 * c["rot"] * min(c["Sq"], 1 << 20)
        return {"bytes": passes * (2 * e * rows * c["D"] + table),
                "flops": passes * 3 * rows * c["rot"]}
    keys = sum(_lens(c))
    seen = keys * 7 / 8 if c["holes"] else keys
    queries = c["B"] * c["H"] * c["Sq"] * c["D"]
    states = 2 * c["Hk"] * keys * c["D"]
    whole = 2 * c["B"] * c["Hk"] * c["Skv"] * c["D"]   # gradients are written for every key
    moved = 2 * queries + states
    if c["train"]:
        moved += 2 * queries + whole                   # dout and dq; dk and dv
    return {"bytes": e * moved, "flops": 4.0 * c["H"] * c["Sq"] * seen * c["D"] *
            (3.5 if c["train"] else 1.0)}


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _exact_table(st):
    """Each pair of channels as a point on the circle, axis by axis."""
    c, dev, (T, H, W) = st["case"], st["device"], st["grid"]
    token = torch.arange(T * H * W, device=dev)
    index = (token // (H * W), token // W % H, token % W)
    cols = []
    for axis, d in enumerate(_triple(c["axes"], ",")):
        at = index[axis].double() + st["start"][axis]
        for i in range(d // 2):
            base, size = THETA, 1.0
            if c["method"] == "ntk" and d > 2:
                base = THETA * math.pow(c["factor"], d / (d - 2.0))
            f = math.exp(-2.0 * i / d * math.log(base))
            if c["method"] == "linear":
                f /= c["factor"]
            elif c["method"] == "yarn":
                turns = c["original"] * f / (2.0 * math.pi)
                g = min(1.0, max(0.0, (turns - 1.0) / 31.0))
                f = (1.0 - g) * f / c["factor"] + g * f
                size = 1.0 + 0.1 * math.log(c["factor"])
            cols.append(torch.polar(torch.full_like(at, size), at * f))
    z = torch.stack(cols, dim=1)
    return [z.real.contiguous(), z.imag.contiguous()]


def _exact_turn(x, turn, rot, interleaved):
    """Pairs of channels as complex numbers, times the token's unit numbers."""
    y = x.detach().double()
    head = y[..., :rot]
    pairs = head.unflatten(-1, (rot // 2, 2)) if interleaved else \
        head.unflatten(-1, (2, rot // 2)).transpose(-2, -1)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z if interleaved else z.transpose(-2, -1)
    return torch.cat((z.flatten(-2), y[..., rot:]), dim=-1)


def _exact_rotary(st):
    c = st["case"]
    turn = torch.complex(st["cos"].double(), st["sin"].double())
    if st["positions"] is not None:
        rows = torch.cat((turn, torch.ones_like(turn[:1])))   # index -1: the unit row
        turn = rows[st["positions"].long()][:, None]
    out = [_exact_turn(st[x], turn, c["rot"], c["interleaved"]) for x in ("q", "k")]
    if c["train"]:
        out += [_exact_turn(st[x], turn.conj(), c["rot"], c["interleaved"]) for x in ("dq", "dk")]
    return out


def _exact_cross(st):
    """Head by head over the valid keys alone."""
    c = st["case"]
    valid = _valid(st)[:, 0, 0]
    group = c["H"] // c["Hk"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    dq = torch.zeros_like(out) if c["train"] else None
    dk, dv = (torch.zeros(st["k"].shape, dtype=torch.float64, device=out.device)
              if c["train"] else None for _ in range(2))
    for b in range(c["B"]):
        on = valid[b].nonzero().flatten()
        if not on.numel():
            continue
        for h in range(c["H"]):
            g = h // group
            q = st["q"][b, h].detach().double()
            k, v = (st[x][b, g].detach()[on].double() for x in ("k", "v"))
            p = torch.softmax(q @ k.t().contiguous() * st["scale"], dim=-1)
            out[b, h] = p @ v
            if not c["train"]:
                continue
            do = st["do"][b, h].double()
            dp = do @ v.t().contiguous()
            ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True)) * st["scale"]
            dq[b, h] = ds @ k
            dk[b, g].index_add_(0, on, ds.t().contiguous() @ q)
            dv[b, g].index_add_(0, on, p.t().contiguous() @ do)
    return [out, dq, dk, dv] if c["train"] else out


def exact(case, seed):
    st = prepare(case, seed)
    return {"table": _exact_table, "rotary": _exact_rotary, "cross": _exact_cross}[case["op"]](st)
