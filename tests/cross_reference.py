"""Cross attention in 64 bits, with the bounds its kernels have to stay in.

The bounds follow the kernels' roundings, to first order, element by element.
u is half an eps of the type, e = 2^-24 the rounding of an fp32 operation:

* a score is a sum of D products in fp32: off by at most D e sum|q||k| scale,
  and its exponent by a few e of its size; E is the largest of these, so a weight
  p is off by 2 E relative (its row's largest score and its own), and by N e in
  the row sum: R = 4 E + (N + 16) e, N the keys (queries for dK and dV);
* p is rounded to T for P V and P^T dO, dS for dS K and dS^T Q: u each, and what
  is smaller than T's subnormals is lost, half of one at most (Z); so is a weight
  below 2^-126, which the exponential unit makes 0, and an operand below 2^-126,
  which the matrix unit may take as 0 (2^-125 for both);
* delta is taken from O as stored in T and what that left over, rounded to T:
  off by u^2 sum|dO||O|, and by what O itself is off before it is stored;
* every result is rounded to T once: u (half the smallest subnormal below).
"""

import torch


def reference(q, k, v, do=None, lens=None, mask=None, scale=None):
    """([out, dq, dk, dv], [their bounds]) in float64, [B, H, S, D] each; the
    gradients only with ``do``."""
    dt, (b, h, sq, d) = q.dtype, q.shape
    hk, n = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    u, e = torch.finfo(dt).eps / 2, 2.0 ** -24
    floor = torch.finfo(dt).tiny * u
    Z = floor + 2.0 ** -125
    f = lambda *s: torch.zeros(s, dtype=torch.float64, device=q.device)   # noqa: E731
    out, t_out, dq, t_dq = (f(b, h, sq, d) for _ in range(4))
    dk, t_dk, dv, t_dv = (f(b, hk, n, d) for _ in range(4))
    for i in range(b):
        ok = torch.ones(n, dtype=torch.bool, device=q.device)
        if lens is not None:
            ok &= torch.arange(n, device=q.device) < int(lens[i])
        if mask is not None:
            ok &= mask[i]
        on = ok.nonzero().flatten()
        if not on.numel():
            continue
        for j in range(h):
            g = j // (h // hk)
            Q = q[i, j].double()
            K, V = k[i, g][on].double(), v[i, g][on].double()
            s = Q @ K.t().contiguous() * scale
            E = (Q.abs() @ K.abs().t().contiguous()).max() * abs(scale) * (d + 4) * e
            p = torch.softmax(s, -1)
            o = p @ V
            R = 4 * E + (on.numel() + 16) * e
            av = p @ V.abs()
            out[i, j], t_out[i, j] = o, (u + R) * av + u * o.abs() + Z * V.abs().sum(0) + floor
            if do is None:
                continue
            R = R + (sq * (h // hk) + 16) * e
            G = do[i, j].double()
            dp = G @ V.t().contiguous()
            delta = (G * o).sum(-1, keepdim=True)
            e_dp = (d + 4) * e * (G.abs() @ V.abs().t().contiguous())
            e_delta = ((u + R) * (G.abs() * av) + (u * u + 2 * d * e) * (G * o).abs()
                       + Z * G.abs()).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            t_ds = (u + R) * ds.abs() + p * (e_dp + e_delta + 2 * e * (dp.abs() + delta.abs())) + \
                Z * (dp.abs() + delta.abs() + 1)
            dq[i, j] = ds @ K * scale
            t_dq[i, j] = t_ds @ K.abs() * abs(scale) + (u + 4 * e) * dq[i, j].abs() + floor
            dk[i, g].index_add_(0, on, ds.t().contiguous() @ Q * scale)
            t_dk[i, g].index_add_(0, on, t_ds.t().contiguous() @ Q.abs() * abs(scale))
            dv[i, g].index_add_(0, on, p.t().contiguous() @ G)
            t_dv[i, g].index_add_(0, on, (u + R) * (p.t().contiguous() @ G.abs()) +
                                Z * G.abs().sum(0))
    if do is None:
        return [out], [t_out]
    t_dk += (u + 4 * e) * dk.abs() + floor
    t_dv += (u + 4 * e) * dv.abs() + floor
    return [out, dq, dk, dv], [t_out, t_dq, t_dk, t_dv]
