"""Definitions of the operators for token sequences in 64 bits on the CPU, and how far a result in `dtype` may be from them.

The bounds are arithmetic, element by element.  u is half a step of the type (its rounding, relative).  A result is rounded once (u); the
weights P and dS are rounded to a 16-bit type before the second product (another u of each term); what is left is fp32: a sum of n
terms is off by at most n 2^-24 of the sum of their magnitudes, a score of magnitude s that is off by e moves its
weight by the factor exp(e), and the hardware's exp2 is off by 2^-21 relative with its argument's rounding.  fp16 has an
absolute floor too: half of its smallest step, 2^-25, for every value that is rounded.  The other types' floor is fp32's smallest
normal number, 2^-126: what is below it is held as zero or with fewer bits -- a weight exp(s - m) with s - m < -88 among
scores of hundreds is such a value, and so is a gradient made of such weights, which no relative bound covers."""
import math

import torch

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
E32 = 2.0 ** -24


def floor_of(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def visible(n, W, ns, length):
    i = torch.arange(n)
    d = i[:, None] - i[None, :]
    return (d >= 0) & ((d < W) | (i[None, :] < ns)) & (i[:, None] < length) & (i[None, :] < length)


def rotate(x, pos, tables, inverse=False):
    """x [B,H,N,C]; pos [A,N] or [B,A,N]."""
    x = x.double()
    y = x.clone()
    if pos.dim() == 2:
        pos = pos[None].expand(x.shape[0], -1, -1)
    at = 0
    for a, t in enumerate(tables):
        R = t.shape[1]
        p = pos[:, a].long()
        cs = t.double()[p.clamp(0, t.shape[0] - 1)][:, None]
        c, s = cs[..., 0], cs[..., 1] * (-1 if inverse else 1)
        on = (p >= 0)[:, None, :, None]
        u, w = x[..., at:at + R], x[..., at + R:at + 2 * R]
        y[..., at:at + R] = torch.where(on, u * c - w * s, u)
        y[..., at + R:at + 2 * R] = torch.where(on, u * s + w * c, w)
        at += 2 * R
    return y


def rotate_bound(x, pos, tables, dtype, inverse=False):
    """|y - rotate(x)|: two products and a sum in fp32, one rounding."""
    m = rotate(x, pos, tables, inverse).abs()
    mag = x.double().abs()
    at = 0
    for t in tables:
        R = t.shape[1]
        pair = mag[..., at:at + R] + mag[..., at + R:at + 2 * R]
        mag[..., at:at + R], mag[..., at + R:at + 2 * R] = pair, pair
        at += 2 * R
    return HALF[dtype] * m * (1 + 4 * E32) + 4 * E32 * mag + floor_of(dtype)


def attention(q, k, v, lens, W, ns, scale, do=None, dtype=None):
    """(values, bounds): dicts with o, lse and, with `do`, dq, dk, dv."""
    dtype = dtype or q.dtype
    q, k, v = (t.double() for t in (q, k, v))
    B, Hq, N, d = q.shape
    Hkv, dv_ = k.shape[1], v.shape[3]
    G = Hq // Hkv
    u, tiny = HALF[dtype], floor_of(dtype)
    u2 = u if dtype != torch.float32 else 0.0            # the second rounding, of P and dS
    val = dict(o=torch.zeros(B, Hq, N, dv_, dtype=torch.float64), lse=torch.full((B, Hq, N), -math.inf, dtype=torch.float64))
    err = {n: torch.zeros_like(t) for n, t in val.items()}
    if do is not None:
        do = do.double()
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            val[n], err[n] = torch.zeros_like(t), torch.zeros_like(t)
    for b in range(B):
        n = N if lens is None else max(0, min(N, int(lens[b])))
        see = visible(n, W, ns, n)
        for h in range(Hq):
            g = h // G
            Q, K, V = q[b, h, :n], k[b, g, :n], v[b, g, :n]
            S = (Q @ K.T * scale).masked_fill(~see, -math.inf)
            P = torch.softmax(S, -1) if n else S
            serr = ((d + 3) * E32 * (Q.abs() @ K.abs().T) * abs(scale)).masked_fill(~see, 0)
            smax = serr.amax(-1, keepdim=True) if n else serr
            # exp of a score that is off by serr, of a sum of n such terms, of a result divided by it
            tau = 2 * smax + (2 * n + 16) * E32 + 2.0 ** -20 + 4 * E32 * S.masked_fill(~see, 0).abs()
            val["o"][b, h, :n] = O = P @ V
            PV = P @ V.abs()
            eo = ((P * (u2 + tau) + tiny) * see) @ V.abs()
            err["o"][b, h, :n] = u * O.abs() + eo * (1 + u) + tiny
            val["lse"][b, h, :n] = torch.logsumexp(S, -1) / math.log(2) if n else 0
            err["lse"][b, h, :n] = (smax[:, 0] + tau.amax(-1)) * 1.5 + 4 * E32 * val["lse"][b, h, :n].abs() if n else 0
            if do is None:
                continue
            D = do[b, h, :n]
            dP = D @ V.T
            delta = (D * O).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            # delta is made from the rounded o; the backward pass takes P from the lse, which is off too
            edelta = ((u * O.abs() + eo + tiny) * D.abs()).sum(-1, keepdim=True) + (dv_ + 3) * E32 * (O.abs() * D.abs()).sum(-1, keepdim=True)
            edP = (dv_ + 3) * E32 * (D.abs() @ V.abs().T)
            eP = P * (2 * tau) + tiny * see
            eS = (dS.abs() * u2 + eP * (dP - delta).abs() + P * (edP + edelta + 2 * E32 * (dP.abs() + delta.abs()))) * (1 + u) + tiny * see
            eSn = eS + (n * G + 8) * E32 * dS.abs()
            val["dq"][b, h, :n] = dS @ K * scale
            err["dq"][b, h, :n] = eSn @ K.abs() * abs(scale)
            val["dk"][b, g, :n] += dS.T @ Q * scale
            err["dk"][b, g, :n] += eSn.T @ Q.abs() * abs(scale)
            val["dv"][b, g, :n] += P.T @ D
            err["dv"][b, g, :n] += ((P * (u2 + (n * G + 8) * E32) + eP + tiny) * see).T @ D.abs()
    for x in ("dq", "dk", "dv"):
        if x in val:
            err[x] = err[x] * (1 + u) + u * val[x].abs() + tiny
    return val, err


def decode(q, k, v, W, ns, scale, dtype=None):
    """One sequence: q [Hq, d] at the last of the n positions of k, v [Hkv, n, .] -> (o, bound) [Hq, dv]."""
    n = k.shape[1]
    qq = torch.zeros(1, q.shape[0], n, q.shape[1], dtype=q.dtype)
    qq[0, :, n - 1] = q
    val, err = attention(qq, k[None], v[None], None, W, ns, scale, dtype=dtype or q.dtype)
    return val["o"][0, :, n - 1], err["o"][0, :, n - 1]


def check(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), f"{what}: other infinities"
    over = ((got - want).abs() - bound)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, (
        f"{what}: {int((over > 0).sum())} values beyond their bound, worst {float(((got - want).abs() / bound.clamp(min=1e-300))[fin].max()):.3g} times")
