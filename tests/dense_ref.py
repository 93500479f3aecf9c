"""Plain 64-bit forms of the dense operators (linear, qk_norm_rope, sparse_attention) on the CPU, each with the bound of
what a correct fp32-accumulating implementation may differ by, derived from the operation counts.

u(t) = eps(t) / 2 is half a step of type t relative to the value; one fp32 operation is off by at most 2^-24 of its result.
Matrix products: a sum of n products of 16-bit (or exact 8-bit) values is off by at most n 2^-23 sum |x w| (each of n
additions rounds once, and up to twice inside the matrix instruction); fp32 products add one rounding each: the same.
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}  # half the last subnormal step (at least)


def act64(y, act):
    if act == "relu":
        return torch.clamp(y, min=0)
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return 0.5 * y * torch.erfc(-y * math.sqrt(0.5))
    if act == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def linear(x, w, bias=None, *, a_scale=1.0, w_scale=None, act="none", residual=None, out_dtype):
    """(result, bound). Activations have slopes of at most 1.13 and are evaluated within 2^-20 |y| + 2^-20 |act(y)| (erf and
    tanh within 2e-7 absolute, exp2 and reciprocal within 1 ulp each, their argument within 2^-23 |y| relative)."""
    x, w = x.cpu().double(), w.cpu().double()
    sc = torch.ones(w.shape[0], dtype=torch.float64) if w_scale is None else w_scale.cpu().double()
    sc = sc * a_scale
    y = (x @ w.t()) * sc
    size = (x.abs() @ w.abs().t()) * sc.abs()
    err = (x.shape[1] + 4) * 2.0 ** -23 * size
    if bias is not None:
        y = y + bias.cpu().double()
        err = err + 2.0 ** -23 * (y.abs() + size)
    z = act64(y, act)
    if act != "none":
        err = 1.13 * err + 2.0 ** -20 * (y.abs() * torch.exp(-y.abs() / 4) + z.abs()) + 2.0 ** -22 * y.abs()
    if residual is not None:
        z = z + residual.cpu().double()
        err = err + 2.0 ** -23 * z.abs()
    return z, err * 1.01 + U[out_dtype] * (z.abs() + err) + TINY[out_dtype]


def norm_rope(x, weight, bias, coords, freqs, *, layer, interleaved, eps=1e-6):
    """(result, bound): a norm's factors are within 2^-20 relative (sums of up to 128 squares, one root, one division), the
    centred value within 2^-21 of the row's largest, a turn's sine and cosine within 2^-21."""
    t = x.dtype
    x = x.cpu().double()
    D = x.shape[-1]
    u = x - x.mean(-1, keepdim=True) if layer else x
    big = x.abs().amax(-1, keepdim=True)
    r = 1 / torch.sqrt((u * u).mean(-1, keepdim=True) + eps)
    w = torch.ones(D, dtype=torch.float64) if weight is None else weight.cpu().double()
    b = torch.zeros(D, dtype=torch.float64) if bias is None else bias.cpu().double()
    y = u * r * w + b
    err = 2.0 ** -20 * (y.abs() + b.abs() + (u * r * w).abs()) + (2.0 ** -21 * big * r * w.abs() if layer else 0)
    ang = coords.cpu()[:, 1:].double() @ freqs.cpu().double().t()  # [M, P]
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    P = freqs.shape[0]
    ia = torch.arange(P) * 2 if interleaved else torch.arange(P)
    ib = ia + 1 if interleaved else ia + D // 2
    z, e = y.clone(), err.clone()
    a, b2 = y[..., ia], y[..., ib]
    both = a.abs() + b2.abs()
    z[..., ia] = a * c - b2 * s
    z[..., ib] = a * s + b2 * c
    e[..., ia] = e[..., ib] = err[..., ia] + err[..., ib] + 2.0 ** -20 * both
    return z, e + U[t] * (z.abs() + e) + TINY[t]


def attention(q, k, v, offsets, kv_offsets=None, *, index=None, kv_index=None, coords=None, kv_coords=None,
              slopes=None, kv_mask=None, cap=0.0, scale=None):
    """(result, bound, covered rows). A score x is off by at most dx: its product's D 2^-23 sum |q k|, 2^-22 of the cap, and
    2^-22 of itself and its bias. A weight is then off by (2 max dx + u + n 2^-22 + 2^-21) of itself, u for its rounding to
    the inputs' type (fp16: or half its last subnormal step, with a sum of weights of at least 1), and so is the result
    of sum p |v|, before its own rounding."""
    t = q.dtype
    q, k, v = (a.cpu().double() for a in (q, k, v))
    Mq, Hq, D = q.shape
    Mk, Hk = k.shape[:2]
    own = kv_offsets is None
    if own:
        kv_offsets, kv_index, kv_coords = offsets, index, coords
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros((Mq, Hq, D), dtype=torch.float64)
    tol = torch.full((Mq, Hq, D), TINY[t], dtype=torch.float64)
    covered = torch.zeros(Mq, dtype=torch.bool)
    qi = torch.arange(Mq) if index is None else index.cpu().long()
    ki = torch.arange(Mk) if kv_index is None else kv_index.cpu().long()
    seen = torch.ones(Mk, dtype=torch.bool) if kv_mask is None else kv_mask.cpu().bool()
    qo, ko = offsets.cpu().clamp(0, len(qi)).tolist(), kv_offsets.cpu().clamp(0, len(ki)).tolist()
    of = torch.arange(Hq) // (Hq // Hk)
    for s in range(len(qo) - 1):
        qr, kr = qi[qo[s]:qo[s + 1]], ki[ko[s]:ko[s + 1]]
        qr = qr[(qr >= 0) & (qr < Mq)]
        kr = kr[(kr >= 0) & (kr < Mk)]
        kr = kr[seen[kr]]
        covered[qr] = True
        if not len(qr):
            continue
        if not len(kr):
            out[qr] = 0
            continue
        qs, ks, vs = q[qr].transpose(0, 1), k[kr][:, of].transpose(0, 1), v[kr][:, of].transpose(0, 1)
        x = qs @ ks.transpose(1, 2) * scale
        dx = (D + 4) * 2.0 ** -23 * scale * (qs.abs() @ ks.abs().transpose(1, 2))
        if cap:
            x = cap * torch.tanh(x / cap)
            dx = dx + 2.0 ** -22 * cap
        dx = dx + 2.0 ** -22 * x.abs()
        if slopes is not None:
            far = (coords.cpu()[qr][:, None, 1:].double() - kv_coords.cpu()[kr][None, :, 1:].double()).abs()
            sl = slopes.cpu().double()
            b = (sl[:, None, None, :] * far[None]).sum(-1)
            x = x - b
            dx = dx + 2.0 ** -21 * (sl.abs()[:, None, None, :] * far[None]).sum(-1) + 2.0 ** -22 * x.abs()
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
        # keys that cannot matter (weight below 2^-60) do not count towards the largest score error
        dmax = torch.where(p > 2.0 ** -60, dx, torch.zeros_like(dx)).amax(-1, keepdim=True)
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        o = p @ vs
        n = len(kr)
        rel = torch.expm1(2 * dmax) + U[t] + n * 2.0 ** -22 + 2.0 ** -21
        e = rel * (p @ vs.abs())
        if t == torch.float16:
            e = e + n * 2.0 ** -25 * vs.abs().amax(1, keepdim=True)
        out[qr] = o.transpose(0, 1)
        tol[qr] = (e + U[t] * (o.abs() + e) + TINY[t]).transpose(0, 1)
    return out, tol, covered


def assert_within(got, want, tol, what=""):
    got = got.detach().cpu().double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN at other places ({int(torch.isnan(got).sum())}, {int(nan.sum())})"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    far = torch.where(nan | inf, torch.zeros_like(want), (got - want).abs() - tol)
    worst = int(far.argmax()) if far.numel() else 0
    assert not far.numel() or float(far.max()) <= 0, (
        f"{what}: {int((far > 0).sum())} of {far.numel()} outside; worst {got.flatten()[worst]:.9g} for "
        f"{want.flatten()[worst]:.9g} +- {tol.flatten()[worst]:.3g} at {worst}")
