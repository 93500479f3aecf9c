"""Plain 64-bit forms of the conditional layer's operators (group_norm, route, grouped_linear, combine, lora_linear) on the CPU,
each with the bound of what a correct implementation may differ by, derived from the operation counts (see dense_ref)."""
import torch

from dense_ref import TINY, U, act64, linear


def segments(offsets, P):
    o = offsets.cpu().clamp(0, P).tolist()
    return list(zip(o, o[1:]))


def _activated(y, err, act, out_dtype):
    """Of act(y), y off by err, evaluated and rounded: the terms of dense_ref.linear."""
    z = act64(y, act)
    if act != "none":
        err = 1.13 * err + 2.0 ** -20 * (y.abs() * torch.exp(-y.abs() / 4) + z.abs()) + 2.0 ** -22 * y.abs()
    return z, err


def _rounded(z, err, out_dtype):
    return z, err * 1.01 + U[out_dtype] * (z.abs() + err) + TINY[out_dtype]


def group_norm(x, groups, weight=None, bias=None, *, offsets=None, eps=1e-5, act="none", out_dtype=None):
    """(result, bound, covered rows). With sums in 64 bits mean and var are off by n 2^-53 of E[x^2] (n values summed one by one at
    the most); the rest is five fp32 operations: the difference, the root's and the scale's rounding, product and sum."""
    out_dtype = out_dtype or x.dtype
    x = x.cpu().double()
    M, C = x.shape
    offsets = torch.tensor([0, M]) if offsets is None else offsets
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.cpu().double()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.cpu().double()
    out, tol = torch.zeros((M, C), dtype=torch.float64), torch.zeros((M, C), dtype=torch.float64)
    covered = torch.zeros(M, dtype=torch.bool)
    for a, e in segments(offsets, M):
        if e <= a:
            continue
        covered[a:e] = True
        u = x[a:e].reshape(e - a, groups, C // groups)
        mean = u.mean(dim=(0, 2), keepdim=True)
        square = (u * u).mean(dim=(0, 2), keepdim=True)
        d = u - mean
        var = (d * d).mean(dim=(0, 2), keepdim=True)
        r = 1 / torch.sqrt(var + eps)
        n = (e - a) * (C // groups)
        off = (n + 8) * 2.0 ** -53  # of E[x^2]
        # relative error of r from var's; the mean's, over the spread
        rel = off * square / (var + eps) + 2.0 ** -22
        y = (d * r).reshape(e - a, C) * w
        err = (rel * (d * r).abs() + off * square.sqrt() * r).reshape(e - a, C) * w.abs() + 2.0 ** -22 * y.abs()
        y = y + b
        err = err + 2.0 ** -23 * (y.abs() + b.abs())
        z, err = _activated(y, err, act, out_dtype)
        out[a:e], tol[a:e] = _rounded(z, err, out_dtype)
    return out, tol, covered


def route(logits, k, *, score="softmax", normalize=False, mask=None):
    """(weights, bound, experts, offsets, pairs, rows); whole numbers are exact. An exponential is off by 2^-22 and 2^-23 of its
    argument, a sum of E by E 2^-23, quotients by 2^-24 each."""
    x = logits.cpu().double()
    M, E = x.shape
    there = ~torch.isnan(x) & (x > float("-inf"))
    by = torch.where(there, x, torch.full_like(x, float("-inf")))
    order = torch.sort(by, dim=-1, descending=True, stable=True).indices
    # (a logit that is not chosen comes last, also behind one of the least finite value)
    order = order.gather(1, torch.sort((~there).gather(1, order).to(torch.int8), dim=-1, stable=True).indices)[:, :k]
    ok = there.gather(1, order)
    v = x.gather(1, order)
    if score == "softmax":
        top = by.amax(-1, keepdim=True)
        top = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
        w = torch.exp(v - top) / torch.exp(x - top).sum(-1, keepdim=True)
        rel = 2.0 ** -20 + E * 2.0 ** -23 + 2.0 ** -22 * (v - top).abs().nan_to_num(0, 0, 0)
    else:
        # (over their sum: of their logarithms, for sigmoids far below the least number are not lost beside each other)
        w = torch.sigmoid(v)
        if normalize:
            log = torch.where(ok, torch.nn.functional.logsigmoid(v), torch.full_like(v, float("-inf")))
            top = log.amax(-1, keepdim=True)
            w = torch.where(torch.isinf(top), torch.zeros_like(w), torch.exp(log - top))
        rel = 2.0 ** -20 + 2.0 ** -22 * v.abs().clamp(max=200).nan_to_num(0, 0, 0)
    w = torch.where(ok, w, torch.zeros_like(w))
    if normalize:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
        rel = rel + rel.amax(-1, keepdim=True) + k * 2.0 ** -23
    experts = torch.where(ok, order, -1)
    if mask is not None:
        on = mask.cpu().bool()[:, None]
        w, experts = torch.where(on, w, torch.zeros_like(w)), torch.where(on, experts, -1)
    flat = experts.reshape(-1).tolist()
    lists = [[] for _ in range(E)]
    for i, e in enumerate(flat):
        if e >= 0:
            lists[e].append(i)
    pairs = [i for group in lists for i in group]
    offsets = torch.tensor([0] + [len(group) for group in lists]).cumsum(0)
    pairs = torch.tensor(pairs + [-1] * (M * k - len(pairs)), dtype=torch.int32).reshape(-1)
    rows = torch.where(pairs < 0, -1, torch.div(pairs, max(k, 1), rounding_mode="floor")).to(torch.int32)
    return w, rel * w.abs() + 2.0 ** -100, experts.to(torch.int32), offsets, pairs, rows


def grouped_linear(x, w, offsets, bias=None, *, index=None, out_index=None, act="none", residual=None, out_dtype, rows=None):
    """(result, bound, rows that a position gives)."""
    P = x.shape[0] if index is None else index.shape[0]
    rows = P if rows is None else rows
    N = w.shape[1]
    out, tol = torch.zeros((rows, N), dtype=torch.float64), torch.zeros((rows, N), dtype=torch.float64)
    given = torch.zeros(rows, dtype=torch.bool)
    xc, res = x.cpu(), None if residual is None else residual.cpu()
    at = torch.arange(P) if index is None else index.cpu().long()
    to = torch.arange(P) if out_index is None else out_index.cpu().long()
    for s, (a, e) in enumerate(segments(offsets, P)):
        i, o = at[a:max(a, e)], to[a:max(a, e)]
        ok = (i >= 0) & (i < x.shape[0]) & (o >= 0) & (o < rows)
        i, o = i[ok], o[ok]
        if not len(i):
            continue
        out[o], tol[o] = linear(xc[i], w[s], None if bias is None else bias[s], act=act, residual=None if res is None else res[o],
                                out_dtype=out_dtype)
        given[o] = True
    return out, tol, given


def combine(y, weights, *, residual=None, out_dtype):
    """k products and sums one behind the other: each rounds once (a multiply-add), at most at the sum of the sizes."""
    y, w = y.cpu().double(), weights.cpu().double()[:, :, None]
    term = torch.where(w == 0, torch.zeros_like(y), w * y)
    z, size = term.sum(1), term.abs().sum(1)
    if residual is not None:
        z, size = z + residual.cpu().double(), size + residual.cpu().double().abs()
    return _rounded(z, (y.shape[1] + 2) * 2.0 ** -24 * size, out_dtype)


def lora_linear(x, w, down, up, adapter, bias=None, *, offsets=None, scale=None, act="none", residual=None, out_dtype):
    """(result, bound). The low products are off by (K + 4) 2^-23 of their sum of sizes, 2^-23 for the scale, and what their parts leave
    out: 2^-24 of them, or of the row's largest (fp16) and of 2^-24; then r products (three parts each at most) in fp32."""
    M, K = x.shape
    xd, wd = x.cpu().double(), w.cpu().double()
    y, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    err = (K + 4) * 2.0 ** -23 * size
    where = torch.full((M,), -1)
    ids = adapter.cpu().tolist()
    for s, (a, e) in enumerate(segments(offsets, M) if offsets is not None else [(m, m + 1) for m in range(M)]):
        where[a:max(a, e)] = ids[s] if 0 <= ids[s] < down.shape[0] else -1
    for i in range(down.shape[0]):
        m = where == i
        if not bool(m.any()):
            continue
        c = 1.0 if scale is None else float(scale[i])
        A, B = down[i].cpu().double(), up[i].cpu().double()
        h, hs = c * (xd[m] @ A.t()), abs(c) * (xd[m].abs() @ A.abs().t())
        he = (K + 5) * 2.0 ** -23 * hs + 2.0 ** -22 * h.abs().amax(-1, keepdim=True)
        low, lows = h @ B.t(), h.abs() @ B.abs().t()
        y[m] += low
        err[m] += he @ B.abs().t() + (3 * down.shape[1] + 4) * 2.0 ** -23 * (size[m] + lows) + (K + 4) * 2.0 ** -23 * lows
    if bias is not None:
        y = y + bias.cpu().double()
        err = err + 2.0 ** -23 * (y.abs() + size)
    z, err = _activated(y, err, act, out_dtype)
    if residual is not None:
        z = z + residual.cpu().double()
        err = err + 2.0 ** -23 * z.abs()
    return _rounded(z, err, out_dtype)
