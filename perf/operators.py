"""The dense operators around the sparse convolutions, as a user's program calls them: `ops.linear` and `ops.linear_i8`
(a product with bias, activation and residual), `ops.qk_norm_rope` (the norms of queries and keys per head with the rotation
by voxel coordinates) and `ops.sparse_attention` (attention inside each frame or pool cell).

`listed()` names twelve cases, `draw(rng)` gives more of the same ranges, `prepare` makes a case's inputs, `run` is one
call, `work` the bytes and operations it cannot do without, and `exact` the same result in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2, "int8": 1}


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # One row through a projection (a frame's pooled token): the smallest call, all latency.
        {"name": "linear_token", "op": "linear", "dtype": "fp16", "M": 1, "K": 1024, "N": 1024, "bias": True,
         "act": "silu", "residual": "", "out": "fp16"},
        # The teacher U-Net's NearestUp linear at its fourth level, with the skip added onto the fp32 stream.
        {"name": "linear_up", "op": "linear", "dtype": "fp16", "M": 11_213, "K": 512, "N": 256, "bias": True,
         "act": "none", "residual": "fp32", "out": "fp32"},
        # A level's features widened in fp32, as the modules run without autocast: one row per pixel of 240x320.
        {"name": "linear_fp32", "op": "linear", "dtype": "fp32", "M": 76_800, "K": 64, "N": 128, "bias": True,
         "act": "silu", "residual": "", "out": "fp32"},
        # The encoder's tokens of four frames (1200 each) through the wide half of a transformer block.
        {"name": "linear_tokens", "op": "linear", "dtype": "bf16", "M": 4_800, "K": 1024, "N": 4096, "bias": True,
         "act": "gelu", "residual": "", "out": "bf16"},
        # The int8 refiner's arithmetic on a level of 77k rows, with the skip row.
        {"name": "linear_int8", "op": "linear", "dtype": "int8", "M": 76_811, "K": 256, "N": 256, "bias": True,
         "act": "silu", "residual": "fp16", "out": "fp16"},
        # Queries and keys of every pixel's voxel at 240x320, 8 heads of 32, slices of one (M, 3, H, D) product.
        {"name": "rope_pixels", "op": "rope", "dtype": "fp16", "M": 76_800, "Hq": 8, "Hkv": 8, "D": 32,
         "norm": "rms", "interleaved": False},
        # The same of one row, with grouped heads.
        {"name": "rope_token", "op": "rope", "dtype": "bf16", "M": 1, "Hq": 16, "Hkv": 4, "D": 64, "norm": "layer",
         "interleaved": True},
        # Attention inside the pool cells of 16^3 of a 240x320 surface (1 to 256 voxels a cell), biased by distance.
        {"name": "attention_cells", "op": "attention", "dtype": "fp16", "B": 1, "H": 240, "W": 320, "cell": 16,
         "Hq": 8, "Hkv": 8, "D": 32, "bias": True, "mask": False, "cap": 0.0, "queries": 0},
        # Attention inside each of four frames of a coarse level, with the invalid pixels' rows masked.
        {"name": "attention_frames", "op": "attention", "dtype": "bf16", "B": 4, "H": 45, "W": 61, "cell": 0,
         "Hq": 8, "Hkv": 8, "D": 64, "bias": False, "mask": True, "cap": 0.0, "queries": 0},
        # A whole level of 120x160 voxels, C = 256 in four heads, biased by distance: the largest.
        {"name": "attention_level", "op": "attention", "dtype": "bf16", "B": 1, "H": 120, "W": 160, "cell": 0,
         "Hq": 4, "Hkv": 4, "D": 64, "bias": True, "mask": False, "cap": 0.0, "queries": 0},
        # One pooled query per frame over that frame's level (8 frames of 120x160), grouped heads: keys and values
        # are read once and that is all.
        {"name": "attention_query", "op": "attention", "dtype": "fp16", "B": 8, "H": 120, "W": 160, "cell": 0,
         "Hq": 16, "Hkv": 4, "D": 64, "bias": False, "mask": True, "cap": 0.0, "queries": 1},
        # Full precision with capped scores, in odd-sized pool cells.
        {"name": "attention_fp32", "op": "attention", "dtype": "fp32", "B": 2, "H": 61, "W": 83, "cell": 24,
         "Hq": 4, "Hkv": 2, "D": 40, "bias": True, "mask": True, "cap": 30.0, "queries": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "rope", "attention", "attention", "attention"])
    if op == "linear":
        dtype = rng.choice(["fp32", "fp16", "bf16", "int8"])
        K, N = _log_int(rng, 16, 1024), _log_int(rng, 16, 4096)
        if rng.random() < 0.7:  # widths of the networks at hand; otherwise odd ones
            K, N = max(16, K // 16 * 16), max(16, N // 16 * 16)
        flops = 4e10 if dtype != "fp32" else 4e9
        M = _log_int(rng, 1, min(307_200, flops / (2 * K * N), 2e8 / (K + 3 * N)))
        return {"op": op, "dtype": dtype, "M": M, "K": K, "N": N, "bias": rng.random() < 0.8,
                "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                "residual": rng.choice(["", "fp32", dtype if dtype != "int8" else "fp16"]),
                "out": rng.choice(["fp32", dtype if dtype != "int8" else "fp16"])}
    if op == "rope":
        Hkv = rng.choice([1, 2, 4, 8])
        Hq, D = Hkv * rng.choice([1, 1, 2, 4]), rng.choice([16, 32, 40, 64, 96, 128])
        return {"op": op, "dtype": rng.choice(["fp32", "fp16", "bf16"]), "M": _log_int(rng, 1, 4e7 / ((Hq + Hkv) * D)),
                "Hq": Hq, "Hkv": Hkv, "D": D, "norm": rng.choice(["rms", "layer"]), "interleaved": rng.random() < 0.5}
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq, D = Hkv * rng.choice([1, 1, 2, 4]), rng.choice([16, 32, 40, 64, 96, 128])
    case = {"op": op, "dtype": dtype, "Hq": Hq, "Hkv": Hkv, "D": D, "bias": rng.random() < 0.6,
            "mask": rng.random() < 0.4, "cap": rng.choice([0.0, 0.0, 30.0])}
    kind = rng.choice(["cells", "cells", "frames", "query"])
    pairs = 4e11 / (4 * Hq * D) / (16 if dtype == "fp32" else 1)  # of a query and a key
    if kind == "cells":
        cell = rng.choice([2, 4, 8, 16, 32])
        n = _log_int(rng, 500, min(76_800, 2e8 / ((Hq + Hkv) * D), pairs / cell ** 2, 3e8 / (Hq * cell ** 2)))
        H = _log_int(rng, max(8, n / 640), min(480, n / 8))
        return {**case, "B": 1, "H": H, "W": max(1, n // H), "cell": cell, "queries": 0}
    if kind == "frames":
        B = rng.choice([1, 2, 3, 5])
        n = _log_int(rng, 1, min(19_200, math.sqrt(pairs / B), math.sqrt(1.4e9 / (Hq * B))))
        H = _log_int(rng, 1, math.sqrt(n))
        return {**case, "B": B, "H": H, "W": max(1, n // H), "cell": 0, "queries": 0}
    B, q = rng.choice([1, 2, 8, 33]), rng.choice([1, 1, 3, 8])
    n = _log_int(rng, 1, min(160_000, 7e7 / (Hkv * D)) / B)
    H = _log_int(rng, 1, math.sqrt(n))
    return {**case, "B": B, "H": H, "W": max(1, n // H), "cell": 0, "queries": q}


# ------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _scene(g, B, H, W):
    """Voxel coordinates (b, x, y, z) int32 of B depth maps, one voxel a pixel in raster order: a sloped floor with waves
    and some nearer boxes, z in steps of 1/128 of log depth."""
    x = torch.arange(H, device=DEVICE, dtype=torch.float32).view(1, H, 1)
    y = torch.arange(W, device=DEVICE, dtype=torch.float32).view(1, 1, W)
    r = torch.rand((B, 8), device=DEVICE, generator=g)
    c = lambda k: r[:, k].view(B, 1, 1)  # noqa: E731
    logz = 0.8 + c(0) - 0.6 * x / max(H, 8) + 0.05 * torch.sin(6.3 * (c(1) + (1 + c(2)) * y / max(W, 8)))
    box = ((x / H - c(3)).abs() < 0.15) & ((y / W - c(4)).abs() < 0.2)
    logz = torch.where(box, logz - 0.2 - 0.3 * c(5), logz)
    z = torch.round(logz * 128).to(torch.int32)
    z = z - z.amin(dim=(1, 2), keepdim=True)
    b = torch.arange(B, device=DEVICE, dtype=torch.int32).view(B, 1, 1).expand(B, H, W)
    xi, yi = x.to(torch.int32).expand(B, H, W), y.to(torch.int32).expand(B, H, W)
    return torch.stack([b, xi, yi, z], dim=-1).reshape(-1, 4).contiguous()


def _cells(coords, cell):
    """The pool cells of `cell`^3 voxels: (seg_indices int32, seg_offsets int64), rows in input order within a cell."""
    p = coords.to(torch.int64)
    q = p[:, 1:] // cell
    key = ((p[:, 0] * 100_000 + q[:, 0]) * 100_000 + q[:, 1]) * 100_000 + q[:, 2]
    _, parent, counts = torch.unique(key, return_inverse=True, return_counts=True)
    offsets = torch.zeros(counts.numel() + 1, dtype=torch.int64, device=DEVICE)
    offsets[1:] = counts.cumsum(0)
    return torch.sort(parent, stable=True).indices.to(torch.int32), offsets


def _frames(g, B, n):
    """Offsets of B frames over B n rows, each frame of about n rows (invalid pixels left out of some)."""
    cuts = torch.arange(1, B, device=DEVICE) * n
    cuts = cuts + ((torch.rand(B - 1, device=DEVICE, generator=g) - 0.5) * 0.3 * n).to(torch.int64)
    ends = torch.tensor([0, B * n], dtype=torch.int64, device=DEVICE)
    return torch.cat([ends[:1], cuts, ends[1:]])


def _freqs(D):
    """Rotation frequencies [D / 2, 3] in radians a voxel: the pairs shared out over x, y and z, wavelengths of 2 pi to
    1000 voxels in each."""
    P = D // 2
    f = torch.zeros((P, 3), dtype=torch.float32)
    for p in range(P):
        f[p, p % 3] = 160.0 ** (-(p // 3) / max(1, -(-P // 3)))
    return f.to(DEVICE)


def prepare(case, seed):
    g = _gen(seed)
    randn = lambda *shape: torch.randn(shape, device=DEVICE, generator=g)  # noqa: E731
    s = {"case": case}
    if case["op"] == "linear":
        M, K, N, dt = case["M"], case["K"], case["N"], DTYPES[case["dtype"]]
        if case["dtype"] == "int8":
            s["x"] = torch.randint(-127, 128, (M, K), device=DEVICE, generator=g, dtype=torch.int8)
            s["w"] = torch.randint(-127, 128, (N, K), device=DEVICE, generator=g, dtype=torch.int8)
            s["a_scale"] = 4.0 / 127
            s["w_scale"] = (0.5 + torch.rand((N,), device=DEVICE, generator=g)) / (74 * math.sqrt(K))
        else:
            s["x"] = randn(M, K).to(dt)
            s["w"] = (randn(N, K) / math.sqrt(K)).to(dt)
        s["bias"] = 0.5 * randn(N) if case["bias"] else None
        s["residual"] = randn(M, N).to(DTYPES[case["residual"]]) if case["residual"] else None
        return s
    Hq, Hkv, D, dt = case["Hq"], case["Hkv"], case["D"], DTYPES[case["dtype"]]
    if case["op"] == "rope":
        M = case["M"]
        s["qkv"] = randn(M, Hq + 2 * Hkv, D).to(dt)  # one product's output: q, k and v side by side
        W = 320
        s["coords"] = _scene(g, 1, -(-M // W), W)[:M].contiguous()
        s["freqs"] = _freqs(D)
        s["q_weight"], s["k_weight"] = 1 + 0.2 * randn(D), 1 + 0.2 * randn(D)
        layer = case["norm"] == "layer"
        s["q_bias"], s["k_bias"] = (0.1 * randn(D), 0.1 * randn(D)) if layer else (None, None)
        return s
    B, n, nq = case["B"], case["H"] * case["W"], case["queries"]
    coords = _scene(g, B, case["H"], case["W"])
    rows = B * n
    s["index"] = None
    if case["cell"]:
        s["index"], s["offsets"] = _cells(coords, case["cell"])
    else:
        s["offsets"] = _frames(g, B, n)
    s["coords"] = coords
    s["longest"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # (the program built the table and knows it)
    if nq:  # pooled queries: `nq` a frame, placed at some voxel of it
        s["q_offsets"] = torch.arange(B + 1, device=DEVICE, dtype=torch.int64) * nq
        at = torch.randint(0, n, (B, nq), device=DEVICE, generator=g) + n * torch.arange(B, device=DEVICE).view(B, 1)
        s["q_coords"] = coords[at.view(-1)].contiguous()
        s["q_longest"] = nq
    else:
        s["q_offsets"], s["q_coords"], s["q_longest"] = s["offsets"], coords, s["longest"]
    s["q"] = randn(B * nq if nq else rows, Hq, D).to(dt)
    s["kv"] = randn(rows, 2, Hkv, D).to(dt)  # keys and values side by side
    s["slopes"] = None
    if case["bias"]:  # a geometric series over the heads; z's voxels are finer than a pixel
        h = 0.5 ** (1 + 6 * torch.arange(Hq, device=DEVICE, dtype=torch.float32).view(Hq, 1) / Hq)
        s["slopes"] = (h * torch.tensor([[1.0, 1.0, 0.25]], device=DEVICE)).contiguous()
    s["kv_mask"] = torch.rand((rows,), device=DEVICE, generator=g) > 0.15 if case["mask"] else None
    return s


# --------------------------------------------------------------------------------------------------------- plain forms
def _activate(y, act):
    if act == "relu":
        return torch.clamp(y, min=0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _linear(s):
    c = s["case"]
    y = s["x"].float() @ s["w"].float().t()  # (int8: whole numbers below 2^24, exact in 32 bits)
    if c["dtype"] == "int8":
        y = y * s["a_scale"] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    y = _activate(y, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DTYPES[c["out"]])


def _norm_rope(x, weight, bias, cos, sin, layer, interleaved):
    u = x.float()
    if layer:
        u = u - u.mean(dim=-1, keepdim=True)
    u = u / torch.sqrt((u * u).mean(dim=-1, keepdim=True) + 1e-6) * weight
    if bias is not None:
        u = u + bias
    h = u.shape[-1] // 2
    a, b = (u[..., 0::2], u[..., 1::2]) if interleaved else (u[..., :h], u[..., h:])
    p, q = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([p, q], dim=-1).flatten(-2) if interleaved else torch.cat([p, q], dim=-1)
    return y.to(x.dtype)


def _rope(s):
    c = s["case"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    t = (s["coords"][:, None, 1:].double() * s["freqs"].double()).sum(dim=-1)[:, None, :]  # angles in 64 bits
    cos, sin = torch.cos(t).float(), torch.sin(t).float()
    layer = c["norm"] == "layer"
    return (_norm_rope(s["qkv"][:, :Hq], s["q_weight"], s["q_bias"], cos, sin, layer, c["interleaved"]),
            _norm_rope(s["qkv"][:, Hq:Hq + Hkv], s["k_weight"], s["k_bias"], cos, sin, layer, c["interleaved"]))


def _padded(offsets, longest, index):
    """[S, longest] rows of each segment (0 behind its end) and which of them there are."""
    at = torch.arange(longest, device=DEVICE)
    there = at < (offsets[1:] - offsets[:-1])[:, None]
    rows = torch.where(there, offsets[:-1, None] + at, 0)
    return (rows if index is None else index.long()[rows]), there


def _attention(s):
    c = s["case"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    kr, kin = _padded(s["offsets"], s["longest"], s["index"])
    qr, qin = (kr, kin) if not c["queries"] else _padded(s["q_offsets"], s["q_longest"], None)
    head = torch.arange(Hq, device=DEVICE) // (Hq // Hkv)
    q = s["q"].float()[qr].permute(0, 2, 1, 3).contiguous()  # [S, Hq, Lq, D]
    k = s["kv"][:, 0].float()[kr][:, :, head].permute(0, 2, 3, 1).contiguous()
    v = s["kv"][:, 1].float()[kr][:, :, head].permute(0, 2, 1, 3).contiguous()
    x = torch.matmul(q, k) * (1 / math.sqrt(D))
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    if s["slopes"] is not None:
        qc, kc = s["q_coords"][qr][:, :, None, 1:], s["coords"][kr][:, None, :, 1:]
        far = (qc - kc).abs().float()  # [S, Lq, Lk, 3]
        w = s["slopes"].view(1, Hq, 3, 1, 1)
        x = x - w[:, :, 0] * far[:, None, :, :, 0]
        x = x - w[:, :, 1] * far[:, None, :, :, 1]
        x = x - w[:, :, 2] * far[:, None, :, :, 2]
    seen = kin if s["kv_mask"] is None else kin & s["kv_mask"][kr]
    x = torch.where(seen[:, None, None, :], x, -math.inf)
    m = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(m), 0.0, m))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    out = torch.empty(s["q"].shape, dtype=torch.float32, device=DEVICE)
    out[qr[qin]] = o.permute(0, 2, 1, 3)[qin]
    return out.to(s["q"].dtype)


def run(s):
    c = s["case"]
    if own:
        from promptmoge_amd import ops

        out = DTYPES.get(c.get("out", ""))
        if c["op"] == "linear" and c["dtype"] == "int8":
            return ops.linear_i8(s["x"], s["w"], s["bias"], a_scale=s["a_scale"], w_scale=s["w_scale"], act=c["act"],
                                 residual=s["residual"], out_dtype=out)
        if c["op"] == "linear":
            return ops.linear(s["x"], s["w"], s["bias"], act=c["act"], residual=s["residual"], out_dtype=out)
        if c["op"] == "rope":
            return ops.qk_norm_rope(s["qkv"][:, :c["Hq"]], s["qkv"][:, c["Hq"]:c["Hq"] + c["Hkv"]], s["coords"],
                                    s["freqs"], q_weight=s["q_weight"], k_weight=s["k_weight"], q_bias=s["q_bias"],
                                    k_bias=s["k_bias"], norm=c["norm"], eps=1e-6, interleaved=c["interleaved"])
        if c["queries"]:
            return ops.sparse_attention(s["q"], s["kv"][:, 0], s["kv"][:, 1], s["q_offsets"], s["offsets"],
                                        coords=s["q_coords"], kv_coords=s["coords"], slopes=s["slopes"],
                                        kv_mask=s["kv_mask"], cap=c["cap"])
        return ops.sparse_attention(s["q"], s["kv"][:, 0], s["kv"][:, 1], s["offsets"], index=s["index"],
                                    coords=s["coords"], slopes=s["slopes"], kv_mask=s["kv_mask"], cap=c["cap"])
    return {"linear": _linear, "rope": _rope, "attention": _attention}[c["op"]](s)


# ----------------------------------------------------------------------------------------------------- work and results
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        b = (M * K + N * K) * e + M * N * BYTES[case["out"]]
        b += 4 * N * (bool(case["bias"]) + (case["dtype"] == "int8"))
        b += M * N * BYTES[case["residual"]] if case["residual"] else 0
        return {"bytes": b, "flops": 2 * M * K * N}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "rope":
        M = case["M"]
        return {"bytes": 2 * M * (Hq + Hkv) * D * e + 16 * M + 6 * D * 4, "flops": M * (Hq + Hkv) * D * 10}
    s = _gen(0)
    rows = case["B"] * case["H"] * case["W"]
    if case["cell"]:  # the lengths of this scene's cells
        offsets = _cells(_scene(s, case["B"], case["H"], case["W"]), case["cell"])[1]
        lengths = (offsets[1:] - offsets[:-1]).double()
        pairs, queries = float((lengths * lengths).sum()), rows
    else:
        queries = case["B"] * case["queries"] if case["queries"] else rows
        pairs = queries * rows / case["B"]
    b = (2 * queries * Hq + 2 * rows * Hkv) * D * e
    b += 16 * (rows + (queries if case["queries"] else 0)) if case["bias"] else 0
    b += rows if case["mask"] else 0
    b += 4 * rows if case["cell"] else 0
    return {"bytes": b, "flops": 4 * Hq * D * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = torch.nn.functional.linear(s["x"].double(), s["w"].double())
        if case["dtype"] == "int8":
            y *= s["w_scale"].double() * s["a_scale"]
        if s["bias"] is not None:
            y += s["bias"].double()
        act = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu,
               "gelu": torch.nn.functional.gelu,
               "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]]
        y = act(y)
        return y if s["residual"] is None else y + s["residual"].double()
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["op"] == "rope":
        xyz = s["coords"][:, 1:].double()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), xyz @ s["freqs"].double().t())
        outs = []
        for x, w, b in ((s["qkv"][:, :Hq], s["q_weight"], s["q_bias"]),
                        (s["qkv"][:, Hq:Hq + Hkv], s["k_weight"], s["k_bias"])):
            x = x.double()
            if case["norm"] == "layer":
                u = torch.nn.functional.layer_norm(x, (D,), w.double(), b.double(), 1e-6)
            else:
                u = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
            u = u.unflatten(-1, (D // 2, 2)) if case["interleaved"] else u.unflatten(-1, (2, D // 2)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(u.contiguous()) * turn[:, None])
            outs.append((z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2))
        return tuple(outs)
    q, k, v = s["q"].double(), s["kv"][:, 0].double(), s["kv"][:, 1].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    ko, qo = s["offsets"].tolist(), s["q_offsets"].tolist()
    whole = torch.arange(k.shape[0], device=DEVICE) if s["index"] is None else s["index"].long()
    seen = torch.ones(k.shape[0], dtype=torch.bool, device=DEVICE) if s["kv_mask"] is None else s["kv_mask"]
    for i in range(len(ko) - 1):
        kr = whole[ko[i]:ko[i + 1]]
        qr = torch.arange(qo[i], qo[i + 1], device=DEVICE) if case["queries"] else kr
        kr = kr[seen[kr]]
        if not kr.numel() or not qr.numel():
            continue
        for h0 in range(0, Hq, Hq if len(qr) * len(kr) < 1e7 else 1):
            hs = slice(h0, Hq if len(qr) * len(kr) < 1e7 else h0 + 1)
            of = torch.arange(Hq, device=DEVICE)[hs] // (Hq // Hkv)
            x = torch.matmul(q[qr][:, hs].transpose(0, 1), k[kr][:, of].permute(1, 2, 0).contiguous()) / math.sqrt(D)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if s["slopes"] is not None:
                d = (s["q_coords"][qr][:, None, 1:] - s["coords"][kr][None, :, 1:]).abs().double()
                x = x - torch.tensordot(s["slopes"][hs].double(), d, dims=([1], [2]))
            out[qr, hs] = torch.matmul(torch.softmax(x, dim=-1), v[kr][:, of].transpose(0, 1).contiguous()).transpose(0, 1)
    return out
