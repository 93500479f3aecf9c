"""The dense operators (ops.linear, linear_i8, qk_norm_rope, sparse_attention) where calls are unusual: addresses, extremes,
tables that do not hold what they should, launches larger than a grid."""
import math

import pytest
import torch

import dense_ref as ref
from conftest import announce
from promptmoge_amd import _lib, ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F16, BF16, F32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H", [1, 2])
def test_heads_at_odd_addresses(gpu, dt, H):
    """Contiguous tensors that start at an odd element: the results of their aligned copies, bit for bit."""
    g = gen(3)
    M, D = 70, 32
    off = torch.tensor([0, 30, 70], device=gpu)
    c, f = torch.randint(0, 50, (M, 4), generator=g, dtype=torch.int32).to(gpu), torch.rand((D // 2, 3), generator=g).to(gpu)
    q, k, v = (randn(g, M * H * D + 1).to(dt).to(gpu)[1:].view(M, H, D) for _ in range(3))
    announce(f"heads at odd addresses {dt} {H}")
    got, want = ops.qk_norm_rope(q, k, c, f), ops.qk_norm_rope(q.clone(), k.clone(), c, f)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(ops.sparse_attention(q, k, v, off), ops.sparse_attention(q.clone(), k.clone(), v.clone(), off))


@pytest.mark.parametrize("dt", TYPES)
def test_results_beside_their_inputs_in_one_buffer(gpu, dt):
    """Outputs in other columns of the inputs' own rows; what lies beside them stays."""
    g = gen(4)
    M, D = 90, 32
    announce(f"results beside inputs {dt}")
    buf = randn(g, M, 160).to(dt).to(gpu)
    w = randn(g, 64, 64).to(dt).to(gpu)
    want = ops.linear(buf[:, 16:80].clone(), w)
    keep = buf.clone()
    ops.linear(buf[:, 16:80], w, out=buf[:, 80:144])
    assert torch.equal(buf[:, 80:144], want) and torch.equal(buf[:, :80], keep[:, :80]) and torch.equal(buf[:, 144:], keep[:, 144:])
    x = randn(g, M, 8, D).to(dt).to(gpu)
    c, f = torch.randint(0, 50, (M, 4), generator=g, dtype=torch.int32).to(gpu), torch.rand((D // 2, 3), generator=g).to(gpu)
    keep = x.clone()
    want = ops.qk_norm_rope(keep[:, :2], keep[:, 2:3], c, f)
    ops.qk_norm_rope(x[:, :2], x[:, 2:3], c, f, out=(x[:, 4:6], x[:, 6:7]))
    assert torch.equal(x[:, 4:6], want[0]) and torch.equal(x[:, 6:7], want[1])
    assert torch.equal(x[:, :4], keep[:, :4]) and torch.equal(x[:, 7:], keep[:, 7:])
    off = torch.tensor([0, 40, M], device=gpu)
    want = ops.sparse_attention(keep[:, :2], keep[:, 2:4], keep[:, 4:6], off)
    x = keep.clone()
    ops.sparse_attention(x[:, :2], x[:, 2:4], x[:, 4:6], off, out=x[:, 6:])
    assert torch.equal(x[:, 6:], want) and torch.equal(x[:, :6], keep[:, :6])


@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_i8_largest_sums(gpu, M):
    """All codes -128 over the longest k: sums of 2^31 - 2^14, exact in fp32 (17 bits times 2^14)."""
    announce(f"linear_i8 largest sums, M={M}")
    x = torch.full((M, 131_071), -128, dtype=torch.int8, device=gpu)
    w = torch.full((70, 131_071), -128, dtype=torch.int8, device=gpu)
    w[::2] = 127
    got = ops.linear_i8(x, w)
    assert bool((got[:, 1::2] == float(2 ** 31 - 2 ** 14)).all()) and bool((got[:, ::2] == float(-128 * 127 * 131_071)).all())


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("M", [5, 700])
def test_linear_activations_of_infinities(gpu, act, out, M):
    """What the formula gives for +-inf and NaN, whatever the result's type and the kernel's form."""
    announce(f"linear activations of infinities {act} {out} {M}")
    x = torch.zeros(M, 64, device=gpu)
    x[:, 0] = torch.tensor([math.inf, -math.inf, math.nan, 1e30, -1e30], device=gpu).repeat(M // 5)
    w = torch.zeros(48, 64, device=gpu)
    w[:, 0] = 1
    want = {"none": [math.inf, -math.inf, math.nan, math.inf, -math.inf], "relu": [math.inf, 0, math.nan, math.inf, 0]}.get(
        act, [math.inf, math.nan, math.nan, math.inf, 0])  # (-inf times 0)
    if out != F16:  # (1e30 is finite there)
        big = float(torch.tensor(1e30).to(out))
        want = [w_ if i < 3 or w_ == 0 else math.copysign(big, w_) for i, w_ in enumerate(want)]
    got = ops.linear(x, w, act=act, out_dtype=out).cpu()
    want = torch.tensor(want).repeat(M // 5).view(M, 1).expand(M, 48).to(out)
    assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0)), (got[:5, 0], want[:5, 0])


@pytest.mark.parametrize("out", [F16, BF16])
def test_linear_gelu_in_the_negative_tail(gpu, out):
    """gelu of each number from -14 to 9 in 16-bit results: within 0.6 of a step (half a step for the rounding, and an evaluation
    of a tenth of a step at most) of the value, subnormal steps included. In bf16, whose subnormal numbers are fp32's, values
    below the smallest normal one may be 0: the exponential has none."""
    announce(f"gelu tail {out}")
    y = torch.linspace(-14.0, 9.0, 64 * 4096).view(-1, 64)
    eye = torch.eye(64, device=gpu)
    got = ops.linear(y.to(gpu), eye, act="gelu", out_dtype=out).cpu().double()
    want = ref.act64(y.double(), "gelu")
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-300)))) * torch.finfo(out).eps
    least = torch.finfo(out).tiny * (torch.finfo(out).eps if out == F16 else 1 / 0.6)
    far = (got - want).abs() / step.clamp(min=least)
    assert float(far.max()) <= 0.6, (float(far.max()), float(y.flatten()[far.argmax()]))


def test_linear_fp32_activations_far_out(gpu):
    """silu and gelu_tanh in fp32 results, relative to their own value from -85 (-8.5) to 40: y / (1 + exp(-z)) with an
    exponential and a reciprocal of 1 ulp (2 x 2^-24) and four more roundings, 2^-21 together; gelu_tanh's z is up to five roundings
    off (constants counted half), |z| 5 x 2^-24 of the exponential."""
    y = torch.linspace(-85.0, 40.0, 64 * 4096).view(-1, 64)
    eye = torch.eye(64, device=gpu)
    announce("linear fp32 silu, gelu_tanh far out")
    got = ops.linear(y.to(gpu), eye, act="silu").cpu().double()
    want = ref.act64(y.double(), "silu")
    assert float(((got - want).abs() / want.abs()).max()) <= 2.0 ** -21
    y = (y / 10).float()
    got = ops.linear(y.to(gpu), eye, act="gelu_tanh").cpu().double()
    yd = y.double()
    z = 2 * math.sqrt(2 / math.pi) * (yd + 0.044715 * yd ** 3)
    want = yd / (1 + torch.exp(-z))
    assert float(((got - want).abs() / (want.abs() * (2.0 ** -21 + 5 * 2.0 ** -24 * z.abs()))).max()) <= 1.0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cap", [0.5, 30.0, 200.0, 256.0, 300.0, 1e4, 1e6, 1e8, 1e30])
@pytest.mark.parametrize("few", [False, True])
def test_attention_caps_of_any_size(gpu, dt, cap, few):
    """One query on two keys whose scores are 0 and x: the result tells the capped score, for x from far below the cap to beyond
    it. The weight e^t / (1 + e^t) of t = cap tanh(x / cap) is off by a quarter of t's error at most: |x| 2^-20 for its few
    roundings, and below a cap of 256, where the 16-bit types take a form whose error is the cap's, 2^-21 cap for these."""
    g = gen(2)
    n = 64
    x = (torch.rand(n, generator=g) * 12 - 6).to(dt)
    x[:6] = torch.tensor([0.0, 1e-3, -1e-3, 0.25, 6.0, -6.0]).to(dt)
    q = torch.zeros(n, 1, 32, dtype=dt)
    q[:, 0, 0] = x
    k, v = torch.zeros(2 * n, 1, 32, dtype=dt), torch.zeros(2 * n, 1, 32, dtype=dt)
    k[1::2, 0, 0], v[1::2] = 1, 1
    off, koff = torch.arange(n + 1), torch.arange(n + 1) * 2
    if few:  # (a block per segment: long segments, the same key again and again)
        k, v = k.view(n, 2, 1, 32).repeat(1, 100, 1, 1).view(-1, 1, 32), v.view(n, 2, 1, 32).repeat(1, 100, 1, 1).view(-1, 1, 32)
        koff = torch.arange(n + 1) * 200
    announce(f"attention cap {cap} {dt} few={few}")
    got = ops.sparse_attention(q.to(gpu), k.to(gpu), v.to(gpu), off.to(gpu), koff.to(gpu), cap=cap, scale=1.0).cpu().double()
    xd = x.double()
    want = torch.sigmoid(cap * torch.tanh(xd / cap)).view(n, 1, 1).expand(n, 1, 32)
    terr = xd.abs() * 2.0 ** -20 + (2.0 ** -21 * cap if cap < 256 and dt != F32 else 0.0)
    # each weight is rounded to the type, and the result; sums of 2 or 200 weights
    tol = want * (1 - want) * 1.01 * terr.view(n, 1, 1) + want * (2 * ref.U[dt] + 2.0 ** -20 + (200 if few else 2) * 2.0 ** -22) + ref.TINY[dt]
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D,bias,mask", [(32, False, False), (64, False, True), (64, True, False), (128, False, False)])
@pytest.mark.parametrize("queries", [1, 70, 8192])
def test_attention_many_small_weights(gpu, dt, D, bias, mask, queries):
    """One key of weight 1 and 150,000 of 2^-25.3, values all 1: the result is 1 within the type's half step and the roundings of
    the two sums in fp32, which hold 1: a matrix step of 16 keys (fp32: 2) and a lane's sum of 32 round by 2^-24 each. (fp16
    holds numbers down to 2^-25: small weights kept as such would all be lost, 0.36 % of the sum, three times that, where the
    keys are not split over blocks: the 16 heads of the most queries.)"""
    n = 150_000
    announce(f"attention small weights {dt} D={D} bias={bias} mask={mask} queries={queries}")
    k, v = torch.zeros(n, 1, D, dtype=dt), torch.ones(n, 1, D, dtype=dt)
    low = -25.3 / 1.4426950408889634
    queries = 20_000 if D == 128 and queries > 100 else queries
    heads = 16 if queries > 100 else 1
    q = torch.ones(queries, heads, D, dtype=dt)
    kw = dict(scale=1.0 / D)
    if bias:
        kc = torch.zeros(n, 4, dtype=torch.int32)
        kc[:, 1] = 5
        kc[77, 1] = 0
        kw |= dict(coords=torch.zeros(queries, 4, dtype=torch.int32).to(gpu), kv_coords=kc.to(gpu), slopes=torch.tensor([[-low / 5, 0.0, 0.0]] * heads, device=gpu))
    else:
        k[:] = low
        k[77] = 0
    if mask:
        m = torch.ones(n, dtype=torch.bool)
        m[1000:2000] = False
        kw["kv_mask"] = m.to(gpu)
    off, koff = torch.tensor([0, queries]), torch.tensor([0, n])
    got = ops.sparse_attention(q.to(gpu), k.to(gpu), v.to(gpu), off.to(gpu), koff.to(gpu), **kw).double()
    # (and half a step of the small weights' own share, 2^-8)
    assert float((got - 1).abs().max()) <= ref.U[dt] * (1 + 2.0 ** -8) + (n / (2 if dt == F32 else 16) + n / 32) * 2.0 ** -24


def used_before(gpu, nbytes):
    """Leaves freed memory that is full of NaN where the next new tensors come from."""
    x = torch.full((nbytes // 4,), math.nan, device=gpu)
    y = [torch.full((n,), math.nan, device=gpu) for n in (1 << 8, 1 << 12, 1 << 16, 1 << 18)]
    torch.cuda.synchronize()
    del x, y


TABLES = {
    "an index out of range": lambda M, g: (torch.tensor([0, M // 3, M]), torch.where(torch.rand(M, generator=g) < 0.2, torch.randint(-9, 2 * M, (M,), generator=g), torch.randperm(M, generator=g)).int()),
    "one row named by all": lambda M, g: (torch.tensor([0, M]), torch.full((M,), 5, dtype=torch.int32)),
    "rows named twice": lambda M, g: (torch.tensor([0, M // 2, M]), torch.randint(0, M, (M,), generator=g).int()),
    "more positions than rows": lambda M, g: (torch.tensor([0, M // 2, 3 * M]), torch.randint(0, M // 2, (3 * M,), generator=g).int()),
    "fewer positions than rows": lambda M, g: (torch.tensor([0, 3, M // 4]), torch.randperm(M, generator=g)[:M // 4].int()),
    "no position": lambda M, g: (torch.tensor([0, 0]), torch.zeros(0, dtype=torch.int32)),
    "segments of a part": lambda M, g: (torch.tensor([M // 5, M // 2, M - 7]), torch.randperm(M, generator=g).int()),
}


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M", [12, 60, 900])
@pytest.mark.parametrize("name", list(TABLES))
@pytest.mark.parametrize("few", [False, True])
def test_attention_new_results_are_written_whole(gpu, dt, M, name, few):
    """Rows that no position of a segment names are 0, in memory that held NaN; a row that several name has the result of one."""
    g = gen(M)
    H, D = 2, 32
    off, idx = TABLES[name](M, g)
    q = randn(g, M, H, D).to(dt).to(gpu)
    if few:  # (few queries on many keys: a block per segment)
        S, Mk = len(off) - 1, 300 * len(idx) + 600
        kv = randn(g, Mk, 2, H, D).to(dt).to(gpu)
        koff, args = torch.arange(S + 1) * (Mk // S), {}
    else:
        kv = randn(g, M, 2, H, D).to(dt).to(gpu)
        koff, args = off, {"kv_index": idx.to(gpu)}
    announce(f"attention whole results {dt} {M} {name} few={few}")
    used_before(gpu, 1 << 22)
    got = ops.sparse_attention(q, kv[:, 0], kv[:, 1], off.to(gpu), koff.to(gpu), index=idx.to(gpu), **args).cpu()
    assert not bool(torch.isnan(got).any())
    seg = torch.full((M,), -1)
    named = {}
    for s in range(len(off) - 1):
        for p in range(int(off[s]), min(int(off[s + 1]), len(idx))):
            if 0 <= int(idx[p]) < M:
                named.setdefault(int(idx[p]), set()).add(s)
    outside = {int(r) for p, r in enumerate(idx.tolist()) if not (int(off[0]) <= p < int(off[-1]))}
    rest = torch.tensor([r not in named for r in range(M)])
    assert not bool(got[rest].any())
    for s in range(len(off) - 1):  # each segment's rows, as if its queries alone were there
        rows = torch.tensor([r for r in range(M) if named.get(r) == {s} and r not in outside], dtype=torch.int64)
        if not len(rows):
            continue
        one = torch.tensor([0, len(rows)])
        ks = koff[s:s + 2].clamp(max=len(idx)) if not few else koff[s:s + 2]
        want, tol, _ = ref.attention(q[rows.to(gpu)], kv[:, 0], kv[:, 1], one, ks, **({} if few else {"kv_index": idx}))
        ref.assert_within(got[rows], want, tol)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("off", [[700, 100, 650, 2 ** 62], [900, -1, 2 ** 40, 0], [-(2 ** 62), 2 ** 62, 5, 880], [0, 900, 300, 900, 100]])
@pytest.mark.parametrize("kind", ["long", "split", "few", "short"])
def test_attention_falling_offsets_leave_no_row_unwritten(gpu, dt, off, kind):
    """What falling offsets give is not said, but it comes from no memory that nobody wrote."""
    g = gen(7)
    H, D = 2, 32
    M = {"long": 900, "split": 900, "few": 900, "short": 900}[kind]
    off = torch.tensor(off)
    if kind == "short":  # (many short segments: tiles through all of them)
        off = torch.cat([off, torch.randint(-50, 1000, (40,), generator=g)])
    q = randn(g, M, H, D).to(dt).to(gpu)
    if kind == "few":
        off = torch.cat([off, torch.randint(-50, 1000, (160,), generator=g)])
        Mk = 200_000
        kv = randn(g, 1000, 2, H, D).to(dt).to(gpu).repeat(200, 1, 1, 1)
        koff = torch.arange(len(off)) * (Mk // len(off))
    elif kind == "split":
        kv = randn(g, 1000, 2, H, D).to(dt).to(gpu).repeat(40, 1, 1, 1)
        koff = torch.arange(len(off)) * 10_000
    else:
        kv, koff = randn(g, M, 2, H, D).to(dt).to(gpu), off
    for idx in (None, torch.randperm(M, generator=g).int().to(gpu)):
        announce(f"attention falling offsets {kind} {off.tolist()[:5]} {dt} index={idx is not None}")
        used_before(gpu, 1 << 24)
        got = ops.sparse_attention(q, kv[:, 0], kv[:, 1], off.to(gpu), koff.to(gpu), index=idx)
        assert not bool(torch.isnan(got).any())
        if kind != "few":  # (there two blocks may work on one row)
            assert float(got.abs().max()) <= 1.02 * float(kv[:, 1].abs().max())  # (an average of values, or 0)
        out = torch.full((M + 64, H, D), 7.0, dtype=dt, device=gpu)
        used_before(gpu, 1 << 24)
        ops.sparse_attention(q, kv[:, 0], kv[:, 1], off.to(gpu), koff.to(gpu), index=idx, out=out[32:-32])
        assert not bool(torch.isnan(out).any())
        assert bool((out[:32] == 7).all()) and bool((out[-32:] == 7).all())


@pytest.mark.parametrize("fall", [False, True])
def test_attention_many_long_segments_with_a_fall(gpu, fall):
    """More segments than a block looks through itself: a kernel looks for a fall in front of it."""
    g = gen(17)
    S, L, H, D = 700, 170, 1, 32
    M = S * L
    off = torch.arange(S + 1) * L
    if fall:
        off[333], off[334] = off[334].item(), off[333].item()
    q, kv = randn(g, M, H, D).to(F16).to(gpu), randn(g, M, 2, H, D).to(F16).to(gpu)
    announce(f"attention many long segments, fall={fall}")
    used_before(gpu, 1 << 25)
    got = ops.sparse_attention(q, kv[:, 0], kv[:, 1], off.to(gpu))
    assert not bool(torch.isnan(got).any())
    if not fall:
        want, tol, _ = ref.attention(q, kv[:, 0], kv[:, 1], off)
        ref.assert_within(got, want, tol)


def test_attention_whole_results_captured_and_replayed(gpu):
    """Marks of named rows live in the call's workspace: a graph's replays with another index each give that index's result."""
    g = gen(21)
    M, H, D = 500, 2, 32
    q, kv = randn(g, M, H, D).to(F16).to(gpu), randn(g, M, 2, H, D).to(F16).to(gpu)
    off = torch.tensor([0, 200, M], device=gpu)
    idx = torch.arange(M, dtype=torch.int32, device=gpu)
    announce("attention whole results in a graph")
    call = lambda: ops.sparse_attention(q, kv[:, 0], kv[:, 1], off, index=idx)  # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for k in range(5):
        new = torch.randperm(M, generator=g).int()
        new[k::7] = torch.tensor([-1, M, 0, 2 ** 31 - 1, 3], dtype=torch.int32)[k]
        if k == 2 or k == 4:  # (a row named twice has either's result: named by none instead)
            new[new == (0 if k == 2 else 3)] = -1
        idx.copy_(new)
        y.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        want, tol, covered = ref.attention(q, kv[:, 0], kv[:, 1], off, index=new)
        assert not bool(y.cpu()[~covered].any())
        ref.assert_within(y, want, tol)
        torch.cuda.synchronize()
        assert torch.equal(y, call())


def test_linear_more_rows_than_a_grid_holds(gpu):
    """2^30 rows in tiles of 64 would be 2^32 threads."""
    M = 2 ** 30 + 77
    announce(f"linear of {M} rows")
    x = torch.zeros((M, 1), dtype=F16, device=gpu)
    at = torch.tensor([0, 1, 63, 64, 2 ** 29, 2 ** 30 - 65, 2 ** 30 - 64, 2 ** 30 - 1, 2 ** 30, M - 1], device=gpu)
    x[at, 0] = torch.arange(1, 11, dtype=F16, device=gpu)
    r = torch.zeros((M, 1), dtype=F16, device=gpu)
    r[at, 0] = 0.5
    got = ops.linear(x, torch.full((1, 1), 3.0, dtype=F16, device=gpu), residual=r, out=r)
    assert torch.equal(got[at, 0].cpu(), 3 * torch.arange(1, 11, dtype=F16) + 0.5)
    got[at] = 0
    assert not any(bool(part.any()) for part in got.split(2 ** 28))


def test_rope_more_rows_than_a_grid_holds(gpu):
    """2^26 rows of 64 pairs, four a block, would be 2^32 threads."""
    M, D = 2 ** 26 + 70, 128
    announce(f"rope of {M} rows")
    q = torch.zeros((M, 1, D), dtype=F16, device=gpu)
    c = torch.zeros((M, 4), dtype=torch.int32, device=gpu)
    at = torch.tensor([0, 3, 4, 2 ** 25, 2 ** 26 - 5, 2 ** 26 - 4, 2 ** 26 - 1, 2 ** 26, M - 1], device=gpu)
    g = gen(1)
    q[at] = randn(g, 9, 1, D).to(F16).to(gpu)
    c[at] = torch.randint(0, 500, (9, 4), generator=g, dtype=torch.int32).to(gpu)
    f = torch.rand((D // 2, 3), generator=g).to(gpu)
    want, tol = ref.norm_rope(q[at], None, None, c[at], f, layer=False, interleaved=False)
    ops.qk_norm_rope(q, None, c, f, out=(q, None))
    ref.assert_within(q[at], want, tol)
    q[at] = 0
    assert not any(bool(part.any()) for part in q.split(2 ** 23))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D", [16, 64, 96])
@pytest.mark.parametrize("kw", [dict(), dict(bias=True), dict(mask=True), dict(cap=5.0, mask=True), dict(bias=True, cap=1e4), dict(few=True, mask=True)])
def test_attention_precise(gpu, dt, D, kw):
    """precise: the fp32 form's bounds on the same numbers, and one rounding to the type at the end. The weights' two parts leave 2^-14 of
    a weight in bf16 (2^-8 of a second part of up to 2^-7 + 2^-8 of it) and less in fp16."""
    g = gen(D)
    lengths = torch.tensor([0, 3, 300, 700, 1000]) if not kw.get("few") else torch.tensor([0, 1, 3])
    M = int(lengths[-1])
    Mk = 20_000 if kw.get("few") else M
    koff = torch.tensor([0, 9000, Mk]) if kw.get("few") else lengths
    q, k, v = (randn(g, m, 2, D).to(dt) for m in (M, Mk, Mk))
    a = dict(cap=kw.get("cap", 0.0))
    if kw.get("bias"):
        a |= dict(coords=torch.randint(0, 40, (M, 4), generator=g, dtype=torch.int32), slopes=0.2 * torch.rand((2, 3), generator=g))
        a["kv_coords"] = a["coords"]
    if kw.get("mask"):
        a["kv_mask"] = torch.rand(Mk, generator=g) > 0.3
    announce(f"attention precise {dt} {D} {kw}")
    dev = {n: t.to(gpu) if isinstance(t, torch.Tensor) else t for n, t in a.items()}
    got = ops.sparse_attention(q.to(gpu), k.to(gpu), v.to(gpu), lengths.to(gpu), koff.to(gpu), precise=True, **dev)
    want, tol, _ = ref.attention(q.float(), k.float(), v.float(), lengths, koff, **a)
    size, _, _ = ref.attention(q.float(), k.float(), v.float().abs(), lengths, koff, **a)  # sum of p |v|
    ref.assert_within(got, want, tol + 2.0 ** -14 * size * (dt != F32) + ref.U[dt] * want.abs() * 1.01 + ref.TINY[dt])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("kw", [dict(), dict(precise=True), dict(cap=1e4), dict(cap=20.0)])
def test_attention_infinite_values_that_count(gpu, dt, D, kw):
    """An average with +inf is +inf, with -inf -inf, with both NaN: in the columns they are in, and there alone."""
    g = gen(D)
    n = 200
    q, k, v = (randn(g, n, 2, D) for _ in range(3))
    q, k = (t.div(4).to(dt) for t in (q, k))  # (weights far from any underflow)
    v[50, 0, 3], v[70, 1, 5], v[20, 0, 6], v[120, 0, 6] = math.inf, -math.inf, math.inf, -math.inf
    v = v.to(dt)
    off = torch.tensor([0, 150, n])
    announce(f"attention infinite values {dt} {D} {kw}")
    got = ops.sparse_attention(q.to(gpu), k.to(gpu), v.to(gpu), off.to(gpu), **kw).cpu()
    want, tol, _ = ref.attention(q, k, v, off, cap=kw.get("cap", 0.0))
    tol = torch.nan_to_num(tol, nan=0.0, posinf=0.0)
    assert bool(torch.isinf(want[:150, 0, 3]).all()) and bool(torch.isnan(want[:150, 0, 6]).all())
    ref.assert_within(got, want, tol)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("straight", [True, False])
@pytest.mark.parametrize("positions", [0, 1, 40, 64])
def test_attention_zero_rest_of_the_c_entry(gpu, dt, straight, positions):
    """Fewer positions than rows without an index, and results of any stride: the other rows are 0, what lies between them stays."""
    import ctypes as C
    g = gen(positions)
    M, H, D = 64, 2, 40
    code, es = {F32: _lib.TYPE_F32, F16: _lib.TYPE_F16, BF16: _lib.TYPE_BF16}[dt], torch.finfo(dt).bits // 8
    q, k, v = (randn(g, M, H, D).to(dt).to(gpu) for _ in range(3))
    buf = torch.full((M, H + 1, D + 4), math.nan, dtype=dt, device=gpu)
    out = torch.full((M, H, D), math.nan, dtype=dt, device=gpu) if straight else buf[:, :H, :D]
    off = torch.tensor([0, positions // 2, max(positions - 3, positions // 2)], device=gpu)
    a = _lib.AttentionArgs(type=code, Hq=H, Hk=H, D=D, q=q.data_ptr(), q_row=H * D, q_head=D, k=k.data_ptr(), k_row=H * D, k_head=D,
                           v=v.data_ptr(), v_row=H * D, v_head=D, out=out.data_ptr(), out_row=out.stride(0), out_head=out.stride(1),
                           q_rows=M, k_rows=M, q_positions=positions, k_positions=positions, segments=2, q_offsets=off.data_ptr(),
                           k_offsets=off.data_ptr(), scale=D ** -0.5, zero_rest=1)
    lib = _lib.lib()
    need = lib.pmg_attention_workspace_bytes(C.byref(a))
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=gpu)
    announce(f"attention zero_rest {dt} straight={straight} positions={positions}")
    _lib.check(lib.pmg_attention(C.byref(a), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    want, tol, covered = ref.attention(q, k, v, off)
    assert not bool(out.cpu()[~covered].any())
    ref.assert_within(out, want, tol)
    if not straight:
        assert bool(torch.isnan(buf[:, H]).all()) and bool(torch.isnan(buf[:, :, D:]).all())


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("S,L,Lk,Hq,Hk,index", [
    (100, 800, 800, 16, 1, True),      # shares of the rows that take several rounds of bits
    (70, 200, 3000, 1, 1, False),      # keys split: parts that nobody wrote
    (90, 200, 2000, 2, 1, True),
    (1100, 1000, 40, 1, 1, True),      # more rows than a sweep goes through: filled first
    (1100, 1000, 40, 1, 1, False),
    (70, 20_000, 300, 1, 1, False)])
@pytest.mark.parametrize("fall", [False, True])
def test_attention_many_segments_with_tables_that_miss_rows(gpu, dt, S, L, Lk, Hq, Hk, index, fall):
    """More segments than a block looks through, with offsets that fall and an index that does not name every row."""
    g = torch.Generator(device=gpu).manual_seed(S + L)
    D = 32
    M, Mk = S * L, S * Lk
    off, koff = torch.arange(S + 1, device=gpu) * L, torch.arange(S + 1, device=gpu) * Lk
    if fall:
        off[S // 2], off[S // 2 + 1] = off[S // 2 + 1].item(), off[S // 2].item()
        off[5] = M
        off[S - 3] = -7
    q = torch.randn((M, Hq, D), device=gpu, generator=g).to(dt)
    k, v = (torch.randn((Mk, Hk, D), device=gpu, generator=g).to(dt) for _ in range(2))
    kw = {}
    if index:
        idx = torch.randperm(M, device=gpu, generator=g).int()
        idx[::9] = -1
        idx[1::50] = 2 ** 31 - 1
        kw["index"] = idx
    announce(f"attention tables that miss rows {dt} {S} x {L} on {Lk}, {Hq}/{Hk}, index={index} fall={fall}")
    used_before(gpu, M * Hq * D * q.element_size())
    got = ops.sparse_attention(q, k, v, off, koff, **kw)
    assert not bool(torch.isnan(got).any())
    assert float(got.abs().max()) <= 1.02 * float(v.abs().max())
    if index:
        named = torch.zeros(M, dtype=torch.bool, device=gpu)
        named[idx[(idx >= 0) & (idx < M)].long()] = True
        assert not bool(got[~named].any()) and (fall or bool(got[named].any(-1).all()))
    if not fall:  # some segments' rows
        for s in (0, 1, S // 2, S - 1):
            rows = torch.arange(s * L, (s + 1) * L, device=gpu)
            if index:
                rows = idx[rows]
                rows = rows[(rows >= 0) & (rows < M)].long()
            rows = rows[:200]
            ks = slice(s * Lk, (s + 1) * Lk)
            want, tol, _ = ref.attention(q[rows], k[ks], v[ks], torch.tensor([0, len(rows)]), torch.tensor([0, Lk]))
            ref.assert_within(got[rows], want, tol)
