"""The conditional layer's operators (ops.group_norm, route, grouped_linear, combine, lora_linear) against their plain 64-bit
forms, with the bounds that layer_ref derives from the operation counts."""
import math

import pytest
import torch

import layer_ref as ref
from conftest import announce
from dense_ref import assert_within
from promptmoge_amd import ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F16, BF16, F32]
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g)


def cuts(gpu, *sizes, start=0):
    return (torch.tensor((0,) + sizes).cumsum(0) + start).to(torch.int64).to(gpu)


# ---------------------------------------------------------------------------------------------------------- group norm
def check_norm(gpu, sizes, C, groups, dt, *, out_dtype=None, act="none", affine=True, spread=1.0, mean=0.0, start=0, behind=0, x=None, seed=0, eps=1e-5):
    g = gen(seed)
    M = start + sum(sizes) + behind
    x = (randn(g, M, C) * spread + mean).to(dt).to(gpu) if x is None else x
    w, b = ((1 + 0.2 * randn(g, C)).to(gpu), randn(g, C).to(gpu)) if affine else (None, None)
    off = cuts(gpu, *sizes, start=start)
    announce(f"group_norm sizes={sizes[:6]} C={C} groups={groups} {dt} out={out_dtype} act={act} start={start} behind={behind}")
    got = ops.group_norm(x, groups, w, b, offsets=off, eps=eps, act=act, out_dtype=out_dtype)
    assert got.dtype == (out_dtype or dt) and got.shape == (M, C)
    want, tol, covered = ref.group_norm(x, groups, w, b, offsets=off, eps=eps, act=act, out_dtype=out_dtype)
    assert_within(got, want, tol, f"{sizes[:6]} {C} {groups}")
    assert not bool(got.cpu()[~covered].any())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sizes,C,groups", [
    ((1,), 64, 16), ((1,) * 8, 256, 32), ((1, 0, 2, 5), 48, 16), ((7,), 5, 5), ((3, 40), 15, 5), ((100,), 75, 1), ((37, 63), 600, 8),
    ((513,), 64, 32), ((5, 511, 300), 512, 32), ((50,), 4096, 1), ((20, 9), 2001, 3), ((64,), 33, 11), ((2000,), 64, 4), ((1100, 1400), 96, 12),
    ((4097,), 40, 40), ((3000, 1, 0, 2500), 130, 13), ((1500,), 4096, 32), ((1300, 900), 1001, 7)])
def test_norm_sizes(gpu, dt, sizes, C, groups):
    check_norm(gpu, sizes, C, groups, dt, seed=C)


@pytest.mark.parametrize("dt", [F16, F32])
def test_norm_large(gpu, dt):
    """Several tiles a segment and several segments a tile's length, checked on a sample of segments' rows in 64 bits."""
    check_norm(gpu, (30_000, 4_000, 11), 64, 16, dt, act="silu", seed=3)
    check_norm(gpu, (9_000, 9_100, 8_800, 9_050), 128, 32, dt, seed=4)


@pytest.mark.parametrize("C,groups", [(256, 32), (64, 16), (24, 8), (7, 7), (512, 1), (4096, 2), (320, 5)])
def test_norm_many_short_segments(gpu, C, groups):
    g = gen(C)
    sizes = tuple(torch.randint(0, 9, (3000,), generator=g).tolist())
    check_norm(gpu, sizes, C, groups, F16, start=2, behind=3)
    check_norm(gpu, (1,) * 700, C, groups, F32, act="gelu_tanh", out_dtype=BF16)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt,out", [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F16, F32), (F32, BF16)])
def test_norm_epilogues(gpu, act, dt, out):
    check_norm(gpu, (70, 30), 96, 8, dt, out_dtype=out, act=act, affine=act != "relu", seed=1)
    check_norm(gpu, (1500,), 96, 8, dt, out_dtype=out, act=act, affine=act != "relu", seed=2)


@pytest.mark.parametrize("dt", TYPES)
def test_norm_rows_of_no_segment(gpu, dt):
    """Rows in front of the first and behind the last segment are 0 in a new result and left alone in a given one."""
    for sizes, C, G in (((20, 30), 64, 8), ((1200, 700), 64, 8), ((), 64, 8), ((0, 0), 64, 8)):
        check_norm(gpu, sizes, C, G, dt, start=9, behind=77, act="silu")
        x = randn(gen(1), 86 + sum(sizes), C).to(dt).to(gpu)
        out = torch.full_like(x, 7.0)
        ops.group_norm(x, G, offsets=cuts(gpu, *sizes, start=9), out=out)
        want, tol, covered = ref.group_norm(x, G, offsets=cuts(gpu, *sizes, start=9))
        want[~covered], tol[~covered] = 7.0, 0.0
        assert_within(out, want, tol)


def test_norm_mean_far_from_zero(gpu):
    """A mean of 3000 times the spread, large and small values: sums in fp32 would lose all of it."""
    for sizes in ((300,), (5000,)):
        check_norm(gpu, sizes, 64, 8, F32, mean=3000.0, seed=5)
        check_norm(gpu, sizes, 64, 8, BF16, mean=100.0, seed=5)
        check_norm(gpu, sizes, 64, 8, F32, spread=1e18, mean=1e18, seed=6)
        check_norm(gpu, sizes, 64, 8, F32, spread=1e-12, seed=7, eps=1e-30)


def test_norm_constant_and_special_values(gpu):
    for n in (40, 2000):
        x = torch.randn(2 * n, 64, generator=gen(1)).to(gpu)
        x[:, 8:16] = 0.1  # a group without spread
        x[3, 20], x[n + 5, 40] = float("nan"), float("inf")
        off = cuts(gpu, n, n)
        announce(f"group_norm special {n}")
        got = ops.group_norm(x, 8, offsets=off)
        bad = torch.zeros(2 * n, 64, dtype=torch.bool)
        bad[:n, 16:24] = True  # that segment's group alone
        bad[n:, 40:48] = True
        assert torch.equal(torch.isnan(got.cpu()), bad)
        assert float(got[:, 8:16].abs().max()) < 1e-5


def test_norm_strides_in_place_and_odd_addresses(gpu):
    g = gen(8)
    big = randn(g, 1300, 3, 100).to(F16).to(gpu)
    for n in (200, 1300):
        for x in (big[:n, 1, :96], big[:n, 2, 3:99], big[:n, 0, 4:100]):
            check_norm(gpu, (n,), 96, 12, F16, x=x, act="silu")
    for n in (50, 1300):
        x = randn(g, n, 64).to(gpu)
        want, tol, _ = ref.group_norm(x, 8, act="gelu")
        announce("group_norm in place")
        got = ops.group_norm(x, 8, act="gelu", out=x)
        assert got is x
        assert_within(x, want, tol)
    buf = torch.full((700, 160), 3.0, dtype=BF16, device=gpu)
    x = randn(g, 700, 64).to(BF16).to(gpu)
    ops.group_norm(x, 4, out=buf[:, 65:129])
    want, tol, _ = ref.group_norm(x, 4)
    assert_within(buf[:, 65:129], want, tol)
    assert bool((buf[:, :65] == 3).all()) and bool((buf[:, 129:] == 3).all())
    assert ops.group_norm(x[:0], 4).shape == (0, 64)


def test_norm_offsets_beyond_32_bits(gpu):
    M, C = 2_200_000, 1024
    announce("group_norm of 2.25e9 elements")
    x = torch.zeros((M, C), dtype=F16, device=gpu)
    x[-300:] = randn(gen(1), 300, C).to(F16).to(gpu)
    off = torch.tensor([0, M - 300, M], device=gpu)
    got = ops.group_norm(x, 32, offsets=off, out=x)
    want, tol, _ = ref.group_norm(randn(gen(1), 300, C).to(F16), 32)
    assert_within(got[-300:], want, tol)
    assert not bool(got[:-300].any())


# --------------------------------------------------------------------------------------------------------------- route
def check_route(logits, k, *, score="softmax", normalize=False, mask=None):
    M, E = logits.shape
    announce(f"route M={M} E={E} k={k} {logits.dtype} {score} normalize={normalize} mask={mask is not None}")
    got = ops.route(logits, k, score=score, normalize=normalize, mask=mask)
    weights, tol, experts, offsets, pairs, rows = ref.route(logits, k, score=score, normalize=normalize, mask=mask)
    assert torch.equal(got.experts.cpu(), experts)
    assert torch.equal(got.offsets.cpu(), offsets)
    assert torch.equal(got.pairs.cpu(), pairs)
    assert torch.equal(got.rows.cpu(), rows)
    assert got.weights.dtype == F32
    assert_within(got.weights, weights, tol, f"weights {M} {E} {k}")
    return got


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,E,k", [(0, 8, 2), (1, 1, 1), (1, 64, 4), (5, 3, 3), (33, 8, 2), (100, 16, 16), (64, 32, 32), (7, 1024, 32), (1000, 64, 8), (4097, 8, 2),
                                   (3000, 5, 1), (2500, 257, 6), (900, 1000, 3), (9001, 24, 4), (20_000, 2, 2)])
def test_route_sizes(gpu, dt, M, E, k):
    x = randn(gen(M + E), M, E).to(dt).to(gpu)
    check_route(x, k)
    check_route(x, k, score="sigmoid", normalize=True)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("M", [50, 6000])
def test_route_masks(gpu, score, normalize, M):
    g = gen(2)
    x = randn(g, M, 12).to(gpu)
    for share in (0.0, 0.3, 1.0):
        mask = (torch.rand(M, generator=g) >= share).to(gpu)
        check_route(x, 3, score=score, normalize=normalize, mask=mask)
        check_route(x, 3, score=score, normalize=normalize, mask=mask.to(torch.uint8) * 5)


@pytest.mark.parametrize("M", [40, 5000])
def test_route_equal_and_absent_logits(gpu, M):
    g = gen(3)
    x = torch.randint(-1, 2, (M, 20), generator=g).float()  # many equal ones, 0 and -0 among them
    x = torch.where((x == 0) & (torch.rand(M, 20, generator=g) < 0.5), -0.0, x)
    check_route(x.to(gpu), 6)
    x = randn(g, M, 20)
    x[torch.rand(M, 20, generator=g) < 0.6] = float("-inf")  # some rows keep fewer than six, some none
    x[1] = float("-inf")
    x[2] = torch.finfo(F32).min
    x[3, :19] = torch.finfo(F32).min
    for normalize in (False, True):
        for score in ("softmax", "sigmoid"):
            check_route(x.to(gpu), 6, score=score, normalize=normalize)
    assert not bool(ops.route(x[1:2].to(gpu), 6, normalize=True).weights.any())
    low = torch.tensor([[-87.5, -88.0, -90.0, -200.0], [-1000.0, -1001.0, -1000.0, -3e38], [-3e38, -3e38, -3e38, -3e38]]).to(gpu)
    check_route(low, 2, score="sigmoid", normalize=True)
    check_route(low, 4, score="sigmoid", normalize=True)


def test_route_values_that_are_no_numbers(gpu):
    x = randn(gen(4), 30, 9)
    x[2, 3] = float("nan")
    x[5] = float("nan")
    x[7, 1] = float("inf")
    x[8, 2], x[8, 4] = float("inf"), float("nan")
    for normalize in (False, True):
        for score in ("softmax", "sigmoid"):
            check_route(x.to(gpu), 2, score=score, normalize=normalize)


def test_route_uneven_loads_and_strides(gpu):
    """All rows to one expert; rows of a wider tensor."""
    x = torch.zeros(5000, 40)
    x[:, 17] = 5.0
    check_route(x.to(gpu), 1)
    big = randn(gen(5), 3000, 50).to(BF16).to(gpu)
    check_route(big[:, 3:44], 4)
    check_route(big[::3, 10:], 4)


# ------------------------------------------------------------------------------------------------------------- experts
def check_grouped(gpu, offsets, Mx, K, N, dt, *, index=None, out_index=None, rows=None, bias=True, act="none", residual=None, out_dtype=None,
                  seed=0, x=None, sample=None):
    g = gen(seed)
    S = offsets.shape[0] - 1
    out_dtype = out_dtype or dt
    x = randn(g, Mx, K).to(dt).to(gpu) if x is None else x
    w = (randn(g, S, N, K) / math.sqrt(K)).to(dt).to(gpu)
    b = randn(g, S, N).to(gpu) if bias else None
    P = Mx if index is None else index.shape[0]
    rows = P if rows is None else rows
    r = randn(g, rows, N).to(residual).to(gpu) if residual else None
    announce(f"grouped_linear S={S} P={P} Mx={Mx} K={K} N={N} {dt} index={index is not None} out_index={out_index is not None} act={act} residual={residual}")
    kw = dict(index=index, out_index=out_index, act=act, residual=r)
    want, tol, given = ref.grouped_linear(x, w, offsets, b, rows=rows, out_dtype=out_dtype, **kw)
    if out_index is None:
        got = ops.grouped_linear(x, w, offsets, b, out_dtype=out_dtype, **kw)
        assert got.dtype == out_dtype and got.shape == (rows, N)
        assert_within(got, want, tol, f"{S} {P} {K} {N}")
    out = torch.full((rows, N), 7.0, dtype=out_dtype, device=gpu)
    assert ops.grouped_linear(x, w, offsets, b, out=out, **kw) is out
    want[~given], tol[~given] = 7.0, 0.0
    assert_within(out, want, tol, f"into out {S} {P} {K} {N}")


SIZES = [((1,), 64, 16), ((0, 3, 0, 1), 128, 48), ((5, 1, 9), 72, 40), ((16, 17, 15), 256, 64), ((2, 2, 1, 3, 0, 0, 4, 1), 1024, 200), ((40, 70), 64, 64),
         ((129, 0, 64, 63), 320, 130), ((600, 3), 200, 96), ((300, 300, 310), 512, 264), ((1, 900), 40, 33), ((64,) * 9, 96, 128)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sizes,K,N", SIZES)
def test_grouped_sizes(gpu, dt, sizes, K, N):
    check_grouped(gpu, cuts(gpu, *sizes), sum(sizes), K, N, dt, seed=K + N)


@pytest.mark.parametrize("table", [[0, 500, 200, 900], [900, 0, 300, 100], [-5, 700, 2 ** 40, 50], [2 ** 62, -2 ** 62, 0, 1200], [1000, 1000, 0, 0]])
def test_falling_offsets_stay_inside(gpu, table):
    """What the rows get is not said, but nothing around them is touched, and segments that do rise have theirs where no other takes
    their rows."""
    M, g = 1200, gen(3)
    off = torch.tensor(table, device=gpu)
    x = randn(g, M, 64).to(F16).to(gpu)
    w = randn(g, 3, 64, 64).to(F16).to(gpu)
    down, up = randn(g, 2, 8, 64).to(F16).to(gpu), randn(g, 2, 64, 8).to(F16).to(gpu)
    ids = torch.tensor([0, 1, 0], dtype=torch.int32, device=gpu)
    few = torch.tensor(table, device=gpu).clamp(-1, 40)
    calls = [lambda o, x, off: ops.group_norm(x, 8, offsets=off, out=o), lambda o, x, off: ops.grouped_linear(x, w, off, out=o),
             lambda o, x, off: ops.lora_linear(x, w[0], down, up, ids, offsets=off, out=o)]
    for i, f in enumerate(calls):
        for rows, offsets in ((M, off), (40, few)):
            announce(f"falling offsets {table} call {i} rows {rows}")
            buf = torch.full((rows + 64, 96), 7.0, dtype=F16, device=gpu)
            f(buf[32:32 + rows, 16:80], x[:rows], offsets)
            buf[32:32 + rows, 16:80] = 7.0
            assert bool((buf == 7.0).all())
            assert f(None, x[:rows], offsets).shape == (rows, 64)


def test_many_segments(gpu):
    """More of them than a wave looks at twice, most of them empty."""
    g = gen(11)
    sizes = torch.zeros(9000, dtype=torch.int64)
    sizes[torch.randint(0, 9000, (60,), generator=g)] = torch.randint(1, 30, (60,), generator=g)
    check_grouped(gpu, cuts(gpu, *sizes.tolist(), start=3), int(sizes.sum()) + 10, 32, 24, F16)
    check_lora(gpu, tuple(sizes.tolist()), 32, 24, 8, 5, F16, start=3, behind=7)
    check_norm(gpu, tuple(sizes.tolist()), 64, 8, F16, start=3, behind=7)
    sizes[[100, 5000]] = 3000
    check_lora(gpu, tuple(sizes.tolist()), 32, 24, 8, 5, F16)
    check_norm(gpu, tuple((sizes * 600).tolist()[4990:5010]) + (1,) * 100, 8, 8, F16)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sizes,K,N", [((1, 2), 1, 1), ((5, 0, 4), 3, 64), ((300, 7), 7, 33), ((70, 90), 65, 1), ((2000, 97), 130, 129), ((70,), 1021, 77)])
def test_grouped_odd_widths(gpu, dt, sizes, K, N):
    check_grouped(gpu, cuts(gpu, *sizes), sum(sizes), K, N, dt, seed=1, residual=dt)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt,out,res", [(F16, F16, None), (BF16, BF16, BF16), (F32, F32, F32), (F16, F32, F32), (BF16, F16, F32)])
@pytest.mark.parametrize("sizes", [(3, 0, 5), (700, 900, 650)])
def test_grouped_epilogues(gpu, act, dt, out, res, sizes):
    check_grouped(gpu, cuts(gpu, *sizes), sum(sizes), 128, 96, dt, act=act, residual=res, out_dtype=out, bias=act != "relu", seed=3)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,E,k,K,N", [(3, 8, 2, 64, 40), (200, 4, 2, 96, 72), (1500, 6, 3, 72, 136), (40, 64, 4, 128, 64)])
def test_grouped_by_a_router(gpu, dt, M, E, k, K, N):
    """Rows gathered (index), and results put in their pairs' places (out_index), with rows that the mask leaves out."""
    g = gen(M)
    mask = (torch.rand(M, generator=g) > 0.2).to(gpu)
    for m in (None, mask):
        r = ops.route(randn(g, M, E).to(gpu), k, mask=m)
        check_grouped(gpu, r.offsets, M, K, N, dt, index=r.rows, act="silu")
        check_grouped(gpu, r.offsets, M * k, K, N, dt, out_index=r.pairs)
        check_grouped(gpu, r.offsets, M, K, N, dt, index=r.rows, out_index=r.pairs, residual=F32, rows=M * k + 3)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("start,behind", [(0, 30), (9, 0), (100, 700)])
def test_grouped_positions_of_no_segment(gpu, dt, start, behind):
    for sizes in ((5, 0, 3), (200, 300), ()):
        check_grouped(gpu, cuts(gpu, *sizes, start=start), start + sum(sizes) + behind, 64, 72, dt)


@pytest.mark.parametrize("sizes", [(6, 10), (400, 300)])
def test_grouped_rows_outside(gpu, sizes):
    """Positions whose row of x or of the result does not exist give nothing; no row of x at all gives nothing anywhere."""
    g, P = gen(6), sum(sizes)
    index = torch.randint(0, 50, (P,), generator=g, dtype=torch.int32)
    index[::5], index[2::7] = -1, 50
    check_grouped(gpu, cuts(gpu, *sizes), 50, 64, 48, F16, index=index.to(gpu))
    to = torch.randperm(P, generator=g).to(torch.int32)
    to[::4], to[1::6] = -3, P + 9
    check_grouped(gpu, cuts(gpu, *sizes), P, 64, 48, F16, out_index=to.to(gpu), residual=F16)
    check_grouped(gpu, cuts(gpu, *sizes), 50, 64, 48, F16, index=index.to(gpu), out_index=to.to(gpu))
    check_grouped(gpu, cuts(gpu, *sizes), 0, 64, 48, F16, index=index.to(gpu))


def test_grouped_strides_and_in_place(gpu):
    g = gen(9)
    big = randn(g, 500, 3, 160).to(F16).to(gpu)
    off = cuts(gpu, 100, 0, 390, start=4)
    for x in (big[:, 1, :128], big[:, 1, 3:131], big[:, 2, 32:]):
        check_grouped(gpu, off, 500, 128, 72, F16, x=x, residual=F32)
    index = torch.randint(0, 250, (500,), generator=g, dtype=torch.int32).to(gpu)
    check_grouped(gpu, off, 250, 128, 72, F16, x=big[::2, 2, 32:], index=index)
    announce("grouped_linear into the residual")
    x, w = big[:, 0, :128], (randn(g, 3, 72, 128) / 11).to(F16).to(gpu)
    res = randn(g, 500, 144).to(gpu)
    keep = res.clone()
    want, tol, given = ref.grouped_linear(x, w, off, residual=res[:, 72:], out_dtype=F32)
    ops.grouped_linear(x, w, off, residual=res[:, 72:], out=res[:, 72:])
    want[~given], tol[~given] = keep.cpu().double()[:, 72:][~given], 0.0
    assert_within(res[:, 72:], want, tol)
    assert torch.equal(res[:, :72], keep[:, :72])
    assert ops.grouped_linear(x[:0], w, torch.zeros(4, dtype=torch.int64, device=gpu)).shape == (0, 72)
    assert not bool(ops.grouped_linear(x, w[:0], torch.zeros(1, dtype=torch.int64, device=gpu)).any())


def test_grouped_padding_is_not_read(gpu):
    """K ends inside the last tile, rows and columns inside a block: what lies behind is NaN and must not count."""
    for dt in TYPES:
        for sizes, K, N in (((130, 60), 72, 130), ((5, 9), 72, 20), ((900, 700), 40, 200)):
            announce(f"grouped padding {dt} {sizes} {K} {N}")
            P, g = sum(sizes), gen(5)
            xb = torch.full((P + 8, K + 24), float("nan"), dtype=dt, device=gpu)
            wb = torch.full((2 * N * K + 4096,), float("nan"), dtype=dt, device=gpu)
            xb[:P, :K] = randn(g, P, K).to(dt).to(gpu)
            wb[:2 * N * K] = randn(g, 2 * N * K).to(dt).to(gpu)
            x, w = xb[:P, :K], wb[:2 * N * K].view(2, N, K)
            want, tol, _ = ref.grouped_linear(x, w, cuts(gpu, *sizes), out_dtype=dt)
            assert_within(ops.grouped_linear(x, w, cuts(gpu, *sizes)), want, tol)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("sizes,K,N", [((1500, 40, 2600, 660), 1024, 1030), ((4000, 3900), 264, 776), ((20_000, 13_000), 64, 520)])
def test_grouped_large(gpu, dt, sizes, K, N):
    """Every tile shape, rows gathered, checked on a sample of positions in 64 bits."""
    P, S = sum(sizes), len(sizes)
    g = torch.Generator(device=gpu).manual_seed(P)
    x = torch.randn((P // 2, K), device=gpu, generator=g).to(dt)
    w = (torch.randn((S, N, K), device=gpu, generator=g) / math.sqrt(K)).to(dt)
    b = torch.randn((S, N), device=gpu, generator=g)
    index = torch.randint(0, P // 2, (P,), device=gpu, generator=g, dtype=torch.int32)
    announce(f"grouped large {dt} {sizes} {K} {N}")
    got = ops.grouped_linear(x, w, cuts(gpu, *sizes), b, index=index, act="gelu")
    at = 0
    for s, n in enumerate(sizes):
        rows = torch.cat([torch.arange(0, n, 41), torch.arange(max(0, n - 66), n)]).to(gpu) + at
        want, tol = ref.linear(x[index[rows].long()], w[s], b[s], act="gelu", out_dtype=dt)
        assert_within(got[rows], want, tol, f"segment {s}")
        at += n


@pytest.mark.parametrize("dt,sizes,K,N", [(F16, (23, 17), 64, 40), (F16, (41, 19), 1032, 40), (F16, (7001, 4999), 64, 136), (BF16, (300, 2200), 64, 3000),
                                          (BF16, (2101, 2099), 128, 3000), (F16, (3001, 1199), 520, 1000), (F32, (1, 39), 264, 40), (F32, (5000, 1003), 520, 136),
                                          (F32, (20, 30), 64, 40), (F32, (3001, 2999), 64, 264)])
def test_grouped_tile_shapes(gpu, dt, sizes, K, N):
    check_grouped(gpu, cuts(gpu, *sizes, start=3), sum(sizes) + 70, K, N, dt, residual=F32)


@pytest.mark.parametrize("S", [61, 62, 63, 126, 253, 254, 255])
def test_numbers_of_segments(gpu, S):
    """Around those up to which a block counts the tiles itself: empty segments, rows in front and behind."""
    g = gen(S)
    sizes = torch.randint(0, 70, (S,), generator=g)
    sizes[torch.randint(0, S, (S // 4,), generator=g)] = 0
    sizes[0], sizes[-1] = 33, 129
    for start, behind in ((0, 0), (70, 300)):
        M = start + int(sizes.sum()) + behind
        for dt in (F16, F32):
            check_grouped(gpu, cuts(gpu, *sizes.tolist(), start=start), M, 64, 72, dt)
        check_lora(gpu, tuple(sizes.tolist()), 128, 72, 8, 5, F16, start=start, behind=behind)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_mostly_positions_of_no_segment(gpu, dt):
    check_grouped(gpu, cuts(gpu, 40, 0, 90, start=9000), 20_000, 64, 72, dt)
    check_lora(gpu, (40, 0, 90), 64, 72, 8, 2, dt, start=9000, behind=9000)


def test_grouped_offsets_beyond_32_bits(gpu):
    """Rows in order behind 4 GiB, and indexed ones (which are read element by element there)."""
    M, K = 2_200_000, 1024
    announce("grouped_linear x of 2.25e9 elements")
    x = torch.zeros((M, K), dtype=F16, device=gpu)
    x[-300:] = randn(gen(1), 300, K).to(F16).to(gpu)
    w = (randn(gen(2), 2, 16, K) / 32).to(F16).to(gpu)
    got = ops.grouped_linear(x, w, torch.tensor([0, M - 150, M], device=gpu))
    want, tol, _ = ref.grouped_linear(x[-300:], w, torch.tensor([0, 150, 300]), out_dtype=F16)
    assert_within(got[-300:], want, tol)
    assert not bool(got[:-300].any())
    for n in (300, 20):
        index = torch.arange(M - n, M, device=gpu, dtype=torch.int32)
        got = ops.grouped_linear(x, w, torch.tensor([0, n // 2, n], device=gpu), index=index)
        want, tol, _ = ref.grouped_linear(x[-n:], w, torch.tensor([0, n // 2, n]), out_dtype=F16)
        assert_within(got, want, tol)


def test_grouped_special_values(gpu):
    for n in (20, 300):
        x = torch.randn(n, 64, generator=gen(2)).to(gpu)
        x[3, 5] = float("nan")
        w = torch.randn(2, 33, 64, generator=gen(3)).to(gpu)
        w[1, 4, 9] = float("inf")
        got = ops.grouped_linear(x, w, cuts(gpu, n // 2, n - n // 2))
        bad = torch.zeros(n, 33, dtype=torch.bool)
        bad[3] = True
        bad[n // 2:, 4] = True
        assert torch.equal(~torch.isfinite(got.cpu()), bad)


# ------------------------------------------------------------------------------------------------------------- combine
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,k,N", [(1, 1, 1), (1, 4, 1024), (0, 2, 16), (33, 2, 64), (100, 3, 37), (1000, 8, 256), (77, 32, 130), (5000, 2, 256)])
def test_combine(gpu, dt, M, k, N):
    g = gen(M + N)
    y, w = randn(g, M, k, N).to(dt), torch.rand((M, k), generator=g)
    gone = torch.rand((M, k), generator=g) < 0.2
    w[gone] = 0.0
    y[gone] = float("nan")  # (not read)
    y, w = y.to(gpu), w.to(gpu)
    for res, out in ((None, dt), (F32, F32), (dt, dt), (BF16, F16)):
        r = randn(g, M, N).to(res).to(gpu) if res else None
        announce(f"combine M={M} k={k} N={N} {dt} residual={res} out={out}")
        got = ops.combine(y, w, residual=r, out_dtype=out)
        assert got.dtype == out and got.shape == (M, N)
        want, tol = ref.combine(y, w, residual=r, out_dtype=out)
        assert_within(got, want, tol)


def test_combine_strides_and_in_place(gpu):
    g = gen(5)
    big = randn(g, 300, 4, 200).to(F16).to(gpu)
    w = torch.rand((300, 3), generator=g).to(gpu)
    for y in (big[:, 1:, 8:136], big[:, :3, 3:131], big[:, 1:, :128], big.permute(1, 0, 2)[:3].permute(1, 0, 2)[:, :, :128]):
        res = randn(g, 300, 160).to(gpu)
        keep = res.clone()
        want, tol = ref.combine(y, w, residual=res[:, 32:], out_dtype=F32)
        announce(f"combine strides {y.stride()}")
        ops.combine(y, w, residual=res[:, 32:], out=res[:, 32:])
        assert_within(res[:, 32:], want, tol)
        assert torch.equal(res[:, :32], keep[:, :32])


# ------------------------------------------------------------------------------------------------------------ adapters
def check_lora(gpu, sizes, K, N, r, A, dt, *, start=0, behind=0, rows=False, bias=True, scale=True, act="none", residual=None, out_dtype=None, seed=0, x=None, big=1.0):
    g = gen(seed)
    M = start + sum(sizes) + behind
    out_dtype = out_dtype or dt
    x = (randn(g, M, K) * big).to(dt).to(gpu) if x is None else x
    w = (randn(g, N, K) / math.sqrt(K)).to(dt).to(gpu)
    down, up = (randn(g, A, r, K) / math.sqrt(K)).to(dt).to(gpu), (randn(g, A, N, r) / math.sqrt(r)).to(dt).to(gpu)
    off = None if rows else cuts(gpu, *sizes, start=start)
    ids = torch.randint(-1, A + 1, (M if rows else len(sizes),), generator=g, dtype=torch.int32).to(gpu)  # -1 and A: none
    sc = (0.25 + torch.rand(A, generator=g)).to(gpu) if scale else None
    b = randn(g, N).to(gpu) if bias else None
    res = randn(g, M, N).to(residual).to(gpu) if residual else None
    announce(f"lora_linear sizes={sizes[:6]} rows={rows} K={K} N={N} r={r} A={A} {dt} act={act} residual={residual} out={out_dtype}")
    kw = dict(offsets=off, scale=sc, act=act, residual=res, out_dtype=out_dtype)
    got = ops.lora_linear(x, w, down, up, ids, b, **kw)
    assert got.dtype == out_dtype and got.shape == (M, N)
    want, tol = ref.lora_linear(x, w, down, up, ids, b, **kw)
    assert_within(got, want, tol, f"{sizes[:6]} {K} {N} {r}")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("r", [1, 4, 8, 16, 20, 48, 64, 128])
@pytest.mark.parametrize("sizes,K,N", [((1, 3), 64, 16), ((20, 0, 7, 33), 128, 72), ((200, 131), 256, 136), ((64, 64, 700), 72, 260)])
def test_lora_ranks_and_sizes(gpu, dt, r, sizes, K, N):
    check_lora(gpu, sizes, K, N, r, 3, dt, seed=r)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N,r", [(1, 1024, 64, 8), (33, 1024, 200, 16), (17, 72, 48, 4), (130, 256, 1024, 32), (700, 64, 264, 8), (2500, 40, 130, 16),
                                     (64, 2056, 40, 16), (8, 2056, 40, 8), (8, 64, 1000, 1), (3, 130, 33, 13), (4, 1024, 96, 16), (5, 33, 7, 12),
                                     (2, 1024, 1000, 16), (9, 64, 40, 7)])
def test_lora_of_single_rows(gpu, dt, M, K, N, r):
    check_lora(gpu, (1,) * M, K, N, r, 7, dt, rows=True, seed=M)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("r", [8, 24, 64, 100])
def test_lora_of_many_single_rows(gpu, dt, r):
    """Blocks of 16 rows that have one adapter, several in runs, or as many as there are."""
    M, K, N, A = 4500, 64, 40, 19
    g = gen(r)
    x, w = randn(g, M, K).to(dt).to(gpu), (randn(g, N, K) / 8).to(dt).to(gpu)
    down, up = (randn(g, A, r, K) / 8).to(dt).to(gpu), (randn(g, A, N, r) / math.sqrt(r)).to(dt).to(gpu)
    for run in (1, 5, 16, 700):
        ids = torch.randint(-2, A + 2, (M // run + 1,), generator=g, dtype=torch.int32).repeat_interleave(run)[:M].contiguous().to(gpu)
        announce(f"lora_linear {dt} r={r}: runs of {run}")
        assert_within(ops.lora_linear(x, w, down, up, ids), *ref.lora_linear(x, w, down, up, ids, out_dtype=dt))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sizes,K,N,r", [((1, 2), 1, 1, 1), ((5, 90), 3, 64, 2), ((300, 200), 65, 33, 5), ((130, 100), 130, 129, 7), ((70,), 1021, 77, 3)])
def test_lora_odd_widths(gpu, dt, sizes, K, N, r):
    check_lora(gpu, sizes, K, N, r, 2, dt, residual=dt)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt,out,res", [(F16, F16, None), (BF16, BF16, BF16), (F32, F32, F32), (F16, F32, F32), (BF16, F32, F16)])
def test_lora_epilogues(gpu, act, dt, out, res):
    for sizes in ((9, 4), (300, 150)):
        check_lora(gpu, sizes, 128, 96, 16, 2, dt, act=act, residual=res, out_dtype=out, bias=act != "relu", scale=act != "silu", seed=3)


@pytest.mark.parametrize("dt", TYPES)
def test_lora_rows_of_no_segment(gpu, dt):
    for sizes in ((5, 0, 9), (200, 300), (), (0,)):
        check_lora(gpu, sizes, 64, 72, 8, 2, dt, start=11, behind=140)


def test_lora_low_products_keep_their_accuracy(gpu):
    """Low products far above and below fp16's range, beside a projection of 0: parts of a row are scaled by its largest."""
    for dt in (F16, BF16):
        for e in (-18, -8, 0, 8, 12):
            g = gen(e + 20)
            x = (randn(g, 300, 64) * 2.0 ** min(e, 8)).to(dt).to(gpu)
            down = (randn(g, 2, 16, 64) * 2.0 ** min(e, 8)).to(dt).to(gpu)
            up = (randn(g, 2, 40, 16) * 2.0 ** (-2 * min(e, 8))).clamp(-6e4, 6e4).to(dt).to(gpu)
            w = torch.zeros(40, 64, dtype=dt, device=gpu)
            sc = torch.tensor([1.0, 2.0 ** (max(e, 8) - 8)], device=gpu)
            ids = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
            announce(f"lora range {dt} {e}")
            got = ops.lora_linear(x, w, down, up, ids, offsets=cuts(gpu, 100, 200), scale=sc, out_dtype=F32)
            want, tol = ref.lora_linear(x, w, down, up, ids, offsets=cuts(gpu, 100, 200), scale=sc, out_dtype=F32)
            assert_within(got, want, tol)


def test_lora_special_values(gpu):
    for sizes in ((9, 11), (150, 200)):
        n = sum(sizes)
        x = torch.randn(n, 64, generator=gen(2))
        x[3, 5], x[7, 2] = float("nan"), float("inf")
        x = x.to(F16).to(gpu)
        w, down, up = (torch.randn(*s, generator=gen(3)).to(F16).to(gpu) for s in ((40, 64), (2, 8, 64), (2, 40, 8)))
        got = ops.lora_linear(x, w, down, up, torch.tensor([1, -1], dtype=torch.int32, device=gpu), offsets=cuts(gpu, *sizes))
        bad = torch.zeros(n, 40, dtype=torch.bool)
        bad[[3, 7]] = True
        assert torch.equal(~torch.isfinite(got.cpu()), bad)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_lora_large(gpu, dt):
    """Large tiles, checked on a sample of rows in 64 bits."""
    sizes, K, N, r = (1200, 1100, 1300, 1200), 1024, 1024, 16
    g = torch.Generator(device=gpu).manual_seed(1)
    M = sum(sizes)
    x = torch.randn((M, K), device=gpu, generator=g).to(dt)
    w = (torch.randn((N, K), device=gpu, generator=g) / 32).to(dt)
    down, up = (torch.randn((3, r, K), device=gpu, generator=g) / 32).to(dt), (torch.randn((3, N, r), device=gpu, generator=g) / 4).to(dt)
    res = torch.randn((M, N), device=gpu, generator=g).to(dt)
    ids = torch.tensor([2, 0, -1, 1], dtype=torch.int32, device=gpu)
    announce(f"lora large {dt}")
    got = ops.lora_linear(x, w, down, up, ids, offsets=cuts(gpu, *sizes), residual=res)
    rows = torch.cat([torch.arange(0, M, 37), torch.arange(1190, 1210), torch.arange(M - 70, M)]).unique().to(gpu)
    one = ids.repeat_interleave(torch.tensor(sizes, device=gpu))[rows]
    want, tol = ref.lora_linear(x[rows], w, down, up, one, residual=res[rows], out_dtype=dt)
    assert_within(got[rows], want, tol)


def test_lora_strides_and_in_place(gpu):
    g = gen(4)
    big = randn(g, 400, 3, 160).to(F16).to(gpu)
    for sizes in ((4,) * 100, (180, 220)):
        for x in (big[:, 1, :128], big[:, 1, 3:131], big[:, 2, 32:]):
            check_lora(gpu, sizes, 128, 72, 8, 2, F16, x=x, residual=F32)
    x, w = big[:, 0, :128], (randn(g, 72, 128) / 11).to(F16).to(gpu)
    down, up = (randn(g, 2, 8, 128) / 11).to(F16).to(gpu), randn(g, 2, 72, 8).to(F16).to(gpu)
    ids, off = torch.tensor([1, 0], dtype=torch.int32, device=gpu), cuts(gpu, 190, 200, start=3)
    res = randn(g, 400, 72).to(gpu)
    want, tol = ref.lora_linear(x, w, down, up, ids, offsets=off, residual=res, out_dtype=F32)
    announce("lora_linear into the residual")
    assert ops.lora_linear(x, w, down, up, ids, offsets=off, residual=res, out=res) is res
    assert_within(res, want, tol)
    assert ops.lora_linear(x[:0], w, down, up, ids[:0]).shape == (0, 72)
    none = ops.lora_linear(x, w, down[:0], up[:0], ids, offsets=off)  # no adapters at all
    assert_within(none, *ref.linear(x, w, out_dtype=F16))


# --------------------------------------------------------------------------------------------------- a layer of them all
def make_layer(gpu, g, C, H, E, r, A, dt):
    t = lambda *s: (randn(g, *s) / math.sqrt(s[-1])).to(dt).to(gpu)  # noqa: E731
    return dict(gamma=(1 + 0.1 * randn(g, C)).to(gpu), beta=(0.1 * randn(g, C)).to(gpu), router=randn(g, E, C).to(dt).to(gpu) / math.sqrt(C), up=t(E, H, C),
                up_b=(0.1 * randn(g, E, H)).to(gpu), dn=t(E, C, H), dn_b=(0.1 * randn(g, E, C)).to(gpu), w=t(C, C), a=t(A, r, C), b=t(A, C, r))


def layer(p, x, offsets, mask, adapter, k=2):
    """A conditional block of a batch of frames: norm, router, experts, their sum onto the stream, a projection with the frames' adapters."""
    M, C = x.shape
    h = ops.group_norm(x, 8, p["gamma"], p["beta"], offsets=offsets, act="silu")
    r = ops.route(ops.linear(h, p["router"], out_dtype=F32), k, normalize=True, mask=mask)
    u = ops.grouped_linear(h, p["up"], r.offsets, p["up_b"], index=r.rows, act="gelu")
    y = ops.grouped_linear(u, p["dn"], r.offsets, p["dn_b"], out_index=r.pairs, out=x.new_empty((M * k, C)))
    z = ops.combine(y.view(M, k, C), r.weights, residual=x)
    return ops.lora_linear(z, p["w"], p["a"], p["b"], adapter, offsets=offsets, residual=z), (h, r, u, y, z)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sizes", [(1, 1, 1), (40, 0, 90), (700, 900)])
def test_layer_of_all(gpu, dt, sizes):
    """Each step against its plain form on what the step before gave."""
    g = gen(7)
    C, H, E, k = 64, 96, 6, 2
    p = make_layer(gpu, g, C, H, E, 8, 3, dt)
    M = sum(sizes)
    x, off, mask = randn(g, M, C).to(dt).to(gpu), cuts(gpu, *sizes), (torch.rand(M, generator=g) > 0.2).to(gpu)
    ids = torch.tensor([2, 0, -1][:len(sizes)], dtype=torch.int32, device=gpu)
    announce(f"layer {dt} {sizes}")
    out, (h, r, u, y, z) = layer(p, x, off, mask, ids)
    assert_within(h, *ref.group_norm(x, 8, p["gamma"], p["beta"], offsets=off, act="silu")[:2])
    logits = ops.linear(h, p["router"], out_dtype=F32)
    weights, tol, experts, offsets, pairs, rows = ref.route(logits, k, normalize=True, mask=mask)
    assert torch.equal(r.pairs.cpu(), pairs) and torch.equal(r.rows.cpu(), rows) and torch.equal(r.offsets.cpu(), offsets)
    assert_within(r.weights, weights, tol)
    assert_within(u, *ref.grouped_linear(h, p["up"], offsets, p["up_b"], index=rows, act="gelu", out_dtype=dt)[:2])
    want, tol, given = ref.grouped_linear(u, p["dn"], offsets, p["dn_b"], out_index=pairs, rows=M * k, out_dtype=dt)
    assert_within(y[given.to(gpu)], want[given], tol[given])
    assert_within(z, *ref.combine(y.view(M, k, C), r.weights, residual=x, out_dtype=dt))
    assert torch.equal(z[~mask], x[~mask])
    assert_within(out, *ref.lora_linear(z, p["w"], p["a"], p["b"], ids, offsets=off, residual=z, out_dtype=dt))


def test_layer_in_a_graph_and_on_two_streams(gpu):
    """Captured and replayed on new inputs with eager work in between, and two of them at once on streams of their own: each time
    the bits of the eager call."""
    g = gen(8)
    sizes = (900, 300, 1200)
    p = make_layer(gpu, g, 64, 128, 8, 16, 3, F16)
    M = sum(sizes)
    xs = [randn(g, M, 64).to(F16).to(gpu) for _ in range(4)]
    off, mask = cuts(gpu, *sizes), (torch.rand(M, generator=g) > 0.1).to(gpu)
    ids = torch.tensor([1, 2, 0], dtype=torch.int32, device=gpu)
    want = [layer(p, x, off, mask, ids)[0].clone() for x in xs]
    torch.cuda.synchronize()
    graphs, ins, outs = [], [], []
    for i in range(2):
        x = xs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(p, x, off, mask, ids)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        announce(f"layer captured {i}")
        with torch.cuda.graph(graph):
            out = layer(p, x, off, mask, ids)[0]
        graphs.append(graph), ins.append(x), outs.append(out)
    for round_ in range(3):
        for i in range(4):
            ins[0].copy_(xs[i]), ins[1].copy_(xs[3 - i])
            announce(f"layer replayed {round_} {i}")
            graphs[0].replay(), graphs[1].replay()
            again = layer(p, xs[i], off, mask, ids)[0]
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[3 - i]) and torch.equal(again, want[i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = {}
    announce("layer on two streams")
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = layer(p, xs[i], off, mask, ids)[0]
    torch.cuda.synchronize()
    for i in range(4):
        assert torch.equal(got[i], want[i])
