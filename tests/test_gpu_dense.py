"""The dense operators (ops.linear, linear_i8, qk_norm_rope, sparse_attention) against their plain 64-bit forms, with the
bounds that dense_ref derives from the operation counts."""
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


# ------------------------------------------------------------------------------------------------------------- linear
def check_linear(gpu, M, K, N, dt, *, bias=True, act="none", residual=None, out_dtype=None, seed=0, x=None, w=None):
    g = gen(seed)
    x = randn(g, M, K).to(dt).to(gpu) if x is None else x
    w = (randn(g, N, K) / math.sqrt(K)).to(dt).to(gpu) if w is None else w
    b = randn(g, N).to(gpu) if bias else None
    r = randn(g, M, N).to(residual).to(gpu) if residual else None
    out_dtype = out_dtype or dt
    announce(f"linear M={M} K={K} N={N} {dt} act={act} residual={residual} out={out_dtype}")
    got = ops.linear(x, w, b, act=act, residual=r, out_dtype=out_dtype)
    assert got.dtype == out_dtype and got.shape == (M, N)
    want, tol = ref.linear(x, w, b, act=act, residual=r, out_dtype=out_dtype)
    ref.assert_within(got, want, tol, f"{M}x{K}x{N}")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 64, 16), (1, 1024, 1000), (3, 72, 40), (17, 128, 48), (33, 1024, 64), (64, 256, 513),
                                   (200, 40, 96), (129, 320, 130), (1000, 64, 64), (700, 512, 260), (5000, 96, 128),
                                   (9001, 72, 200)])
def test_linear_sizes(gpu, dt, M, K, N):
    check_linear(gpu, M, K, N, dt, seed=M + K + N)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,K,N", [(4099, 200, 1030), (4800, 1024, 4096), (8200, 1024, 2056), (20_000, 264, 776), (33_000, 64, 520)])
def test_linear_large(gpu, dt, M, K, N):
    """Every tile shape, with rows, columns and k that end inside a tile; checked on a sample of rows in 64 bits."""
    g = torch.Generator(device=gpu).manual_seed(M)
    x = torch.randn((M, K), device=gpu, generator=g).to(dt)
    w = (torch.randn((N, K), device=gpu, generator=g) / math.sqrt(K)).to(dt)
    b, r = torch.randn(N, device=gpu, generator=g), torch.randn((M, N), device=gpu, generator=g).to(dt)
    announce(f"linear large {dt} {M} {K} {N}")
    got = ops.linear(x, w, b, act="gelu", residual=r)
    rows = torch.cat([torch.arange(0, M, 37), torch.arange(M - 70, M)]).to(gpu)
    want, tol = ref.linear(x[rows], w, b, act="gelu", residual=r[rows], out_dtype=dt)
    ref.assert_within(got[rows], want, tol)


@pytest.mark.parametrize("dt", [F16, BF16, torch.int8])
@pytest.mark.parametrize("M,K,N", [(9_700, 1024, 1000), (30_001, 272, 264), (19_300, 816, 200), (4_777, 4096, 520)])
def test_linear_large_of_middle_tiles(gpu, dt, M, K, N):
    """Tiles of 128 rows, with and without a residual read ahead; checked on a sample of rows in 64 bits."""
    g = torch.Generator(device=gpu).manual_seed(M)
    i8 = dt == torch.int8
    if i8:
        x = torch.randint(-127, 128, (M, K), device=gpu, generator=g, dtype=dt)
        w = torch.randint(-127, 128, (N, K), device=gpu, generator=g, dtype=dt)
        kw = dict(a_scale=4.0 / 127, w_scale=(0.5 + torch.rand(N, device=gpu, generator=g)) / (74 * math.sqrt(K)), out_dtype=F16)
    else:
        x = torch.randn((M, K), device=gpu, generator=g).to(dt)
        w = (torch.randn((N, K), device=gpu, generator=g) / math.sqrt(K)).to(dt)
        kw = dict(out_dtype=dt)
    b = torch.randn(N, device=gpu, generator=g)
    rows = torch.cat([torch.arange(0, M, 41), torch.arange(M - 130, M)]).to(gpu)
    for r in (None, torch.randn((M, N), device=gpu, generator=g).to(F16)):
        announce(f"linear middle tiles {dt} {M} {K} {N} residual={r is not None}")
        got = (ops.linear_i8 if i8 else ops.linear)(x, w, b, act="silu", residual=r, **kw)
        want, tol = ref.linear(x[rows], w, b, act="silu", residual=None if r is None else r[rows], **kw)
        ref.assert_within(got[rows], want, tol)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (5, 3, 64), (300, 7, 33), (9000, 3, 64), (2000, 65, 1), (4097, 130, 129), (70, 1021, 77)])
def test_linear_odd_widths(gpu, dt, M, K, N):
    check_linear(gpu, M, K, N, dt, seed=1, residual=dt)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt,out,res", [(F16, F16, None), (BF16, BF16, BF16), (F32, F32, F32), (F16, F32, F32), (BF16, F16, F32)])
@pytest.mark.parametrize("M", [7, 2500])
def test_linear_epilogues(gpu, act, dt, out, res, M):
    check_linear(gpu, M, 128, 96, dt, act=act, residual=res, out_dtype=out, bias=act != "relu", seed=3)


@pytest.mark.parametrize("M,K,N,act,res,out", [(1, 64, 16, "none", None, F32), (50, 48, 33, "silu", F16, F16), (77, 80, 16, "none", F32, BF16),
                                               (3000, 256, 256, "silu", F16, F16), (9001, 1024, 130, "gelu", F32, F32),
                                               (300, 17, 40, "none", None, F32)])
def test_linear_i8(gpu, M, K, N, act, res, out):
    g = gen(7)
    x = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8).to(gpu)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).to(gpu)
    ws, b = (torch.rand(N, generator=g) / (74 * math.sqrt(K))).to(gpu), randn(g, N).to(gpu)
    r = randn(g, M, N).to(res).to(gpu) if res else None
    announce(f"linear_i8 {M} {K} {N} {act} {res} {out}")
    got = ops.linear_i8(x, w, b, a_scale=0.03, w_scale=ws, act=act, residual=r, out_dtype=out)
    want, tol = ref.linear(x, w, b, a_scale=0.03, w_scale=ws, act=act, residual=r, out_dtype=out)
    ref.assert_within(got, want, tol)
    exact = ops.linear_i8(x, w)  # the sums themselves: exact in fp32 below 2^24
    assert torch.equal(exact.cpu().double(), x.cpu().double() @ w.cpu().double().t())


def test_linear_strides_in_place_and_views(gpu):
    g = gen(11)
    big = randn(g, 500, 3, 160).to(F16).to(gpu)
    w = randn(g, 72, 128).to(F16).to(gpu)
    check_linear(gpu, 500, 128, 72, F16, x=big[:, 1, :128], w=w, residual=F32)  # rows of 480 elements, 16-byte aligned
    check_linear(gpu, 500, 128, 72, F16, x=big[:, 1, 3:131], w=w)  # not aligned
    check_linear(gpu, 250, 128, 72, F16, x=big[::2, 2, 32:], w=w)
    announce("linear into the residual and into a strided view")
    x = big[:, 0, :128]
    res = randn(g, 500, 144).to(gpu)
    keep = res.clone()
    want, tol = ref.linear(x, w, residual=res[:, 72:], out_dtype=F32)
    got = ops.linear(x, w, residual=res[:, 72:], out=res[:, 72:])
    assert got.data_ptr() == res[:, 72:].data_ptr()
    ref.assert_within(res[:, 72:], want, tol)
    assert torch.equal(res[:, :72], keep[:, :72])
    assert ops.linear(x[:0], w).shape == (0, 72)


def test_linear_zero_padding_is_not_read(gpu):
    """K ends inside the last tile of 128 bytes, M and N inside a block: what lies behind is NaN and must not count."""
    for dt in TYPES:
        for M, K, N in ((130, 72, 130), (20, 72, 20), (4000, 40, 200)):
            announce(f"linear padding {dt} {M} {K} {N}")
            xb = torch.full((M + 8, K + 24), float("nan"), dtype=dt, device=gpu)
            wb = torch.full((N * K + 4096,), float("nan"), dtype=dt, device=gpu)
            g = gen(5)
            xb[:M, :K] = randn(g, M, K).to(dt).to(gpu)
            wb[:N * K] = randn(g, N * K).to(dt).to(gpu)
            x, w = xb[:M, :K], wb[:N * K].view(N, K)
            want, tol = ref.linear(x, w, out_dtype=dt)
            ref.assert_within(ops.linear(x, w), want, tol)


def test_linear_special_values(gpu):
    x = torch.randn(40, 64, generator=gen(2)).to(gpu)
    x[3, 5], x[7, 1] = float("nan"), float("inf")
    w = torch.randn(33, 64, generator=gen(3)).to(gpu)
    for act in ("none", "relu", "silu", "gelu"):
        announce(f"linear special {act}")
        got = ops.linear(x, w, act=act)
        assert bool(torch.isnan(got[3]).all()) and not bool(torch.isnan(got[[0, 1, 2, 4, 5, 6]]).any())
        assert not bool(torch.isfinite(got[7, ((w[:, 1] > 0))]).any())


def test_linear_offsets_beyond_32_bits(gpu):
    M, K = 2_200_000, 1024
    announce("linear x of 2.25e9 elements")
    x = torch.zeros((M, K), dtype=torch.int8, device=gpu)
    x[-300:] = torch.randint(-127, 128, (300, K), generator=gen(1), dtype=torch.int8).to(gpu)
    w = torch.randint(-127, 128, (16, K), generator=gen(2), dtype=torch.int8).to(gpu)
    got = ops.linear_i8(x, w)
    assert torch.equal(got[-300:].cpu().double(), x[-300:].cpu().double() @ w.cpu().double().t())
    assert not bool(got[:-300].any())


def test_linear_refusals(gpu):
    x, w = torch.zeros(8, 64, dtype=F16, device=gpu), torch.zeros(16, 64, dtype=F16, device=gpu)
    for f, msg in [(lambda: ops.linear(x.double(), w), "float32"), (lambda: ops.linear(x, w.float()), "w must be"),
                   (lambda: ops.linear(x, w[:, :32]), "contiguous"), (lambda: ops.linear(x[:, :32], w), "input channels"),
                   (lambda: ops.linear(x, w, act="tanh"), "act must"), (lambda: ops.linear(x[0], w), "2-D"),
                   (lambda: ops.linear(x, w, w[:, 0]), "bias must"), (lambda: ops.linear(x.t().contiguous().t(), w), "contiguous rows"),
                   (lambda: ops.linear(x[:1].expand(8, 64), w), "overlap"),
                   (lambda: ops.linear(x, w, residual=x), "residual must"),
                   (lambda: ops.linear(x, w, out=x[:, :16]), "overlap"),
                   (lambda: ops.linear(x, w, out=x.new_zeros(8, 8)), "out must"),
                   (lambda: ops.linear_i8(x, w), "int8"), (lambda: ops.linear(x, w, out_dtype=torch.float64), "float32")]:
        with pytest.raises(ValueError, match=msg):
            f()
    with pytest.raises(RuntimeError, match="inference-only"):
        ops.linear(x.requires_grad_(), w)
    with torch.no_grad():
        assert ops.linear(x, w).shape == (8, 16)


# --------------------------------------------------------------------------------------------------------------- rope
def coords_of(g, M, top=600):
    c = torch.randint(0, top, (M, 4), generator=g, dtype=torch.int32)
    c[:, 0] = 0
    return c


def freqs_of(g, P):
    return torch.rand((P, 3), generator=g)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,Hq,Hk,D,P,norm,inter", [
    (1, 1, 1, 8, 4, "rms", False), (1, 16, 4, 64, 32, "layer", True), (77, 8, 8, 32, 16, "rms", False), (33, 6, 2, 40, 20, "layer", False),
    (300, 3, 1, 128, 64, "rms", True), (129, 5, 5, 96, 48, "rms", False), (50, 4, 0, 64, 32, "rms", False), (64, 2, 2, 16, 5, "layer", True),
    (64, 2, 2, 64, 10, "rms", False), (40, 2, 1, 24, 0, "rms", False), (1000, 1, 1, 56, 28, "layer", True)])
def test_rope(gpu, dt, M, Hq, Hk, D, P, norm, inter):
    g = gen(M + D)
    qkv = randn(g, M, Hq + 2 * max(Hk, 1), D).to(dt).to(gpu)
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hk] if Hk else None
    c, f = coords_of(g, M).to(gpu), freqs_of(g, P).to(gpu)
    w = [(1 + 0.2 * randn(g, D)).to(gpu) for _ in range(2)]
    b = [(0.1 * randn(g, D)).to(gpu) if norm == "layer" else None for _ in range(2)]
    announce(f"rope {dt} M={M} {Hq}/{Hk} D={D} P={P} {norm} inter={inter}")
    keep = qkv.clone()
    qo, ko = ops.qk_norm_rope(q, k, c, f, q_weight=w[0], k_weight=w[1], q_bias=b[0], k_bias=b[1], norm=norm, interleaved=inter)
    assert torch.equal(keep, qkv)
    for x, o, ww, bb in ((q, qo, w[0], b[0]), (k, ko, w[1], b[1])):
        if x is None:
            assert o is None
            continue
        want, tol = ref.norm_rope(x, ww, bb, c, f, layer=norm == "layer", interleaved=inter)
        ref.assert_within(o, want, tol)
    # in place
    ops.qk_norm_rope(q, k, c, f, q_weight=w[0], k_weight=w[1], q_bias=b[0], k_bias=b[1], norm=norm, interleaved=inter, out=(q, k))
    assert torch.equal(q, qo) and (k is None or torch.equal(k, ko))
    assert torch.equal(qkv[:, Hq + Hk:], keep[:, Hq + Hk:])


def test_rope_far_positions_and_plain_weights(gpu):
    g = gen(5)
    M, D = 64, 64
    q = randn(g, M, 2, D).to(gpu)
    c = torch.randint(-2 ** 31, 2 ** 31 - 1, (M, 4), generator=g, dtype=torch.int64).to(torch.int32).to(gpu)
    f = freqs_of(g, 32).to(gpu)
    announce("rope far positions")
    qo, _ = ops.qk_norm_rope(q, None, c, f)
    want, tol = ref.norm_rope(q, None, None, c, f, layer=False, interleaved=False)
    # three products of 2^31 and their sum in 64 bits: an angle is off by less than 2^-19 turns' radians on either side
    ref.assert_within(qo, want, tol + 2.0 ** -18 * want.abs().amax(-1, keepdim=True))


def test_rope_misaligned_views_and_zero_rows(gpu):
    g = gen(9)
    base = randn(g, 30, 2 * 24 + 1).to(F16).to(gpu)
    q = base[:, 1:].unflatten(1, (2, 24))
    c, f = coords_of(g, 30).to(gpu), freqs_of(g, 12).to(gpu)
    announce("rope misaligned")
    qo, _ = ops.qk_norm_rope(q, None, c, f)
    want, tol = ref.norm_rope(q, None, None, c, f, layer=False, interleaved=False)
    ref.assert_within(qo, want, tol)
    assert ops.qk_norm_rope(q[:0], None, c[:0], f)[0].shape == (0, 2, 24)
    z, _ = ops.qk_norm_rope(torch.zeros_like(q), None, c, f, eps=1e-6)
    assert not bool(z.any())


def test_rope_refusals(gpu):
    q = torch.zeros(4, 2, 16, device=gpu)
    c, f = torch.zeros(4, 4, dtype=torch.int32, device=gpu), torch.zeros(8, 3, device=gpu)
    for fn, msg in [(lambda: ops.qk_norm_rope(q.double(), None, c, f), "float32"), (lambda: ops.qk_norm_rope(q, q.half(), c, f), "k must"),
                    (lambda: ops.qk_norm_rope(q, None, c[:3], f), "coords"), (lambda: ops.qk_norm_rope(q, None, c.long(), f), "coords"),
                    (lambda: ops.qk_norm_rope(q, None, c, f.double()), "freqs"), (lambda: ops.qk_norm_rope(q, None, c, f, norm="l2"), "norm"),
                    (lambda: ops.qk_norm_rope(q, None, c, f, q_weight=torch.ones(8, device=gpu)), "q_weight"),
                    (lambda: ops.qk_norm_rope(q, q, c, f, out=(q, None)), "out"), (lambda: ops.qk_norm_rope(q[0], None, c, f), "rows")]:
        with pytest.raises(ValueError, match=msg):
            fn()
    with pytest.raises(_lib.PmgError, match="pairs"):
        ops.qk_norm_rope(q, None, c, torch.zeros(9, 3, device=gpu))
    with pytest.raises(_lib.PmgError, match="multiple of 8"):
        ops.qk_norm_rope(q[:, :, :12], None, c, f[:4])


# ---------------------------------------------------------------------------------------------------------- attention
def offsets_of(lengths, start=0):
    o = [start]
    for n in lengths:
        o.append(o[-1] + n)
    return torch.tensor(o, dtype=torch.int64)


def check_attention(gpu, dt, lengths, Hq, Hk, D, *, kv_lengths=None, start=0, tail=0, perm=False, bias=False, mask=0.0, cap=0.0,
                    scale=None, top=40, seed=0, spread=1.0, edit=None):
    g = gen(seed)
    off = offsets_of(lengths, start)
    Mq = int(off[-1]) + tail
    q = (spread * randn(g, Mq, Hq, D)).to(dt).to(gpu)
    kw = {"cap": cap, "scale": scale}
    koff, Mk = None, Mq
    if kv_lengths is not None:
        koff = offsets_of(kv_lengths)
        Mk = int(koff[-1])
    kv = randn(g, Mk, 2, Hk, D).to(dt).to(gpu)
    if perm:
        kw["index"] = torch.randperm(Mq, generator=g).to(torch.int32).to(gpu)
        if koff is not None:
            kw["kv_index"] = torch.randperm(Mk, generator=g).to(torch.int32).to(gpu)
    if bias:
        kw["coords"] = coords_of(g, Mq, top).to(gpu)
        if koff is not None:
            kw["kv_coords"] = coords_of(g, Mk, top).to(gpu)
        kw["slopes"] = (0.3 * torch.rand((Hq, 3), generator=g)).to(gpu)
    if mask:
        kw["kv_mask"] = (torch.rand(Mk, generator=g) >= mask).to(gpu)
    off = off.to(gpu)
    koff = koff.to(gpu) if koff is not None else None
    if edit:
        edit(q, kv, kw)
    announce(f"attention {dt} lengths={lengths[:8]} kv={kv_lengths and kv_lengths[:8]} {Hq}/{Hk} D={D} perm={perm} bias={bias} mask={mask} cap={cap}")
    got = ops.sparse_attention(q, kv[:, 0], kv[:, 1], off, koff, **kw)
    want, tol, covered = ref.attention(q, kv[:, 0], kv[:, 1], off, koff, **kw)
    ref.assert_within(got, want, tol)
    return q, kv, off, koff, kw, got


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lengths", [[1], [2, 0, 0, 5, 1, 1, 30], [31, 33, 64, 1], [300], [0, 700, 3, 0], [130, 129, 1, 257], [4] * 60])
@pytest.mark.parametrize("D", [32, 64])
def test_attention_lengths(gpu, dt, lengths, D):
    check_attention(gpu, dt, lengths, 2, 2, D, seed=sum(lengths) + D)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Hq,Hk,D", [(1, 1, 8), (3, 1, 16), (4, 2, 40), (5, 5, 24), (6, 2, 96), (8, 1, 128), (2, 1, 56), (33, 1, 64)])
@pytest.mark.parametrize("perm,bias,mask,cap", [(False, False, 0.0, 0.0), (True, True, 0.3, 0.0), (True, False, 0.3, 5.0), (False, True, 0.0, 20.0)])
def test_attention_heads_and_options(gpu, dt, Hq, Hk, D, perm, bias, mask, cap):
    check_attention(gpu, dt, [37, 0, 65, 1, 90], Hq, Hk, D, perm=perm, bias=bias, mask=mask, cap=cap, tail=9, start=3, seed=Hq + D)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("q,kv", [([1], [1]), ([1], [5000]), ([1, 1, 1], [700, 0, 3000]), ([1] * 40, [200] * 40), ([3, 0, 8, 1], [900, 40, 0, 1500]),
                                  ([1] * 70, [3] * 70), ([0, 100], [4000, 10]), ([40], [9000]), ([2, 2], [0, 0]), ([600, 1], [1, 600])])
def test_attention_few_queries(gpu, dt, q, kv):
    """Pooled queries on long frames: a block per segment, keys split over blocks; and the other way round."""
    check_attention(gpu, dt, q, 4, 2, 64, kv_lengths=kv, seed=len(q))
    check_attention(gpu, dt, q, 4, 4, 40, kv_lengths=kv, perm=True, bias=True, mask=0.4, seed=len(q))


@pytest.mark.parametrize("dt", TYPES)
def test_attention_long(gpu, dt):
    check_attention(gpu, dt, [2500, 1100], 2, 1, 64, bias=True, mask=0.2, perm=True, seed=3)
    check_attention(gpu, dt, [1300], 1, 1, 128, seed=4)
    check_attention(gpu, dt, [900, 900], 4, 4, 32, bias=True, top=500, seed=5)


@pytest.mark.parametrize("dt", TYPES)
def test_attention_rising_scores(gpu, dt):
    """Scores that grow along the keys by far more than a tile's range: the running maximum moves again and again."""
    def edit(q, kv, kw):
        n = kv.shape[0]
        q[:] = 1
        kv[:, 0] = (torch.arange(n, device=q.device, dtype=torch.float32) * (40.0 / n)).to(dt).view(n, 1, 1)
    check_attention(gpu, dt, [600], 2, 2, 32, scale=0.5, edit=edit)
    def down(q, kv, kw):
        edit(q, kv, kw)
        kv[:, 0] = kv[:, 0].flip(0)
    check_attention(gpu, dt, [600], 2, 2, 32, scale=0.5, edit=down)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_attention_scores_that_jump(gpu, dt, D):
    """Runs of keys whose scores lie up to 2^60 weights above the ones before, under a mask and under a bias."""
    def edit(q, kv, kw):
        n = kv.shape[0]
        q[:] = 1
        kv[:, 0] = (torch.arange(n, device=q.device) // 45 % 7 * 5.0).to(dt).view(n, 1, 1)
    check_attention(gpu, dt, [500], 2, 2, D, scale=1.0 / D, mask=0.2, edit=edit)
    check_attention(gpu, dt, [500, 300], 2, 2, D, scale=1.0 / D, bias=True, edit=edit)


@pytest.mark.parametrize("dt", TYPES)
def test_attention_first_keys_far_away(gpu, dt):
    """The first keys' scores lie thousands below the later ones' (and below 2^-128 of anything): they set the running
    maximum first and then count for nothing."""
    def edit(q, kv, kw):
        kw["coords"][:, 1:] = 5
        kw["coords"][:96, 1] = 20_000  # keys 0 .. 95 of the first segment, queries there included
        kw["coords"][500:560, 3] = -30_000
    check_attention(gpu, dt, [400, 300], 2, 2, 32, bias=True, edit=edit)
    check_attention(gpu, dt, [3, 2], 2, 2, 64, kv_lengths=[3000, 900], bias=True, top=5, edit=lambda q, kv, kw: (
        kw["kv_coords"].__setitem__((slice(0, 2900), 2), 9_000), kw["kv_coords"].__setitem__((slice(3000, 3500), 2), 9_000)))


@pytest.mark.parametrize("dt", TYPES)
def test_attention_masked_rows_hold_anything(gpu, dt):
    """Invalid rows' keys and values may be infinite or NaN; a segment whose rows are all invalid gives 0, also for queries
    that are NaN themselves."""
    def edit(q, kv, kw):
        m = torch.ones(kv.shape[0], dtype=torch.bool, device=q.device)
        m[::3] = False
        m[64:100] = False  # the second segment, whole
        kw["kv_mask"] = m
        kv[~m] = float("nan")
        kv[6], kv[9] = float("inf"), -float("inf")
        q[70] = float("nan")
    for kw in (dict(), dict(bias=True), dict(cap=4.0)):
        _, _, _, _, _, got = check_attention(gpu, dt, [64, 36, 50], 2, 1, 32, edit=edit, **kw)
        assert not bool(got[64:100].any())
    got = check_attention(gpu, dt, [1, 1], 2, 1, 32, kv_lengths=[3000, 3000], edit=lambda q, kv, kw: (kv.__setitem__(slice(0, 3000), float("nan")), kw.__setitem__("kv_mask", torch.arange(6000, device=q.device) >= 3000)))[-1]
    assert not bool(got[0].any())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lengths", [[5, 6, 7, 8], [20, 100, 30], [600, 520, 700], [64, 64, 64]])
def test_attention_segments_do_not_touch(gpu, dt, lengths):
    """A frame with NaN and infinite values changes nothing in its neighbours, which share its blocks."""
    clean = check_attention(gpu, dt, lengths, 2, 2, 32, seed=1)[-1]
    off = [0]
    for n in lengths:
        off.append(off[-1] + n)
    def edit(q, kv, kw):
        kv[off[1]:off[2]] = float("nan")
        kv[off[1] + 1, 1] = float("inf")
    got = check_attention(gpu, dt, lengths, 2, 2, 32, seed=1, edit=edit)[-1]
    assert bool(torch.isnan(got[off[1]:off[2]]).all())
    for a, b in zip(off[:1] + off[2:-1], off[1:2] + off[3:]):
        # (the same keys in the same order, but tiles may start at another key: equal within a rounding of either)
        d = (got[a:b].double() - clean[a:b].double()).abs()
        assert bool((d <= 4 * ref.U[dt] * clean[a:b].double().abs() + 2e-3 * (dt != F32) + 1e-6).all())


def test_attention_bad_tables_are_absent_rows(gpu):
    """Offsets behind the rows, falling offsets and indices outside the rows: never read or written."""
    g = gen(4)
    M, H, D = 100, 2, 32
    q, kv = randn(g, M, H, D).to(F16).to(gpu), randn(g, M, 2, H, D).to(F16).to(gpu)
    idx = torch.randperm(M, generator=g).to(torch.int32)
    idx[10], idx[20], idx[60] = -1, M, 2 ** 31 - 1
    off = torch.tensor([0, 40, 1000], dtype=torch.int64)
    for dt in TYPES:
        announce(f"attention bad tables {dt}")
        out = torch.full((M, H, D), 7.0, dtype=dt, device=gpu)
        got = ops.sparse_attention(q.to(dt), kv[:, 0].to(dt), kv[:, 1].to(dt), off.to(gpu), index=idx.to(gpu), out=out)
        want, tol, covered = ref.attention(q.to(dt), kv[:, 0].to(dt), kv[:, 1].to(dt), off, index=idx)
        want[~covered], tol[~covered] = 7.0, 0.0
        ref.assert_within(got, want, tol)
        announce(f"attention falling offsets {dt}")
        got = ops.sparse_attention(q.to(dt), kv[:, 0].to(dt), kv[:, 1].to(dt), torch.tensor([50, 10, -5, 2 ** 62], device=gpu))
        assert bool(torch.isfinite(got).all())
    announce("attention few queries, bad tables")
    big = randn(g, 5000, 2, H, D).to(F16).to(gpu)
    got = ops.sparse_attention(q[:3], big[:, 0], big[:, 1], torch.tensor([0, 1, 3], device=gpu), torch.tensor([-7, 2500, 9999], device=gpu))
    want, tol, _ = ref.attention(q[:3], big[:, 0], big[:, 1], torch.tensor([0, 1, 3]), torch.tensor([0, 2500, 5000]))
    ref.assert_within(got, want, tol)


@pytest.mark.parametrize("few", [False, True])
def test_attention_rows_outside_segments(gpu, few):
    g = gen(6)
    M, H, D = 90, 2, 32
    q = randn(g, M, H, D).to(BF16).to(gpu)
    Mk = 8000 if few else M
    kv = randn(g, Mk, 2, H, D).to(BF16).to(gpu)
    off = torch.tensor([4, 6, 9], dtype=torch.int64) if few else torch.tensor([4, 30, 70], dtype=torch.int64)
    koff = torch.tensor([0, 5000, Mk], dtype=torch.int64) if few else off
    args = (q, kv[:, 0], kv[:, 1], off.to(gpu), koff.to(gpu))
    want, tol, covered = ref.attention(q, kv[:, 0], kv[:, 1], off, koff)
    announce(f"attention rows outside, few={few}")
    got = ops.sparse_attention(*args)
    ref.assert_within(got, want, tol)
    assert not bool(got[~covered].any())
    out = torch.full_like(q, 3.0)
    ops.sparse_attention(*args, out=out)
    assert bool((out[~covered] == 3.0).all()) and torch.equal(out[covered], got[covered])
    # no segment at all, no key at all, no query at all
    assert not bool(ops.sparse_attention(q, q, q, torch.zeros(1, dtype=torch.int64, device=gpu)).any())
    none = ops.sparse_attention(q, kv[:0, 0], kv[:0, 1], off.to(gpu), torch.zeros(3, dtype=torch.int64, device=gpu))
    assert not bool(none.any())
    assert ops.sparse_attention(q[:0], kv[:, 0], kv[:, 1], torch.zeros(3, dtype=torch.int64, device=gpu), koff.to(gpu)).shape == (0, H, D)


def test_attention_index_shorter_than_rows(gpu):
    g = gen(8)
    q, kv = randn(g, 60, 2, 32).to(F16).to(gpu), randn(g, 60, 2, 2, 32).to(F16).to(gpu)
    idx = torch.randperm(60, generator=g)[:25].to(torch.int32).to(gpu)
    off = torch.tensor([0, 10, 25], dtype=torch.int64, device=gpu)
    announce("attention short index")
    got = ops.sparse_attention(q, kv[:, 0], kv[:, 1], off, index=idx)
    want, tol, covered = ref.attention(q, kv[:, 0], kv[:, 1], off, index=idx)
    ref.assert_within(got, want, tol)
    assert not bool(got[~covered].any())


def test_attention_strides_and_far_coordinates(gpu):
    g = gen(12)
    qkv = randn(g, 150, 3, 4, 33).to(F16).to(gpu)  # rows and heads of odd strides: copied
    c = torch.randint(-2 ** 22, 2 ** 22, (150, 4), generator=g, dtype=torch.int32).to(gpu)
    sl = (torch.rand((4, 3), generator=g) * 1e-6).to(gpu)
    off = torch.tensor([0, 70, 150], dtype=torch.int64, device=gpu)
    q, k, v = qkv[:, 0, :, :32], qkv[:, 1, :, :32], qkv[:, 2, :, :32]
    announce("attention strides, far coordinates")
    got = ops.sparse_attention(q, k, v, off, coords=c, slopes=sl)
    want, tol, _ = ref.attention(q, k, v, off, coords=c, slopes=sl)
    ref.assert_within(got, want, tol)
    heads_first = qkv[..., :32].permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)  # (rows, 3, heads, width), head stride largest
    got2 = ops.sparse_attention(heads_first[:, 0], heads_first[:, 1], heads_first[:, 2], off, coords=c, slopes=sl)
    assert torch.equal(got, got2)


def test_attention_offsets_beyond_32_bits(gpu):
    Mk, D = 17_500_000, 128
    announce("attention keys of 2.24e9 elements")
    kv = torch.zeros((2, Mk, 1, D), dtype=F16, device=gpu)
    g = gen(2)
    kv[:, -400:] = randn(g, 2, 400, 1, D).to(F16).to(gpu)
    q = randn(g, 2, 1, D).to(F16).to(gpu)
    off, koff = torch.tensor([0, 1, 2], device=gpu), torch.tensor([0, Mk - 400, Mk], device=gpu)
    got = ops.sparse_attention(q, kv[0], kv[1], off, koff)
    want, tol, _ = ref.attention(q[1:], kv[0, -400:], kv[1, -400:], torch.tensor([0, 1]), torch.tensor([0, 400]))
    ref.assert_within(got[1:], want, tol)
    assert not bool(got[0].any())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lengths,Hq,Hk,D", [([200, 0, 385, 128, 256, 1], 2, 1, 32), ([1000], 1, 1, 64), ([129, 300, 90, 300], 3, 3, 40),
                                             ([2600, 1, 0, 2300], 1, 1, 64), ([500] * 70, 1, 1, 32)])
def test_attention_long_segments_with_rows_around(gpu, dt, lengths, Hq, Hk, D):
    """Segments of many rows, whose tiles start where they start, with rows before, between masked keys and behind."""
    check_attention(gpu, dt, lengths, Hq, Hk, D, start=37, tail=300, mask=0.2, seed=D)
    check_attention(gpu, dt, lengths, Hq, Hk, D, start=128, tail=1, perm=True, bias=True, seed=D + 1)


def test_attention_falling_offsets_of_long_segments(gpu):
    g = gen(8)
    M, H, D = 900, 2, 32
    q, kv = randn(g, M, H, D).to(F16).to(gpu), randn(g, M, 2, H, D).to(F16).to(gpu)
    for off in ([700, 100, 650, 2 ** 62], [900, -1, 2 ** 40, 0], [-(2 ** 62), 2 ** 62, 5, 880]):
        for dt in TYPES:
            announce(f"attention falling offsets {off} {dt}")
            # (offsets have to rise: rows that these miss may be left as they were, but nothing else happens)
            out = torch.full((M + 64, H, D), 7.0, dtype=dt, device=gpu)
            ops.sparse_attention(q.to(dt), kv[:, 0].to(dt), kv[:, 1].to(dt), torch.tensor(off, device=gpu), out=out[32:-32])
            assert bool(torch.isfinite(out).all()) and bool((out[:32] == 7).all()) and bool((out[-32:] == 7).all())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_attention_one_query_not_finite(gpu, dt, value):
    """Every other row of its tile is what it is without it, masked keys or not."""
    g = gen(9)
    M, H, D = 300, 2, 64
    q, kv = randn(g, M, H, D).to(dt).to(gpu), randn(g, M, 2, H, D).to(dt).to(gpu)
    off, mask = torch.tensor([0, 300]), torch.rand(M, generator=g) > 0.3
    want, tol, _ = ref.attention(q, kv[:, 0], kv[:, 1], off, kv_mask=mask)
    bad = q.clone()
    bad[7, :, 3], bad[200, 1] = value, value
    announce(f"attention query {value} {dt}")
    got = ops.sparse_attention(bad, kv[:, 0], kv[:, 1], off.to(gpu), kv_mask=mask.to(gpu))
    rest = torch.ones(M, dtype=torch.bool)
    rest[[7, 200]] = False
    ref.assert_within(got[rest.to(gpu)], want[rest], tol[rest])
    assert bool(torch.isnan(got[7]).any()) and bool(torch.isnan(got[200, 1]).any())


def test_attention_keys_of_almost_4_gib(gpu):
    Mk, D = 16_700_000, 128
    announce("attention keys of 4.28e9 bytes")
    kv = torch.zeros((2, Mk, 1, D), dtype=F16, device=gpu)
    g = gen(2)
    kv[:, -400:] = randn(g, 2, 400, 1, D).to(F16).to(gpu)
    kv[:, -100] = float("nan")
    q = randn(g, 200, 1, D).to(F16).to(gpu)
    mask = torch.ones(Mk, dtype=torch.bool, device=gpu)
    mask[-100] = False
    off, koff = torch.tensor([0, 200], device=gpu), torch.tensor([Mk - 400, Mk], device=gpu)
    got = ops.sparse_attention(q, kv[0], kv[1], off, koff, kv_mask=mask)
    want, tol, _ = ref.attention(q, kv[0, -400:], kv[1, -400:], torch.tensor([0, 200]), torch.tensor([0, 400]), kv_mask=mask[-400:])
    ref.assert_within(got, want, tol)


def test_attention_refusals(gpu):
    q = torch.zeros(8, 4, 16, device=gpu)
    o = torch.tensor([0, 8], device=gpu)
    sl = torch.zeros(4, 3, device=gpu)
    for f, msg in [(lambda: ops.sparse_attention(q, q.half(), q, o), "q's type"), (lambda: ops.sparse_attention(q, q[:, :3], q[:, :3], o), "multiple"),
                   (lambda: ops.sparse_attention(q, q[:5], q[:5], o), "without kv_offsets"), (lambda: ops.sparse_attention(q, q, q, o.int()), "offsets must"),
                   (lambda: ops.sparse_attention(q, q, q, o, o[:1]), "same length"), (lambda: ops.sparse_attention(q, q, q, o, index=o), "index must"),
                   (lambda: ops.sparse_attention(q, q, q, o, slopes=sl), "slopes need"), (lambda: ops.sparse_attention(q, q, q, o, slopes=sl[:2]), "slopes must"),
                   (lambda: ops.sparse_attention(q, q, q, o, kv_mask=o), "kv_mask must"), (lambda: ops.sparse_attention(q, q, q, o, out=q), "overlap"),
                   (lambda: ops.sparse_attention(q, q, q, o, out=q.half()), "out must"), (lambda: ops.sparse_attention(q, q, q, o, kv_index=o.int()), "go with"),
                   (lambda: ops.sparse_attention(q, q[..., :8], q[..., :8], o), "got")]:
        with pytest.raises(ValueError, match=msg):
            f()
    with pytest.raises(_lib.PmgError, match="scale"):
        ops.sparse_attention(q, q, q, o, scale=-1.0)
    with pytest.raises(_lib.PmgError, match="multiple of 8"):
        ops.sparse_attention(q[..., :12], q[..., :12], q[..., :12], o)
    with pytest.raises(RuntimeError, match="inference-only"):
        ops.sparse_attention(q, q, q.clone().requires_grad_(), o)


# ----------------------------------------------------------------------------------------------------------- together
def layer(x, coords, off, idx, p, H, D):
    """One attention layer on the rows of pool cells, as a user writes it: norm, product, norms and rotation, attention,
    product with the residual, then the wide half."""
    h = ops.ln_silu_f16(x, p["g"], p["b"])
    qkv = ops.linear(h, p["wqkv"], p["bqkv"]).view(-1, 3, H, D)
    q, k = ops.qk_norm_rope(qkv[:, 0], qkv[:, 1], coords, p["freqs"], q_weight=p["qw"], k_weight=p["kw"])
    o = ops.sparse_attention(q, k, qkv[:, 2], off, index=idx, coords=coords, slopes=p["slopes"])
    x = ops.linear(o.view(-1, H * D), p["wo"], p["bo"], residual=x, out_dtype=F32)
    h = ops.ln_silu_f16(x, p["g"], p["b"])
    h = ops.linear(h, p["w1"], p["b1"], act="gelu")
    return ops.linear(h, p["w2"], p["b2"], residual=x, out_dtype=F32)


def make_layer(gpu, seed=0, H=4, D=32, hw=(40, 56), cell=8):
    g = gen(seed)
    C = H * D
    rows, cols = hw
    i, j = torch.meshgrid(torch.arange(rows), torch.arange(cols), indexing="ij")
    z = ((i + 2 * j) // 7 + (torch.rand(hw, generator=g) * 3).long()).to(torch.int32)
    coords = torch.stack([torch.zeros_like(z), i.int(), j.int(), z], -1).view(-1, 4).contiguous().to(gpu)
    shape = (1, rows, cols, int(z.max()) + 1)
    _, _, seg, off = ops.pool_cache(coords, shape, (cell,) * 3, (1,) + tuple(-(-s // cell) for s in shape[1:]))
    M = rows * cols
    mat = lambda n, k: (randn(g, n, k) / math.sqrt(k)).to(F16).to(gpu)  # noqa: E731
    vec = lambda n: (0.1 * randn(g, n)).to(gpu)  # noqa: E731
    p = {"g": 1 + vec(C), "b": vec(C), "wqkv": mat(3 * C, C), "bqkv": vec(3 * C), "freqs": freqs_of(g, D // 2).to(gpu), "qw": 1 + vec(D),
         "kw": 1 + vec(D), "slopes": (0.2 * torch.rand((H, 3), generator=g)).to(gpu), "wo": mat(C, C), "bo": vec(C), "w1": mat(2 * C, C),
         "b1": vec(2 * C), "w2": mat(C, 2 * C), "b2": vec(C)}
    x = randn(g, M, C).to(gpu)
    return x, coords, off, seg, p, H, D


def layer64(x, coords, off, idx, p, H, D):
    d = lambda t: t.cpu().double()  # noqa: E731
    def ln(v):
        y = torch.nn.functional.layer_norm(v, (v.shape[-1],), d(p["g"]), d(p["b"]), 1e-6)
        return y * torch.sigmoid(y)
    x = d(x)
    qkv = (ln(x) @ d(p["wqkv"]).t() + d(p["bqkv"])).view(-1, 3, H, D)
    q, _ = ref.norm_rope(qkv[:, 0].float(), p["qw"], None, coords, p["freqs"], layer=False, interleaved=False)
    k, _ = ref.norm_rope(qkv[:, 1].float(), p["kw"], None, coords, p["freqs"], layer=False, interleaved=False)
    o, _, _ = ref.attention(q.float(), k.float(), qkv[:, 2].float(), off, index=idx, coords=coords, slopes=p["slopes"])
    x = x + o.view(-1, H * D) @ d(p["wo"]).t() + d(p["bo"])
    h = ref.act64(ln(x) @ d(p["w1"]).t() + d(p["b1"]), "gelu")
    return x + h @ d(p["w2"]).t() + d(p["b2"])


def test_layer_on_pool_cells(gpu):
    """The operators together on a pool cache's cells. Each of the chain's eleven roundings to fp16 is at most 2^-11 of a value
    of unit size (the norms keep them so), and enters the result through matrices of unit gain: the 2-norm of the
    difference stays below 11 x 2^-11 / sqrt(3) (a uniform rounding's root mean square) of the result's, twice that allowed."""
    a = make_layer(gpu)
    announce("attention layer on pool cells")
    got, want = layer(*a), layer64(*a)
    assert float((got.cpu().double() - want).norm() / want.norm()) < 2 * 11 * 2.0 ** -11 / math.sqrt(3)


def test_layer_captured_and_replayed(gpu):
    """Captured once (allocations included), replayed with changed inputs and eager work between: the eager results, bit for bit."""
    x, coords, off, idx, p, H, D = make_layer(gpu, 1)
    announce("layer in a graph")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        layer(x, coords, off, idx, p, H, D)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(x, coords, off, idx, p, H, D)
    for k in range(4):
        x.copy_(randn(gen(40 + k), *x.shape))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer(x, coords, off, idx, p, H, D)), k


def test_split_attention_captured_twice_and_replayed_at_once(gpu):
    """Two graphs of the split form, replayed on two streams at a time: each has a workspace of its own."""
    g = gen(3)
    H, D, Mk = 4, 64, 40_000
    kv = randn(g, Mk, 2, H, D).to(F16).to(gpu)
    off, koff = torch.tensor([0, 1, 2], device=gpu), torch.tensor([0, 15_000, Mk], device=gpu)
    qs = [randn(g, 2, H, D).to(F16).to(gpu) for _ in range(2)]
    announce("split attention, two graphs")
    eager = [ops.sparse_attention(q, kv[:, 0], kv[:, 1], off, koff) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.sparse_attention(q, kv[:, 0], kv[:, 1], off, koff))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in qs]
    for k in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e), k


def test_same_bits_on_every_call_and_stream(gpu):
    x, coords, off, idx, p, H, D = make_layer(gpu, 2)
    announce("layer on other streams")
    first = layer(x, coords, off, idx, p, H, D)
    torch.cuda.synchronize()
    for _ in range(3):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            y = layer(x, coords, off, idx, p, H, D)
        s.synchronize()
        assert torch.equal(first, y)
