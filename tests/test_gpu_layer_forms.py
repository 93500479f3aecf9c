"""Every kernel of grouped_linear and lora_linear at sizes that take it (layer_forms), against 64 bits on a sample of rows: those around
the segments' borders, and every so many."""
import math

import pytest
import torch

import layer_ref as ref
from conftest import announce
from dense_ref import assert_within
from layer_forms import OF_16_BITS, OF_32_BITS, SEGMENTS, form_of
from promptmoge_amd import _lib, ops
from test_layer_forms import PARTS, low_case

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CASES = [(F16, i) for i in range(len(OF_16_BITS))] + [(BF16, i) for i in range(len(OF_16_BITS))] + [(F32, i) for i in range(len(OF_32_BITS))]
EPILOGUES = [("none", None, None), ("gelu", F32, F32), ("silu", None, "own"), ("gelu_tanh", F32, None), ("relu", None, F32)]  # act, out, residual


def table(gpu, g, M, S):
    """Offsets of S segments of different lengths, one of them empty, with rows in front and behind."""
    cut = torch.sort(torch.randint(1, M - 2, (S + 1,), generator=g)).values
    cut[0], cut[-1] = min(3, M // 8), M - min(5, M // 8)
    cut = torch.cummax(cut.clamp(max=int(cut[-1])), 0).values
    if S > 2:
        cut[2] = cut[1]
    return cut.to(torch.int64).to(gpu)


@pytest.mark.parametrize("dt,i", CASES)
def test_every_kernel(gpu, dt, i):
    bits = 32 if dt == F32 else 16
    (M, K, N, rank, S), form = (OF_32_BITS if bits == 32 else OF_16_BITS)[i]
    assert form_of(_lib.lib(), bits, M, K, N, rank, S) == form
    act, out, res = EPILOGUES[i % len(EPILOGUES)]
    out, res = out or dt, dt if res == "own" else res
    g, d = torch.Generator().manual_seed(i), torch.Generator(device=gpu).manual_seed(i)
    t = lambda *shape, by=1.0: (torch.randn(shape, device=gpu, generator=d) / by).to(dt)  # noqa: E731
    announce(f"{('grouped', 'lora')[rank > 0]} {dt} M={M} K={K} N={N} rank={rank} S={S} form={form} {act} {out} {res}")
    x = t(M, K)
    r = torch.randn((M, N), device=gpu, generator=d).to(res) if res else None
    off = None if S is None else table(gpu, g, M, S)
    ends = torch.tensor([0, M]) if off is None else off.cpu()
    around = torch.cat([torch.arange(int(e) - 66, int(e) + 66) for e in ends[:6]] + [torch.arange(M - 140, M), torch.arange(0, M, 101)])
    rows = around[(around >= 0) & (around < M)].unique()
    segment = torch.full((M,), -1)
    if off is None:
        segment = torch.arange(M)
    else:
        for s in range(S):
            segment[int(ends[s]):int(ends[s + 1])] = s
    of, rows = segment[rows], rows.to(gpu)
    some = r[rows] if r is not None else None
    if not rank:
        w, b = t(S, N, K, by=math.sqrt(K)), torch.randn((S, N), device=gpu, generator=d)
        got = ops.grouped_linear(x, w, off, b, act=act, residual=r, out_dtype=out)
        assert not bool(got[(segment < 0).to(gpu)].any())
        for s in range(S):
            m = of == s
            if bool(m.any()):
                mine = m.to(gpu)
                assert_within(got[rows[mine]], *ref.linear(x[rows[mine]], w[s], b[s], act=act, residual=None if some is None else some[mine], out_dtype=out), f"segment {s}")
        return
    A = 5
    w, b, sc = t(N, K, by=math.sqrt(K)), torch.randn((N,), device=gpu, generator=d), 0.25 + torch.rand((A,), device=gpu, generator=d)
    down, up = t(A, rank, K, by=math.sqrt(K)), t(A, N, rank, by=math.sqrt(rank))
    ids = torch.randint(-1, A, (M if S is None else S,), generator=g, dtype=torch.int32)
    got = ops.lora_linear(x, w, down, up, ids.to(gpu), b, offsets=off, scale=sc, act=act, residual=r, out_dtype=out)
    one = torch.where(of < 0, torch.tensor(-1, dtype=torch.int32), ids[of.clamp(min=0)])
    assert_within(got[rows], *ref.lora_linear(x[rows], w, down, up, one, b, scale=sc, act=act, residual=some, out_dtype=out))


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,rank,S", [(300, 40, 16, 2), (700, 300, 8, 3), (2500, 2350, 24, 3), (300, 33, 5, 2), (50, 40, 16, None), (7, 40, 8, None), (4300, 40, 16, None)])
def test_low_products_are_carried_to_24_bits(gpu, dt, M, N, rank, S):
    """Low products that are whole numbers of up to 23 bits, exact in fp32, beside a projection of 0: each result is one of them times a
    power of two, so that nothing hides what their parts leave out (that fewer parts exceed the bound: test_layer_forms)."""
    K = 128
    (x, down, up, sc, ids, off), _, want, tol = low_case(M, K, N, rank, S, dt)
    form = form_of(_lib.lib(), 32 if dt == F32 else 16, M, K, N, rank, S)
    assert (form[0] == SEGMENTS) == (S is not None and rank % 8 == 0)
    announce(f"lora parts {dt} M={M} N={N} rank={rank} S={S} form={form} parts={PARTS[dt]}")
    got = ops.lora_linear(x.to(gpu), torch.zeros((N, K), dtype=dt, device=gpu), down.to(gpu), up.to(gpu), ids.to(gpu), offsets=None if off is None else off.to(gpu),
                          scale=sc.to(gpu), out_dtype=F32)
    assert_within(got, want, tol)


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("S", [3, None])
def test_an_infinite_low_product_leaves_the_others_finite(gpu, dt, S):
    """An adapter with an infinity: its rows' results are infinite, of the sign that `up` gives that one, for the others (above fp16's
    largest) stay finite beside it."""
    M, K, N, rank, g = 200, 64, 24, 8, torch.Generator().manual_seed(1)
    x, down = torch.randint(1, 9, (M, K), generator=g) * 128.0, torch.randint(1, 9, (2, rank, K), generator=g) * 128.0
    up = torch.where(torch.rand(2, N, rank, generator=g) < 0.5, -2.0, 2.0)
    down[1, 0, 5] = float("inf")
    x, down, up, w = x.to(dt), down.to(dt), up.to(dt), torch.zeros((N, K), dtype=dt)
    off, ids = (None, torch.arange(M, dtype=torch.int32) // 70 % 2) if S is None else (torch.tensor([0, 70, 140, M]), torch.tensor([0, 1, 0], dtype=torch.int32))
    announce(f"lora infinite low product {dt} S={S}")
    got = ops.lora_linear(x.to(gpu), w.to(gpu), down.to(gpu), up.to(gpu), ids.to(gpu), offsets=None if off is None else off.to(gpu), out_dtype=F32)
    want, tol = ref.lora_linear(x, w, down, up, ids, offsets=off, out_dtype=F32)
    assert int(torch.isinf(want).sum()) == 70 * N and not bool(torch.isnan(want).any())
    assert_within(got, want, tol)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("S", [3, None])
def test_low_products_near_the_largest_float(gpu, dt, S):
    """Up to fp32's largest, above bf16's: sums of two exact products, 2^127 (1 + k / 128) + 2^119 l / 16 with k < 128 and l < 16, by up of
    2^-20, so that a result is one of them (bounds: those of the 24-bit test)."""
    M, K, N, rank, g = 200, 64, 24, 8, torch.Generator().manual_seed(2)
    x, down = torch.zeros(M, K), torch.zeros(1, rank, K)
    x[:, 0], x[:, 1] = 2.0 ** 60 * (1 + torch.randint(0, 128, (M,), generator=g) / 128), 2.0 ** 60 * torch.randint(0, 16, (M,), generator=g) / 16
    x[::5, 0], x[::5, 1] = 2.0 ** 60 * (1 + 127 / 128), 2.0 ** 60 * 15 / 16
    down[:, :, 0], down[:, :, 1] = 2.0 ** 67, 2.0 ** 59
    up = torch.zeros(1, N, rank)
    up[:, torch.arange(N), torch.arange(N) % rank] = 2.0 ** -20
    low = x.double() @ down[0].double().t()
    assert float(low.max()) <= torch.finfo(F32).max and float(low.max()) > torch.finfo(BF16).max
    want = low[:, torch.arange(N) % rank] * 2.0 ** -20
    x, down, up, w = x.to(dt), down.to(dt), up.to(dt), torch.zeros((N, K), dtype=dt)
    off, ids = (None, torch.zeros(M, dtype=torch.int32)) if S is None else (torch.tensor([0, 70, 140, M]), torch.zeros(3, dtype=torch.int32))
    announce(f"lora large low products {dt} S={S}")
    got = ops.lora_linear(x.to(gpu), w.to(gpu), down.to(gpu), up.to(gpu), ids.to(gpu), offsets=None if off is None else off.to(gpu), out_dtype=F32)
    assert_within(got, want, (2.0 ** -24 + 3 * 2.0 ** -23) * want.abs())
