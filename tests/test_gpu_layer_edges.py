"""The conditional layer's operators where rows lie unevenly: most of them in one segment or in none, and tables that fall."""
import pytest
import torch

import layer_ref as ref
from conftest import announce
from dense_ref import assert_within
from promptmoge_amd import _lib, ops
from test_gpu_layer import check_norm, cuts, gen, randn

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def microseconds(f, n=10, rounds=5):
    """Of one of n calls one behind the other, the least of a few rounds."""
    f()
    best = float("inf")
    for _ in range(rounds):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1000 / n)
    return best


# ---------------------------------------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("dt,out", [(F16, F16), (F32, BF16)])
@pytest.mark.parametrize("sizes,start,behind,C,groups", [
    ((1,) * 40, 0, 9000, 64, 16), ((1,) * 40, 7000, 0, 24, 8), ((3, 0, 2) * 20, 3000, 6001, 130, 13), ((200, 300, 100), 500, 400, 256, 32), ((0,) * 30, 0, 15_000, 33, 11),
    ((0, 0), 300, 701, 4096, 2), ((), 0, 500, 64, 8), ((1,) * 1500, 999, 100_001, 7, 7),
    ((1, 0) * 1300, 700, 9001, 24, 4)])
def test_norm_most_rows_in_no_segment(gpu, dt, out, sizes, start, behind, C, groups):
    """Rows in front and behind, many times the segments' own, in a new result, and left alone in a given one."""
    check_norm(gpu, sizes, C, groups, dt, out_dtype=out, act="silu", start=start, behind=behind)
    M = start + sum(sizes) + behind
    x, off = randn(gen(2), M, C).to(dt).to(gpu), cuts(gpu, *sizes, start=start)
    given = torch.full((M, C), 7.0, dtype=out, device=gpu)
    ops.group_norm(x, groups, offsets=off, out=given)
    assert bool((given[:start] == 7).all()) and bool((given[start + sum(sizes):] == 7).all())


@pytest.mark.parametrize("S,n,rows,C", [(1000, 20, 40_000, 256), (1000, 1, 501_000, 64)])
def test_norm_rows_of_no_segment_are_everybodys(gpu, S, n, rows, C):
    """A buffer of fixed size whose segments fill a part of it takes no longer than with segments that fill it (one block going
    over the rest alone: 12 and more times as long)."""
    x = randn(gen(1), rows, C).to(F16).to(gpu)
    some, all_ = cuts(gpu, *(n,) * S), cuts(gpu, *(rows // S,) * S)
    announce(f"group_norm {S} segments of {n} in {rows} rows, timed")
    few, full = microseconds(lambda: ops.group_norm(x, 16, offsets=some)), microseconds(lambda: ops.group_norm(x, 16, offsets=all_))
    assert few < 3 * full, f"{few:.0f} us, {full:.0f} with all rows in segments"


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("short,n,long_,C,groups", [(300, 1, 60_000, 64, 16), (3000, 1, 20_000, 64, 16), (200, 3, 30_001, 40, 5), (40, 300, 9001, 256, 32), (1200, 2, 9000, 130, 13)])
def test_norm_one_long_segment_among_short_ones(gpu, dt, short, n, long_, C, groups):
    """In the form of one launch, which goes by the mean length: first, last and in the middle, by a block and by a wave."""
    for at in (0, short // 2, short):
        check_norm(gpu, (n,) * at + (long_,) + (n,) * (short - at), C, groups, dt, act="silu", mean=3.0, seed=at)


@pytest.mark.parametrize("dt,out", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("sizes", [(30,), (300, 20), (1,) * 70 + (40,), (2000,), (9000, 7000)])
def test_norm_spreads_at_the_ends_of_the_range(gpu, dt, out, sizes):
    """Values up to the type's largest, of either sign, whose differences overflow fp32, and down to its least without eps, whose
    spread's reciprocal does; groups in the middle of the range beside them."""
    M, C, G, g = sum(sizes), 64, 8, gen(len(sizes))
    largest = torch.finfo(dt).max
    big = torch.where(torch.rand(M, C, generator=g) < 0.3, -largest, largest) * (1 - torch.rand(M, C, generator=g) / 64)
    for by, eps in (({0: big, 3: big}, 1e-5), ({1: randn(g, M, C) * 1e-38, 7: randn(g, M, C) * 1e-36}, 0.0), ({2: big, 5: randn(g, M, C) * 1e-37}, 0.0)):
        x = randn(g, M, C)
        for group, v in by.items():
            x[:, 8 * group:8 * group + 8] = v[:, 8 * group:8 * group + 8]
        check_norm(gpu, sizes, C, G, dt, out_dtype=out, act="silu", x=x.to(dt).to(gpu), eps=eps)


# ------------------------------------------------------------------------------------------------------ falling offsets
def falling(S, M, seed):
    """A table that rises and falls, with bounds far outside the rows."""
    o = torch.randint(0, M + 1, (S + 1,), generator=gen(seed), dtype=torch.int64)
    o[seed % (S + 1)], o[(seed + 2) % (S + 1)] = 2 ** 62, -2 ** 62
    return o


def framed(gpu, M, C_, dt=F16):
    """(a buffer of sevens, the M rows inside it that a call writes)."""
    buf = torch.full((M + 64, C_ + 32), 7.0, dtype=dt, device=gpu)
    return buf, buf[32:32 + M, 16:16 + C_]


def untouched(buf, inside):
    inside.fill_(7.0)
    assert bool((buf == 7.0).all())


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("S,M", [(2, 30_000), (4, 60_001), (3, 8000)])
def test_falling_offsets_of_two_launches_stay_inside(gpu, S, M, seed):
    """The norm whose workspace is addressed from the bounds: what the rows get is not said, but nothing else is written, here nor
    in memory behind the workspace."""
    x, off = randn(gen(seed), M, 64).to(F16).to(gpu), falling(S, M, seed).to(gpu)
    for out in (None, framed(gpu, M, 64)):
        to = torch.full((M, 64), 7.0, dtype=F16, device=gpu) if out is None else out[1]
        args = _lib.GROUP_NORM_PACK.pack(_lib.TYPE_F16, x.data_ptr(), 64, M, 64, 16, 0, 0, off.data_ptr(), S, 1e-5, 0, to.data_ptr(), _lib.TYPE_F16, to.stride(0), out is None)
        need = _lib.lib().pmg_group_norm_workspace_bytes(args)
        assert need > 0
        ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device=gpu)
        announce(f"group_norm falling S={S} M={M} seed={seed}")
        assert _lib.lib().pmg_group_norm(args, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
        assert bool((ws[need:] == 77).all())
        if out is not None:
            untouched(*out)


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("S", [40, 63, 130, 254, 255, 300])
def test_falling_offsets_of_many_segments_stay_inside(gpu, S, seed):
    """By one and by four segments a lane, and by the search of more."""
    M, g = 9000, gen(seed)
    off, x = falling(S, M, seed).to(gpu), randn(g, M, 64).to(F16).to(gpu)
    w, down, up = randn(g, S, 64, 64).to(F16).to(gpu), randn(g, 2, 8, 64).to(F16).to(gpu), randn(g, 2, 64, 8).to(F16).to(gpu)
    ids = torch.randint(-1, 2, (S,), generator=g, dtype=torch.int32).to(gpu)
    index = torch.randint(0, M, (M,), generator=g, dtype=torch.int32).to(gpu)
    calls = [lambda o: ops.group_norm(x, 8, offsets=off, out=o), lambda o: ops.grouped_linear(x, w, off, out=o), lambda o: ops.grouped_linear(x, w, off, index=index, out=o),
             lambda o: ops.lora_linear(x, w[0], down, up, ids, offsets=off, out=o)]
    for i, f in enumerate(calls):
        announce(f"falling offsets S={S} seed={seed} call {i}")
        buf, inside = framed(gpu, M, 64)
        f(inside)
        untouched(buf, inside)
        assert f(None).shape == (M, 64)


# --------------------------------------------------------------------------------------------------------------- route
@pytest.mark.parametrize("M,E,k", [(1, 16, 2), (64, 1024, 32), (65, 16, 2), (100, 8, 2), (300, 64, 4), (5000, 16, 2), (5000, 1024, 1)])
def test_route_keeps_little_beside_its_tables(gpu, M, E, k):
    r = ops.route(randn(gen(1), M, E).to(gpu), k)
    kept = sum({t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in r}.values())
    assert kept <= sum(t.nbytes for t in r) + 4 * min((M + 15) // 16 * (E + 1), 32_768)
