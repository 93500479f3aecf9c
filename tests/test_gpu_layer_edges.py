"""The conditional layer's operators where rows lie unevenly: most of them in one segment or in none, and tables that fall."""
import pytest
import torch

import layer_ref as ref
from conftest import announce
from dense_ref import assert_within
from promptmoge_amd import ops
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
