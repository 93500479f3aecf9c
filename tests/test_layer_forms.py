"""Which kernel takes a call of grouped_linear and lora_linear, and what route asks for, asked of the library without a GPU."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from layer_forms import EXPERTS, FEW, ROWS, SEGMENTS, cases, form_of
from promptmoge_amd import _lib
from test_layer_abi import grouped_args, lora_args, refused, route_args

CSRC = Path(__file__).resolve().parents[1] / "promptmoge_amd" / "csrc"


def shapes(bits):
    """The tiles' shapes as the library's table has them: (rows, columns, places)."""
    text = (CSRC / "pmg_grouped.h").read_text()
    table = re.search(rf"kShapes{bits}\[6\]\[3\] = \{{(.*)\}};", text).group(1)
    return [tuple(int(v) for v in row.split(",")) for row in re.findall(r"\{([^{}]*)\}", table)]


@pytest.mark.parametrize("bits", [16, 32])
def test_the_sizes_take_the_kernels_they_stand_for(libpmg, bits):
    for sizes, form in cases(bits):
        assert form_of(libpmg, bits, *sizes) == form, (bits, sizes)


@pytest.mark.parametrize("bits", [16, 32])
def test_every_kernel_has_sizes(bits):
    named = {form for _, form in cases(bits)}
    every = {(kind, *shape, 1) for kind in (EXPERTS, SEGMENTS, ROWS) for shape in shapes(bits)}
    every |= {(kind, 64, 64, 1, 0) for kind in (EXPERTS, ROWS)} | {(FEW, 8, 32, 0, vec) for vec in (0, 1)}
    every |= {(EXPERTS, 16, 32, 0, 1), (EXPERTS, 16, 16, 0, 0), (ROWS, 16, 16, 0, 1), (ROWS, 16, 16, 0, 0)}
    assert len(shapes(bits)) == (6 if bits == 16 else 3) and named == every


def test_forms_of_refused_and_empty_calls(libpmg):
    form = (C.c_int * 5)()
    refused(libpmg, libpmg.pmg_debug_grouped_form(None, form), "null")
    refused(libpmg, libpmg.pmg_debug_grouped_form(C.byref(grouped_args()), None), "null")
    refused(libpmg, libpmg.pmg_debug_grouped_form(C.byref(grouped_args(K=0)), form), "K must")
    refused(libpmg, libpmg.pmg_debug_lora_form(None, form), "null")
    refused(libpmg, libpmg.pmg_debug_lora_form(C.byref(lora_args(rank=0)), form), "rank")
    assert libpmg.pmg_debug_grouped_form(C.byref(grouped_args(positions=0)), form) == _lib.PMG_OK
    assert libpmg.pmg_debug_lora_form(C.byref(lora_args(M=0)), form) == _lib.PMG_OK


PARTS = {torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}  # that a type's low products are carried in


def low_case(M, K, N, rank, S, dt):
    """(x, down, up, scale, adapters, offsets) of a call whose low products are whole numbers below 2^23 (255^2 K), the sums of which no
    order rounds in fp32, times a power of two; each column of `up` has one power of two, so that a result is one of them. Then
    (them, a column's, times what), the result, and its bound: 2^-24 of it for what the parts leave out, 2^-23 for each of their up to three sums."""
    g = torch.Generator().manual_seed(M + rank)
    whole = lambda *shape: torch.randint(0, 256, shape, generator=g).to(dt)  # noqa: E731
    A = 3
    x, down = whole(M, K), whole(A, rank, K)
    up = torch.zeros((A, N, rank))
    column = torch.arange(N) % rank
    up[:, torch.arange(N), column] = 2.0 ** torch.randint(-6, 5, (A, N), generator=g)
    sc = torch.tensor([1.0, 2.0 ** -9, -4.0])
    ids = torch.randint(0, A, (M if S is None else S,), generator=g, dtype=torch.int32)
    off = None if S is None else (torch.arange(S + 1) * M // S).to(torch.int64)
    of = ids.long() if S is None else ids.long().repeat_interleave(off[1:] - off[:-1])
    low = torch.einsum("mk,mrk->mr", x.double(), down.double()[of]) * sc.double()[of][:, None]
    by = up.sum(-1).double()[of]
    want = low[:, column] * by
    return (x, down, up.to(dt), sc, ids, off), (low, column, by), want, (2.0 ** -24 + 3 * 2.0 ** -23) * want.abs()


def in_parts(low, dt, n):
    """Values carried as the sum of n of dt; fp16: scaled by a power of two that brings the row's largest to 2^14 .. 2^15."""
    by = 2.0 ** (14 - torch.floor(torch.log2(low.abs().amax(-1, keepdim=True)))) if dt == torch.float16 else torch.ones(1, dtype=torch.float64)
    rest, total = (low * by).float(), torch.zeros_like(low)
    for _ in range(n):
        part = rest.to(dt)
        total, rest = total + part.double(), rest - part.float()
    return total / by


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,rank,S", [(300, 40, 16, 2), (700, 300, 8, 3)])
def test_fewer_parts_would_be_seen(dt, M, N, rank, S):
    """The bound that the GPU's low products are held to is exceeded in most places by one part less, and kept by all of them."""
    _, (low, column, by), want, tol = low_case(M, 128, N, rank, S, dt)
    far = lambda n: ((in_parts(low, dt, n)[:, column] * by - want).abs() > tol).double().mean()  # noqa: E731
    assert float(far(PARTS[dt])) == 0.0 and float(far(PARTS[dt] - 1)) > 0.5


def test_routes_need_a_count_of_each_expert_for_16_rows_at_the_most(libpmg):
    """What the wrapper gives them beside its tables."""
    for E in (1, 2, 3, 8, 16, 63, 64, 65, 100, 128, 129, 256, 300, 512, 513, 1000, 1024):
        for k in {1, min(E, 2), min(E, 5), min(E, 9), min(E, 17), min(E, 32)}:
            for M in (*range(65, 400), 500, 1000, 1023, 1025, 4095, 4097, 8191, 8193, 20_000, 76_800, 1_000_000):
                need = libpmg.pmg_route_workspace_bytes(C.byref(route_args(M=M, E=E, ld=E, k=k)))
                assert need <= 4 * min((M + 15) // 16 * (E + 1), 32_768), (M, E, k)
