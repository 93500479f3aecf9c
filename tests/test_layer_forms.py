"""Which kernel takes a call of grouped_linear and lora_linear, asked of the library without a GPU."""
import ctypes as C
import re
from pathlib import Path

import pytest

from layer_forms import EXPERTS, FEW, ROWS, SEGMENTS, cases, form_of
from promptmoge_amd import _lib
from test_layer_abi import grouped_args, lora_args, refused

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
