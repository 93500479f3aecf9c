"""Refusals of the conditional layer's entry points on the host, without a GPU: nothing is launched."""
import ctypes as C

import pytest
import torch

from promptmoge_amd import _lib, ops

D16 = 1 << 12  # an address that is never dereferenced: validation fails first
F16, F32 = _lib.TYPE_F16, _lib.TYPE_F32
BIG = (1 << 31) - 512


def norm_args(**kw):
    a = _lib.GroupNormArgs(F16, D16, 64, 5000, 64, 8, None, None, D16, 2, 1e-5, 0, D16, F16, 64, 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def route_args(**kw):
    a = _lib.RouteArgs(F32, D16, 16, 10_000, 16, 2, 0, 0, None, D16, D16, D16, D16, D16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def grouped_args(**kw):
    a = _lib.GroupedLinearArgs(F16, D16, 64, 100, D16, 100, 3, 64, 32, D16, None, None, None, 0, None, 0, 0, D16, F16, 32, 100, 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def combine_args(**kw):
    a = _lib.CombineArgs(F16, D16, 128, 64, 10, 2, 64, D16, None, 0, 0, D16, F16, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def lora_args(**kw):
    a = _lib.LoraLinearArgs(F16, D16, 64, 100, 64, 32, D16, D16, D16, 8, 4, None, D16, D16, 3, None, 0, None, 0, 0, D16, F16, 32)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(libpmg, code, msg):
    assert code == _lib.PMG_E_INVALID
    assert msg in libpmg.pmg_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "type"), (dict(out_type=3), "out_type"), (dict(act=5), "activation"), (dict(M=-1), "M out"), (dict(M=BIG - 1536), "M out"),
    (dict(C=0), "C must"), (dict(C=4104, groups=1, ldx=5000, ldo=5000), "C must"), (dict(groups=0), "C must"), (dict(groups=7), "C must"),
    (dict(ldx=63), "strides"), (dict(ldo=63), "strides"), (dict(segments=-1), "segments"), (dict(offsets=None), "one segment"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(x=None), "null"), (dict(out=None), "null"),
    (dict(x=D16 + 1), "aligned"), (dict(out=D16 + 1), "aligned"), (dict(weight=D16 + 2), "aligned"), (dict(bias=D16 + 2), "aligned"),
    (dict(offsets=D16 + 4), "aligned")])
def test_group_norm_refusals(libpmg, kw, msg):
    refused(libpmg, libpmg.pmg_group_norm(C.byref(norm_args(**kw)), D16, 1 << 30, None), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "type"), (dict(E=0), "E must"), (dict(E=1025, ld=1025), "E must"), (dict(k=0), "k 1"), (dict(k=17), "k 1"), (dict(k=33, E=64, ld=64), "k 1"),
    (dict(M=-1), "E must"), (dict(M=BIG // 2), "M k"), (dict(ld=15), "strides"), (dict(score=2), "score"), (dict(logits=None), "null"), (dict(weights=None), "null"),
    (dict(experts=None), "null"), (dict(offsets=None), "null"), (dict(pairs=None), "null"), (dict(rows=None), "null"), (dict(logits=D16 + 2), "aligned"),
    (dict(offsets=D16 + 4), "aligned"), (dict(rows=D16 + 2), "aligned")])
def test_route_refusals(libpmg, kw, msg):
    refused(libpmg, libpmg.pmg_route(C.byref(route_args(**kw)), D16, 1 << 30, None), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "type"), (dict(out_type=3), "out_type"), (dict(act=5), "activation"), (dict(K=0), "K must"), (dict(K=131073, ldx=200_000), "K must"),
    (dict(N=0), "N 1"), (dict(N=(1 << 22) + 1, ldo=1 << 23), "N 1"), (dict(ldx=63), "strides"), (dict(ldx=1 << 22), "strides"), (dict(ldo=31), "strides"),
    (dict(residual=D16, ldr=31), "strides"), (dict(residual=D16, ldr=32, residual_type=3), "residual_type"), (dict(residual=D16 + 2, ldr=32), "aligned"),
    (dict(positions=-1), "out of range"), (dict(positions=BIG), "out of range"), (dict(x_rows=-1), "out of range"), (dict(out_rows=BIG), "out of range"),
    (dict(segments=-1), "segments"), (dict(segments=1 << 24), "segments"), (dict(positions=101), "more positions"), (dict(out_rows=99), "more positions"),
    (dict(out_index=D16), "zero_rest"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(out=None), "null"), (dict(offsets=None), "null"),
    (dict(x=D16 + 1), "aligned"), (dict(w=D16 + 1), "aligned"), (dict(bias=D16 + 2), "aligned"), (dict(offsets=D16 + 4), "aligned"),
    (dict(index=D16 + 2), "aligned")])
def test_grouped_linear_refusals(libpmg, kw, msg):
    refused(libpmg, libpmg.pmg_grouped_linear(C.byref(grouped_args(**kw)), None), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "type"), (dict(out_type=3), "out_type"), (dict(M=-1), "M,"), (dict(M=1 << 31), "M,"), (dict(k=0), "k ("), (dict(k=33), "k ("), (dict(N=0), "N (1"),
    (dict(N=(1 << 24) + 1, ldo=1 << 25), "N (1"), (dict(y_row=-1), "strides"), (dict(y_slot=-1), "strides"), (dict(ldo=63), "strides"), (dict(residual=D16, ldr=63), "strides"),
    (dict(y=None), "null"), (dict(weights=None), "null"), (dict(out=None), "null"), (dict(y=D16 + 1), "aligned"), (dict(weights=D16 + 2), "aligned"),
    (dict(residual=D16, ldr=64, residual_type=3), "residual_type"), (dict(residual=D16 + 2, ldr=64), "aligned")])
def test_combine_refusals(libpmg, kw, msg):
    refused(libpmg, libpmg.pmg_combine(C.byref(combine_args(**kw)), None), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "type"), (dict(out_type=3), "out_type"), (dict(act=-1), "activation"), (dict(M=-1), "M out"), (dict(M=BIG), "M out"), (dict(K=0), "K must"),
    (dict(N=0), "N 1"), (dict(ldx=63), "strides"), (dict(ldo=31), "strides"), (dict(rank=0), "rank"), (dict(rank=129), "rank"), (dict(adapters=-1), "adapters"),
    (dict(segments=-1), "segments"), (dict(offsets=None), "every row"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(down=None), "null"), (dict(up=None), "null"),
    (dict(adapter=None), "null"), (dict(out=None), "null"), (dict(x=D16 + 1), "aligned"), (dict(up=D16 + 1), "aligned"), (dict(scale=D16 + 2), "aligned"),
    (dict(adapter=D16 + 2), "aligned"), (dict(offsets=D16 + 4), "aligned"), (dict(residual=D16, ldr=31), "strides")])
def test_lora_linear_refusals(libpmg, kw, msg):
    refused(libpmg, libpmg.pmg_lora_linear(C.byref(lora_args(**kw)), D16, 1 << 30, None), msg)


def test_workspaces_are_asked_for_and_checked(libpmg):
    for entry, args, asked in (("pmg_group_norm", norm_args(), True), ("pmg_route", route_args(), True), ("pmg_lora_linear", lora_args(), True),
                               ("pmg_lora_linear", lora_args(segments=1, M=2000), True), ("pmg_group_norm", norm_args(M=100), False), ("pmg_route", route_args(M=10), False)):
        need = getattr(libpmg, entry + "_workspace_bytes")(C.byref(args))
        assert (need > 0) == asked
        if asked:
            for ws, n in ((None, need), (D16, need - 1), (D16 + 2, need)):
                refused(libpmg, getattr(libpmg, entry)(C.byref(args), ws, n, None), "workspace")
    for entry, bad in (("pmg_group_norm", norm_args(groups=7)), ("pmg_route", route_args(k=0)), ("pmg_lora_linear", lora_args(rank=0))):
        assert getattr(libpmg, entry + "_workspace_bytes")(C.byref(bad)) == 0
        assert getattr(libpmg, entry + "_workspace_bytes")(None) == 0


def test_workspaces_that_the_wrappers_do_not_ask_for(libpmg):
    """Short segments' norms and one block's routes need none; other routes 32,768 counts at the most; adapters at most 6 r + 4 bytes
    a row and 512."""
    for S in (1, 3, 1000):
        for M in (1, 512 * S - 1, 512 * S):
            assert libpmg.pmg_group_norm_workspace_bytes(C.byref(norm_args(M=M, segments=S))) == 0
    for E in (1, 2, 16, 300, 1024):
        for k in {1, min(E, 2), min(E, 32)}:
            for M in (0, 1, 63, 64):
                assert libpmg.pmg_route_workspace_bytes(C.byref(route_args(M=M, E=E, ld=E, k=k))) == 0
    for type_ in (0, 1, 2):
        for M, S in ((1, 1), (7, 7), (8, 8), (9, 9), (5000, 2), (1 << 20, 9)):
            for r in (1, 8, 9, 16, 17, 128):
                few = lora_args(type=type_, M=M, segments=M, rank=r, offsets=None)
                assert (libpmg.pmg_lora_linear_workspace_bytes(C.byref(few)) == 0) == (M <= 8 and r <= 16 and M * r <= 64)
                a = lora_args(type=type_, M=M, segments=S, rank=r)
                assert 0 < libpmg.pmg_lora_linear_workspace_bytes(C.byref(a)) <= (6 * r + 4) * M + 512


def test_workspaces_stay_small(libpmg):
    for M, S in ((1 << 20, 1), ((1 << 31) - 2049, 5), (1 << 24, 1 << 12)):
        assert libpmg.pmg_group_norm_workspace_bytes(C.byref(norm_args(M=M, segments=S, C=4096, groups=32, ldx=4096, ldo=4096))) < 1 << 23
    for M, E in ((1 << 20, 1024), (1 << 29, 8)):
        assert libpmg.pmg_route_workspace_bytes(C.byref(route_args(M=M, E=E, ld=E))) <= 1 << 17


def test_null_args_and_empty_calls(libpmg):
    for f in (lambda p: libpmg.pmg_group_norm(p, None, 0, None), lambda p: libpmg.pmg_route(p, None, 0, None), lambda p: libpmg.pmg_grouped_linear(p, None),
              lambda p: libpmg.pmg_combine(p, None), lambda p: libpmg.pmg_lora_linear(p, None, 0, None)):
        assert f(None) == _lib.PMG_E_INVALID
    assert libpmg.pmg_group_norm(C.byref(norm_args(M=0, x=None, out=None)), None, 0, None) == _lib.PMG_OK
    assert libpmg.pmg_grouped_linear(C.byref(grouped_args(positions=0, x=None, out=None)), None) == _lib.PMG_OK
    assert libpmg.pmg_combine(C.byref(combine_args(M=0, y=None, out=None)), None) == _lib.PMG_OK
    assert libpmg.pmg_lora_linear(C.byref(lora_args(M=0, x=None, out=None)), None, 0, None) == _lib.PMG_OK


def test_host_tensors_are_refused():
    x, w, o = torch.zeros(4, 8), torch.zeros(2, 16, 8), torch.tensor([0, 1, 4])
    i = torch.zeros(2, dtype=torch.int32)
    for f in (lambda: ops.group_norm(x, 2), lambda: ops.route(x, 2), lambda: ops.grouped_linear(x, w, o), lambda: ops.combine(w, torch.zeros(2, 16)),
              lambda: ops.lora_linear(x, w[0], torch.zeros(2, 4, 8), torch.zeros(2, 16, 4), i, offsets=o)):
        with pytest.raises(ValueError, match="GPU tensor"):
            f()
