"""Refusals of the dense operators' entry points on the host, without a GPU: nothing is launched."""
import ctypes as C

import pytest
import torch

from promptmoge_amd import _lib, ops

D16 = 1 << 12  # an address that is never dereferenced: validation fails first


def linear_args(**kw):
    a = _lib.LinearArgs(_lib.TYPE_F16, D16, 64, D16, 10, 64, 32, 1.0, None, None, 0, None, 0, 0, D16, _lib.TYPE_F16, 32)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def rope_args(**kw):
    a = _lib.RopeArgs(_lib.TYPE_F16, 10, 4, 2, 64, 32, D16, 256, 64, D16, 128, 64, D16, 256, 64, D16, 128, 64, D16, D16,
                      None, None, None, None, 0, 0, 1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attention_args(**kw):
    a = _lib.AttentionArgs(_lib.TYPE_F16, 4, 2, 64, D16, 256, 64, D16, 128, 64, D16, 128, 64, D16, 256, 64, 100, 100, 100,
                           100, 3, D16, D16, None, None, None, None, None, None, 0.125, 0.0, 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(type=4), "type"), (dict(out_type=3), "out_type"), (dict(act=5), "activation"), (dict(M=-1), "M out of range"),
    (dict(M=1 << 31), "M out of range"), (dict(K=0), "K must"), (dict(K=131073, ldx=200000), "K must"), (dict(N=0), "N"),
    (dict(ldx=63), "strides"), (dict(ldo=31), "strides"), (dict(ldx=1 << 22), "strides"), (dict(x=None), "null"),
    (dict(out=None), "null"), (dict(x=D16 + 1), "aligned"), (dict(out=D16 + 1), "aligned"), (dict(bias=D16 + 2), "aligned"),
    (dict(residual=D16, residual_type=3, ldr=32), "residual_type"), (dict(residual=D16, ldr=31), "strides"),
    (dict(residual=D16 + 2, residual_type=0, ldr=32), "aligned"),
])
def test_linear_refusals(libpmg, kw, msg):
    assert libpmg.pmg_linear(C.byref(linear_args(**kw)), None) == _lib.PMG_E_INVALID
    assert msg in libpmg.pmg_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "type"), (dict(M=-1), "M"), (dict(Hq=0), "heads"), (dict(Hk=-1), "heads"), (dict(D=60), "multiple of 8"),
    (dict(D=136), "multiple of 8"), (dict(D=0), "multiple of 8"), (dict(pairs=33), "pairs"), (dict(pairs=-1), "pairs"),
    (dict(eps=-1.0), "eps"), (dict(q=None), "null"), (dict(k_out=None), "null"), (dict(coords=None), "coords"),
    (dict(freqs=None), "coords"), (dict(q=D16 + 4), "groups of 4"), (dict(q_row=258), "groups of 4"),
    (dict(k_out_head=66), "groups of 4"),
])
def test_rope_refusals(libpmg, kw, msg):
    assert libpmg.pmg_qk_norm_rope(C.byref(rope_args(**kw)), None) == _lib.PMG_E_INVALID
    assert msg in libpmg.pmg_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(type=3), "type"), (dict(Hq=3), "heads"), (dict(Hk=0), "heads"), (dict(D=60), "multiple of 8"),
    (dict(D=136), "multiple of 8"), (dict(q_rows=-1), "negative"), (dict(segments=-1), "negative"),
    (dict(k_rows=1 << 31, k_positions=100), "2^31"), (dict(q_positions=101), "more query positions"),
    (dict(k_positions=101), "more key positions"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(cap=-1.0), "cap"), (dict(q=None), "null"), (dict(k=None), "null"),
    (dict(q_offsets=None), "null"), (dict(slopes=D16), "coordinates"), (dict(q=D16 + 8), "16 bytes"),
    (dict(v_row=132), "16 bytes"), (dict(out_row=258), "groups of 4"),
    (dict(slopes=D16, q_coords=D16 + 4, k_coords=D16), "16-byte"),
])
def test_attention_refusals(libpmg, kw, msg):
    assert libpmg.pmg_attention(C.byref(attention_args(**kw)), None, 0, None) == _lib.PMG_E_INVALID
    assert msg in libpmg.pmg_last_error().decode()


def test_attention_workspace_is_asked_for_and_checked(libpmg):
    """Few queries on many keys are split over the keys: the call says how much it needs, and refuses less."""
    a = attention_args(q_rows=8, q_positions=8, segments=8, k_rows=100_000, k_positions=100_000)
    need = libpmg.pmg_attention_workspace_bytes(C.byref(a))
    assert need >= 2 * 8 * 4 * (64 * 4 + 8)
    for ws, n in ((None, need), (D16, need - 1), (D16 + 8, need)):
        assert libpmg.pmg_attention(C.byref(a), ws, n, None) == _lib.PMG_E_INVALID
        assert b"workspace" in libpmg.pmg_last_error()
    assert libpmg.pmg_attention_workspace_bytes(C.byref(attention_args())) == 0
    assert libpmg.pmg_attention_workspace_bytes(C.byref(attention_args(D=60))) == 0
    assert libpmg.pmg_attention_workspace_bytes(None) == 0


@pytest.mark.parametrize("rows,heads,width,segments", [(19_200, 4, 64, 1), (76_800, 8, 64, 1), (300_000, 8, 128, 1), (1_000_000, 32, 128, 3), (5_000, 8, 96, 20)])
def test_attention_workspace_stays_small(libpmg, rows, heads, width, segments):
    a = attention_args(Hq=heads, Hk=heads, D=width, q_rows=rows, q_positions=rows, k_rows=rows, k_positions=rows, segments=segments)
    assert libpmg.pmg_attention_workspace_bytes(C.byref(a)) <= 1 << 28


def test_null_args_and_empty_calls(libpmg):
    for f in (lambda p: libpmg.pmg_linear(p, None), lambda p: libpmg.pmg_qk_norm_rope(p, None),
              lambda p: libpmg.pmg_attention(p, None, 0, None)):
        assert f(None) == _lib.PMG_E_INVALID
    assert libpmg.pmg_linear(C.byref(linear_args(M=0, x=None, out=None)), None) == _lib.PMG_OK
    assert libpmg.pmg_qk_norm_rope(C.byref(rope_args(M=0, q=None, k=None)), None) == _lib.PMG_OK
    assert libpmg.pmg_attention(C.byref(attention_args(q_rows=0, q_positions=0)), None, 0, None) == _lib.PMG_OK


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(16, 8)
    c = torch.zeros(4, 4, dtype=torch.int32)
    h = torch.zeros(4, 2, 8)
    for f in (lambda: ops.linear(x, w), lambda: ops.linear_i8(x.to(torch.int8), w.to(torch.int8)),
              lambda: ops.qk_norm_rope(h, h, c, torch.zeros(4, 3)),
              lambda: ops.sparse_attention(h, h, h, torch.tensor([0, 4]))):
        with pytest.raises(ValueError, match="GPU tensor"):
            f()
