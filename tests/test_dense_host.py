"""What the dense operators' Python entries decide on the host before anything is launched. The tensors here say that they
are on a GPU and are not; nothing may reach a kernel."""
import ctypes as C
import inspect

import pytest
import torch

from promptmoge_amd import _lib, ops
from test_dense_abi import D16, attention_args, linear_args

F16, F32 = torch.float16, torch.float32


class OnGpu(torch.Tensor):
    """A host tensor that says it is on GPU 0."""
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda:0"))

    def get_device(self):
        return 0


def on_gpu(t):
    return t.as_subclass(OnGpu)


class Reached(Exception):
    """The call would have been launched."""


@pytest.fixture
def no_launch(monkeypatch):
    def stop(d, name, *args):
        raise Reached(name)
    monkeypatch.setattr(ops, "_on", stop)
    monkeypatch.setattr(ops, "_entry", lambda name: lambda args: 0)


def zeros(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


def calls():
    """(entry, every tensor argument by name, the others)."""
    i32 = torch.int32
    yield "linear", dict(x=zeros(4, 16), w=zeros(8, 16), bias=zeros(8, dtype=F32), residual=zeros(4, 8), out=zeros(4, 8)), {}
    yield "linear_i8", dict(x=zeros(4, 16, dtype=torch.int8), w=zeros(8, 16, dtype=torch.int8), bias=zeros(8, dtype=F32),
                            w_scale=zeros(8, dtype=F32), residual=zeros(4, 8), out=zeros(4, 8, dtype=F32)), {}
    vec = {n: zeros(16, dtype=F32) for n in ("q_weight", "k_weight", "q_bias", "k_bias")}
    yield "qk_norm_rope", dict(q=zeros(4, 2, 16), k=zeros(4, 1, 16), coords=zeros(4, 4, dtype=i32), freqs=zeros(8, 3, dtype=F32),
                               out=(zeros(4, 2, 16), zeros(4, 1, 16)), **vec), {}
    off = torch.tensor([0, 4])
    yield "sparse_attention", dict(
        q=zeros(4, 2, 16), k=zeros(6, 1, 16), v=zeros(6, 1, 16), offsets=off, kv_offsets=torch.tensor([0, 6]),
        index=torch.arange(4, dtype=i32), kv_index=torch.arange(6, dtype=i32), coords=zeros(4, 4, dtype=i32),
        kv_coords=zeros(6, 4, dtype=i32), slopes=zeros(2, 3, dtype=F32), kv_mask=zeros(6, dtype=torch.bool), out=zeros(4, 2, 16)), {}


def everywhere(v):
    return tuple(on_gpu(t) for t in v) if isinstance(v, tuple) else on_gpu(v)


PLACES = [(name, place, part) for name, args, _ in calls() for place, v in args.items() for part in (range(len(v)) if isinstance(v, tuple) else [None])]


@pytest.mark.parametrize("name,place,part", PLACES)
def test_one_host_tensor_is_refused_in_every_place(no_launch, name, place, part):
    args, kw = next((a, k) for n, a, k in calls() if n == name)
    every = {n: everywhere(v) for n, v in args.items()}
    with pytest.raises(Reached):
        getattr(ops, name)(**every, **kw)
    one = dict(every)
    one[place] = args[place] if part is None else tuple(args[place][i] if i == part else t for i, t in enumerate(every[place]))
    with pytest.raises(ValueError, match="GPU tensor"):
        getattr(ops, name)(**one, **kw)
    several = {n: v if n == place else args[n] for n, v in every.items()}  # only that one on the GPU
    with pytest.raises(ValueError, match="GPU tensor"):
        getattr(ops, name)(**several, **kw)


def test_the_places_are_all_there_are():
    for name, args, kw in calls():
        named = set(inspect.signature(getattr(ops, name)).parameters)
        rest = {"act", "out_dtype", "a_scale", "norm", "eps", "interleaved", "cap", "scale", "precise"}
        assert named - rest == set(args)


@pytest.mark.parametrize("make", [
    lambda b: b[1:97].view(3, 2, 16),                                       # contiguous, but at an odd element
    lambda b: b[:96].view(3, 2, 16)[:, :1].as_strided((3, 1, 16), (32, 17, 1)),  # one head, whose stride means nothing
    lambda b: b[4:52].view(1, 3, 16).as_strided((1, 3, 16), (51, 16, 1)),    # one row
    lambda b: b[:102].view(3, 34)[:, 1:33].unflatten(1, (2, 16)),            # odd columns
    lambda b: b[:96].view(3, 16, 2).transpose(1, 2),                         # heads not contiguous
])
def test_heads_off_their_units_are_copied(make):
    t = make(torch.arange(128, dtype=torch.float32).to(F16))
    for unit in (8, 16):
        c = ops._heads(t, "q", unit)
        assert torch.equal(c, t) and c.data_ptr() % unit == 0 and c.stride(2) == 1
        assert c.stride(0) * 2 % unit == 0 and c.stride(1) * 2 % unit == 0
    straight = torch.zeros(3, 2, 16, dtype=F16)
    assert ops._heads(straight, "q", 16) is straight


def test_an_out_off_its_units_is_refused(no_launch):
    for shape in ((5, 2, 16), (5, 1, 16)):
        n = shape[0] * shape[1] * 16
        x = on_gpu(zeros(*shape))
        c, f = on_gpu(zeros(5, 4, dtype=torch.int32)), on_gpu(zeros(8, 3, dtype=F32))
        odd = on_gpu(zeros(n + 8)[1:n + 1].view(shape))
        with pytest.raises(ValueError, match="groups of 4"):
            ops.qk_norm_rope(x, None, c, f, out=(odd, None))
        with pytest.raises(ValueError, match="groups of 4"):
            ops.sparse_attention(x, x, x, on_gpu(torch.tensor([0, 5])), out=odd)


def test_overlap_of_strided_tensors_is_that_of_their_elements():
    """Against the sets of bytes themselves, over slices of one buffer; a doubtful pair may count as overlapping only where rows
    of different strides (or more than one axis that leaves gaps) are laced into each other."""
    buf = torch.zeros(4, 6, 10)
    views = [buf[:, a:b] for a, b in ((0, 2), (2, 4), (1, 3), (5, 6))] + [buf[:, :, 2:4], buf[:, :, 4:8], buf[1:2], buf[:0], buf[2:, 1:3],
             buf.view(24, 10)[:, :5], buf.view(24, 10)[:, 5:], buf.view(24, 10)[3:9, 4:6], buf.view(-1)[7:30],
             buf.permute(1, 0, 2)[:3], buf.permute(1, 0, 2)[3:], buf.view(4, 60)[:, 12:40], buf.view(4, 60)[:, 40:], buf.view(4, 60)[:1, :40]]
    sets = [{v.data_ptr() + 4 * sum(i * s for i, s in zip(at, v.stride())) for at in torch.cartesian_prod(*[torch.arange(n) for n in v.shape]).view(-1, v.ndim).tolist()}
            if v.numel() else set() for v in views]
    for a, sa in zip(views, sets):
        for b, sb in zip(views, sets):
            truth = bool(sa & sb)
            assert ops._overlap(a, b) or not truth
            wide = [max((s for n, s in zip(v.shape, v.stride()) if n > 1), default=0) for v in (a, b)]
            if not truth and a.ndim == 2 and b.ndim == 2 and wide[0] == wide[1]:
                assert not ops._overlap(a, b), (a.shape, a.stride(), b.shape, b.stride())


def test_disjoint_columns_of_one_buffer_are_taken(no_launch):
    buf = on_gpu(zeros(5, 64))
    w = on_gpu(zeros(32, 32))
    with pytest.raises(Reached):
        ops.linear(buf[:, :32], w, out=buf[:, 32:])
    with pytest.raises(Reached):
        ops.linear(buf[:, :32], on_gpu(zeros(16, 32)), residual=buf[:, 32:48], out=buf[:, 48:])
    for a, b in ((0, 31), (1, 0), (8, 24)):
        with pytest.raises(ValueError, match="overlap"):
            ops.linear(buf[:, a:a + 32], w, out=buf[:, b:b + 32])
    qk = on_gpu(zeros(5, 6, 16))
    c, f = on_gpu(zeros(5, 4, dtype=torch.int32)), on_gpu(zeros(8, 3, dtype=F32))
    with pytest.raises(Reached):  # q and k side by side, in and out
        ops.qk_norm_rope(qk[:, :2], qk[:, 2:3], c, f, out=(qk[:, 3:5], qk[:, 5:]))
    with pytest.raises(Reached):  # the same in place
        ops.qk_norm_rope(qk[:, :2], qk[:, 2:3], c, f, out=(qk[:, :2], qk[:, 2:3]))
    hq = on_gpu(zeros(3, 5, 16)).permute(1, 0, 2)  # heads first
    with pytest.raises(Reached):
        ops.qk_norm_rope(hq[:, :2], hq[:, 2:], c, f, out=(hq[:, :2], hq[:, 2:]))
    with pytest.raises(Reached):
        ops.sparse_attention(qk[:, :2], qk[:, 2:4], qk[:, 2:4], on_gpu(torch.tensor([0, 5])), out=qk[:, 4:])
    with pytest.raises(ValueError, match="overlap"):
        ops.sparse_attention(qk[:, :2], qk[:, 2:4], qk[:, 2:4], on_gpu(torch.tensor([0, 5])), out=qk[:, 3:5])
    with pytest.raises(ValueError, match="overlap"):  # k would be read while q, the same rows, is written
        ops.qk_norm_rope(qk[:, :2], qk[:, :2], c, f, out=(qk[:, :2], on_gpu(zeros(5, 2, 16))))
    with pytest.raises(ValueError, match="overlap"):
        ops.qk_norm_rope(qk[:, :2], qk[:, 2:4], c, f, out=(qk[:, 2:4], qk[:, :2]))
    with pytest.raises(ValueError, match="must not overlap"):
        ops.qk_norm_rope(qk[:, :2], qk[:, 2:4], c, f, out=(on_gpu(zeros(5, 2, 16)),) * 2)


@pytest.mark.parametrize("name,place", [
    ("linear", "bias"), ("linear_i8", "bias"), ("linear_i8", "w_scale"), ("qk_norm_rope", "coords"), ("qk_norm_rope", "freqs"),
    ("qk_norm_rope", "q_weight"), ("qk_norm_rope", "k_weight"), ("qk_norm_rope", "q_bias"), ("qk_norm_rope", "k_bias"),
    ("sparse_attention", "offsets"), ("sparse_attention", "kv_offsets"), ("sparse_attention", "index"), ("sparse_attention", "kv_index"),
    ("sparse_attention", "coords"), ("sparse_attention", "kv_coords"), ("sparse_attention", "slopes"), ("sparse_attention", "kv_mask")])
def test_an_out_on_another_argument_is_refused(no_launch, name, place):
    """A block would write what another one still reads."""
    args = next(a for n, a, _ in calls() if n == name)
    args = {n: everywhere(v) for n, v in args.items()}
    bytes_ = torch.zeros(4096, dtype=torch.uint8)
    t = args[place]
    args[place] = on_gpu(bytes_[:t.numel() * t.element_size()].view(t.dtype).view(t.shape))
    lay = lambda o: on_gpu(bytes_[:o.numel() * o.element_size()].view(o.dtype).view(o.shape))  # noqa: E731
    for which in range(len(args["out"])) if isinstance(args["out"], tuple) else [None]:
        out = args["out"]
        out = lay(out) if which is None else tuple(lay(o) if i == which else o for i, o in enumerate(out))
        with pytest.raises(ValueError, match="overlap"):
            getattr(ops, name)(**{**args, "out": out})


def test_an_out_whose_own_rows_overlap_is_refused(no_launch):
    """Different results would be written to one place."""
    x, off = on_gpu(zeros(6, 2, 16)), on_gpu(torch.tensor([0, 6]))
    c, f = on_gpu(zeros(6, 4, dtype=torch.int32)), on_gpu(zeros(8, 3, dtype=F32))
    big = zeros(512)
    for strides in ((0, 16, 1), (16, 16, 1), (32, 0, 1), (24, 12, 1), (8, 96, 1), (16, 80, 1)):
        out = on_gpu(big.as_strided((6, 2, 16), strides))
        with pytest.raises(ValueError, match="overlap"):
            ops.sparse_attention(x, x, x, off, out=out)
        with pytest.raises(ValueError, match="overlap"):
            ops.qk_norm_rope(x, None, c, f, out=(out, None))
        with pytest.raises(ValueError, match="overlap"):
            ops.qk_norm_rope(x, x, c, f, out=(on_gpu(zeros(6, 2, 16)), out))
    for strides in ((32, 16, 1), (48, 20, 1), (16, 96, 1), (20, 120, 1)):
        out = on_gpu(big.as_strided((6, 2, 16), strides))
        with pytest.raises(Reached):
            ops.sparse_attention(x, x, x, off, out=out)
        with pytest.raises(Reached):
            ops.qk_norm_rope(x, None, c, f, out=(out, None))
    one = on_gpu(big.as_strided((1, 2, 16), (0, 16, 1)))
    with pytest.raises(Reached):
        ops.sparse_attention(x[:1], x[:1], x[:1], off, out=one)


def test_out_dtype_has_to_be_that_of_out(no_launch):
    x, w, q, u = on_gpu(zeros(4, 16)), on_gpu(zeros(8, 16)), on_gpu(zeros(4, 16, dtype=torch.int8)), on_gpu(zeros(8, 16, dtype=torch.int8))
    for out in (F16, F32, torch.bfloat16):
        o = on_gpu(zeros(4, 8, dtype=out))
        for want in (F16, F32, torch.bfloat16):
            for f in (lambda: ops.linear(x, w, out_dtype=want, out=o), lambda: ops.linear_i8(q, u, out_dtype=want, out=o)):
                with pytest.raises(Reached if want == out else ValueError, match=None if want == out else "out_dtype"):
                    f()
        for f in (lambda: ops.linear(x, w, out=o), lambda: ops.linear_i8(q, u, out=o)):  # out says it
            with pytest.raises(Reached):
                f()


@pytest.mark.parametrize("name,place", [(n, p) for n, args, _ in calls() for p, v in args.items() if p != "out" and v.is_floating_point()])
def test_forward_mode_tangents_are_refused(no_launch, name, place):
    """They would be lost in silence. Without a tangent, or outside its level, the call is made."""
    args = next(a for n, a, _ in calls() if n == name)
    every = {n: everywhere(v) for n, v in args.items()}
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(Reached):
            getattr(ops, name)(**every)
        dual = torch.autograd.forward_ad.make_dual(args[place], torch.ones_like(args[place]))
        with pytest.raises(RuntimeError, match="inference-only"):
            getattr(ops, name)(**{**every, place: on_gpu(dual)})
        with pytest.raises(ValueError, match="GPU tensor"):  # on the host as well
            getattr(ops, name)(**{**every, "out": args["out"]})
    with pytest.raises(Reached):
        getattr(ops, name)(**every)


def test_int8_sums_that_could_pass_32_bits_are_refused(libpmg):
    """131,072 products of -128 by -128 are 2^31; one fewer fit."""
    i8 = dict(type=_lib.TYPE_I8, ldx=1 << 18)
    assert (-128) ** 2 * 131_072 > 2 ** 31 - 1 >= (-128) ** 2 * 131_071
    assert libpmg.pmg_linear(C.byref(linear_args(K=131_072, **i8)), None) == _lib.PMG_E_INVALID
    assert b"K must" in libpmg.pmg_last_error()
    assert libpmg.pmg_linear(C.byref(linear_args(K=131_071, M=0, **i8)), None) == _lib.PMG_OK
    assert libpmg.pmg_linear(C.byref(linear_args(K=131_072, M=0, ldx=1 << 18)), None) == _lib.PMG_OK


@pytest.mark.parametrize("kw,msg", [(dict(scale=2e30), "scale"), (dict(cap=2e30), "cap"), (dict(cap=float("nan")), "cap"), (dict(cap=float("inf")), "cap"),
                                    (dict(cap=1e-38), "too small"), (dict(cap=1e-8, scale=1e30), "too small")])
def test_attention_scales_and_caps_out_of_range_are_refused(libpmg, kw, msg):
    """Products of them with log2 e, and their quotient, have to be numbers of fp32."""
    assert libpmg.pmg_attention(C.byref(attention_args(**kw)), None, 0, None) == _lib.PMG_E_INVALID
    assert msg in libpmg.pmg_last_error().decode()


@pytest.mark.parametrize("kw", [dict(q_rows=1 << 30, q_positions=1 << 30, segments=1), dict(q_rows=1 << 27, q_positions=1 << 27, segments=1 << 26, k_rows=(1 << 31) - 65, k_positions=(1 << 31) - 65)])
def test_attention_of_more_blocks_than_a_grid_holds_is_refused(libpmg, kw):
    """(before a launch fails) A grid holds fewer than 2^32 threads."""
    a = attention_args(Hq=32, Hk=32, D=8, k_row=256, v_row=256, **{k: v for k, v in kw.items() if not k.startswith("k_")})
    a.k_rows, a.k_positions = kw.get("k_rows", 1 << 30), kw.get("k_positions", 1 << 30)
    need = libpmg.pmg_attention_workspace_bytes(C.byref(a))
    assert libpmg.pmg_attention(C.byref(a), D16, need, None) == _lib.PMG_E_INVALID
    assert b"too many" in libpmg.pmg_last_error()


def test_attention_positions_close_to_32_bits_are_refused(libpmg):
    """A tile of 64 keys behind the last whole one would count past 2^31."""
    for name in ("q", "k"):
        for n in ((1 << 31) - 1, (1 << 31) - 63):
            a = attention_args(**{f"{name}_rows": n, f"{name}_positions": n})
            assert libpmg.pmg_attention(C.byref(a), None, 0, None) == _lib.PMG_E_INVALID
            assert b"2^31" in libpmg.pmg_last_error()


def test_attention_of_equal_frames_is_not_planned_as_ragged_cells(libpmg):
    """Twelve frames of 800 rows fill the CUs evenly: split, they take a third longer. Ragged cells have an index."""
    rows = dict(type=_lib.TYPE_BF16, Hk=4, D=128, q_rows=9600, q_positions=9600, k_rows=9600, k_positions=9600, segments=12)
    assert libpmg.pmg_attention_workspace_bytes(C.byref(attention_args(**rows))) == 0
    assert libpmg.pmg_attention_workspace_bytes(C.byref(attention_args(q_index=D16, k_index=D16, **rows))) > 0


def test_heads_of_no_width_are_refused_as_other_widths(no_launch, monkeypatch):
    """(by the entry itself: D^-1/2 is not formed)"""
    q, off = on_gpu(zeros(4, 2, 0)), on_gpu(torch.tensor([0, 4]))
    with pytest.raises(Reached):
        ops.sparse_attention(q, q, q, off)
    with pytest.raises(Reached):
        ops.sparse_attention(q, q, q, off, scale=1.0)


@pytest.mark.parametrize("bad", [None, 1.0, [1.0]])
def test_what_is_no_tensor_is_refused_by_name(no_launch, bad):
    every = {n: {m: everywhere(v) for m, v in args.items()} for n, args, _ in calls()}
    for name, first in (("linear", "x"), ("linear_i8", "x"), ("qk_norm_rope", "q"), ("sparse_attention", "q")):
        for place in (first, "out") if bad is not None else (first,):
            wrong = (bad, bad) if (name, place) == ("qk_norm_rope", "out") else bad
            with pytest.raises(ValueError, match="GPU tensor"):
                getattr(ops, name)(**{**every[name], place: wrong})
