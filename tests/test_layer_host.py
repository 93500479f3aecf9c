"""What the conditional layer's Python entries decide on the host before anything is launched. The tensors here say that they are
on a GPU and are not; nothing may reach a kernel."""
import inspect

import pytest
import torch

from promptmoge_amd import ops
from test_dense_host import Reached, everywhere, no_launch, on_gpu, zeros  # noqa: F401

F16, F32, I32 = torch.float16, torch.float32, torch.int32


def calls():
    """(entry, every tensor argument by name, the others)."""
    off = torch.tensor([0, 3, 4])
    yield "group_norm", dict(x=zeros(4, 16), weight=zeros(16, dtype=F32), bias=zeros(16, dtype=F32), offsets=off, out=zeros(4, 16)), dict(groups=4)
    yield "route", dict(logits=zeros(4, 8), mask=zeros(4, dtype=torch.bool)), dict(k=2)
    yield "grouped_linear", dict(x=zeros(5, 16), w=zeros(2, 8, 16), offsets=off, bias=zeros(2, 8, dtype=F32), index=zeros(4, dtype=I32), out_index=zeros(4, dtype=I32),
                                 residual=zeros(6, 8), out=zeros(6, 8)), {}
    yield "combine", dict(y=zeros(4, 2, 16), weights=zeros(4, 2, dtype=F32), residual=zeros(4, 16), out=zeros(4, 16)), {}
    yield "lora_linear", dict(x=zeros(4, 16), w=zeros(8, 16), down=zeros(3, 4, 16), up=zeros(3, 8, 4), adapter=zeros(2, dtype=I32), bias=zeros(8, dtype=F32),
                              offsets=off, scale=zeros(3, dtype=F32), residual=zeros(4, 8), out=zeros(4, 8)), {}


PLACES = [(name, place) for name, args, _ in calls() for place in args]


def of(name):
    args, kw = next((a, k) for n, a, k in calls() if n == name)
    return args, {n: everywhere(v) for n, v in args.items()}, kw


def test_the_places_are_all_there_are():
    rest = {"groups", "eps", "act", "out_dtype", "k", "score", "normalize"}
    for name, args, kw in calls():
        assert set(inspect.signature(getattr(ops, name)).parameters) - rest == set(args)
        assert name in ops.__all__


@pytest.mark.parametrize("name,place", PLACES)
def test_one_host_tensor_is_refused_in_every_place(no_launch, name, place):  # noqa: F811
    args, every, kw = of(name)
    with pytest.raises(Reached):
        getattr(ops, name)(**every, **kw)
    with pytest.raises(ValueError, match="GPU tensor"):
        getattr(ops, name)(**{**every, place: args[place]}, **kw)
    with pytest.raises(ValueError, match="GPU tensor"):
        getattr(ops, name)(**{n: v if n == place else args[n] for n, v in every.items()}, **kw)


@pytest.mark.parametrize("name,place", [(n, p) for n, p in PLACES if p != "out" and next(a for m, a, _ in calls() if m == n)[p].is_floating_point()])
def test_gradients_and_tangents_are_refused(no_launch, name, place):  # noqa: F811
    args, every, kw = of(name)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[place], torch.ones_like(args[place]))
        with pytest.raises(RuntimeError, match="inference-only"):
            getattr(ops, name)(**{**every, place: on_gpu(dual)}, **kw)
    needs = on_gpu(args[place].clone().requires_grad_())
    with pytest.raises(RuntimeError, match="inference-only"):
        getattr(ops, name)(**{**every, place: needs}, **kw)
    with torch.no_grad(), pytest.raises(Reached):
        getattr(ops, name)(**{**every, place: needs}, **kw)


@pytest.mark.parametrize("name,place", [(n, p) for n, p in PLACES if n != "route" and p not in ("out", "residual") and (n, p) != ("group_norm", "x")])
def test_an_out_on_another_argument_is_refused(no_launch, name, place):  # noqa: F811
    """A block would write what another one still reads."""
    args, every, kw = of(name)
    bytes_ = torch.zeros(4096, dtype=torch.uint8)
    lay = lambda t: on_gpu(bytes_[:t.numel() * t.element_size()].view(t.dtype).view(t.shape))  # noqa: E731
    with pytest.raises(ValueError, match="overlap"):
        getattr(ops, name)(**{**every, place: lay(args[place]), "out": lay(args["out"])}, **kw)


@pytest.mark.parametrize("name,place", [("group_norm", "x"), ("grouped_linear", "residual"), ("combine", "residual"), ("lora_linear", "residual")])
def test_an_out_may_be_what_it_stands_for_but_not_overlap_it_otherwise(no_launch, name, place):  # noqa: F811
    args, every, kw = of(name)
    rows, N = args["out"].shape
    buf = on_gpu(zeros(rows + 1, N + 8))
    with pytest.raises(Reached):
        getattr(ops, name)(**{**every, place: buf[:rows, :N], "out": buf[:rows, :N]}, **kw)
    for other in (buf[1:, :N], buf[:rows, 1:N + 1], buf[:rows, 4:N + 4]):
        with pytest.raises(ValueError, match="itself"):
            getattr(ops, name)(**{**every, place: buf[:rows, :N], "out": other}, **kw)
    f32 = on_gpu(zeros(rows, N, dtype=F32))
    with pytest.raises(ValueError, match="itself"):  # of another type
        getattr(ops, name)(**{**every, place: f32, "out": f32.view(-1).view(F16)[:rows * N].view(rows, N)}, **kw)


@pytest.mark.parametrize("name,kw,msg", [
    ("group_norm", dict(groups=3), "multiple of 3"), ("group_norm", dict(groups=0), "groups"), ("group_norm", dict(act="tanh"), "act must"), ("group_norm", dict(x=zeros(4, 4, 4)), "2-D"),
    ("group_norm", dict(x=zeros(4, 16, dtype=torch.float64)), "float32"), ("group_norm", dict(weight=zeros(16)), "weight must"), ("group_norm", dict(bias=zeros(8, dtype=F32)), "bias must"),
    ("group_norm", dict(offsets=zeros(3, dtype=I32)), "offsets must"), ("group_norm", dict(offsets=torch.zeros(0, dtype=torch.int64)), "offsets must"),
    ("group_norm", dict(out=zeros(4, 8)), "out must"), ("group_norm", dict(out_dtype=F32), "out_dtype"), ("group_norm", dict(x=zeros(4, 32)[:, ::2]), "contiguous rows"),
    ("group_norm", dict(x=zeros(1, 16).expand(4, 16)), "overlap"), ("group_norm", dict(out=zeros(1, 16).expand(4, 16)), "overlap"),
    ("route", dict(k=0), "32 a row"), ("route", dict(k=9), "32 a row"), ("route", dict(score="tanh"), "score must"), ("route", dict(mask=zeros(3, dtype=torch.bool)), "mask must"),
    ("route", dict(mask=zeros(4, dtype=F32)), "mask must"), ("route", dict(logits=zeros(4, 1025)), "1 to 1024"), ("route", dict(logits=zeros(4, 0)), "1 to 1024"), ("route", dict(logits=zeros(4, 8, dtype=I32)), "float32"),
    ("grouped_linear", dict(w=zeros(2, 8, 16, dtype=F32)), "w must be"), ("grouped_linear", dict(w=zeros(8, 16)), "contiguous"), ("grouped_linear", dict(w=zeros(2, 8, 12)), "input channels"),
    ("grouped_linear", dict(w=zeros(2, 16, 16).transpose(1, 2)), "contiguous"), ("grouped_linear", dict(offsets=torch.tensor([0, 4])), "segments"), ("grouped_linear", dict(bias=zeros(8, dtype=F32)), "bias must"),
    ("grouped_linear", dict(index=torch.zeros(4, dtype=torch.int64)), "index must"), ("grouped_linear", dict(index=zeros(3, dtype=I32)), "positions"), ("grouped_linear", dict(out=None), "needs out"),
    ("grouped_linear", dict(out_index=None, residual=None), "out must"), ("grouped_linear", dict(out_index=None), "residual must"), ("grouped_linear", dict(residual=zeros(4, 8)), "residual must"), ("grouped_linear", dict(act=None), "act must"), ("grouped_linear", dict(out=zeros(6, 9)), "out must"),
    ("grouped_linear", dict(out=zeros(6), residual=None), "out must"), ("grouped_linear", dict(out=zeros(1, 8).expand(6, 8)), "overlap"),
    ("combine", dict(y=zeros(8, 16)), "y must"), ("combine", dict(y=zeros(4, 16, 2).transpose(1, 2)), "contiguous N"), ("combine", dict(y=zeros(4, 33, 16)), "32 slots"), ("combine", dict(y=zeros(4, 0, 16)), "32 slots"),
    ("combine", dict(weights=zeros(4, 2)), "weights must"), ("combine", dict(weights=zeros(4, 3, dtype=F32)), "weights must"), ("combine", dict(residual=zeros(4, 8)), "residual must"), ("combine", dict(out=zeros(3, 16)), "out must"),
    ("lora_linear", dict(w=zeros(8, 16, dtype=F32)), "must be torch.float16"), ("lora_linear", dict(down=zeros(3, 4, 16, dtype=F32)), "must be torch.float16"), ("lora_linear", dict(w=zeros(8, 12)), "w must"),
    ("lora_linear", dict(down=zeros(3, 4, 12)), "down must"), ("lora_linear", dict(down=zeros(4, 16)), "down must"), ("lora_linear", dict(up=zeros(3, 4, 8)), "up must"), ("lora_linear", dict(up=zeros(2, 8, 4)), "up must"),
    ("lora_linear", dict(adapter=torch.zeros(2, dtype=torch.int64)), "adapter must"), ("lora_linear", dict(adapter=zeros(4, dtype=I32)), "adapter must"), ("lora_linear", dict(offsets=None), "adapter must"),
    ("lora_linear", dict(scale=zeros(2, dtype=F32)), "scale must"), ("lora_linear", dict(bias=zeros(8)), "bias must"), ("lora_linear", dict(down=zeros(3, 129, 16), up=zeros(3, 8, 129)), "rank 1"),
    ("lora_linear", dict(out_dtype=F32), "out_dtype")])
def test_refusals(no_launch, name, kw, msg):  # noqa: F811
    _, every, rest = of(name)
    mine = {k: on_gpu(v) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    with pytest.raises(ValueError, match=msg):
        getattr(ops, name)(**{**every, **rest, **mine})


@pytest.mark.parametrize("bad", [None, 1.0, [1.0]])
def test_what_is_no_tensor_is_refused_by_name(no_launch, bad):  # noqa: F811
    for name, args, kw in calls():
        every = of(name)[1]
        for place in (next(iter(args)), "out") if bad is not None and "out" in args else (next(iter(args)),):
            with pytest.raises(ValueError, match="GPU tensor"):
                getattr(ops, name)(**{**every, place: bad}, **kw)


def test_a_new_result_has_the_type_asked_for(no_launch, monkeypatch):  # noqa: F811
    monkeypatch.setattr(ops, "_on", lambda d, name, *args: None)
    for name, args, kw in calls():
        if name == "route":
            continue
        every = {n: v for n, v in of(name)[1].items() if n not in ("out", "out_index", "residual")}
        assert getattr(ops, name)(**every, **kw).dtype == F16
        for t in (F32, torch.bfloat16):
            assert getattr(ops, name)(**every, **kw, out_dtype=t).dtype == t
        with pytest.raises(ValueError, match="float32"):
            getattr(ops, name)(**every, **kw, out_dtype=torch.float64)
