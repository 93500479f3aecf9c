"""What the dense operators' Python entries decide on the host before anything is launched. The tensors here say that they
are on a GPU and are not; nothing may reach a kernel."""
import inspect

import pytest
import torch

from promptmoge_amd import ops

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
        rest = {"act", "out_dtype", "a_scale", "norm", "eps", "interleaved", "cap", "scale"}
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
