"""The block-scaled e4m3 modules as parts of a model: cast, moved, copied,
reloaded, their buffers replaced between calls."""
import pytest
import torch
from torch import nn

from knurlogic_b200 import Fp8Linear, Fp8SwitchLinear, fp8, grouped_linear
from knurlogic_b200.switch_layers import fp8_descriptor
from tests.test_fp8 import make_weight, make_x

DEV = "cuda:0"

MODULES = [(Fp8Linear, (256, 384)), (Fp8SwitchLinear, (2, 256, 384))]


def _module(cls, shape, seed=1):
    return cls(*make_weight(shape, seed))


# ------------------------------------------------------------------ CPU

@pytest.mark.parametrize("cls,shape", MODULES)
@pytest.mark.parametrize("cast,dtype", [(lambda m: m.to(torch.bfloat16), torch.bfloat16),
                                        (lambda m: m.half(), torch.float16),
                                        (lambda m: m.to("cpu", torch.float64), torch.float64)],
                         ids=["bfloat16", "half", "device and float64"])
def test_a_cast_of_the_model_leaves_the_format(cls, shape, cast, dtype):
    """`model.to(dtype)` converts every floating buffer of a module tree; the
    e4m3 values and their float32 scales are a format, not a precision."""
    m = _module(cls, shape)
    w, s = m.weight.clone(), m.weight_scale_inv.clone()
    tree = cast(nn.Sequential(nn.Linear(4, 4), m))
    assert tree[0].weight.dtype == dtype
    assert m.weight.dtype == torch.float8_e4m3fn and m.weight_scale_inv.dtype == torch.float32
    assert torch.equal(m.weight.view(torch.uint8), w.view(torch.uint8)) and torch.equal(m.weight_scale_inv, s)


@pytest.mark.parametrize("cls,shape", MODULES)
def test_the_descriptor_follows_replaced_buffers(cls, shape):
    """Buffers of another shape at the same addresses: views of their
    beginnings, or new ones where freed ones lay."""
    m = _module(cls, shape)
    d = fp8_descriptor(m)
    assert (d.out_features, d.in_features) == (256, 384)
    at = m.weight.data_ptr()
    if cls is Fp8Linear:
        m.weight, m.weight_scale_inv = m.weight[:128], m.weight_scale_inv[:1]
    else:
        m.weight, m.weight_scale_inv = m.weight[:1].view(1, 384, 256), m.weight_scale_inv[:1].reshape(1, 3, 2)
    d = fp8_descriptor(m)
    assert d.weight == at
    assert (d.out_features, d.in_features) == tuple(m.weight.shape[-2:])
    assert d.num_experts == 1


@pytest.mark.parametrize("cls,shape", MODULES)
def test_replaced_buffers_are_checked(cls, shape):
    def replaced(weight=None, scale=None):
        m = _module(cls, shape)
        fp8_descriptor(m)
        if weight is not None:
            m.weight = weight(m.weight)
        if scale is not None:
            m.weight_scale_inv = scale(m.weight_scale_inv)
        return lambda: fp8_descriptor(m)

    for bad, why in ((replaced(weight=lambda w: w.to(torch.bfloat16)), "float8_e4m3fn"),
                     (replaced(weight=lambda w: w.view(torch.int8)), "float8_e4m3fn"),
                     (replaced(scale=lambda s: s.to(torch.bfloat16)), "float32"),
                     (replaced(weight=lambda w: w[..., :128, :]), "weight_scale_inv"),
                     (replaced(weight=lambda w: w[0] if w.dim() == 3 else w[None],
                               scale=lambda s: s[0] if s.dim() == 3 else s[None]), "OUT, IN"),
                     (replaced(scale=lambda s: s[..., :1, :]), "weight_scale_inv"),
                     (replaced(weight=lambda w: w.transpose(-1, -2), scale=lambda s: s.transpose(-1, -2)), "contiguous"),
                     (replaced(scale=lambda s: s.to("meta")), "meta")):
        with pytest.raises(ValueError, match=why):
            bad()


def test_a_state_dict_assigned_in_another_type_is_refused():
    m, o = _module(*MODULES[0]), _module(*MODULES[0], seed=2)
    m.load_state_dict(o.state_dict())
    assert torch.equal(m.weight.view(torch.uint8), o.weight.view(torch.uint8))
    fp8_descriptor(m)
    m.load_state_dict({k: v.to(torch.bfloat16) for k, v in o.state_dict().items()}, assign=True)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        fp8_descriptor(m)


# ------------------------------------------------------------------ GPU
# The kernels' own waits cannot be made to run out without a fault, so the
# tests raise the device's word themselves, by an ordinary copy.

@pytest.mark.gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_a_wait_that_ran_out_is_reported_once(monkeypatch, mode):
    monkeypatch.setattr(fp8, "_status", {})
    with mode():
        m = Fp8Linear(*make_weight((144, 272), 1, DEV))
        x = make_x(3, 272, 1, DEV)
        y = m(x)
        fp8.check_status(DEV)
        fp8._status[0].fill_(1)
        m(x)                                            # a later call does not clear it
    with pytest.raises(TimeoutError, match="ran out"):
        fp8.check_status()
    fp8.check_status(DEV)
    assert torch.equal(m(x), y)
    fp8.check_status(torch.device(DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("place", [lambda: Fp8Linear(*make_weight((144, 272), 1, DEV)),
                                   lambda: Fp8Linear(*make_weight((144, 272), 1)).to(DEV)], ids=["made", "moved"])
def test_a_captured_first_call_has_a_status_word(monkeypatch, place):
    """A module's device has its word before the first call on it, which may
    be a captured one: the graph's kernels are given it."""
    monkeypatch.setattr(fp8, "_status", {})
    m, x = place(), make_x(3, 272, 1, DEV)
    assert list(fp8._status) == [0]
    given = []
    call = fp8.call_on
    monkeypatch.setattr(fp8, "call_on", lambda dev, name, *a: (given.append(a[-1]), call(dev, name, *a)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m(x)
    g.replay()
    assert given == [fp8._status[0].data_ptr()]
    assert torch.equal(y, m(x))


@pytest.mark.gpu
def test_a_captured_first_grouped_call_runs_without_one(monkeypatch):
    """No module came before it: the call is captured all the same, with no
    word to raise, and leaves none of the graph's memory behind as one."""
    w = torch.randn(3, 32, 64, device=DEV).to(torch.bfloat16)
    x, off = make_x(50, 64, 1, DEV), torch.tensor([0, 10, 10, 50], dtype=torch.int32, device=DEV)
    ref = grouped_linear(x, w, off)
    monkeypatch.setattr(fp8, "_status", {})
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = grouped_linear(x, w, off)
    g.replay()
    assert torch.equal(y, ref) and not fp8._status
    fp8.check_status(DEV)


@pytest.mark.gpu
def test_a_cast_model_gives_the_same_product():
    m, x = Fp8Linear(*make_weight((144, 272), 1, DEV)), make_x(5, 272, 2, DEV)
    y = m(x)
    assert torch.equal(m.to(torch.bfloat16)(x), y) and torch.equal(m.cpu().half().to(DEV)(x), y)


@pytest.mark.gpu
def test_a_product_follows_replaced_buffers():
    """The first 128 outputs, from a view of the weights' beginning, and
    nothing written behind them."""
    m, x = Fp8Linear(*make_weight((400, 272), 1, DEV)), make_x(5, 272, 2, DEV)
    y = m(x)
    m.weight, m.weight_scale_inv = m.weight[:128], m.weight_scale_inv[:1]
    assert torch.equal(m(x), y[:, :128])
    m.weight = m.weight.to(torch.bfloat16)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        m(x)
