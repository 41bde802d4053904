"""The block-scaled e4m3 modules as parts of a model: cast, moved, copied,
reloaded, their buffers replaced between calls."""
import pytest
import torch
from torch import nn

from knurlogic_b200 import Fp8Linear, Fp8SwitchLinear
from knurlogic_b200.switch_layers import fp8_descriptor
from tests.test_fp8 import make_weight

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
