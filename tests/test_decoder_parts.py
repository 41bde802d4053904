"""The decoder's parts as Python objects: what a program reads off them,
copies and stores."""
import copy
import pickle
from dataclasses import replace

import pytest
import torch

from knurlogic_b200 import Fp8Linear, decoder

TINY = decoder.CONFIGS["tiny"]
P = "model.layers.0.self_attn."
PROJECTIONS = {"wq": "q_proj", "wk": "k_proj", "wv": "v_proj", "wo": "o_proj"}


@pytest.fixture(scope="module")
def bf16():
    w = decoder.make_weights(replace(TINY, mtp=False), seed=1)
    return w, decoder.Attention(w, P, TINY)


def test_bf16_projections_are_the_state_dicts_tensors(bf16):
    w, a = bf16
    for n, leaf in PROJECTIONS.items():
        assert getattr(a, n) is w[f"{P}{leaf}.weight"]


def test_an_attention_block_pickles(bf16):
    w, a = bf16
    b = pickle.loads(pickle.dumps(a))
    for n, leaf in PROJECTIONS.items():
        assert torch.equal(getattr(b, n), w[f"{P}{leaf}.weight"])


def test_a_copied_attention_block_has_its_own_weights(bf16):
    w, a = bf16
    b = copy.deepcopy(a)
    for n in PROJECTIONS:
        assert torch.equal(getattr(b, n), getattr(a, n))
        assert getattr(b, n).data_ptr() != getattr(a, n).data_ptr()


def test_a_copied_block_scaled_attention_block_has_its_own_weights():
    cfg = replace(TINY, fp8=True, mtp=False)
    a = decoder.Attention(decoder.make_weights(cfg, seed=1), P, cfg)
    b = copy.deepcopy(a)
    for n in PROJECTIONS:
        x, y = getattr(a, n), getattr(b, n)
        assert isinstance(x, Fp8Linear) and isinstance(y, Fp8Linear)
        assert torch.equal(x.weight.view(torch.uint8), y.weight.view(torch.uint8))
        assert x.weight.data_ptr() != y.weight.data_ptr()
