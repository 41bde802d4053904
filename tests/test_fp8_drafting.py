"""Drafted decoding of a model in the block-scaled format, against plain
greedy decoding; and one row's product in calls of other sizes."""
from dataclasses import replace

import numpy as np
import pytest
import torch

from knurlogic_b200 import Fp8Linear, decoder
from tests.test_fp8 import f64, linear_64, make_weight, make_x

DEV = "cuda:0"
TINY = decoder.CONFIGS["tiny"]
CFG = replace(TINY, fp8=True, moe=replace(TINY.moe, quant="fp8"))


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("k", [1, 2, 3])
def test_drafting_emits_the_plain_greedy_tokens(k, graphs):
    model = decoder.build(CFG, seed=5, device=DEV)
    prompts = torch.randint(0, CFG.vocab, (4, 16), generator=torch.Generator().manual_seed(5)).to(DEV)
    plain = decoder.generate_greedy(model, prompts, 24)
    drafted, stats = decoder.generate_mtp(model, prompts, 24, k=k, graphs=graphs)
    assert torch.equal(drafted, plain)
    assert stats["steps"] > 0 and stats["drafted"] == stats["steps"] * 4 * k
    assert 0 <= stats["accepted"] <= stats["drafted"]


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(4096, 4096), (528, 2064), (272, 144)])
def test_a_row_in_calls_of_other_sizes(N, K):
    """The number of rows picks the kernel's mode and how many CTAs share a
    tile's sum, so a row's float32 sum may be added in another order: each
    order is within the bar of test_fp8, two within twice that; the values of
    the other rows change nothing."""
    m = Fp8Linear(*make_weight((N, K), 3, DEV))
    x = make_x(2600, K, 4, DEV)
    row = x[:1].clone()
    one = f64(m(row, out_dtype=torch.float32))
    _, mag = linear_64(row, m.weight, m.weight_scale_inv)
    bar = 2 * (K + 4) * 2.0 ** -23 * mag
    for T in (2, 33, 64, 128, 129, 300, 1001, 2600):
        y = m(x[:T], out_dtype=torch.float32)
        assert np.all(np.abs(f64(y[:1]) - one) <= bar), T
        others = torch.cat([row, make_x(T - 1, K, T, DEV)])
        assert torch.equal(m(others, out_dtype=torch.float32)[:1], y[:1]), T
