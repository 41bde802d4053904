"""Block-scaled e4m3 and grouped products at the edges of what their
documentation allows (tolerances as in test_fp8)."""
import numpy as np
import pytest
import torch

from knurlogic_b200 import Fp8Linear, fp8, grouped_linear
from tests.test_fp8 import (check, f64, grouped_64, linear_64, make_weight, make_x, quantize_64, spread, weight_64)

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(1, 4096, 4096), (1, 16, 144), (40, 528, 2064), (300, 1040, 400)])
def test_repeated_calls_give_the_same_bits(T, N, K):
    """Dense products fetch their first weights while the quantizer before
    them still runs; calls behind one another, one set of inputs in turn with
    another, neither meet nor run into a bounded wait."""
    m = Fp8Linear(*make_weight((N, K), T, DEV))
    xs = [make_x(T, K, i, DEV) for i in range(2)]
    first = [m(x) for x in xs]
    for x, y in zip(xs, first):
        check(y, *linear_64(x, m.weight, m.weight_scale_inv), K)
    for x, y in [(xs[i % 2], m(xs[i % 2])) for i in range(200)]:
        assert torch.equal(y, first[0] if x is xs[0] else first[1])
    fp8.check_status(DEV)


OFFSETS = {
    "falling": lambda P: [0, P, 0, P],                     # the last group would have every row a second time
    "a fall in the middle": lambda P: [2, P // 2, P // 4, P - 1, P - 1],
    "all the way down": lambda P: [P, P // 2, 1, 0],       # every group empty
    "past both ends": lambda P: [-9, P + 50, -3, P + 7, 4],
    "many": lambda P: [(7 * e * e) % (P + 1) for e in range(201)],
}


@pytest.mark.gpu
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("P", [3, 40, 700, 1500])
@pytest.mark.parametrize("kind", OFFSETS)
def test_offsets_that_fall_back_name_no_row_twice(kind, P, quant):
    """An offset below an earlier one counts as the largest before it."""
    off = OFFSETS[kind](P)
    rising = np.maximum.accumulate(np.clip(off, 0, P))
    E, N, K = len(off) - 1, 144, 528
    x = make_x(P, K, P, DEV)
    if quant:
        w, s = make_weight((E, N, K), E, DEV)
        q, xs = quantize_64(f64(x))
        ref, mag = grouped_64(q * spread(xs, K), weight_64(f64(w), f64(s)), rising)
    else:
        w, s = torch.empty(E, N, K, device=DEV).normal_(0, 0.05).to(torch.bfloat16), None
        ref, mag = grouped_64(f64(x), f64(w), rising)
    out = torch.full((P, N), 7.0, dtype=torch.bfloat16, device=DEV)
    grouped_linear(x, w, torch.tensor(off, dtype=torch.int32, device=DEV), weight_scale_inv=s, out=out)
    a, b = int(rising[0]), int(rising[-1])
    assert (out[:a] == 7).all() and (out[b:] == 7).all()
    if a < b:
        check(out[a:b], ref[a:b], mag[a:b], K)
    fp8.check_status(DEV)
