"""Block-scaled e4m3 and grouped products at the edges of what their
documentation allows (tolerances as in test_fp8)."""
import pytest
import torch

from knurlogic_b200 import Fp8Linear, fp8
from tests.test_fp8 import check, linear_64, make_weight, make_x

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
