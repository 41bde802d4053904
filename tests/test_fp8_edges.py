"""Block-scaled e4m3 and grouped products at the edges of what their
documentation allows (tolerances as in test_fp8)."""
import numpy as np
import pytest
import torch

from knurlogic_b200 import Fp8Linear, Fp8SwitchLinear, SwitchGLU, fp8, grouped_linear, quantize_fp8
from tests.conftest import assert_bf16_close, to_np
from tests.test_fp8 import (check, experts_64, f64, grouped_64, linear_64, make_weight, make_x, quantize_64, spread,
                            weight_64)

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


def _glu(E, H, I):
    w = make_weight((E, I, H), 1, DEV), make_weight((E, I, H), 2, DEV), make_weight((E, H, I), 3, DEV)
    return SwitchGLU(*(Fp8SwitchLinear(*p) for p in w)), w


@pytest.mark.gpu
@pytest.mark.parametrize("E", [8, 1024])
def test_pairs_of_no_expert_among_many(E):
    """From 4096 pairs the sort is spread over CTAs: ids outside the experts
    take no place there either, and an expert named twice by a token has both
    its pairs."""
    T, k, H, I = 2100, 3, 64, 32
    glu, w = _glu(E, H, I)
    x = make_x(T, H, 1, DEV)
    idx = np.random.default_rng(E).integers(0, E, (T, k)).astype(np.int32)
    idx[7] = idx[7, 0]
    idx[5, 1], idx[6], idx[T - 1, 2] = -1, (E, 1 << 30, -(1 << 31)), E
    ok = (idx >= 0) & (idx < E)
    y = to_np(glu(x, torch.from_numpy(idx).to(DEV)))
    assert np.array_equal(y[7, 0], y[7, 1]) and np.array_equal(y[7, 0], y[7, 2])
    ref = experts_64(f64(x), idx, *w)
    assert_bf16_close(y[ok], ref[ok], f"pairs of no expert, {E} experts")


@pytest.mark.gpu
def test_more_tokens_than_a_launch_takes():
    """8192 tokens a launch: the rest is a launch of its own."""
    E, k, H, I = 8, 2, 64, 32
    glu, w = _glu(E, H, I)
    x = make_x(8200, H, 1, DEV)
    idx = np.random.default_rng(1).integers(0, E, (8200, k)).astype(np.int32)
    y = glu(x, torch.from_numpy(idx).to(DEV))
    assert_bf16_close(to_np(y), experts_64(f64(x), idx, *w), "8200 tokens")
    rows = glu.down_proj(make_x(8200, I, 2, DEV).view(8200, 1, I), torch.from_numpy(idx[:, 0]).to(DEV)).view(8200, H)
    q, xs = quantize_64(f64(make_x(8200, I, 2)))
    xv, wv = q * spread(xs, I), weight_64(f64(w[2][0]), f64(w[2][1]))
    at = idx[:, 0]
    check(rows, np.einsum("rk,rnk->rn", xv, wv[at]), np.einsum("rk,rnk->rn", np.abs(xv), np.abs(wv[at])), I)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """More than 2^31 values quantized, and more than 2^31 outputs."""
    K = 4096
    x = make_x(64, K, 1, DEV).repeat(8300, 1)                  # 2.18e9 values
    q, s = quantize_fp8(x)
    rq, rs = quantize_fp8(x[:64])
    assert torch.equal(q[-64:].view(torch.uint8), rq.view(torch.uint8)) and torch.equal(s[-64:], rs)
    del q, s
    m = Fp8Linear(*make_weight((16, K), 2, DEV))
    check(m(x)[-64:], *linear_64(x[-64:], m.weight, m.weight_scale_inv), K)
    del x
    m = Fp8Linear(*make_weight((65536, 128), 3, DEV))
    x = make_x(64, 128, 4, DEV).repeat(520, 1)                 # 2.18e9 outputs
    ref = linear_64(x[-64:], m.weight, m.weight_scale_inv)
    check(m(x)[-64:], *ref, 128)
    off = torch.tensor([0, 5, x.shape[0]], dtype=torch.int32, device=DEV)
    w = torch.stack([m.weight[:32768].view(torch.uint8)] * 2).view(torch.float8_e4m3fn)
    y = grouped_linear(torch.cat([x, x]), w, off * 2, weight_scale_inv=torch.stack([m.weight_scale_inv[:256]] * 2))
    check(y[-64:], ref[0][:, :32768], ref[1][:, :32768], 128)
    fp8.check_status(DEV)
