"""A decoder whose projections, LM head and experts are block-scaled e4m3
(`DecoderConfig.fp8`, `MoEConfig.quant` "fp8"): the operators of the format
together, as the model runs them."""
from dataclasses import replace

import numpy as np
import pytest
import torch

from knurlogic_b200 import Fp8Linear, Fp8SwitchLinear, SparseMoeBlock, decoder, synth
from knurlogic_b200.moe import dense_weight
from tests.conftest import assert_bf16_close, to_np
from tests.test_fp8 import f64, linear_64, make_weight

DEV = "cuda:0"
TINY = decoder.CONFIGS["tiny"]
CFG = replace(TINY, fp8=True, moe=replace(TINY.moe, quant="fp8"))


def test_weight_names_and_modules():
    w = decoder.make_weights(CFG, seed=1)
    p = "model.layers.0.self_attn."
    assert w[p + "q_proj.weight"].dtype == torch.float8_e4m3fn
    assert w[p + "q_proj.weight_scale_inv"].shape == (CFG.heads * 2 * CFG.head_dim // 128, CFG.hidden // 128)
    assert isinstance(decoder.Attention(w, p, CFG).wo, Fp8Linear)
    assert not isinstance(decoder.Attention(decoder.make_weights(TINY, seed=1), p, TINY).wo, Fp8Linear)
    assert w["lm_head.weight_scale_inv"].shape == (CFG.vocab // 128, CFG.hidden // 128)


def test_a_block_scaled_shared_expert_is_restored():
    wt, sc = make_weight((144, 272), 3)
    d = {"a.weight": wt, "a.weight_scale_inv": sc, "b.weight": wt}
    ref = wt.float() * sc.repeat_interleave(128, 0)[:144].repeat_interleave(128, 1)[:, :272]
    assert torch.equal(dense_weight(d, "a"), ref.to(torch.bfloat16))
    with pytest.raises(ValueError, match="weight_scale_inv"):
        dense_weight(d, "b")
    moe = replace(CFG.moe, shared_inter=0)
    w = synth.make_weights(moe, seed=1)
    assert isinstance(SparseMoeBlock.from_weights(w, moe.top_k).switch_mlp.up_proj, Fp8SwitchLinear)
    del w["mlp.switch_mlp.up_proj.weight_scale_inv"]
    with pytest.raises(KeyError, match="weight_scale_inv"):
        SparseMoeBlock.from_weights(w, moe.top_k)


class _Linear64:
    """The projection by the 64-bit formula, rounded once to bf16."""

    def __init__(self, m: Fp8Linear):
        self.m = m

    def __call__(self, x):
        ref, _ = linear_64(x.reshape(-1, x.shape[-1]), self.m.weight, self.m.weight_scale_inv)
        return torch.from_numpy(ref).to(torch.bfloat16).to(x.device).view(*x.shape[:-1], -1)


@pytest.mark.gpu
@pytest.mark.parametrize("B,L", [(1, 1), (2, 7), (3, 50)])
def test_attention_matches_64_bit_projections(B, L):
    """The attention block with its four projections on the kernels and by
    the 64-bit formula: bf16 neighbours where a float32 sum rounds the other
    way, within the layer bar of conftest."""
    w = {k: v.to(DEV) for k, v in decoder.make_weights(CFG, seed=4).items()}
    a, b = (decoder.Attention(w, "model.layers.0.self_attn.", CFG) for _ in range(2))
    for n in ("wq", "wk", "wv", "wo"):
        setattr(b, n, _Linear64(getattr(a, n)))
    x = torch.randn(B, L, CFG.hidden, generator=torch.Generator().manual_seed(L)).to(torch.bfloat16).to(DEV)
    out = [m(x, decoder.KVCache(B, 64, CFG.kv_heads, CFG.head_dim, DEV), 0) for m in (a, b)]
    assert_bf16_close(to_np(out[0]), to_np(out[1]), f"fp8 attention B{B} L{L}")


@pytest.mark.gpu
def test_head_logits_and_generation():
    model = decoder.build(CFG, seed=2, device=DEV)
    prompts = torch.randint(0, CFG.vocab, (3, 20), generator=torch.Generator().manual_seed(0)).to(DEV)
    normed, _ = model(prompts, model.new_caches(3, 24, DEV), 0)
    lg = model.fp8_head(normed, out_dtype=torch.float32)
    ref, mag = linear_64(normed.reshape(-1, CFG.hidden), model.lm_head, model.fp8_head.weight_scale_inv)
    assert np.all(np.abs(f64(lg).reshape(ref.shape) - ref) <= (CFG.hidden + 4) * 2.0 ** -23 * mag)
    assert torch.equal(model.logits(normed), lg.to(torch.bfloat16))
    eager = decoder.generate_greedy(model, prompts, 8)
    assert torch.equal(decoder.generate_greedy(model, prompts, 8, graphs=True), eager)
    toks, stats = decoder.generate_mtp(model, prompts, 8, k=2)
    assert toks.shape == (3, 8) and stats["steps"] > 0
