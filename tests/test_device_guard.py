"""Every call runs on its tensors' device and that device's current stream,
whichever device is current: two devices' default streams have the same
handle, so a launch under the wrong device would not be noticed by it."""
import contextlib
import ctypes

import pytest
import torch

from knurlogic_b200 import (Fp8Linear, Fp8SwitchLinear, SparseMoeBlock, SwitchGLU, _lib, decoder, fp8, gemma4, moe,
                            quantize_fp8, switch_layers, synth)
from knurlogic_b200.switch_layers import GeGLU
from tests.test_fp8 import make_weight


@pytest.fixture
def two_devices(monkeypatch):
    """A stand-in for two GPUs with device 0 current; what was called is
    recorded as (name, the device current then, the stream given)."""
    seen, now = [], [0]

    @contextlib.contextmanager
    def device(i):
        before, now[0] = now[0], i
        yield
        now[0] = before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(switch_layers, "c_stream", lambda d: ("stream of", d.index))
    monkeypatch.setattr(_lib, "call", lambda name, *a: seen.append((name, now[0], a[-1])))
    return seen


def test_an_entry_point_runs_under_its_device(two_devices):
    for i in (0, 1, 0):
        switch_layers.call_on(torch.device("cuda", i), "entry", ctypes.c_int(1))
    assert two_devices == [("entry", i, ("stream of", i)) for i in (0, 1, 0)]


def test_every_module_calls_on_its_inputs_device(monkeypatch):
    seen = []
    for m in (switch_layers, fp8, gemma4, moe, decoder):
        monkeypatch.setattr(m, "call_on", lambda d, name, *a: seen.append((name, d)))
        monkeypatch.setattr(m, "require_cuda", lambda *ts: None)
    monkeypatch.setattr(_lib, "call", lambda name, *a: pytest.fail(f"{name} called on no device in particular"))
    monkeypatch.setattr(fp8, "_rows", lambda x, k: x.reshape(-1, k))
    monkeypatch.setattr(fp8, "_status_word", lambda d: torch.zeros(1, dtype=torch.int32))
    bf = torch.bfloat16
    E, k, H, I = 8, 2, 256, 128
    w = [make_weight(s, 1) for s in ((E, I, H), (E, I, H), (E, H, I))]
    x, idx = torch.zeros(3, H, dtype=bf), torch.zeros(3, k, dtype=torch.int32)
    glu = SwitchGLU(*(Fp8SwitchLinear(*p) for p in w))
    glu(x, idx)
    glu.gate_proj(x.view(3, 1, 1, H), idx)
    gemma4.Experts(SwitchGLU(*(Fp8SwitchLinear(*p) for p in w), activation=GeGLU()))(x, idx, torch.ones(3, k))
    gemma4.Router(torch.zeros(E, H, dtype=bf), torch.ones(H), torch.ones(E), k)(x)
    cfg = synth.MoEConfig("fp8", E, k, H, I, 0, 3, quant="fp8")
    blk = SparseMoeBlock.from_weights(synth.make_weights(cfg, seed=1), k)
    blk(x)
    blk.check_status()
    Fp8Linear(*make_weight((H, H), 2))(x)
    quantize_fp8(x)
    decoder.add_rms_norm(x, None, torch.ones(H), 1e-6)
    assert [n for n, _ in seen] == ["vqmoe_switch_glu", "vqmoe_switch_linear", "vqmoe_moe_experts", "vqmoe_rms_norm",
                                    "vqmoe_router_ex", "vqmoe_sparse_moe_block", "vqmoe_workspace_status",
                                    "vqmoe_grouped_linear", "vqmoe_quantize_fp8", "vqmoe_add_rms_norm"]
    assert all(d == x.device for _, d in seen)


def test_tensors_of_two_devices_are_refused(monkeypatch):
    """(The meta device stands in for a second GPU.)"""
    for m in (switch_layers, gemma4, moe):
        monkeypatch.setattr(m, "call_on", lambda *a: pytest.fail("launched"))
        monkeypatch.setattr(m, "require_cuda", lambda *ts: None)
    E, k, H, I = 8, 2, 256, 128
    cfgs = [synth.MoEConfig(q, E, k, H, I, 0, 3, quant=q) for q in ("vq", "affine", "fp8")]
    cfgs.append(synth.MoEConfig("dense", E, k, H, I, 0, 3, quant="dense"))
    x, idx = torch.zeros(3, H, dtype=torch.bfloat16), torch.zeros(3, k, dtype=torch.int32)
    for cfg in cfgs:
        if cfg.quant == "dense":
            sw = [switch_layers.SwitchLinear(torch.zeros(s)) for s in ((E, I, H), (E, I, H), (E, H, I))]
            blk = SparseMoeBlock(torch.zeros(E, H), SwitchGLU(*sw), k)
        else:
            blk = SparseMoeBlock.from_weights(synth.make_weights(cfg, seed=1), k)
        glu = blk.switch_mlp
        with pytest.raises(ValueError, match="indices are on meta"):
            glu(x, idx.to("meta"))
        with pytest.raises(ValueError, match="indices are on meta"):
            glu.gate_proj(x.view(3, 1, 1, H), idx.to("meta"))
        glu.down_proj.to("meta")
        for call in (lambda: glu(x, idx), lambda: blk(x),
                     lambda: glu.down_proj(torch.zeros(3, 1, 1, I, dtype=torch.bfloat16), idx)):
            with pytest.raises(ValueError, match="weights are on meta"):
                call()
        e = gemma4.Experts(SwitchGLU(glu.gate_proj, glu.up_proj, glu.down_proj, activation=GeGLU()))
        with pytest.raises(ValueError, match="weights are on meta"):
            e(x, idx, torch.ones(3, k))
