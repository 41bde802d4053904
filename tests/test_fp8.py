"""Block-scaled e4m3 products and ragged grouped products (`quantize_fp8`,
`Fp8Linear`, `grouped_linear`, `Fp8SwitchLinear`) against plain 64-bit
implementations of their formulas.

Tolerances. The products of two e4m3 (or bf16) values are exact in float32;
what a kernel may lose against the 64-bit sum is its float32 additions, at
most 2^-23 of the running sum of magnitudes each whatever their order (a
truncating adder's bound; rounding halves it), the two scalings of a block's
sum (2^-24 each), and the one rounding of the output (2^-8 of the value for
bf16, none more for float32). With S the sum of the terms' magnitudes and K
terms that is |got - ref| <= half * |ref| + (K + 4) 2^-23 S.
Quantization is exact: its values and scales are compared bit for bit.
"""
import copy

import numpy as np
import pytest
import torch

from knurlogic_b200 import (Fp8Linear, Fp8SwitchLinear, SparseMoeBlock, SwitchGLU, _lib, fp8, gemma4,
                            grouped_linear, quantize_fp8, synth, tensor_split)
from knurlogic_b200.switch_layers import GeGLU
from oracle import moe_ref as R
from tests.conftest import assert_bf16_close, to_np

DEV = "cuda:0"


# ------------------------------------------------------------- references

def e4m3_64(v):
    """Nearest e4m3 value of float64 numbers up to 448, ties to even."""
    a = np.abs(v)
    _, ex = np.frexp(np.maximum(a, 2.0 ** -6))
    step = np.ldexp(1.0, ex - 4)
    return np.sign(v) * np.minimum(np.rint(a / step) * step, 448.0)


def quantize_64(x):
    """(values, scales) of float64 rows, groups of 128."""
    rows, K = x.shape
    G = -(-K // 128)
    q, s = np.zeros((rows, K)), np.zeros((rows, G), np.float32)
    for g in range(G):
        v = x[:, 128 * g:128 * g + 128]
        a = np.maximum(np.abs(v).max(1), 2.0 ** -100)
        q[:, 128 * g:128 * g + 128] = e4m3_64(448.0 * v / a[:, None])
        s[:, g] = a / 448.0
    return q, s.astype(np.float64)


def spread(s, n):
    return np.repeat(s, 128, axis=-1)[..., :n]


def weight_64(w, s):
    """Block-scaled weights [.., N, K] as float64."""
    n, k = w.shape[-2:]
    full = np.repeat(np.repeat(s.astype(np.float64), 128, axis=-2)[..., :n, :], 128, axis=-1)[..., :k]
    return w.astype(np.float64) * full


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def make_weight(shape, seed, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(shape, generator=g) * 110).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand((*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128)), generator=g) * 2e-4 + 1e-4
    return w.to(dev), s.to(dev)


def make_x(rows, k, seed, dev="cpu"):
    g = torch.Generator().manual_seed(1000 + seed)
    ch = torch.exp(0.7 * torch.randn(k, generator=g))
    return (torch.randn(rows, k, generator=g) * ch).to(torch.bfloat16).to(dev)


def check(got, ref, mag, K, f32=False):
    got = f64(got)
    assert got.shape == ref.shape
    assert np.isfinite(got).all()
    bar = (0.0 if f32 else 2.0 ** -8) * np.abs(ref) + (K + 4) * 2.0 ** -23 * mag + 1e-37
    over = np.abs(got - ref) > bar
    assert not over.any(), f"{over.sum()} of {over.size} off, worst {np.max(np.abs(got - ref) / bar):.2f} of the bar"


# ------------------------------------------------------------------ CPU

def test_argument_refusals():
    w, s = make_weight((144, 272), 1)
    m = Fp8Linear(w, s)
    assert (m.out_features, m.in_features) == (144, 272) and s.shape == (2, 3)
    with pytest.raises(ValueError, match="weight_scale_inv"):
        Fp8Linear(w, s[:, :2])
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        Fp8Linear(w.float(), s)
    with pytest.raises(ValueError, match="multiples of 16"):
        Fp8Linear(w[:, :264], s)
    with pytest.raises(RuntimeError, match="CUDA"):
        m(torch.zeros(1, 272, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match=r"\[E, OUT, IN\]"):
        Fp8SwitchLinear(w, s)
    e = Fp8SwitchLinear(w[None], s[None])
    assert (e.num_experts, e.output_dims, e.input_dims) == (1, 144, 272)
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_fp8(torch.zeros(4, 128, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="CUDA"):
        grouped_linear(torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(2, 16, 16, dtype=torch.bfloat16),
                       torch.zeros(3, dtype=torch.int32))


def _c_linear(E=2, N=256, K=256, fmt=_lib.FMT_FP8_BLOCK, **kw):
    return _lib.Linear(format=fmt, num_experts=E, out_features=N, in_features=K, weight=4096, scales=4096,
                       group_size=kw.pop("group_size", 128), **kw)


def _status(d, x=4096, rows=4, pitch=256, off=4096, out=4096, dt=0, ws=4096, n=1 << 30):
    lib = _lib.lib()
    import ctypes
    return _lib.STATUS[lib.vqmoe_grouped_linear(ctypes.byref(d), x, rows, pitch, off, out, dt, ws, n, None, None)]


def test_c_refusals_before_any_launch():
    lib = _lib.lib()
    import ctypes
    assert _status(_c_linear(K=264)) == "BAD_SHAPE"
    assert _status(_c_linear(N=264)) == "BAD_SHAPE"
    assert _status(_c_linear(group_size=64)) == "BAD_FORMAT"
    assert _status(_c_linear(fmt=_lib.FMT_VQ_U8)) == "BAD_FORMAT"
    assert _status(_c_linear(), pitch=250) == "BAD_SHAPE"
    assert _status(_c_linear(), pitch=260) == "BAD_SHAPE"
    assert _status(_c_linear(), rows=-1) == "BAD_SHAPE"
    assert _status(_c_linear(E=2048)) == "BAD_SHAPE"
    assert _status(_c_linear(), off=None) == "BAD_POINTER"
    assert _status(_c_linear(), x=None) == "BAD_POINTER"
    assert _status(_c_linear(), out=4100) == "BAD_POINTER"
    assert _status(_c_linear(), ws=None) == "BAD_POINTER"
    assert _status(_c_linear(), dt=2) == "BAD_FORMAT"
    assert _status(_c_linear(), n=16) == "WORKSPACE_TOO_SMALL"
    assert _status(_c_linear(), rows=0) == "OK"
    d = _c_linear()
    assert lib.vqmoe_grouped_linear_workspace_size(ctypes.byref(d), 4) >= 4 * 256 + 4 * 2 * 4
    assert lib.vqmoe_grouped_linear_workspace_size(ctypes.byref(_c_linear(fmt=0)), 4) == 0
    st = lib.vqmoe_quantize_fp8
    assert _lib.STATUS[st(4096, 4, 100, 104, 4096, 4096, None)] == "BAD_SHAPE"
    assert _lib.STATUS[st(4096, 4, 128, 100, 4096, 4096, None)] == "BAD_SHAPE"
    assert _lib.STATUS[st(4098, 4, 128, 128, 4096, 4096, None)] == "BAD_POINTER"
    assert _lib.STATUS[st(None, 0, 128, 128, None, None, None)] == "OK"


def test_a_glu_takes_the_format_on_all_linears_or_none():
    import ctypes
    g, u, d = _c_linear(E=2, N=128, K=256), _c_linear(E=2, N=128, K=256), _c_linear(E=2, N=256, K=128, fmt=0)
    st = _lib.lib().vqmoe_switch_glu(ctypes.byref(g), ctypes.byref(u), ctypes.byref(d), 4096, 4096, 4, 2, 4096, 4096,
                                     1 << 30, None)
    assert _lib.STATUS[st] == "BAD_FORMAT"


def test_split_rules_for_block_scaled_weights():
    def shapes(h, i):
        out = {}
        for n, (o, k) in {"gate": (i, h), "up": (i, h), "down": (h, i)}.items():
            out[f"mlp.switch_mlp.{n}_proj.weight"] = (8, o, k)
            out[f"mlp.switch_mlp.{n}_proj.weight_scale_inv"] = (8, -(-o // 128), -(-k // 128))
        return out
    assert tensor_split.refusals(shapes(2048, 768), 2) == []
    assert tensor_split.refusals(shapes(2048, 768), 3) == []
    bad = tensor_split.refusals(shapes(2048, 768), 4)           # 192 rows a rank: scale blocks cut in two
    assert len(bad) >= 3 and any("128" in b for b in bad)


# ------------------------------------------------------------- quantize

@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 128), (5, 144), (7, 2000), (64, 2048), (1001, 336), (2, 8192)])
def test_quantize_is_exact(rows, cols):
    x = make_x(rows, cols, rows + cols, DEV)
    q, s = quantize_fp8(x)
    rq, rs = quantize_64(f64(x))
    assert np.array_equal(f64(q), rq)
    assert np.array_equal(f64(s), rs)


@pytest.mark.gpu
def test_quantize_ties_and_extremes():
    """Every pair of 8-bit significands as (value, largest): many quotients
    fall exactly half way between two e4m3 values; and the smallest, largest
    and zero groups."""
    a = 1.0 + torch.arange(128) / 128.0
    x = torch.empty(128, 256)
    for sc in range(2):
        x[:, 128 * sc:128 * sc + 128] = (1.0 + torch.arange(128) / 128.0)[None, :] * (2.0 ** -(sc + 1))
        x[:, 128 * sc] = a
    x = torch.cat([x, torch.zeros(1, 256), torch.full((1, 256), 2.0 ** -110), torch.full((1, 256), 3.38e38),
                   -x[:1] * 2.0 ** 126, x[:1] * 2.0 ** -99]).to(torch.bfloat16).to(DEV)
    q, s = quantize_fp8(x)
    rq, rs = quantize_64(f64(x))
    assert np.array_equal(f64(q), rq) and np.array_equal(f64(s), rs)


@pytest.mark.gpu
def test_quantize_strides_shapes_and_non_finite_groups():
    big = make_x(40, 512, 3, DEV)
    for v in (big[:, 128:400], big[::2, :256], big[:, 8:24], big.t()[:, :32].contiguous().t()[:, :256], big[:0],
              big[:, 4:36], big.view(4, 10, 512), big[0]):
        q, s = quantize_fp8(v)
        assert q.shape == v.shape and s.shape == (*v.shape[:-1], -(-v.shape[-1] // 128))
        rq, rs = quantize_64(f64(v).reshape(-1, v.shape[-1])) if v.numel() else (np.zeros(q.shape), np.zeros(s.shape))
        assert np.array_equal(f64(q).reshape(rq.shape), rq) and np.array_equal(f64(s).reshape(rs.shape), rs)
    x = make_x(4, 384, 4, DEV)
    x[0, 5], x[1, 200], x[2, 383] = float("nan"), float("inf"), float("-inf")
    s = quantize_fp8(x)[1].isnan().cpu()
    want = torch.zeros(4, 3, dtype=torch.bool)
    want[0, 0] = want[1, 1] = want[2, 2] = True
    assert torch.equal(s, want)


# ------------------------------------------------------------ Fp8Linear

def linear_64(x, w, s):
    q, xs = quantize_64(f64(x))
    xv, wv = q * spread(xs, x.shape[1]), weight_64(f64(w), f64(s))
    return xv @ wv.T, np.abs(xv) @ np.abs(wv).T


LINEAR = [(1, 16, 16), (1, 4096, 2048), (2, 128, 128), (3, 144, 272), (16, 256, 4096), (17, 272, 1360), (33, 528, 512),
          (64, 1024, 2048), (65, 400, 144), (100, 2048, 640), (128, 256, 2000), (129, 272, 2000), (300, 528, 384),
          (257, 16, 128), (640, 768, 1040), (2600, 2064, 528)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", LINEAR)
def test_linear_matches_64_bits(T, N, K):
    w, s = make_weight((N, K), T + N + K, DEV)
    x = make_x(T, K, T, DEV)
    m = Fp8Linear(w, s)
    ref, mag = linear_64(x, w, s)
    check(m(x), ref, mag, K)
    check(m(x, out_dtype=torch.float32), ref, mag, K, f32=True)
    fp8.check_status(x.device)


@pytest.mark.gpu
def test_linear_shapes_strides_and_streams():
    w, s = make_weight((144, 272), 5, DEV)
    m = Fp8Linear(w, s)
    assert m(torch.empty(0, 272, dtype=torch.bfloat16, device=DEV)).shape == (0, 144)
    assert m(torch.empty(2, 0, 272, dtype=torch.bfloat16, device=DEV)).shape == (2, 0, 144)
    big = make_x(24, 600, 6, DEV)
    for v in (big[:, 8:280], big[:, 3:275], big[::3, :272]):
        ref, mag = linear_64(v, w, s)
        check(m(v), ref, mag, 272)
    y = m(big[:, :272].reshape(2, 3, 4, 272))
    assert y.shape == (2, 3, 4, 144)
    assert torch.equal(y.view(24, 144), m(big[:, :272]))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        z = m(big[:, :272])
    st.synchronize()
    assert torch.equal(z, y.view(24, 144))
    with pytest.raises(TypeError, match="bfloat16"):
        m(big.float()[:, :272])
    with pytest.raises(ValueError, match="features"):
        m(big)


@pytest.mark.gpu
def test_a_copied_module_has_its_own_weights():
    w, s = make_weight((144, 272), 5, DEV)
    m, x = Fp8Linear(w, s), make_x(3, 272, 1, DEV)
    y = m(x)
    c = copy.deepcopy(m)
    m.weight.view(torch.uint8).zero_()
    assert torch.equal(c(x), y) and not m(x).any()
    e = Fp8SwitchLinear(w[None].clone(), s[None])
    e.descriptor()
    assert "_descriptor" in e.__dict__ and "_descriptor" not in copy.deepcopy(e).__dict__


@pytest.mark.gpu
def test_calls_on_two_streams_do_not_meet():
    """Workspaces are each call's own: products and experts interleaved on
    two streams give what they give alone."""
    m = Fp8Linear(*make_weight((528, 1040), 5, DEV))
    glu = SwitchGLU(*(Fp8SwitchLinear(*make_weight(sh, i, DEV)) for i, sh in
                      enumerate([(8, 256, 1040), (8, 256, 1040), (8, 1040, 256)])))
    xs = [make_x(T, 1040, T, DEV) for T in (3, 40, 300, 700)]
    idx = [torch.randint(0, 8, (x.shape[0], 2), device=DEV, dtype=torch.int32) for x in xs]
    alone = [(m(x), glu(x, i)) for x, i in zip(xs, idx)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for j, (x, i) in enumerate(zip(xs, idx)):
            with torch.cuda.stream(streams[j % 2]):
                got.append((j, m(x), glu(x, i)))
    torch.cuda.synchronize()
    for j, a, b in got:
        assert torch.equal(a, alone[j][0]) and torch.equal(b, alone[j][1])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 64, 200])
def test_linear_replays_in_a_graph(T):
    w, s = make_weight((528, 1040), T, DEV)
    m = Fp8Linear(w, s)
    x = make_x(T, 1040, 1, DEV)
    m(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m(x)
    for seed in (2, 3):
        x.copy_(make_x(T, 1040, seed, DEV))
        g.replay()
        assert torch.equal(y, m(x))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 8, 200])
def test_a_non_finite_input_stays_in_its_row(T):
    w, s = make_weight((144, 272), 7, DEV)
    m = Fp8Linear(w, s)
    x = make_x(T + 2, 272, 8, DEV)
    clean = m(x)
    x[1, 150] = float("inf")
    y = m(x)
    assert y[1].isnan().all()
    keep = [i for i in range(T + 2) if i != 1]
    assert torch.equal(y[keep], clean[keep])


# ------------------------------------------------------- grouped_linear

def counts_of(kind, E, P, seed):
    g = np.random.default_rng(seed)
    if kind == "uniform":
        return np.bincount(g.integers(0, E, P), minlength=E)
    if kind == "one":
        c = np.zeros(E, np.int64)
        c[E // 2] = P
        return c
    if kind == "skew":
        p = 1.0 / np.arange(1, E + 1) ** 1.2
        return np.bincount(g.choice(E, P, p=p / p.sum()), minlength=E)
    return np.zeros(E, np.int64)


def grouped_64(x, w, off):
    ref, mag = np.zeros((x.shape[0], w.shape[1])), np.zeros((x.shape[0], w.shape[1]))
    for e in range(w.shape[0]):
        a, b = off[e], off[e + 1]
        ref[a:b], mag[a:b] = x[a:b] @ w[e].T, np.abs(x[a:b]) @ np.abs(w[e]).T
    return ref, mag


GROUPED = [("uniform", 4, 1, 16, 16), ("uniform", 8, 40, 144, 272), ("skew", 16, 300, 272, 400),
           ("one", 5, 260, 128, 128), ("uniform", 128, 512, 256, 512), ("skew", 7, 900, 528, 336),
           ("uniform", 1, 129, 256, 144), ("uniform", 1024, 700, 16, 64), ("none", 6, 12, 32, 32),
           ("one", 200, 17, 720, 1360), ("skew", 3, 1500, 400, 1040),
           # several tiles a CTA, more scale blocks than accumulators
           ("uniform", 128, 600, 768, 1168), ("skew", 100, 2000, 640, 2064),
           # many rows a group: CTA pairs, the last pair half empty
           ("skew", 2, 1500, 400, 1040), ("uniform", 2, 1410, 1296, 272)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,E,P,N,K", GROUPED)
@pytest.mark.parametrize("quant", [False, True])
def test_grouped_matches_64_bits(kind, E, P, N, K, quant):
    cnt = counts_of(kind, E, P, E + P)
    lead, tail = 3, 5                                   # rows before the first and behind the last group
    off = lead + np.concatenate([[0], np.cumsum(cnt)])
    rows = int(off[-1]) + tail
    x = make_x(rows, K, P, DEV)
    offs = torch.from_numpy(off.astype(np.int32)).to(DEV)
    if quant:
        w, s = make_weight((E, N, K), N + K, DEV)
        q, xs = quantize_64(f64(x))
        ref, mag = grouped_64(q * spread(xs, K), weight_64(f64(w), f64(s)), off)
    else:
        w, s = torch.empty(E, N, K, device=DEV).normal_(0, 0.05).to(torch.bfloat16), None
        ref, mag = grouped_64(f64(x), f64(w), off)
    for dt in (torch.bfloat16, torch.float32):
        out = torch.full((rows, N), 7.0, dtype=dt, device=DEV)
        y = grouped_linear(x, w, offs, weight_scale_inv=s, out=out)
        assert y is out
        assert (out[:lead] == 7).all() and (out[int(off[-1]):] == 7).all()
        a, b = lead, int(off[-1])
        check(out[a:b], ref[a:b], mag[a:b], K, f32=dt == torch.float32)
    if a < b:
        assert torch.equal(grouped_linear(x, w, offs, weight_scale_inv=s)[a:b],
                           grouped_linear(x, w, offs, weight_scale_inv=s, out=torch.empty_like(out, dtype=torch.bfloat16))[a:b])


@pytest.mark.gpu
@pytest.mark.parametrize("P", [20, 900])
def test_grouped_offsets_are_clamped_to_the_rows(P):
    """Offsets outside [0, rows] name no row beyond the tensor."""
    w = torch.empty(3, 32, 64, device=DEV).normal_().to(torch.bfloat16)
    x = make_x(P, 64, 1, DEV)
    off = torch.tensor([-5, 7, 7, P + 1000], dtype=torch.int32, device=DEV)
    y = grouped_linear(x, w, off)
    ref, mag = grouped_64(f64(x), f64(w), [0, 7, 7, P])
    check(y, ref, mag, 64)


@pytest.mark.gpu
def test_grouped_arguments_and_graph():
    w = torch.empty(3, 32, 64, device=DEV).normal_().to(torch.bfloat16)
    off = torch.tensor([0, 10, 10, 50], dtype=torch.int32, device=DEV)
    big = make_x(50, 200, 2, DEV)
    x = big[:, 64:128]                                   # rows at a pitch
    ref, mag = grouped_64(f64(x), f64(w), [0, 10, 10, 50])
    check(grouped_linear(x, w, off), ref, mag, 64)
    assert grouped_linear(x[:0], w, off * 0).shape == (0, 32)
    for bad in (lambda: grouped_linear(x, w, off.long()), lambda: grouped_linear(x, w, off[:3]),
                lambda: grouped_linear(x[:, :48], w, off), lambda: grouped_linear(x, w[0], off),
                lambda: grouped_linear(x, w, off, out=torch.empty(50, 16, dtype=torch.bfloat16, device=DEV)),
                lambda: grouped_linear(x, w.to(torch.float8_e4m3fn), off),
                lambda: grouped_linear(x[0], w, off)):
        with pytest.raises(ValueError):
            bad()
    x = x.contiguous()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = grouped_linear(x, w, off)
    x.copy_(make_x(50, 64, 9, DEV))
    off.copy_(torch.tensor([0, 30, 31, 50]))             # another split of the rows, same graph
    g.replay()
    ref, mag = grouped_64(f64(x), f64(w), [0, 30, 31, 50])
    check(y, ref, mag, 64)


# ------------------------------------------------------ experts, modules

def bf(v):
    return torch.from_numpy(v).to(torch.bfloat16).double().numpy()


def act_64(g, kind):
    if kind == "geglu":
        return 0.5 * g * (1.0 + np.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3)))
    return g / (1.0 + np.exp(-g))


def pair_64(x, w, s):
    q, xs = quantize_64(x)
    return (q * spread(xs, x.shape[1])) @ weight_64(f64(w), f64(s)).T


def experts_64(x, idx, gate, up, down, kind="swiglu"):
    """[T, k, H] of the SwitchGLU; pairs with no such expert stay NaN."""
    T, k = idx.shape
    E = gate[0].shape[0]
    y = np.full((T * k, down[0].shape[1]), np.nan)
    flat = idx.reshape(-1)
    for e in np.unique(flat[(flat >= 0) & (flat < E)]):
        at = np.nonzero(flat == e)[0]
        g = bf(pair_64(x[at // k], gate[0][e], gate[1][e]))
        u = bf(pair_64(x[at // k], up[0][e], up[1][e]))
        y[at] = bf(pair_64(bf(bf(act_64(g, kind)) * u), down[0][e], down[1][e]))
    return y.reshape(T, k, -1)


EXPERTS = [(1, 8, 2, 256, 128), (1, 64, 8, 2048, 768), (3, 16, 4, 272, 144), (24, 16, 4, 512, 256),
           (64, 64, 8, 640, 384), (300, 8, 2, 400, 272), (700, 4, 3, 256, 144), (2100, 8, 2, 128, 128),
           (40, 200, 1, 144, 400), (60, 128, 8, 1168, 384),
           # the smallest widths, more experts a token than eight, CTA pairs
           (2, 8, 2, 16, 16), (5, 16, 9, 64, 16), (40, 40, 32, 128, 32), (900, 2, 2, 272, 144)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,H,I", EXPERTS)
def test_switch_glu_matches_64_bits(T, E, k, H, I):
    """Intermediates round to bf16 and e4m3 in both; the float32 sums now and
    then round to a neighbour there, which the layer bar of conftest covers."""
    gate, up, down = make_weight((E, I, H), 1, DEV), make_weight((E, I, H), 2, DEV), make_weight((E, H, I), 3, DEV)
    kind = "geglu" if T == 24 else "swiglu"
    glu = SwitchGLU(*(Fp8SwitchLinear(*w) for w in (gate, up, down)), activation=GeGLU() if kind == "geglu" else None)
    x = make_x(T, H, T, DEV)
    rng = np.random.default_rng(T)
    idx = np.stack([rng.choice(E, k, replace=False) for _ in range(T)]).astype(np.int32)
    y = glu(x, torch.from_numpy(idx).to(DEV))
    assert y.shape == (T, k, H)
    ref = experts_64(f64(x), idx, gate, up, down, kind)
    assert_bf16_close(to_np(y), ref, f"fp8 glu T{T} E{E} k{k} H{H} I{I}")


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 4, 256, 128), (50, 8, 2, 400, 144), (700, 4, 2, 272, 256),
                                       (1500, 4, 2, 272, 256)])
def test_weighted_experts_match_64_bits(T, E, k, H, I):
    """Gemma-4's `Experts` in the format: bf16(y * w) a pair, summed over the
    slots in float32 and rounded once."""
    gate, up, down = make_weight((E, I, H), 4, DEV), make_weight((E, I, H), 5, DEV), make_weight((E, H, I), 6, DEV)
    m = gemma4.Experts(SwitchGLU(*(Fp8SwitchLinear(*w) for w in (gate, up, down)), activation=GeGLU()))
    x = make_x(T, H, T, DEV)
    rng = np.random.default_rng(T)
    idx = np.stack([rng.choice(E, k, replace=False) for _ in range(T)]).astype(np.int32)
    w = bf(rng.random((T, k)) + 0.1)
    out = m(x, torch.from_numpy(idx).to(DEV), torch.from_numpy(w).to(torch.bfloat16).to(DEV))
    ref = R.combine(experts_64(f64(x), idx, gate, up, down, "geglu"), w)
    assert_bf16_close(to_np(out), ref, f"fp8 weighted experts T{T}")


@pytest.mark.gpu
def test_pairs_of_no_expert_change_nothing_else():
    E, k, H, I = 8, 2, 256, 128
    gate, up, down = make_weight((E, I, H), 1, DEV), make_weight((E, I, H), 2, DEV), make_weight((E, H, I), 3, DEV)
    glu = SwitchGLU(*(Fp8SwitchLinear(*w) for w in (gate, up, down)))
    for T in (5, 400):
        x = make_x(T, H, T, DEV)
        idx = np.random.default_rng(T).integers(0, E, (T, k)).astype(np.int32)
        whole = glu(x, torch.from_numpy(idx).to(DEV))
        idx[1, 0], idx[2, 1], idx[4] = -1, E, (-7, 1 << 30)
        y = glu(x, torch.from_numpy(idx).to(DEV))
        ok = torch.from_numpy((idx >= 0) & (idx < E)).to(DEV)
        assert torch.equal(y[ok], whole[ok])
        allbad = torch.full((T, k), -1, dtype=torch.int32, device=DEV)
        glu(x, allbad)
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,per_pair", [(1, 2, False), (9, 4, False), (33, 4, True), (400, 2, False), (260, 2, True)])
def test_switch_linear_matches_64_bits(T, k, per_pair):
    E, N, K = 6, 272, 400
    w, s = make_weight((E, N, K), 4, DEV)
    m = Fp8SwitchLinear(w, s)
    idx = np.random.default_rng(T).integers(0, E, (T, k)).astype(np.int32)
    x = make_x(T * k if per_pair else T, K, T, DEV)
    xin = x.view(T, k, 1, K) if per_pair else x.view(T, 1, 1, K)
    y = m(xin, torch.from_numpy(idx).to(DEV)).reshape(T * k, N)
    q, xs = quantize_64(f64(x))
    xv = q * spread(xs, K)
    wv = weight_64(f64(w), f64(s))
    rows = np.arange(T * k) if per_pair else np.arange(T * k) // k
    flat = idx.reshape(-1)
    ref = np.stack([wv[e] @ xv[r] for e, r in zip(flat, rows)])
    mag = np.stack([np.abs(wv[e]) @ np.abs(xv[r]) for e, r in zip(flat, rows)])
    check(y, ref, mag, K)


@pytest.mark.gpu
@pytest.mark.parametrize("T,shared", [(1, 0), (16, 256), (600, 256)])
def test_block_from_weights(T, shared):
    """SparseMoeBlock in the format, against the oracle's router, shared
    expert and combine around the 64-bit experts."""
    cfg = synth.MoEConfig("fp8", 16, 4, 512, 256, shared, T, router="uniform", quant="fp8")
    w = synth.make_weights(cfg, seed=11)
    blk = SparseMoeBlock.from_weights({n: t.to(DEV) for n, t in w.items()}, cfg.top_k)
    assert isinstance(blk.switch_mlp.gate_proj, Fp8SwitchLinear)
    x = synth.make_input(cfg, seed=3)
    y = blk(x.to(DEV))
    blk.check_status()
    assert torch.equal(blk(x.to(DEV)), y)
    xn = to_np(x)
    inds, scores, _ = R.router(xn, to_np(w["mlp.gate.weight"]), cfg.top_k)
    sw = [(w[f"mlp.switch_mlp.{n}_proj.weight"], w[f"mlp.switch_mlp.{n}_proj.weight_scale_inv"])
          for n in ("gate", "up", "down")]
    ref = R.combine(experts_64(f64(x), inds, *sw), scores)
    if shared:
        p = {n: to_np(w["mlp." + n + ".weight"]) for n in
             ("shared_expert_gate", "shared_expert.up_proj", "shared_expert.gate_proj", "shared_expert.down_proj")}
        ref = R.bf16(ref.astype(np.float64) + R.shared_expert(xn, *p.values()))
    assert_bf16_close(to_np(y), ref, f"fp8 block T{T}")


@pytest.mark.gpu
def test_quantize_product_and_experts_together():
    """The set as a model uses it: a projection in the format, the block
    after it, and a float32 head, eagerly and replayed from one graph."""
    cfg = synth.MoEConfig("fp8", 16, 4, 512, 256, 256, 24, router="uniform", quant="fp8")
    w = {n: t.to(DEV) for n, t in synth.make_weights(cfg, seed=5).items()}
    blk = SparseMoeBlock.from_weights(w, cfg.top_k)
    proj, head = Fp8Linear(*make_weight((512, 512), 6, DEV)), Fp8Linear(*make_weight((1040, 512), 7, DEV))
    x = make_x(24, 512, 1, DEV)

    def step():
        return head(blk(proj(x)), out_dtype=torch.float32)
    a = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    g.replay()
    assert torch.equal(y, a)
    x.copy_(make_x(24, 512, 2, DEV))
    g.replay()
    assert torch.equal(y, step()) and not torch.equal(y, a)
    ref, mag = linear_64(blk(proj(x)), head.weight, head.weight_scale_inv)
    check(y, ref, mag, 512, f32=True)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2])
def test_tensor_split_cuts(n):
    """The ranks' cuts of a block, their partials summed in float32 and
    rounded once. Each rank rounds its expert outputs and its partial to bf16
    before the sum, so the reference makes the same cuts (the unsplit block
    rounds a pair's whole output once instead: up to n + 1 half steps of the
    partials away, which cancel to many steps of a small output)."""
    cfg = synth.MoEConfig("fp8", 8, 2, 256, 512, 0, 20, router="uniform", quant="fp8")
    w = {k: t.to(DEV) for k, t in synth.make_weights(cfg, seed=9).items()}
    x = synth.make_input(cfg, seed=2).to(DEV)
    inds, scores, _ = R.router(to_np(x), to_np(w["mlp.gate.weight"]), cfg.top_k)
    part, ref = torch.zeros(20, 256, device=DEV), np.zeros((20, 256))
    for r in range(n):
        cut = tensor_split.shard_state_dict(w, r, n)
        blk = SparseMoeBlock.from_weights(cut, cfg.top_k)
        out = torch.empty(20, 256, dtype=torch.float32, device=DEV)
        part += blk.forward_into(x, out)
        sw = [(cut[f"mlp.switch_mlp.{m}_proj.weight"], cut[f"mlp.switch_mlp.{m}_proj.weight_scale_inv"])
              for m in ("gate", "up", "down")]
        ref += R.combine(experts_64(f64(x), inds, *sw), scores)
    assert_bf16_close(to_np(part.to(torch.bfloat16)), R.bf16(ref), "fp8 tensor split")
