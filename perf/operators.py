"""The 8-bit and ragged matrix products of the expert layer, as measured work.

Four operators, each in its plain form (elementary torch operations in 32
bits, rounded once at the end) and, where `own` is set, through the package's
public entry points:

* quantize: a bfloat16 row in groups of 128 -> e4m3 values and one float32
  scale a group: with a the largest |x| (at least 2^-100), s = a / 448 and
  q = e4m3(448 x / a);
* linear: y = x W^T with W in e4m3 and one float32 scale for each 128 x 128
  block (`weight`, `weight_scale_inv` of a block-scaled checkpoint), the
  rows of x quantized as above on the way in;
* grouped: rows in expert order, ragged counts (device offsets), bfloat16
  weights [E, N, K]: y[r] = x[r] W[e]^T for the rows of expert e;
* experts: a SwitchGLU whose three expert linears are e4m3 with block scales.
"""
import math

import torch

own = False

GROUP = 128
LARGEST_FLOPS = 2.0 * 8192 * 8192 * 4096


# ------------------------------------------------------------------ cases

def listed():
    return [
        # the inputs of one decode / draft-verify step of the 2048-wide layer
        {"name": "quantize decode", "op": "quantize", "rows": 64, "cols": 2048},
        # a prompt's hidden states, 4096 wide
        {"name": "quantize prompt", "op": "quantize", "rows": 8192, "cols": 4096},
        # the attention's output projection for a single sequence's next token
        {"name": "linear one token", "op": "linear", "rows": 1, "n": 4096, "k": 4096},
        # queries and output gates of 32 sequences with 3 drafts each
        {"name": "linear verify", "op": "linear", "rows": 128, "n": 8192, "k": 4096},
        # sizes that divide into neither tiles nor scale blocks
        {"name": "linear ragged", "op": "linear", "rows": 1001, "n": 1488, "k": 2000},
        # queries and output gates of an 8192-token prompt
        {"name": "linear prompt", "op": "linear", "rows": 8192, "n": 8192, "k": 4096},
        # 64 decode tokens, top-8 of 128 experts: about four rows an expert
        {"name": "grouped decode", "op": "grouped", "rows": 512, "e": 128, "n": 768, "k": 2048, "zipf": 0.0},
        # few rows over many experts with odd widths: most experts have none
        {"name": "grouped odd", "op": "grouped", "rows": 77, "e": 200, "n": 720, "k": 1360, "zipf": 1.1},
        # a 4096-token prompt, top-8, expert popularity by Zipf's law
        {"name": "grouped prompt", "op": "grouped", "rows": 32768, "e": 128, "n": 768, "k": 2048, "zipf": 1.1},
        # one sequence's next token through the experts
        {"name": "experts one token", "op": "experts", "rows": 1, "e": 128, "top": 8, "h": 2048, "i": 768, "zipf": 0.0},
        # 16 sequences x (1 + 3 drafts)
        {"name": "experts verify", "op": "experts", "rows": 64, "e": 128, "top": 8, "h": 2048, "i": 768, "zipf": 0.0},
        # a 4096-token prompt through the experts
        {"name": "experts prompt", "op": "experts", "rows": 4096, "e": 128, "top": 8, "h": 2048, "i": 768, "zipf": 1.1},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "grouped", "grouped", "experts", "experts"])
    while True:
        if op == "quantize":
            case = {"op": op, "rows": _log(rng, 1, 8192), "cols": _log(rng, 128, 4096, 16)}
        elif op == "linear":
            case = {"op": op, "rows": _log(rng, 1, 8192), "n": _log(rng, 256, 8192, 16), "k": _log(rng, 256, 8192, 16)}
        elif op == "grouped":
            case = {"op": op, "rows": _log(rng, 1, 32768), "e": _log(rng, 4, 256), "n": _log(rng, 256, 2048, 16),
                    "k": _log(rng, 256, 4096, 16), "zipf": rng.choice([0.0, 0.6, 1.1])}
        else:
            e = _log(rng, 8, 256)
            case = {"op": op, "rows": _log(rng, 1, 4096), "e": e, "top": rng.randint(1, min(8, e)),
                    "h": _log(rng, 256, 4096, 16), "i": _log(rng, 128, 1536, 16), "zipf": rng.choice([0.0, 0.6, 1.1])}
        if _plain_flops(case) <= LARGEST_FLOPS and _weight_values(case) <= 128 * 3 * 768 * 2048:
            return case


def _weight_values(c):
    return {"quantize": lambda: 0, "linear": lambda: c["n"] * c["k"], "grouped": lambda: c["e"] * c["n"] * c["k"],
            "experts": lambda: 3 * c["e"] * c["h"] * c["i"]}[c["op"]]()


def _block(pairs, e):
    """Rows of one block of the plain grouped product: near the mean count."""
    b = 8
    while b < 128 and b * e < pairs:
        b *= 2
    return b


def _blocks(pairs, e):
    """A bound on the row blocks of `pairs` rows in `e` groups."""
    return min(pairs, pairs // _block(pairs, e) + e)


def _plain_flops(c):
    if c["op"] == "quantize":
        return 0.0
    if c["op"] == "linear":
        return 2.0 * c["rows"] * c["n"] * c["k"]
    pairs = c["rows"] * c.get("top", 1)
    rows = _blocks(pairs, c["e"]) * _block(pairs, c["e"])
    return 2.0 * rows * (c["n"] * c["k"] if c["op"] == "grouped" else 3 * c["h"] * c["i"])


def _touched(rows, e, zipf, top=1):
    """Expected number of experts that receive a row."""
    p = [(i + 1.0) ** -zipf for i in range(e)]
    s = sum(p)
    return sum(1.0 - max(0.0, 1.0 - min(1.0, top * v / s)) ** rows for v in p)


def work(case):
    c = case
    op = c["op"]
    if op == "quantize":
        n = c["rows"] * c["cols"]
        return {"bytes": 3.0 * n + 4.0 * c["rows"] * -(-c["cols"] // GROUP), "flops": 0.0}
    if op == "linear":
        m, n, k = c["rows"], c["n"], c["k"]
        return {"bytes": 2.0 * m * k + n * k + 4.0 * -(-n // GROUP) * -(-k // GROUP) + 2.0 * m * n,
                "flops": 2.0 * m * n * k}
    if op == "grouped":
        m, n, k = c["rows"], c["n"], c["k"]
        return {"bytes": 2.0 * m * k + 2.0 * n * k * _touched(m, c["e"], c["zipf"]) + 2.0 * m * n,
                "flops": 2.0 * m * n * k}
    m, h, i = c["rows"], c["h"], c["i"]
    pairs = m * c["top"]
    return {"bytes": 2.0 * m * h + 3.0 * h * i * _touched(m, c["e"], c["zipf"], c["top"]) + 2.0 * pairs * h + 4.0 * pairs,
            "flops": 6.0 * pairs * h * i}


# ----------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(rows, cols, g):
    """Hidden states: channels of unlike size, a few of them outliers, and
    tokens of unlike size."""
    ch = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    ch = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.004, 20.0 * ch, ch)
    tok = torch.exp(0.3 * torch.randn(rows, 1, generator=g, device="cuda"))
    return (torch.randn(rows, cols, generator=g, device="cuda") * ch * tok).to(torch.bfloat16)


def _fp8_weight(shape, g):
    """e4m3 weights near the type's range and a scale for each 128 x 128
    block, as a block-quantized checkpoint of N(0, 0.02) weights has."""
    w = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    flat = w.view(-1)
    piece = 1 << 26
    for at in range(0, flat.numel(), piece):
        n = min(piece, flat.numel() - at)
        flat[at:at + n] = (torch.randn(n, generator=g, device="cuda") * 110.0).clamp_(-448.0, 448.0).to(w.dtype)
    sshape = (*shape[:-2], -(-shape[-2] // GROUP), -(-shape[-1] // GROUP))
    return w, (0.7 + 0.6 * torch.rand(sshape, generator=g, device="cuda")) * (0.02 / 110.0)


def _popularity(e, zipf, g):
    p = (torch.arange(1, e + 1, device="cuda", dtype=torch.float32)) ** -zipf
    return p[torch.randperm(e, generator=g, device="cuda")]


def prepare(case, seed):
    c, g = case, _gen(seed)
    op = c["op"]
    if op == "quantize":
        return {"op": op, "x": _activations(c["rows"], c["cols"], g)}
    if op == "linear":
        w, s = _fp8_weight((c["n"], c["k"]), g)
        st = {"op": op, "x": _activations(c["rows"], c["k"], g), "w": w, "s": s}
        if own:
            from knurlogic_b200 import Fp8Linear
            st["module"] = Fp8Linear(w, s)
        return st
    p = _popularity(c["e"], c["zipf"], g)
    if op == "grouped":
        w = (torch.randn(c["e"], c["n"], c["k"], generator=g, device="cuda") * 0.02).to(torch.bfloat16)
        ids = torch.multinomial(p, c["rows"], replacement=True, generator=g)
        off = torch.zeros(c["e"] + 1, dtype=torch.int32, device="cuda")
        off[1:] = torch.bincount(ids, minlength=c["e"]).cumsum(0).to(torch.int32)
        return {"op": op, "x": _activations(c["rows"], c["k"], g), "w": w, "off": off}
    e, h, i = c["e"], c["h"], c["i"]
    st = {"op": op, "x": _activations(c["rows"], h, g)}
    st["gate"], st["up"], st["down"] = (_fp8_weight((e, i, h), g), _fp8_weight((e, i, h), g), _fp8_weight((e, h, i), g))
    st["idx"] = torch.multinomial(p.expand(c["rows"], e), c["top"], generator=g).to(torch.int32)
    if own:
        from knurlogic_b200 import Fp8SwitchLinear, SwitchGLU
        st["module"] = SwitchGLU(*(Fp8SwitchLinear(*st[n]) for n in ("gate", "up", "down")))
    return st


# ------------------------------------------------------------- plain form

def _pad(t, dim):
    """`t` with zeros up to a multiple of the group along `dim`."""
    n = -t.shape[dim] % GROUP
    if not n:
        return t
    shape = list(t.shape)
    shape[dim] = n
    return torch.cat([t, torch.zeros(shape, dtype=t.dtype, device=t.device)], dim)


def _quantize(x):
    """(q e4m3 [rows, cols], scales float32 [rows, groups]). The quotients
    are often exactly half way between two e4m3 values (both are ratios of
    8-bit numbers): in 64 bits, so that none falls to the wrong side."""
    rows, cols = x.shape
    v = _pad(x.double(), 1).view(rows, -1, GROUP)
    a = v.abs().amax(-1).clamp_min(2.0 ** -100)
    q = (v * 448.0 / a[..., None]).to(torch.float8_e4m3fn)
    return q.view(rows, -1)[:, :cols], (a / 448.0).float()


def _values(q, s):
    """What quantized rows stand for, float32."""
    return q.float() * s.repeat_interleave(GROUP, 1)[:, :q.shape[1]]


def _weight_values_of(w, s):
    """What block-scaled weights [..., n, k] stand for, float32."""
    n, k = w.shape[-2:]
    full = s.repeat_interleave(GROUP, -2)[..., :n, :].repeat_interleave(GROUP, -1)[..., :k]
    return w.float() * full


def _grouped(x, weights, off, e):
    """y[r] = x[r] . weights(e)^T for row r of group e: the rows cut into
    blocks of one group each, one batched product over the blocks."""
    rows, k = x.shape
    b = _block(rows, e)
    nb = _blocks(rows, e)
    off = off.long()
    per = (off[1:] - off[:-1] + b - 1) // b
    last = per.cumsum(0)
    blk = torch.arange(nb, device=x.device)
    g = torch.searchsorted(last, blk, right=True).clamp_max(e - 1)
    at = (off[g] + (blk - (last - per)[g]) * b)[:, None] + torch.arange(b, device=x.device)
    ok = (at < off[g + 1][:, None]) & (blk < last[-1])[:, None]
    xb = x[at.clamp(0, rows - 1)] * ok[..., None]
    yb = torch.bmm(xb, weights(g).transpose(1, 2))
    y = torch.zeros((rows + 1, yb.shape[-1]), device=x.device)
    y[torch.where(ok, at, rows)] = yb
    return y[:rows]


def _plain(st):
    op, x = st["op"], st["x"]
    if op == "quantize":
        return _quantize(x)
    if op == "linear":
        return (_values(*_quantize(x)) @ _weight_values_of(st["w"], st["s"]).T).to(torch.bfloat16)
    if op == "grouped":
        w = st["w"]
        return _grouped(x.float(), lambda g: w[g].float(), st["off"], w.shape[0]).to(torch.bfloat16)
    idx = st["idx"]
    top, e = idx.shape[1], st["gate"][0].shape[0]
    ids, order = idx.reshape(-1).long().sort(stable=True)
    off = torch.searchsorted(ids, torch.arange(e + 1, device=x.device))
    xs = _values(*_quantize(x))[order // top]

    def expert(name):
        w, s = st[name]
        return lambda g: _weight_values_of(w.view(torch.uint8)[g].view(w.dtype), s[g])

    gate, up = (_grouped(xs, expert(n), off, e).to(torch.bfloat16).float() for n in ("gate", "up"))
    act = (gate / (1.0 + torch.exp(-gate))).to(torch.bfloat16).float() * up
    y = _grouped(_values(*_quantize(act.to(torch.bfloat16))), expert("down"), off, e).to(torch.bfloat16)
    out = torch.empty_like(y)
    out[order] = y
    return out.view(x.shape[0], top, -1)


def run(state):
    if not own:
        return _plain(state)
    import knurlogic_b200 as kb
    op = state["op"]
    if op == "quantize":
        return kb.quantize_fp8(state["x"])
    if op == "linear":
        return state["module"](state["x"])
    if op == "grouped":
        return kb.grouped_linear(state["x"], state["w"], state["off"])
    return state["module"](state["x"], state["idx"])


# -------------------------------------------------------- in 64 bits, apart

def _e4m3(v):
    """The e4m3 value nearest to each float64 (ties to the even one), |v| up
    to 448: steps of 2^-9 below 2^-6, of an eighth of the power of two above."""
    a = v.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3.0)
    return torch.sign(v) * (torch.round(a / step) * step).clamp_max(448.0)


def _rows64(x):
    """(e4m3 values, scales) of rows in float64."""
    rows, cols = x.shape
    q = torch.zeros((rows, cols), dtype=torch.float64, device=x.device)
    s = torch.zeros((rows, -(-cols // GROUP)), dtype=torch.float64, device=x.device)
    for j in range(s.shape[1]):
        v = x[:, j * GROUP:(j + 1) * GROUP].double()
        a = v.abs().max(1).values.clamp_min(2.0 ** -100)
        s[:, j] = a / 448.0
        q[:, j * GROUP:(j + 1) * GROUP] = _e4m3(448.0 * v / a[:, None])
    return q, s


def _product64(q, s, w, ws):
    """sum over scale groups of s . ws . (q . w^T)."""
    n = w.shape[0]
    y = torch.zeros((q.shape[0], n), dtype=torch.float64, device=q.device)
    for j in range(s.shape[1]):
        part = q[:, j * GROUP:(j + 1) * GROUP] @ w[:, j * GROUP:(j + 1) * GROUP].double().T
        y += part * s[:, j:j + 1] * ws[:, j].double().repeat_interleave(GROUP)[:n]
    return y


def exact(case, seed):
    st = prepare(case, seed)
    op, x = case["op"], st["x"]
    if op == "quantize":
        q, s = _rows64(x)
        return q.to(torch.float8_e4m3fn), s
    if op == "linear":
        return _product64(*_rows64(x), st["w"], st["s"])
    if op == "grouped":
        off = st["off"].tolist()
        return torch.cat([x[a:b].double() @ w.double().T for a, b, w in zip(off, off[1:], st["w"])])
    idx = st["idx"]
    top = idx.shape[1]
    flat = idx.reshape(-1)
    y = torch.zeros((flat.numel(), case["h"]), dtype=torch.float64, device=x.device)
    q, s = _rows64(x)

    def bf(v):
        return v.to(torch.bfloat16).double()

    for e in flat.unique().tolist():
        at = (flat == e).nonzero().view(-1)
        gate, up = (bf(_product64(q[at // top], s[at // top], st[n][0][e], st[n][1][e])) for n in ("gate", "up"))
        act = bf(bf(gate * torch.sigmoid(gate)) * up)
        y[at] = _product64(*_rows64(act), st["down"][0][e], st["down"][1][e])
    return y.view(x.shape[0], top, -1)
