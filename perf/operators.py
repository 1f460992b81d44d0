"""Operators of large language models that the library offers, through its public entry points: the way of a hidden state to a token with
8-bit products.

Four kinds: root-mean-square norm of the residual stream with its 8-bit output (``norm``), a matrix or a gated pair brought into 8 bits
(``quantize``), InnerProduct of 8-bit operands (``product``) and the draw of a token from its logits (``sample``).  8 bits are e4m3 with
an fp32 scale for each block: 128 consecutive columns of one row (activations; scales stored [block][row]) or 128 x 128 (weights;
[row block][column block]).  Every input is made on the GPU from a seed: hidden states ~ N(0, 1) with a few columns that are far larger
than the rest, as residual streams have them; weights ~ N(0, 1/inputs); logits ~ N(0, 2.5) with a few high ones and masked ones.  The
library is forward only.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BLOCK = 128


def listed():
    return [
        # the norm between two layers for one new token: all latency
        dict(name="norm_1x4096", kind="norm", rows=1, cols=4096, type="bf16", out="e4m3", residual=True),
        # the same for a batch of prompts: all bandwidth
        dict(name="norm_8192x5120", kind="norm", rows=8192, cols=5120, type="bf16", out="e4m3", residual=True),
        # the gated activation between the two products of a feed-forward layer, one token
        dict(name="quantize_silu_1x12288", kind="quantize", rows=1, cols=12288, type="bf16", gate="silu", block_rows=1),
        # the same for a batch of prompts
        dict(name="quantize_silu_8192x12288", kind="quantize", rows=8192, cols=12288, type="bf16", gate="silu", block_rows=1),
        # a layer's weights as they are brought into 8 bits at start-up, a last block of rows that is not full
        dict(name="quantize_weights_11000x4096", kind="quantize", rows=11000, cols=4096, type="bf16", gate="none", block_rows=128),
        # one token through a square projection: reads the weights once
        dict(name="product_1x4096x4096", kind="product", rows=1, inputs=4096, outputs=4096, out="bf16", bias=False, act="identity"),
        # a batch of tokens being generated, through the first product of a feed-forward layer
        dict(name="product_48x4096x24576", kind="product", rows=48, inputs=4096, outputs=24576, out="bf16", bias=False, act="identity"),
        # a short prompt through a layer whose sizes are no multiple of anything, with bias and activation, fp32 out
        dict(name="product_517x5000x7100", kind="product", rows=517, inputs=5000, outputs=7100, out="fp32", bias=True, act="relu"),
        # prompts through the first product of a feed-forward layer: the largest case
        dict(name="product_8192x4096x24576", kind="product", rows=8192, inputs=4096, outputs=24576, out="bf16", bias=False, act="identity"),
        # one request's next token, a short list of candidates
        dict(name="sample_1x32000_k50", kind="sample", rows=1, classes=32000, type="fp32", top_k=True, top_p=True, min_p=False),
        # a batch of requests by probability mass alone, logits of 16 bits with many equal values
        dict(name="sample_64x128000_p", kind="sample", rows=64, classes=128000, type="bf16", top_k=False, top_p=True, min_p=False),
        # a large batch where every row has settings of its own, an odd number of classes
        dict(name="sample_256x150001_mixed", kind="sample", rows=256, classes=150001, type="fp32", top_k=True, top_p=True, min_p=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "product", "product", "sample", "sample"])
    if kind == "norm":
        cols = _log_int(rng, 64, 16384)
        rows = _log_int(rng, 1, min(16384, 8192 * 5120 // 2 // cols))
        return dict(kind=kind, rows=rows, cols=cols, type=rng.choice(["bf16", "fp16", "fp32"]), out=rng.choice(["e4m3", "e4m3", "bf16", "fp16", "fp32"]),
                    residual=rng.random() < 0.7)
    if kind == "quantize":
        cols = _log_int(rng, 64, 16384)
        rows = _log_int(rng, 1, min(16384, 8192 * 12288 // 4 // cols))
        gate = rng.choice(["none", "silu", "silu", "gelu"])
        return dict(kind=kind, rows=rows, cols=cols, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), gate=gate,
                    block_rows=128 if gate == "none" and rng.random() < 0.5 else 1)
    if kind == "product":
        inputs, outputs = _log_int(rng, 128, 16384), _log_int(rng, 64, 28672)
        rows = _log_int(rng, 1, max(1, min(8192, 8192 * 4096 * 12288 // (inputs * outputs))))
        return dict(kind=kind, rows=rows, inputs=inputs, outputs=outputs, out=rng.choice(["bf16", "bf16", "fp16", "fp32"]), bias=rng.random() < 0.3,
                    act=rng.choice(["identity", "identity", "relu", "sigmoid"]))
    return dict(kind=kind, rows=_log_int(rng, 1, 128), classes=_log_int(rng, 500, 262144), type=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                top_k=rng.random() < 0.5, top_p=rng.random() < 0.6, min_p=rng.random() < 0.3)


# ---- the 8-bit form ---------------------------------------------------------------------------------------------------------------
def _blocks(v, block_rows):
    """v [rows, cols], padded with zeros, as [row blocks, block_rows, column blocks, 128]."""
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % BLOCK, 0, -rows % block_rows))
    return v.reshape(v.shape[0] // block_rows, block_rows, v.shape[1] // BLOCK, BLOCK)


def _to_8_bits(v, block_rows):
    """(values in e4m3, scales) of an fp32 matrix."""
    rows, cols = v.shape
    b = _blocks(v, block_rows)
    scales = (b.abs().amax((1, 3)) / 448).clamp_min(2.0 ** -126)
    q = (b / scales[:, None, :, None]).to(torch.float8_e4m3fn)
    q = q.reshape(b.shape[0] * block_rows, -1)[:rows, :cols]
    return q, (scales.t().contiguous() if block_rows == 1 else scales)


def _rows_of(rows, cols, dtype, device="cuda"):
    """An empty matrix whose rows start on 16-byte boundaries, as 8-bit matrices have to."""
    return torch.empty(rows, -(-cols // 16) * 16, dtype=dtype, device=device)[:, :cols]


def _hidden(rows, cols, g):
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x[:, torch.randint(0, cols, (max(1, cols // 500),), device="cuda", generator=g)] *= 20
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "norm":
        rows, cols, t = case["rows"], case["cols"], TYPES[case["type"]]
        s["x"] = _hidden(rows, cols, g).to(t)
        s["r"] = (3 * _hidden(rows, cols, g)).to(t) if case["residual"] else None
        s["w"] = (1 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(t)
        s["total"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["y"] = _rows_of(rows, cols, TYPES[case["out"]])
        s["scales"] = torch.empty(-(-cols // BLOCK), rows, device="cuda") if case["out"] == "e4m3" else None
    elif case["kind"] == "quantize":
        rows, cols, t, br = case["rows"], case["cols"], TYPES[case["type"]], case["block_rows"]
        s["x"] = (2 * _hidden(rows, cols * (1 if case["gate"] == "none" else 2), g)).to(t)
        s["q"] = _rows_of(rows, cols, torch.float8_e4m3fn)
        blocks = -(-cols // BLOCK)
        s["scales"] = torch.empty((blocks, rows) if br == 1 else (-(-rows // br), blocks), device="cuda")
    elif case["kind"] == "product":
        rows, k, n = case["rows"], case["inputs"], case["outputs"]
        for name, count, block_rows, scale in (("x", rows, 1, 1.0), ("w", n, BLOCK, k ** -0.5)):
            q, s[name + "_scales"] = _to_8_bits(scale * _hidden(count, k, g), block_rows)
            s[name] = _rows_of(count, k, torch.float8_e4m3fn)
            s[name].copy_(q)
        s["b"] = torch.rand(n, device="cuda", generator=g) - 0.5 if case["bias"] else None
        s["y"] = torch.empty(rows, n, dtype=TYPES[case["out"]], device="cuda")
    else:
        rows, n = case["rows"], case["classes"]
        x = 2.5 * torch.randn(rows, n, device="cuda", generator=g)
        x[:, torch.randint(0, n, (8,), device="cuda", generator=g)] += 9
        x[torch.rand(rows, n, device="cuda", generator=g) < 0.02] = -math.inf
        s["x"] = x.to(TYPES[case["type"]])
        u = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, device="cuda", generator=g)    # noqa: E731
        s["u"] = u(0.0, 1.0)
        # some rows greedy, some with a setting switched off
        s["temperature"] = torch.where(u(0, 1) < 0.1, torch.zeros(rows, device="cuda"), u(0.5, 1.3))
        s["k"] = torch.where(u(0, 1) < 0.2, torch.zeros(rows, device="cuda"), u(1, 200)).int() if case["top_k"] else None
        s["p"] = torch.where(u(0, 1) < 0.2, torch.ones(rows, device="cuda"), u(0.3, 0.99)) if case["top_p"] else None
        s["m"] = torch.where(u(0, 1) < 0.2, torch.zeros(rows, device="cuda"), u(0.001, 0.2)) if case["min_p"] else None
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------------
def run(s):
    kind = s["kind"]
    if own:
        from dlprimitives_b200 import capi
        if kind == "norm":
            capi.rms_norm(s["x"], s["w"], s["y"], residual=s["r"], total=s["total"], scales=s["scales"], eps=1e-6)
            return [t for t in (s["y"], s["scales"], s["total"]) if t is not None]
        if kind == "quantize":
            capi.quantize(s["x"], s["q"], s["scales"], gate=s["gate"], block_rows=s["block_rows"])
            return s["q"], s["scales"]
        if kind == "product":
            capi.scaled_inner_product(s["x"], s["x_scales"], s["w"], s["w_scales"], s["y"], bias=s["b"], activation=s["act"])
            return s["y"]
        capi.sample(s["x"], s["u"], s["tokens"], temperature=s["temperature"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
        return s["tokens"]
    return {"norm": _norm, "quantize": _quantize, "product": _product, "sample": _sample}[kind](s)


def _norm(s):
    h = s["x"].float()
    if s["r"] is not None:
        h = h + s["r"].float()
    v = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6) * s["w"].float()
    out = list(_to_8_bits(v, 1)) if s["scales"] is not None else [v.to(s["y"].dtype)]
    return out + ([h.to(s["x"].dtype)] if s["r"] is not None else [])


def _quantize(s):
    v = s["x"].float()
    if s["gate"] != "none":
        a, up = v[:, :s["cols"]], v[:, s["cols"]:]
        if s["gate"] == "silu":
            v = a / (1 + torch.exp(-a)) * up
        else:
            v = 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a * a * a))) * up
    return _to_8_bits(v, s["block_rows"])


def _product(s):
    k = s["inputs"]
    x = s["x"].float() * s["x_scales"].t().repeat_interleave(BLOCK, 1)[:, :k]
    w = s["w"].float() * s["w_scales"].repeat_interleave(BLOCK, 0)[:s["outputs"]].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ w.t()
    if s["b"] is not None:
        y = y + s["b"]
    if s["act"] == "relu":
        y = y.clamp_min(0)
    elif s["act"] == "sigmoid":
        y = 1 / (1 + torch.exp(-y))
    return y.to(s["y"].dtype)


def _sample(s):
    """In 64 bits: masses next to a border decide which token it is."""
    x = s["x"].double()
    rows, n = x.shape
    top = x.amax(1, keepdim=True)
    t = s["temperature"].double()[:, None]
    mass = torch.where(x == top, 1.0, torch.exp((x - top) / t))
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    m = mass.gather(1, order)
    rank = torch.arange(n, device=x.device)
    kept = (rank == 0) | (t > 0)
    if s["k"] is not None:
        kept = kept & ((rank < s["k"][:, None]) | (s["k"][:, None] <= 0))
    m = m * kept
    if s["p"] is not None:
        before = m.cumsum(1)
        whole = before[:, -1:].clone()
        before = torch.cat([torch.zeros_like(whole), before[:, :-1]], 1)
        p = s["p"].double()[:, None]
        m = m * ((before < p * whole) | (rank == 0) | (p >= 1))
    if s["m"] is not None:
        m = m * (m >= s["m"].double()[:, None].clamp_max(1))
    mass = torch.zeros_like(m).scatter_(1, order, m).cumsum(1)
    token = (mass <= s["u"].double()[:, None] * mass[:, -1:]).sum(1)
    return torch.where(top[:, 0] == -math.inf, -1, token).int()


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------------
def _e4m3(v):
    """v rounded to three binary places behind the leading one (ties to even), steps of 2^-9 below 2^-6; at most 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_8_bits(v, block_rows):
    rows, cols = v.shape
    tall, wide = -(-rows // block_rows), -(-cols // BLOCK)
    big = torch.zeros(tall * block_rows, wide * BLOCK, dtype=torch.float64, device=v.device)
    big[:rows, :cols] = v
    most = big.abs().view(tall, block_rows, wide * BLOCK).amax(1).view(tall, wide, BLOCK).amax(2)
    scale = torch.clamp(most / 448, min=2.0 ** -126)
    over = scale.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return [_e4m3(v / over), scale.T.clone() if block_rows == 1 else scale]


def exact(case, seed):
    s = prepare(case, seed)
    d = lambda t: t.to(torch.float64)   # noqa: E731
    if case["kind"] == "norm":
        h = d(s["x"]) + (d(s["r"]) if case["residual"] else 0)
        v = d(s["w"]) * h / torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + 1e-6)
        return (_exact_8_bits(v, 1) if case["out"] == "e4m3" else [v]) + ([h] if case["residual"] else [])
    if case["kind"] == "quantize":
        v = d(s["x"])
        if case["gate"] != "none":
            a, up = v.chunk(2, 1)
            inner = a if case["gate"] == "silu" else 2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)
            v = a * up * torch.sigmoid(inner)          # (1 + tanh(z)) / 2 is the logistic function of 2 z
        return _exact_8_bits(v, case["block_rows"])
    if case["kind"] == "product":
        k, n = case["inputs"], case["outputs"]
        y = torch.zeros(case["rows"], n, dtype=torch.float64, device="cuda")
        for b in range(-(-k // BLOCK)):
            at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            over = d(s["w_scales"][:, b]).repeat_interleave(BLOCK)[:n]
            y += (d(s["x"][:, at]) * d(s["x_scales"][b])[:, None]) @ (d(s["w"][:, at]) * over[:, None]).T
        if case["bias"]:
            y += d(s["b"])
        return {"identity": lambda v: v, "relu": torch.relu, "sigmoid": torch.sigmoid}[case["act"]](y)
    return None                                          # a token is a whole number: there is nothing between it and the next


def work(case):
    size = {"fp32": 4, "fp16": 2, "bf16": 2, "e4m3": 1}
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        scales = 4 * case["rows"] * -(-case["cols"] // BLOCK) if case["out"] == "e4m3" else 0
        read = size[case["type"]] * (2 if case["residual"] else 1)
        return {"bytes": n * (read + size[case["out"]] + (size[case["type"]] if case["residual"] else 0)) + scales + case["cols"] * size[case["type"]],
                "flops": 6 * n}
    if case["kind"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (size[case["type"]] * (1 if case["gate"] == "none" else 2) + 1) + 4 * n // BLOCK // case["block_rows"],
                "flops": (3 if case["gate"] == "none" else 12) * n}
    if case["kind"] == "product":
        r, k, n = case["rows"], case["inputs"], case["outputs"]
        scales = 4 * -(-k // BLOCK) * (r + -(-n // BLOCK))
        return {"bytes": r * k + n * k + r * n * size[case["out"]] + scales + (4 * n if case["bias"] else 0), "flops": 2 * r * k * n}
    return {"bytes": case["rows"] * (case["classes"] * size[case["type"]] + 20), "flops": 4 * case["rows"] * case["classes"]}
