"""Performance cases of the block-scaled operators of ``aeisu_amd.blocks``, over the range of sizes they serve.

* ``quantize``: rows of FP16 / BF16 values to E4M3 codes with an FP32 scale for each 128 columns
  (``quantize_rows``), as they are, gathered in the experts' order, or gated (SiLU(a) b).
* ``matmul``: E4M3 rows times E4M3 weights with a scale for each 128 x 128 tile.
* ``grouped``: rows sorted by expert times each expert's weights, in E4M3 blocks, FP16 or BF16.

``own`` false computes each in its plain form, elementary torch operations in 32 bits; ``own`` true makes the calls
that a user makes.  Codes are held as uint8 rows padded with zeros to a multiple of 128 columns, the scales of rows as
[blocks, rows], those of weights as [..., row blocks, column blocks].
"""
from __future__ import annotations

import math
import random

import torch

own = False
BLOCK, TOP = 128, 448.0
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1}


def listed():
    return [
        # the activations of eight tokens in flight, quantised ahead of a layer's product: bound by latency
        {"name": "quantize-8x4096", "op": "quantize", "rows": 8, "cols": 4096, "in": "bf16", "source": 0, "gated": False},
        # the input of the upscaler's compress layer: 488 x 280 low pixels of 128 channels, a 1080p frame
        {"name": "quantize-compress-1080p", "op": "quantize", "rows": 136640, "cols": 128, "in": "f16", "source": 0,
         "gated": False},
        # a prompt of 8,192 tokens sent to two experts each: 16,384 rows gathered in the experts' order
        {"name": "quantize-dispatch-16384", "op": "quantize", "rows": 16384, "cols": 4096, "in": "bf16", "source": 8192,
         "gated": False},
        # between an expert's two products: SiLU(a) b of an odd number of rows and a width that ends inside a block
        {"name": "quantize-gated-4099x2750", "op": "quantize", "rows": 4099, "cols": 2750, "in": "bf16", "source": 0,
         "gated": True},
        # one token through one layer: the weights are read once
        {"name": "matmul-1x4096x4096", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "out": "bf16", "bias": False,
         "slope": -1.0},
        # the upscaler's compress layer over a 1080p frame: 128 -> 64 channels, bias and LeakyReLU
        {"name": "matmul-compress-1080p", "op": "matmul", "m": 136640, "n": 64, "k": 128, "out": "f16", "bias": True,
         "slope": 0.1},
        # a short prompt with nothing a multiple of anything, FP32 results
        {"name": "matmul-333x1111x2500-f32", "op": "matmul", "m": 333, "n": 1111, "k": 2500, "out": "f32", "bias": True,
         "slope": -1.0},
        # a long prompt through a wide layer: the largest product
        {"name": "matmul-8192x10240x5120", "op": "matmul", "m": 8192, "n": 10240, "k": 5120, "out": "bf16", "bias": False,
         "slope": -1.0},
        # sixteen rows of tokens in flight over 64 experts: most experts have no row, the others one or two
        {"name": "grouped-16-of-64", "op": "grouped", "t": 16, "e": 64, "n": 2048, "k": 2048, "kind": "e4m3", "out": "bf16",
         "bias": False},
        # a long prompt over 32 experts of uneven load
        {"name": "grouped-16384-of-32", "op": "grouped", "t": 16384, "e": 32, "n": 4096, "k": 2048, "kind": "e4m3",
         "out": "bf16", "bias": False},
        # weights kept in BF16: a prompt over 16 experts
        {"name": "grouped-6000-of-16-bf16", "op": "grouped", "t": 6000, "e": 16, "n": 2816, "k": 2048, "kind": "bf16",
         "out": "bf16", "bias": False},
        # FP16 weights of odd width, few experts, bias and FP32 results
        {"name": "grouped-777-of-7-f16", "op": "grouped", "t": 777, "e": 7, "n": 515, "k": 1003, "kind": "f16", "out": "f32",
         "bias": True},
    ]


def _size(rng, low, high):
    """Over the logarithm of the range; half of them multiples of 40, the others any number."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(40, round(v / 40) * 40) if low >= 40 and rng.random() < 0.5 else round(v)


_MOST_FLOPS = 2 * 8192 * 10240 * 5120
_MOST_WEIGHTS = 64 * 2048 * 2048


def draw(rng):
    op = rng.choice(("quantize", "matmul", "matmul", "grouped", "grouped"))
    if op == "quantize":
        gated = rng.random() < 0.35
        cols = _size(rng, 64, 8192)
        rows = _size(rng, 1, min(140000, 16384 * 4096 // cols // (2 if gated else 1)))
        source = 0 if gated or rng.random() < 0.6 else _size(rng, 1, max(2, rows))
        return {"op": op, "rows": rows, "cols": cols, "in": rng.choice(("f16", "bf16")), "source": source, "gated": gated}
    if op == "matmul":
        n, k = _size(rng, 64, 10240), _size(rng, 64, 8192)
        m = _size(rng, 1, min(140000 if n * k < 1 << 16 else 8192, _MOST_FLOPS // (2 * n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(("bf16", "f16", "f32")), "bias": rng.random() < 0.4,
                "slope": rng.choice((-1.0, -1.0, 0.1))}
    e, n, k = _size(rng, 2, 64), _size(rng, 64, 4096), _size(rng, 64, 4096)
    e = max(2, min(e, _MOST_WEIGHTS // (n * k)))
    t = _size(rng, 1, 16384)
    return {"op": op, "t": t, "e": e, "n": n, "k": k, "kind": rng.choice(("e4m3", "e4m3", "bf16", "f16")),
            "out": rng.choice(("bf16", "f16", "f32")), "bias": rng.random() < 0.4}


# ---- inputs --------------------------------------------------------------------------------------------
def _blocks(cols):
    return -(-cols // BLOCK)


def _shares(e):
    """How often a row goes to each expert: uneven, and from four experts on one that is never chosen."""
    share = [1 / math.sqrt(1 + i) for i in range(e)]
    if e >= 4:
        share[e // 2] = 0.0
    return [s / sum(share) for s in share]


def _activations(rows, cols, g):
    """Normal values, each row with a scale of its own, and one channel in fifty 20 times the others."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    x *= torch.where(torch.rand(1, cols, generator=g, device="cuda") < 0.02, 20.0, 1.0)
    return x


def _weights(n, k, g):
    return torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)


def _codes(x, rows):
    """Codes and scales of a matrix for blocks of ``rows`` x 128; scales [row blocks, column blocks]."""
    n, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -n % rows))
    t = x.view(x.shape[0] // rows, rows, x.shape[1] // BLOCK, BLOCK)
    scale = (t.abs().amax((1, 3)) / TOP).clamp_min(2.0 ** -126)
    codes = (t / scale[:, None, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).view(x.shape)[:n].contiguous(), scale


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s = {"case": dict(case)}
    if case["op"] == "quantize":
        dt = DTYPE[case["in"]]
        s["x"] = _activations(case["source"] or case["rows"], case["cols"] * (2 if case["gated"] else 1), g).to(dt)
        s["rows"] = None
        if case["source"]:
            s["rows"] = torch.randint(case["source"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
        return s
    grouped = case["op"] == "grouped"
    n, k, e = case["n"], case["k"], case["e"] if grouped else 1
    m = case["t"] if grouped else case["m"]
    kind = case.get("kind", "e4m3")
    x = _activations(m, k, g)
    if kind == "e4m3":
        s["x"], scale = _codes(x, 1)
        s["x_scales"] = scale.t().contiguous()
        s["w"] = torch.empty(e, n, _blocks(k) * BLOCK, dtype=torch.uint8, device="cuda")
        s["w_scales"] = torch.empty(e, _blocks(n), _blocks(k), device="cuda")
    else:
        s["x"] = x.to(DTYPE[kind])
        s["w"] = torch.empty(e, n, k, dtype=DTYPE[kind], device="cuda")
    for i in range(e):
        w = _weights(n, k, g)
        if kind == "e4m3":
            s["w"][i], s["w_scales"][i] = _codes(w, BLOCK)
        else:
            s["w"][i] = w.to(DTYPE[kind])
    s["bias"] = torch.randn(e, n, generator=g, device="cuda") if case["bias"] else None
    if grouped:
        pick = torch.multinomial(torch.tensor(_shares(e)), m, replacement=True, generator=torch.Generator().manual_seed(seed))
        s["bounds"] = [0] + torch.bincount(pick, minlength=e).cumsum(0).tolist()     # what a plain loop goes by
        s["offsets"] = torch.tensor(s["bounds"], dtype=torch.int32, device="cuda")
    else:
        for key in ("w", "w_scales", "bias"):
            s[key] = s[key][0] if s[key] is not None else None
    return s


# ---- the plain forms -----------------------------------------------------------------------------------
def _plain_quantize(x, rows, gated):
    y = (x if rows is None else x[rows]).float()
    if gated:
        a, b = y.chunk(2, dim=1)
        y = a / (1 + torch.exp(-a)) * b
    y = torch.nn.functional.pad(y, (0, -y.shape[1] % BLOCK)).view(y.shape[0], -1, BLOCK)
    scale = (y.abs().amax(2) / TOP).clamp_min(2.0 ** -126)
    codes = (y / scale[:, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return {"codes": codes.view(y.shape[0], -1), "scales": scale.t().contiguous()}


def _plain_rows(codes, scales, cols):
    return codes.view(torch.float8_e4m3fn).float()[:, :cols] * scales.t().repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_weight(codes, scales, cols):
    n = codes.shape[0]
    wide = scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :cols]
    return codes.view(torch.float8_e4m3fn).float()[:, :cols] * wide


def _plain_finish(y, bias, slope, dtype):
    y = y if bias is None else y + bias
    return (y if slope < 0 else torch.maximum(y, slope * y)).to(dtype)


def _plain_grouped(s, case):
    k, e4m3 = case["k"], case["kind"] == "e4m3"
    x = _plain_rows(s["x"], s["x_scales"], k) if e4m3 else s["x"].float()
    out = torch.zeros(case["t"], case["n"], dtype=DTYPE[case["out"]], device="cuda")
    for e, (lo, hi) in enumerate(zip(s["bounds"], s["bounds"][1:])):      # one product for each expert that has rows
        if lo < hi:
            w = _plain_weight(s["w"][e], s["w_scales"][e], k) if e4m3 else s["w"][e].float()
            out[lo:hi] = _plain_finish(x[lo:hi] @ w.t(), None if s["bias"] is None else s["bias"][e], -1.0, out.dtype)
    return out


def run(state):
    case = state["case"]
    slope = case.get("slope", -1.0)
    if own:
        from aeisu_amd import blocks
        if case["op"] == "quantize":
            q = blocks.quantize_rows(state["x"], rows=state["rows"], gated=case["gated"])
            return {"codes": q.codes.view(torch.float8_e4m3fn), "scales": q.scales}
        x, w = state["x"], state["w"]
        if case.get("kind", "e4m3") == "e4m3":
            x, w = blocks.QuantRows(x, state["x_scales"], case["k"]), blocks.QuantWeight(w, state["w_scales"], case["k"])
        if case["op"] == "matmul":
            return blocks.matmul(x, w, bias=state["bias"], slope=None if slope < 0 else slope, out_dtype=DTYPE[case["out"]])
        return blocks.grouped_matmul(x, w, state["offsets"], bias=state["bias"], out_dtype=DTYPE[case["out"]])
    if case["op"] == "quantize":
        return _plain_quantize(state["x"], state["rows"], case["gated"])
    if case["op"] == "matmul":
        x = _plain_rows(state["x"], state["x_scales"], case["k"])
        w = _plain_weight(state["w"], state["w_scales"], case["k"])
        return _plain_finish(x @ w.t(), state["bias"], slope, DTYPE[case["out"]])
    return _plain_grouped(state, case)


# ---- what a pass cannot do without ---------------------------------------------------------------------
def work(case):
    if case["op"] == "quantize":
        r, c = case["rows"], case["cols"]
        inputs = c * (2 if case["gated"] else 1) * BYTES[case["in"]]
        seen = case["source"] * (1 - (1 - 1 / case["source"]) ** r) if case["source"] else r     # rows that are picked at all
        return {"bytes": seen * inputs + r * (c + 4 * _blocks(c)) + (4 * r if case["source"] else 0),
                "flops": r * c * (8 if case["gated"] else 3)}
    n, k = case["n"], case["k"]
    m = case["m"] if case["op"] == "matmul" else case["t"]
    kind = case.get("kind", "e4m3")
    experts = 1 if case["op"] == "matmul" else sum(1 - (1 - p) ** m for p in _shares(case["e"]))  # those with a row
    one = n * k * BYTES[kind] + (4 * _blocks(n) * _blocks(k) if kind == "e4m3" else 0) + (4 * n if case["bias"] else 0)
    rows = m * (k * BYTES[kind] + (4 * _blocks(k) if kind == "e4m3" else 0) + n * BYTES[case["out"]])
    return {"bytes": experts * one + rows, "flops": 2 * m * n * k}


# ---- the definition in 64 bits -------------------------------------------------------------------------
def _e4m3_values():
    """The value of each code: sign, four exponent bits with bias 7, three of the mantissa, no infinities."""
    table = []
    for code in range(256):
        e, f = code >> 3 & 15, code & 7
        v = math.ldexp(f, -9) if e == 0 else math.ldexp(8 + f, e - 10)
        table.append(-v if code & 128 else v)
    table[127] = table[255] = math.nan
    return torch.tensor(table, dtype=torch.float64, device="cuda")


def _nearest_e4m3(v):
    """Nearest E4M3 value of each number, ties to even, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_quantize(s, case):
    y = s["x"].double()
    if s["rows"] is not None:
        y = y.index_select(0, s["rows"].long())
    if case["gated"]:
        y = torch.sigmoid(y[:, :case["cols"]]) * y[:, :case["cols"]] * y[:, case["cols"]:]
    nb = _blocks(case["cols"])
    wide = y.new_zeros(y.shape[0], nb * BLOCK)
    wide[:, :case["cols"]] = y
    parts = wide.reshape(-1, nb, BLOCK)
    scale = torch.maximum(parts.abs().amax(-1) / TOP, parts.new_tensor(2.0 ** -126))
    return {"codes": _nearest_e4m3(parts / scale.unsqueeze(-1)).reshape(wide.shape), "scales": scale.t().contiguous()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_quantize(s, case)
    k, n = case["k"], case["n"]
    column = torch.arange(k, device="cuda") // BLOCK
    row = torch.arange(n, device="cuda") // BLOCK
    if case.get("kind", "e4m3") == "e4m3":
        values = _e4m3_values()
        x = values[s["x"][:, :k].long()] * s["x_scales"].double()[column].t()
        weight = lambda c, w: values[c[:, :k].long()] * w.double()[row][:, column]  # noqa: E731
    else:
        x = s["x"].double()
        weight = lambda c, w: c.double()  # noqa: E731
    if case["op"] == "matmul":
        y = torch.mm(x, weight(s["w"], s["w_scales"]).t().contiguous())
        y = y if s["bias"] is None else y + s["bias"].double()
        return torch.where(y < 0, y * case["slope"], y) if case["slope"] >= 0 else y
    y = x.new_zeros(case["t"], n)
    for e in range(case["e"]):
        lo, hi = s["bounds"][e], s["bounds"][e + 1]
        if hi > lo:
            y[lo:hi] = torch.mm(x[lo:hi], weight(s["w"][e], s["w_scales"][e] if "w_scales" in s else None).t().contiguous())
            if s["bias"] is not None:
                y[lo:hi] += s["bias"][e].double()
    return y
