"""Block-scaled operators on the GPU against their definition in 64 bits (tests/_blocks.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import _blocks as O

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def B(gpu):
    from aeisu_amd import blocks
    return blocks


def rng(*key):
    return np.random.default_rng(list(key))


def values(r, *shape):
    """Normal values, rows of different size, some channels 20 times the others."""
    x = r.standard_normal(shape) * np.exp(0.5 * r.standard_normal((*shape[:-1], 1)))
    return x * np.where(r.random(shape[-1]) < 0.02, 20.0, 1.0)


def tensor(a, dtype=F32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


# ---- quantisation -------------------------------------------------------------------------------------------
def check_rows(q, y, what):
    codes, scales = O.quantize(y, 1)
    assert np.array_equal(q.scales.cpu().numpy(), scales.T), what
    assert O.same_codes(q.codes.cpu().numpy(), codes), what


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 4096), (3, 127), (16, 128), (17, 129), (33, 1000), (200, 515)])
def test_quantize_rows_is_the_definition(B, m, k, dtype):
    x = tensor(values(rng(m, k), m, k), dtype)
    check_rows(B.quantize_rows(x), x.cpu().double().numpy(), (m, k, dtype))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_quantize_rows_of_views(B, dtype):
    """Rows at odd addresses, a row stride, an offset; codes and scales of the tensor they are cut from stay."""
    big = tensor(values(rng(5), 40, 701), dtype)
    for view in (big[3:29, 5:5 + 300], big[::2, 1:130], big[:, 700:], big.t()[:0].t()[:, :0]):
        check_rows(B.quantize_rows(view), view.cpu().double().numpy(), view.shape)


def test_quantize_rows_extreme_values(B):
    """Zero rows, denormals, the type's largest and smallest, scales at their floor, values that tie, infinities and NaN."""
    r = rng(6)
    x = values(r, 24, 300).astype(np.float32)
    x[0] = 0
    x[1] *= 1e-42
    x[2] = 3.4e38
    x[3, :128] = np.float32(2.0 ** -149)
    x[4] *= np.float32(1e-36)
    x[5] *= np.float32(1e-38)
    x[6, :128] = np.arange(128) * 3.5 + 3.5                      # scale 1: every code and midpoint between
    x[6, 127] = 448
    x[7, 5], x[7, 200] = np.inf, -np.inf
    x[8, 0], x[8, 299] = np.nan, -np.nan
    x[9] = np.nan
    x[10, 128:256] = np.inf
    x[11] = -0.0
    x[12] *= np.float32(2.0 ** -70)
    x[13] *= np.float32(2.0 ** 100)
    for dtype in (F32, BF16, F16):
        t = torch.from_numpy(x).to(dtype).cuda()
        check_rows(B.quantize_rows(t), t.cpu().double().numpy(), dtype)


def test_quantize_rows_every_quotient_near_a_midpoint(B):
    """Quotients at and beside every midpoint of E4M3, for scales that are no powers of two."""
    codes = np.arange(0x7E)
    from aeisu_amd import fp8
    v = fp8.decode(codes.astype(np.uint8)).astype(np.float64)
    mid = (v + np.append(v[1:], 448.0)) / 2
    rows = []
    for s in rng(7).random(64) * 3 + 0.01:
        for step in (-1, 0, 1):
            y = (mid * s).astype(np.float32)
            y = np.nextafter(y, np.float32(np.inf * step)) if step else y
            rows.append(np.concatenate([y, [np.float32(448 * s)], [np.float32(-448 * s)]])[:128])
    x = np.stack(rows).astype(np.float32)
    check_rows(B.quantize_rows(tensor(x)), x.astype(np.float64), "midpoints")


def test_quantize_rows_gathered(B):
    """Repeated, missing and out-of-range rows; the last give zeros."""
    x = tensor(values(rng(8), 30, 200), BF16)
    index = [3, 3, 29, 0, -1, 30, 7, 2 ** 31 - 1, -2 ** 31] + list(range(29, -1, -1))
    y = np.stack([x[i].cpu().double().numpy() if 0 <= i < 30 else np.zeros(200) for i in index])
    check_rows(B.quantize_rows(x, rows=torch.tensor(index, dtype=torch.int32, device="cuda")), y, "gathered")
    empty = B.quantize_rows(x[:0], rows=torch.zeros(2, dtype=torch.int32, device="cuda"))
    check_rows(empty, np.zeros((2, 200)), "gathered from nothing")
    none = B.quantize_rows(x, rows=torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert none.codes.shape == (0, 256) and none.scales.shape == (2, 0)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (5, 128), (19, 275), (130, 640)])
def test_quantize_rows_gated(B, m, k, dtype):
    """SiLU(a) b has at most 8 roundings of FP32 besides exp's two: 2^-20 of the value, so scales are that close, and
    each code is a nearest one for a quotient that close."""
    x = tensor(values(rng(m, k, 9), m, 2 * k), dtype)
    d = x.cpu().double()
    y = (torch.sigmoid(d[:, :k]) * d[:, :k] * d[:, k:]).numpy()
    q = B.quantize_rows(x, gated=True)
    _, scales = O.quantize(y, 1)
    got = q.scales.cpu().double().numpy().T
    assert (np.abs(got - scales) <= scales * 2.0 ** -20).all()
    value = O.rows_value(q.codes, q.scales, k).numpy()
    wide = np.repeat(got, 128, axis=1)[:, :k]
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(y / wide), 2.0 ** -6))) - 3) * wide
    assert (np.abs(value - y) <= step * 0.5 + np.abs(y) * 2.0 ** -18).all()
    assert not q.codes[:, k:].any()


def test_gate_at_the_ends_of_its_range(B):
    """SiLU of large magnitudes is 0 or the value itself, without overflow of exp; NaN and infinity stay in their place."""
    a = torch.tensor([[-1e30, -200.0, -88.0, 0.0, 88.0, 200.0, 1e30, float("nan"), float("inf"), -3.0]], device="cuda")
    b = torch.full_like(a, 2.0)
    q = B.quantize_rows(torch.cat([a, b], 1), gated=True)
    v = q.dequantize()[0].cpu()
    assert v[7].isnan() and v[8].isnan()
    assert v[0] == 0 and v[1] == 0 and v[6] == pytest.approx(2e30, rel=1e-6)


def test_gate_of_large_products_whose_logistic_underflows(B):
    """exp(a) below the normal numbers of FP32, and above them with b: the result is a normal number and keeps 2^-20."""
    x = torch.cat([-(85 + 80 * torch.rand(40, 128)), 1e38 * (1 + torch.rand(40, 128))], 1)
    x[:, :128] = x[:, :1] + 0.25 * torch.rand(40, 128)
    d = x.double()
    y = (d[:, :128].exp() / (1 + d[:, :128].exp()) * d[:, :128] * d[:, 128:]).numpy()
    y, x = y[np.abs(y).max(1) > 2.0 ** -100], x[np.abs(y).max(1) > 2.0 ** -100]
    assert len(y) >= 10
    q = B.quantize_rows(x.cuda(), gated=True)
    _, scales = O.quantize(y, 1)
    assert (np.abs(q.scales.cpu().double().numpy().T - scales) <= scales * 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 257), (3, 70, 130), (2, 300, 128), (4, 1, 500)])
def test_quantize_weight_is_the_definition(B, shape, dtype):
    w = tensor(values(rng(*shape), *shape), dtype)
    q = B.quantize_weight(w)
    three = w.reshape(-1, *shape[-2:])
    for i in range(three.shape[0]):
        codes, scales = O.quantize(three[i].cpu().double().numpy(), 128)
        assert np.array_equal(q.scales.reshape(-1, *q.scales.shape[-2:])[i].cpu().numpy(), scales)
        assert O.same_codes(q.codes.reshape(-1, *q.codes.shape[-2:])[i].cpu().numpy(), codes)


def test_quantize_weight_of_views(B):
    big = tensor(values(rng(11), 4, 90, 410), F16)
    for v in (big[1:3, 5:80, 3:300], big[:, ::3, :129], big[2, :, 9:]):
        q, want = B.quantize_weight(v), B.quantize_weight(v.contiguous())
        assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)


# ---- products ------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 64, 128), (1, 500, 1111), (2, 129, 300), (15, 16, 64), (16, 128, 128), (17, 127, 129),
         (31, 260, 2050), (33, 48, 640), (64, 64, 256), (65, 193, 1000), (100, 1030, 515), (129, 128, 384),
         (257, 300, 130), (300, 515, 777), (700, 640, 900), (1025, 1100, 260), (2100, 72, 128)]


def operands(B, m, n, k, key=0):
    r = rng(m, n, k, key)
    x = B.quantize_rows(tensor(values(r, m, k), BF16))
    w = B.quantize_weight(tensor(r.standard_normal((n, k)) / k ** 0.5, BF16))
    return x, w, tensor(r.standard_normal(n))


@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(B, m, n, k, out_dtype):
    x, w, bias = operands(B, m, n, k)
    xv, wv = O.rows_value(x.codes, x.scales, k), O.weight_value(w.codes, w.scales, k)
    for b, slope in ((None, None), (bias, 0.1), (None, 0.0)):
        got = B.matmul(x, w, bias=b, slope=slope, out_dtype=out_dtype)
        assert got.dtype == out_dtype and got.shape == (m, n)
        y, mag = O.product(xv, wv, b, slope)
        O.check(got, y, mag, k, True, f"{m}x{n}x{k} {out_dtype} slope {slope}")


def test_matmul_defaults_to_fp16_and_is_repeatable(B):
    x, w, _ = operands(B, 333, 257, 1000)
    a, b = B.matmul(x, w), B.matmul(x, w)
    assert a.dtype == F16 and torch.equal(a, b)


@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 70, 200), (40, 130, 257), (300, 333, 500)])
def test_matmul_of_views_into_a_view(B, m, n, k, out_dtype):
    """Codes, scales and results with row strides and offsets; what lies round the result keeps its value."""
    x, w, bias = operands(B, m, n, k)
    kp = x.codes.shape[1]
    codes = torch.zeros(m + 3, kp + 48, dtype=torch.uint8, device="cuda")
    codes[2:m + 2, 16:16 + kp] = x.codes
    scales = torch.zeros(x.scales.shape[0], m + 7, device="cuda")
    scales[:, 3:3 + m] = x.scales
    wide = torch.full((n, kp + 32), 0x7F, dtype=torch.uint8, device="cuda")
    wide[:, :kp] = w.codes
    xs, ws = B.QuantRows(codes[2:m + 2, 16:16 + kp], scales[:, 3:3 + m], k), B.QuantWeight(wide[:, :kp], w.scales, k)
    want = B.matmul(x, w, bias=bias, out_dtype=out_dtype)
    for left, extra in ((0, 0), (3, 2), (4, 0)):
        page = torch.full((m + 4, n + left + extra), -7.0, dtype=out_dtype, device="cuda")
        got = B.matmul(xs, ws, bias=bias, out=page[2:m + 2, left:left + n])
        assert torch.equal(got, want) and got.data_ptr() == page[2, left:].data_ptr()
        page[2:m + 2, left:left + n] = -7.0
        assert (page == -7).all()


def test_matmul_without_terms(B):
    """No columns: the bias alone; no rows or no results: nothing."""
    x = B.quantize_rows(torch.zeros(5, 0, device="cuda"))
    w = B.quantize_weight(torch.zeros(7, 0, device="cuda"))
    bias = torch.arange(7.0, device="cuda") - 3
    assert torch.equal(B.matmul(x, w, bias=bias, slope=0.5, out_dtype=F32)[4].cpu(),
                       torch.tensor([-1.5, -1, -0.5, 0, 1, 2, 3]))
    x, w, _ = operands(B, 4, 6, 40)
    assert B.matmul(B.quantize_rows(torch.zeros(0, 40, device="cuda")), w).shape == (0, 6)
    assert B.matmul(x, B.quantize_weight(torch.zeros(0, 40, device="cuda"))).shape == (4, 0)


@pytest.mark.parametrize("m,n,k", [(3, 40, 300), (90, 200, 300), (600, 700, 300)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_values_that_are_not_finite_stay_in_their_rows_and_columns(B, m, n, k, out_dtype):
    x = values(rng(1, m), m, k)
    w = rng(2, m).standard_normal((n, k))
    clean = B.matmul(B.quantize_rows(tensor(x)), B.quantize_weight(tensor(w)), out_dtype=out_dtype)
    x[m // 2, 150] = np.inf
    w[n - 1, 299] = np.nan
    got = B.matmul(B.quantize_rows(tensor(x)), B.quantize_weight(tensor(w)), out_dtype=out_dtype)
    assert got[m // 2].isnan().all() and got[:, n - 1].isnan().all()
    rows, cols = [i for i in range(m) if i != m // 2], list(range(n - 128))       # the tile with the NaN has its own scale
    if cols:
        assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
    assert got[rows][:, :n - 1].isfinite().all()


def test_exact_products_when_the_result_is_fp32(B):
    """Large products that cancel, with a small one beside them in the same group of eight: FP32 results keep it."""
    for m, n in ((1, 16), (20, 64), (300, 300)):
        x = torch.zeros(m, 256)
        w = torch.zeros(n, 256)
        x[:, 0], x[:, 8], x[:, 1], x[:, 130] = 448, 448, 1, 448
        w[:, 0], w[:, 8], w[:, 1], w[:, 130] = 448, -448, 1, 448      # every scale is 1
        got = B.matmul(B.quantize_rows(x.cuda()), B.quantize_weight(w.cuda()), out_dtype=F32)
        assert (got == 448 * 448 + 1).all()


# ---- products grouped by expert --------------------------------------------------------------------------------
def offsets_of(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def grouped_case(B, kind, t, e, n, k, key=0):
    r = rng(t, e, n, k, key)
    x, w = values(r, t, k), r.standard_normal((e, n, k)) / max(k, 1) ** 0.5
    bias = tensor(r.standard_normal((e, n)))
    if kind == "e4m3":
        x, w = B.quantize_rows(tensor(x, BF16)), B.quantize_weight(tensor(w, BF16))
        xv, wv = O.rows_value(x.codes, x.scales, k), O.weight_value(w.codes, w.scales, k)
    else:
        dt = F16 if kind == "f16" else BF16
        x, w = tensor(x, dt), tensor(w, dt)
        xv, wv = x.cpu().double(), w.cpu().double()
    return x, w, bias, xv, wv


COUNTS = {
    "one expert": [37], "one row": [0, 0, 1, 0], "uneven": [3, 0, 130, 1, 17, 64, 0, 40], "first empty": [0, 70], "last empty": [65, 0],
    "even": [16] * 9, "large": [300, 513, 2, 700], "many experts": [1, 0, 2] * 45, "singles": [1] * 70,
}


@pytest.mark.parametrize("kind,out_dtype", [("e4m3", BF16), ("e4m3", F32), ("e4m3", F16), ("f16", F16), ("bf16", BF16), ("bf16", F32)])
@pytest.mark.parametrize("name", list(COUNTS))
@pytest.mark.parametrize("n,k", [(130, 200), (64, 129), (300, 512)])
def test_grouped_matmul(B, name, n, k, kind, out_dtype):
    counts = COUNTS[name]
    off = offsets_of(counts)
    x, w, bias, xv, wv = grouped_case(B, kind, sum(counts), len(counts), n, k)
    got = B.grouped_matmul(x, w, off, bias=bias, slope=0.25, out_dtype=out_dtype)
    y, mag = O.grouped(xv, wv, off.tolist(), bias, 0.25)
    O.check(got, y, mag, k, kind == "e4m3", f"{name} {n}x{k} {kind} {out_dtype}")
    assert torch.equal(got, B.grouped_matmul(x, w, off, bias=bias, slope=0.25, out_dtype=out_dtype))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("k", [1, 7, 8, 63, 64, 65, 100, 1003])
def test_grouped_matmul_of_16_bit_rows_that_end_anywhere(B, kind, k):
    off = offsets_of([5, 0, 80, 33])
    x, w, bias, xv, wv = grouped_case(B, kind, 118, 4, 70, k)
    y, mag = O.grouped(xv, wv, off.tolist(), None, None)
    O.check(B.grouped_matmul(x, w, off, out_dtype=F32), y, mag, k, False, f"k {k}")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_grouped_matmul_of_views(B, kind):
    """Rows and weights at addresses that are no multiple of 16 bytes, with NaN round them."""
    off = offsets_of([50, 31, 0, 90])
    x, w, bias, xv, wv = grouped_case(B, kind, 171, 4, 90, 144)
    want = B.grouped_matmul(x, w, off)
    for left, extra in ((1, 2), (8, 8), (3, 5)):
        xb = torch.full((175, 144 + left + extra), float("nan"), dtype=x.dtype, device="cuda")
        wb = torch.full((4, 93, 144 + left + extra), float("nan"), dtype=x.dtype, device="cuda")
        xb[2:173, left:left + 144] = x
        wb[:, 1:91, left:left + 144] = w
        got = B.grouped_matmul(xb[2:173, left:left + 144], wb[:, 1:91, left:left + 144], off)
        y, mag = O.grouped(xv, wv, off.tolist(), None, None)
        O.check(got, y, mag, 144, False, f"view at {left}")
        if left % 8 == 0:
            assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
@pytest.mark.parametrize("t", [40, 900])
def test_rows_of_no_expert_are_zero_and_any_offsets_are_safe(B, kind, t):
    """Rows before the first and after the last offset; offsets that decrease or leave the rows count as the largest up to
    them, kept within the rows, and every row is written."""
    x, w, bias, xv, wv = grouped_case(B, kind, t, 5, 100, 130)
    for raw in ([7, 9, 9, 20, 30, t - 4], [0, 0, 0, 0, 0, 0], [t] * 6, [5, 3, 30, 10, 35, t], [-8, 4, t + 100, 2, 1, 0],
                [2 ** 31 - 1] * 6, [-2 ** 31, 10, 2 ** 31 - 1, -5, 3, 4]):
        seen = np.clip(np.maximum.accumulate(np.array(raw, dtype=np.int64)), 0, t).tolist()
        out = torch.full((t, 100), float("nan"), dtype=F32, device="cuda")
        B.grouped_matmul(x, w, torch.tensor(raw, dtype=torch.int32, device="cuda"), bias=bias, out=out)
        y, mag = O.grouped(xv, wv, seen, bias, None)
        O.check(out, y, mag, 130, kind == "e4m3", str(raw))
        assert not out[:seen[0]].any() and not out[seen[-1]:].any()


@pytest.mark.parametrize("kind", ["e4m3", "f16"])
def test_experts_without_rows_are_not_seen(B, kind):
    """NaN in the weights, scales or bias of an expert without rows, and in another expert's rows, reaches nothing else."""
    off = offsets_of([40, 0, 60, 3])
    x, w, bias, _, _ = grouped_case(B, kind, 103, 4, 80, 128)
    want = B.grouped_matmul(x, w, off, bias=bias)
    bias[1] = float("nan")
    if kind == "e4m3":
        w.codes[1], w.scales[1] = 0x7F, float("nan")
        x.codes[102] = 0x7F
    else:
        w[1], x[102] = float("nan"), float("nan")
    got = B.grouped_matmul(x, w, off, bias=bias)
    assert torch.equal(got[:102], want[:102]) and got[102].isnan().all()


def test_grouped_matmul_agrees_with_matmul(B):
    """One expert with all rows is the plain product."""
    for m in (5, 100, 700):
        x, w, bias = operands(B, m, 200, 400)
        off = torch.tensor([0, m], dtype=torch.int32, device="cuda")
        w3 = B.QuantWeight(w.codes[None], w.scales[None], 400)
        a = B.grouped_matmul(x, w3, off, bias=bias[None], out_dtype=F32)
        y, mag = O.product(O.rows_value(x.codes, x.scales, 400), O.weight_value(w.codes, w.scales, 400), bias, None)
        O.check(a, y, mag, 400, True, f"{m} rows")


# ---- large products: a definition in 64 bits on the GPU ------------------------------------------------------------
def on_gpu(v, cols, tiles):
    """float64 values of codes on the GPU, from the oracle's table"""
    from aeisu_amd import fp8
    table = torch.from_numpy(fp8.DECODE.astype(np.float64)).cuda()
    scale = v.scales.double()
    wide = scale.repeat_interleave(128, -2)[..., :v.codes.shape[-2], :] if tiles else scale.t()
    return table[v.codes[..., :cols].long()] * wide.repeat_interleave(128, -1)[..., :cols]


@pytest.mark.parametrize("out_dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", [(4100, 4000, 1000), (8192, 2050, 130), (300, 20000, 2300), (20000, 16, 512), (8192, 13, 300)])
def test_large_matmul(B, m, n, k, out_dtype):
    g = torch.Generator("cuda").manual_seed(m)
    x = B.quantize_rows(torch.randn(m, k, generator=g, device="cuda"))
    w = B.quantize_weight(torch.randn(n, k, generator=g, device="cuda"))
    bias = torch.randn(n, generator=g, device="cuda")
    xv, wv = on_gpu(x, k, False), on_gpu(w, k, True)
    y, mag = xv @ wv.t() + bias.double(), xv.abs() @ wv.abs().t() + bias.double().abs()
    y = torch.where(y < 0, y * 0.1, y).cpu()
    O.check(B.matmul(x, w, bias=bias, slope=0.1, out_dtype=out_dtype), y, mag.cpu(), k, True, f"{m}x{n}x{k}")


@pytest.mark.parametrize("kind,k,out_dtype", [("e4m3", 900, BF16), ("e4m3", 300, F32), ("bf16", 712, BF16), ("f16", 640, F32), ("f16", 8, F16), ("f16", 1003, F16),
                                              ("bf16", 129, F32)])
@pytest.mark.parametrize("counts", [[2000, 0, 3, 1100, 257, 1, 3000, 120], [4096, 4096], [130] * 40])
def test_large_grouped_matmul(B, counts, kind, k, out_dtype):
    """Enough rows for every tile height, whole and partly filled tiles, halves without rows, steps that end inside a block."""
    e, n, t = len(counts), 1300, sum(counts)
    g = torch.Generator("cuda").manual_seed(k)
    x, w = torch.randn(t, k, generator=g, device="cuda"), torch.randn(e, n, k, generator=g, device="cuda")
    if kind == "e4m3":
        x, w = B.quantize_rows(x), B.quantize_weight(w)
        xv, wv = on_gpu(x, k, False), on_gpu(w, k, True)
    else:
        x, w = (v.to(F16 if kind == "f16" else BF16) for v in (x, w))
        xv, wv = x.double(), w.double()
    off = offsets_of(counts)
    out = torch.full((t + 5, n), float("nan"), dtype=out_dtype, device="cuda")
    xs = B.QuantRows(torch.cat([x.codes, x.codes[:5]]), torch.cat([x.scales, x.scales[:, :5]], 1), k) if kind == "e4m3" \
        else torch.cat([x, x[:5]])
    B.grouped_matmul(xs, w, off, out=out)
    assert not out[t:].any()
    y = torch.zeros(t, n, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(y)
    for i, (lo, hi) in enumerate(zip(off.tolist(), off.tolist()[1:])):
        y[lo:hi], mag[lo:hi] = xv[lo:hi] @ wv[i].t(), xv[lo:hi].abs() @ wv[i].abs().t()
    O.check(out[:t], y.cpu(), mag.cpu(), k, kind == "e4m3", f"{counts[:3]} {kind} {k}")


@pytest.mark.parametrize("kind,out_dtype", [("f16", F16), ("bf16", F32), ("f16", F32)])
@pytest.mark.parametrize("counts,n,k", [([700, 0, 1500, 1, 300], 900, 1001), ([3000, 1100], 515, 2003), ([257] * 9, 1300, 1150),
                                        ([5000], 1030, 777), ([7000, 0, 4000, 1, 1000], 900, 1001), ([3000, 3000, 1000], 1500, 1100)])
def test_large_products_on_rows_that_are_laid_out(B, counts, n, k, kind, out_dtype):
    """Rows and weights at odd addresses with NaN round them, on both sides of where laying them out pays (there for
    certain from five million results on): with the workspace that the library asks for, one that is too small, and none."""
    from aeisu_amd import _lib as L
    import ctypes
    e, t, dtype = len(counts), sum(counts), F16 if kind == "f16" else BF16
    g = torch.Generator("cuda").manual_seed(k)
    xb = torch.full((t + 2, k + 4), float("nan"), dtype=dtype, device="cuda")
    wb = torch.full((e, n + 2, k + 5), float("nan"), dtype=dtype, device="cuda")
    x, w = xb[1:t + 1, 3:k + 3], wb[:, 1:n + 1, 1:k + 1]
    x.copy_(torch.randn(t, k, generator=g, device="cuda"))
    w.copy_(torch.randn(e, n, k, generator=g, device="cuda"))
    bias, off = torch.randn(e, n, generator=g, device="cuda"), offsets_of(counts)
    y = torch.cat([v.double() @ wi.double().t() + b.double() for v, wi, b in zip(x.split(counts), w, bias)])
    mag = torch.cat([v.double().abs() @ wi.double().abs().t() + b.double().abs() for v, wi, b in zip(x.split(counts), w, bias)])
    y = torch.where(y < 0, y * 0.25, y)
    got = B.grouped_matmul(x, w, off, bias=bias, slope=0.25, out_dtype=out_dtype)
    O.check(got, y.cpu(), mag.cpu(), k, False, "with the workspace asked for")
    assert torch.equal(got, B.grouped_matmul(x, w, off, bias=bias, slope=0.25, out_dtype=out_dtype))
    room = torch.empty((t, n), dtype=out_dtype, device="cuda")
    p = L.Product(type=B._TYPES[dtype], out_type=B._TYPES[out_dtype], rows=t, n=n, k=k, x=x.data_ptr(), x_stride=x.stride(0),
                  w=w.data_ptr(), w_stride=w.stride(1), w_expert_stride=w.stride(0), bias=bias.data_ptr(), slope=0.25,
                  out=room.data_ptr(), out_stride=n)
    need = L.lib().aeisu_product_workspace(ctypes.byref(p), e)
    padded = -(-k // 8) * 8
    assert need in (0, -(-t * padded * 2 // 256) * 256 + e * n * padded * 2) and (need or t * n < 5000000)
    for size in (need, need - 1, 0) if need else (0,):
        space = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")
        p.workspace, p.workspace_bytes = space.data_ptr() if size else 0, size
        room.fill_(float("nan"))
        L.check(L.lib().aeisu_grouped_matmul(ctypes.byref(p), off.data_ptr(), e, torch.cuda.current_stream().cuda_stream))
        O.check(room, y.cpu(), mag.cpu(), k, False, f"workspace of {size}")
        assert (space[need if size == need else 0:] == 255).all()
        assert size < need or torch.equal(room, got)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("k", [1003, 1067, 70, 2051])
def test_products_of_few_rows_out_of_line_in_two_halves(B, kind, k):
    """One block for each CU at most: two steps at a time, their number odd and even, the last one partly filled."""
    counts, n = [120, 0, 200, 1, 150, 190, 116], 515
    off = offsets_of(counts)
    x, w, bias, xv, wv = grouped_case(B, kind, sum(counts), len(counts), n, k)
    y, mag = O.grouped(xv, wv, off.tolist(), bias, 0.25)
    got = B.grouped_matmul(x, w, off, bias=bias, slope=0.25, out_dtype=F32)
    O.check(got, y, mag, k, False, f"{kind} k {k}")
    assert torch.equal(got, B.grouped_matmul(x, w, off, bias=bias, slope=0.25, out_dtype=F32))


def test_laid_out_rows_of_one_weight_for_all_experts(B):
    """A weight of expert stride 0, and operands of which only one is out of line."""
    t, e, n, k = 4000, 6, 1000, 1024
    g = torch.Generator("cuda").manual_seed(9)
    x, one = (torch.randn(r, k, generator=g, device="cuda").bfloat16() for r in (t, n))
    w, off = one.expand(e, n, k), offsets_of([900, 0, 1100, 1000, 999, 1])
    want = x.double() @ one.double().t()
    mag = x.double().abs() @ one.double().abs().t()
    shifted = torch.full((t, k + 1), float("nan"), dtype=BF16, device="cuda")[:, 1:]
    shifted.copy_(x)
    for a in (x, shifted):
        O.check(B.grouped_matmul(a, w, off, out_dtype=F32), want.cpu(), mag.cpu(), k, False, "one weight")
    short = x[:, :1021], w[:, :, :1021]              # aligned rows whose columns end inside a piece
    want, mag = short[0].double() @ one[:, :1021].double().t(), short[0].double().abs() @ one[:, :1021].double().abs().t()
    O.check(B.grouped_matmul(*short, off, out_dtype=F32), want.cpu(), mag.cpu(), 1021, False, "short rows")


# ---- memory, streams, graphs ------------------------------------------------------------------------------------
def test_offsets_past_32_bits(B):
    """Operands and results whose rows lie more than 4 GiB apart from first to last."""
    m, n, k, apart = 34, 64, 256, 1 << 27
    x, w, _ = operands(B, m, n, k)
    want = B.matmul(x, w, out_dtype=F32)
    room = torch.empty(m * apart, dtype=torch.uint8, device="cuda")
    codes = room.as_strided((m, k), (apart, 1))
    codes.copy_(x.codes)
    assert torch.equal(B.matmul(B.QuantRows(codes, x.scales, k), w, out_dtype=F32), want)
    out = room.view(torch.float32).as_strided((m, n), (apart // 4, 1), 4096)
    B.matmul(x, w, out=out)
    assert torch.equal(out, want)
    wide = room.as_strided((n // 2, k), (apart, 1), 65536)
    wide.copy_(w.codes[:n // 2])
    assert torch.equal(B.matmul(x, B.QuantWeight(wide, w.scales, k), out_dtype=F32), want[:, :n // 2])
    src = room.view(torch.bfloat16).as_strided((m, k), (apart // 2, 1), 1 << 17)
    src.copy_(torch.randn(m, k))
    a, b = B.quantize_rows(src), B.quantize_rows(src.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    off = torch.tensor([0, 10, m], dtype=torch.int32, device="cuda")
    w16 = torch.randn(2, n, k, device="cuda").bfloat16()
    assert torch.equal(B.grouped_matmul(src, w16, off), B.grouped_matmul(src.contiguous(), w16, off))


@pytest.mark.parametrize("gathered", [False, True])
def test_more_rows_than_a_launch_takes(B, gathered):
    """2^27 rows and some: both sides of where the second launch begins."""
    first, more = 1 << 27, 37
    x = torch.empty(1000 if gathered else first + more, 3, dtype=F16, device="cuda")
    x[:1000].normal_()
    x[-1000:].normal_()
    index = None
    if gathered:
        index = torch.full((first + more,), -1, dtype=torch.int32, device="cuda")
        index[:500] = torch.arange(500, device="cuda", dtype=torch.int32)
        index[-500:] = torch.arange(999, 499, -1, device="cuda", dtype=torch.int32)
    q = B.quantize_rows(x, rows=index)
    for part in (slice(0, 500), slice(first + more - 500, first + more)):
        want = B.quantize_rows(x[index[part].long()] if gathered else x[part])
        assert torch.equal(q.codes[part], want.codes) and torch.equal(q.scales[:, part], want.scales)


def test_work_is_ordered_on_the_given_stream(B):
    x, w, _ = operands(B, 300, 400, 1000)
    src = tensor(values(rng(3), 300, 1000), BF16)
    want = B.matmul(B.quantize_rows(src), w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = src * 1
    got = B.matmul(B.quantize_rows(mine, stream=side), w, stream=side)
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_calls_replay(B):
    """Quantisation and both products in a graph, replayed on changing inputs with other work between."""
    from aeisu_amd.experts import ExpertLayer, route
    r = rng(12)
    layer = ExpertLayer(tensor(r.standard_normal((4, 256, 192)) / 14, BF16), tensor(r.standard_normal((4, 192, 128)) / 11, BF16))
    x, pick = torch.zeros(50, 192, dtype=BF16, device="cuda"), torch.zeros(50, 4, device="cuda")
    _, order, offsets = route(torch.randn(50, 4, device="cuda"), 2)
    token = (order // 2).int()

    def step():
        h = B.grouped_matmul(B.quantize_rows(x, rows=token), layer.gate_up, offsets, out_dtype=BF16)
        return B.grouped_matmul(B.quantize_rows(h, gated=True), layer.down, offsets, out_dtype=F32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(tensor(values(rng(13, i), 50, 192), BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), i


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("t", [1, 77, 700])
def test_expert_layer(B, t, quantized):
    """The layer against its formula in 64 bits: on the weights it holds (their own quantisation error is not the layer's),
    within what quantising the activations twice costs: E4M3 keeps 4 bits, 2^-4 at most and 2^-5.5 in the mean square for
    each, the second of them and the gate's two factors from the first."""
    from aeisu_amd.experts import ExpertLayer, reference
    r = rng(t, 14)
    gate_up, down = tensor(r.standard_normal((6, 320, 200)) / 14, BF16), tensor(r.standard_normal((6, 200, 160)) / 13, BF16)
    x, logits = tensor(r.standard_normal((t, 200)), BF16), tensor(r.standard_normal((t, 6)))
    layer = ExpertLayer(gate_up, down, 2, quantized)
    a, b = (layer.gate_up.dequantize(), layer.down.dequantize()) if quantized else (gate_up, down)
    want = reference(a.cpu().double(), b.cpu().double(), x.cpu().double(), logits.cpu().double(), 2)
    got = layer(x, logits)
    assert got.shape == x.shape and got.dtype == x.dtype
    off = ((got.cpu().double() - want).norm() / want.norm()).item()
    assert off <= (2.0 ** -5.5 * 3 if quantized else 2.0 ** -7), off
