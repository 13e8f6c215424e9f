"""Refusals of the block-scaled operators (no GPU): the C entry points check every argument before any HIP call."""
from __future__ import annotations

import ctypes

import pytest
import torch

from aeisu_amd import _lib as L
from aeisu_amd import blocks as B

P = 1 << 20          # an address that is never touched


def product(**change):
    v = dict(type=L.TYPE_E4M3, out_type=L.TYPE_F16, rows=4, n=8, k=100, x=P, x_stride=128, x_scales=P, x_scales_stride=4, w=P,
             w_stride=128, w_expert_stride=1024, w_scales=P, bias=0, slope=1.0, out=P, out_stride=8)
    v.update(change)
    return L.Product(**v)


@pytest.mark.parametrize("change,message", [
    ({"type": L.TYPE_F32}, "operands"), ({"type": 9}, "operands"), ({"out_type": L.TYPE_E4M3}, "results"),
    ({"rows": -1}, "rows"), ({"n": 1 << 30}, "n out"), ({"k": -5}, "k out"), ({"slope": -0.5}, "slope"),
    ({"slope": float("nan")}, "slope"), ({"slope": float("inf")}, "slope"), ({"out": 0}, "result"), ({"out": P + 1}, "result"),
    ({"out_stride": 7}, "result's row stride"), ({"x": 0}, "operand"), ({"w": 0}, "operand"), ({"x": P + 8}, "16-byte"),
    ({"w": P + 4}, "16-byte"), ({"x_stride": 100}, "x's row stride"), ({"x_stride": 136}, "16-byte"), ({"w_stride": 112}, "w's row stride"),
    ({"x_scales": 0}, "scales"), ({"w_scales": P + 2}, "scales"), ({"w_expert_stride": -1}, "expert stride"), ({"bias": P + 1}, "bias"),
    ({"type": L.TYPE_BF16, "x": P + 1}, "operand"), ({"type": L.TYPE_F16, "x_stride": 99}, "x's row stride"),
    ({"k": 200, "x_stride": 256, "w_stride": 256, "x_scales_stride": 3}, "stride of x's scales"),
])
def test_products_are_refused(change, message):
    lib = L.lib()
    p = product(**change)
    assert lib.aeisu_matmul(ctypes.byref(p), None) == L.AEISU_ERR_INVALID_ARGUMENT
    assert message in lib.aeisu_last_error().decode()
    assert lib.aeisu_grouped_matmul(ctypes.byref(p), P, 3, None) == L.AEISU_ERR_INVALID_ARGUMENT


def test_grouped_products_are_refused():
    lib = L.lib()
    p = product()
    for offsets, experts, stride in ((0, 3, 1024), (P + 2, 3, 1024), (P, 0, 1024), (P, 65536, 1024), (P, 3, 1030)):
        p.w_expert_stride = stride
        assert lib.aeisu_grouped_matmul(ctypes.byref(p), offsets, experts, None) == L.AEISU_ERR_INVALID_ARGUMENT
    assert lib.aeisu_matmul(None, None) == L.AEISU_ERR_INVALID_ARGUMENT


def test_workspaces_are_checked_and_asked_for():
    """A workspace has to be aligned; it is asked for by large 16-bit products out of line, and by no other."""
    lib = L.lib()
    for change in ({"workspace": P + 8, "workspace_bytes": 64}, {"workspace": P, "workspace_bytes": -1}):
        p = product(**change)
        assert lib.aeisu_matmul(ctypes.byref(p), None) == L.AEISU_ERR_INVALID_ARGUMENT
        assert "workspace" in lib.aeisu_last_error().decode()

    def need(experts=4, **change):
        v = dict(type=L.TYPE_BF16, rows=16000, n=2000, k=2000, x_stride=2000, w_stride=2000, w_expert_stride=4000000, out_stride=2000)
        v.update(change)
        return lib.aeisu_product_workspace(ctypes.byref(product(**v)), experts)
    assert need() == 0                                                     # in line
    assert need(k=1999) == (16000 + 4 * 2000) * 2000 * 2                   # columns that end inside a piece
    assert need(x=P + 2) == need(w=P + 2) == need(k=1999)                  # rows that start inside one
    assert need(k=1999, w_expert_stride=0) == (16000 + 2000) * 2000 * 2    # one weight for all
    assert need(k=1999, rows=2) == 0                                       # less work than laying out
    assert need(k=1999, x_stride=100) == 0 and need(k=1999, experts=70000) == 0 and need(k=1999, rows=0) == 0
    assert need(0, k=1999) == (16000 + 2000) * 2000 * 2                    # one weight, no offsets
    assert lib.aeisu_product_workspace(None, 4) == 0
    assert lib.aeisu_product_workspace(ctypes.byref(product(rows=16000)), 4) == 0


def test_nothing_to_do_is_no_error():
    lib = L.lib()
    assert lib.aeisu_matmul(ctypes.byref(product(rows=0, x=0, w=0, out=0)), None) == L.AEISU_OK
    assert lib.aeisu_matmul(ctypes.byref(product(n=0, x=0, w=0, out=0)), None) == L.AEISU_OK
    assert lib.aeisu_quantize_rows(0, L.TYPE_F16, 0, 0, 10, 0, 0, 0, 0, 0, 0, 0, None) == L.AEISU_OK
    assert lib.aeisu_quantize_weight(0, L.TYPE_F16, 2, 0, 5, 0, 0, 0, 0, None) == L.AEISU_OK


@pytest.mark.parametrize("change", [
    {"type": L.TYPE_E4M3}, {"x_rows": -1}, {"cols": 1 << 30}, {"rows": 5}, {"x": 0}, {"x": P + 1}, {"x_stride": 99},
    {"codes": 0}, {"codes": P + 8}, {"codes_stride": 100}, {"codes_stride": 136}, {"scales": 0}, {"scales": P + 2},
    {"index": P + 1}, {"gated": 1}, {"cols": 300, "x_stride": 300, "codes_stride": 384, "scales_stride": 3},
])
def test_quantize_rows_is_refused(change):
    v = dict(x=P, type=L.TYPE_F16, x_rows=4, x_stride=100, cols=100, gated=0, index=0, rows=4, codes=P, codes_stride=128, scales=P,
             scales_stride=4)
    v.update(change)
    assert L.lib().aeisu_quantize_rows(*v.values(), None) == L.AEISU_ERR_INVALID_ARGUMENT
    assert L.lib().aeisu_last_error()


@pytest.mark.parametrize("change", [{"type": 7}, {"experts": 70000}, {"n": -1}, {"w": 0}, {"row_stride": 99}, {"expert_stride": -1},
                                    {"codes": P + 1}, {"scales": 0}])
def test_quantize_weight_is_refused(change):
    v = dict(w=P, type=L.TYPE_F16, experts=2, n=4, k=100, expert_stride=400, row_stride=100, codes=P, scales=P)
    v.update(change)
    assert L.lib().aeisu_quantize_weight(*v.values(), None) == L.AEISU_ERR_INVALID_ARGUMENT


def rows(m=4, k=100):
    return B.QuantRows(torch.zeros(m, 128, dtype=torch.uint8), torch.zeros(1, m), k)


def weight(n=8, k=100, lead=()):
    return B.QuantWeight(torch.zeros(*lead, n, 128, dtype=torch.uint8), torch.zeros(*lead, 1, 1), k)


@pytest.mark.parametrize("make", [
    lambda: B.QuantRows(torch.zeros(4, 128), torch.zeros(1, 4), 100),                                # codes of another type
    lambda: B.QuantRows(torch.zeros(4, 100, dtype=torch.uint8), torch.zeros(1, 4), 100),             # not padded
    lambda: B.QuantRows(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 1), 100),             # scales the other way
    lambda: B.QuantRows(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4), -1),
    lambda: B.QuantWeight(torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(1, 2), 100),
    lambda: B.QuantWeight(torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.float16), 100),
    lambda: B.QuantWeight(torch.zeros(128, dtype=torch.uint8), torch.zeros(1, 1), 100),
    lambda: B.quantize_rows(torch.zeros(4, 8)),                                                      # not on the GPU
    lambda: B.quantize_rows(torch.zeros(4, 8, dtype=torch.int32)),
    lambda: B.quantize_weight(torch.zeros(8)),
    lambda: B.matmul(rows(), weight()),                                                              # not on the GPU
    lambda: B.matmul(rows(k=99), weight()),
    lambda: B.matmul(rows(), weight(lead=(2,))),
    lambda: B.matmul(torch.zeros(4, 8).half(), torch.zeros(8, 8).half()),
    lambda: B.grouped_matmul(rows(), weight(), torch.zeros(3, dtype=torch.int32)),
    lambda: B.grouped_matmul(rows(), torch.zeros(2, 8, 100).half(), torch.zeros(3, dtype=torch.int32)),
    lambda: B.grouped_matmul(torch.zeros(4, 8).half(), torch.zeros(2, 8, 8).bfloat16(), torch.zeros(3, dtype=torch.int32)),
    lambda: B.grouped_matmul(torch.zeros(4, 8), torch.zeros(2, 8, 8), torch.zeros(3, dtype=torch.int32)),
    lambda: B.grouped_matmul(rows(), weight(lead=(2,)), [0, 1, 2]),
])
def test_python_refuses(make):
    with pytest.raises(ValueError):
        make()


def test_expert_layer_refuses():
    from aeisu_amd.experts import ExpertLayer
    for a, b, k in (((2, 6, 8), (2, 8, 4), 1), ((2, 5, 8), (2, 8, 2), 1), ((2, 6, 8), (2, 8, 3), 0), ((2, 6, 8), (2, 8, 3), 3)):
        with pytest.raises(ValueError):
            ExpertLayer(torch.zeros(a).half(), torch.zeros(b).half(), k, quantized=False)
    layer = ExpertLayer(torch.zeros(2, 6, 8).half(), torch.zeros(2, 8, 3).half(), 1, quantized=False)
    for x, logits in ((torch.zeros(4, 7).half(), torch.zeros(4, 2)), (torch.zeros(4, 8), torch.zeros(4, 2)),
                      (torch.zeros(4, 8).half(), torch.zeros(4, 3))):
        with pytest.raises(ValueError):
            layer(x, logits)


def test_routing_sorts_by_expert_and_ties_go_to_the_lower():
    from aeisu_amd.experts import route
    logits = torch.tensor([[1.0, 1, 0], [0, 5, 5], [2, 2, 2], [0, 0, 9]])
    shares, order, offsets = route(logits, 2)
    assert offsets.tolist() == [0, 3, 6, 8] and offsets.dtype == torch.int32
    assert order.tolist() == [0, 4, 7, 1, 2, 5, 3, 6]
    assert torch.allclose(shares.sum(1), torch.ones(4))
