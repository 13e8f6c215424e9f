"""Block-scaled operators: quantisation to E4M3 with a scale for each 128 columns, and matrix products of such operands.

``quantize_rows`` turns activations into ``QuantRows`` (E4M3 codes, one FP32 scale for each row and 128 columns) and
``quantize_weight`` weights into ``QuantWeight`` (one scale for each tile of 128 x 128); ``matmul`` multiplies the two, and
``grouped_matmul`` multiplies rows sorted by expert with each expert's weight, in E4M3 blocks or kept in FP16 / BF16.
``aeisu_amd.experts`` puts them together.

    w = quantize_weight(weight)                       # once: [n, k], or [experts, n, k]
    y = matmul(quantize_rows(x), w, bias=b, slope=0.1, out_dtype=torch.float16)

Sums are held in FP32 and rounded once to the result's type.  Products of E4M3 operands with an FP32 result are exact;
with a 16-bit result they may run on the FP8 matrix unit, whose rounding (about 2e-5 of the result) lies below the
result's own.  All work is enqueued on ``stream`` (default: torch's current one) and nothing waits for it.  Arguments
that cannot be served raise ``ValueError``.  The HIP kernels of ``libaeisu_amd.so`` do all arithmetic; there is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import _lib as L

BLOCK = 128
_TYPES = {torch.float16: L.TYPE_F16, torch.float32: L.TYPE_F32, torch.bfloat16: L.TYPE_BF16}


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


class QuantRows:
    """E4M3 rows: value[r, c] = codes[r, c] * scales[c // 128, r].

    ``codes`` uint8 [rows, >= padded], columns ``cols`` up to the next multiple of 128 holding code 0; ``scales``
    float32 [ceil(cols / 128), rows].  Rows of codes are 16-byte aligned; both may be views with a row stride.
    """

    __slots__ = ("codes", "scales", "cols")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int):
        _require(codes.dtype == torch.uint8 and codes.ndim == 2 and scales.dtype == torch.float32 and scales.ndim == 2,
                 "codes are uint8 [rows, padded columns], scales float32 [blocks, rows]")
        nb = -(-cols // BLOCK)
        _require(cols >= 0 and codes.shape[1] >= nb * BLOCK and scales.shape == (nb, codes.shape[0]),
                 f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold rows of {cols} columns")
        _require(codes.device == scales.device, "codes and scales lie on different devices")
        self.codes, self.scales, self.cols = codes, scales, cols

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.cols))

    @property
    def device(self):
        return self.codes.device

    def dequantize(self) -> torch.Tensor:
        """The values in float32."""
        wide = self.scales.t().repeat_interleave(BLOCK, 1)[:, :self.cols]
        return self.codes[:, :self.cols].contiguous().view(torch.float8_e4m3fn).float() * wide


class QuantWeight:
    """E4M3 weights: value[.., n, k] = codes[.., n, k] * scales[.., n // 128, k // 128].

    ``codes`` uint8 [n, >= padded] or [experts, n, >= padded], columns ``cols`` up to the next multiple of 128 holding
    code 0, rows 16-byte aligned; ``scales`` float32, contiguous.
    """

    __slots__ = ("codes", "scales", "cols")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int):
        _require(codes.dtype == torch.uint8 and codes.ndim in (2, 3) and scales.dtype == torch.float32,
                 "codes are uint8 [(experts,) n, padded columns], scales float32")
        nb = -(-cols // BLOCK)
        want = (*codes.shape[:-2], -(-codes.shape[-2] // BLOCK), nb)
        _require(cols >= 0 and codes.shape[-1] >= nb * BLOCK and scales.shape == want and scales.is_contiguous(),
                 f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold rows of {cols} columns")
        _require(codes.device == scales.device, "codes and scales lie on different devices")
        self.codes, self.scales, self.cols = codes, scales, cols

    @property
    def shape(self):
        return torch.Size((*self.codes.shape[:-1], self.cols))

    @property
    def device(self):
        return self.codes.device

    def dequantize(self) -> torch.Tensor:
        """The values in float32."""
        n = self.codes.shape[-2]
        wide = self.scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :self.cols]
        return self.codes[..., :self.cols].contiguous().view(torch.float8_e4m3fn).float() * wide


# ---- calls ---------------------------------------------------------------------------------------------
def _stream(device: torch.device, stream: Optional[torch.cuda.Stream]) -> int:
    if stream is None:
        return torch.cuda.current_stream(device).cuda_stream
    _require(stream.device == device, f"the stream belongs to {stream.device}, the tensors to {device}")
    return stream.cuda_stream


def _call(device: torch.device, fn, *args) -> None:
    if device.index == torch.cuda.current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(device):
            rc = fn(*args)
    if rc:
        L.check(rc)


def _new(shape, dtype, device, stream) -> torch.Tensor:
    """A result of a call on ``stream``: its memory may be reused for work on the current stream only, and the
    other stream's work is not awaited by it."""
    t = torch.empty(shape, dtype=dtype, device=device)
    if stream is not None:
        t.record_stream(stream)
    return t


def _on_device(t: torch.Tensor, device: torch.device, what: str) -> None:
    _require(t.device == device, f"{what} lies on {t.device}, not on {device}")


def quantize_rows(x: torch.Tensor, rows: Optional[torch.Tensor] = None, gated: bool = False,
                  stream: Optional[torch.cuda.Stream] = None) -> QuantRows:
    """[m, k] float16 / bfloat16 / float32 -> E4M3 rows with a scale for each 128 columns.

    ``rows`` (int32 indices) gathers: row r of the result is row rows[r] of ``x``, zeros where the index lies outside it.
    ``gated`` takes [m, 2 k] and quantises SiLU(a) * b of the two halves.  A block's scale is its largest finite
    magnitude / 448 (at least 2^-126); codes are to nearest, ties to even; a value that is not finite becomes NaN in
    its own place.  The columns of ``x`` have to be adjacent, its rows may lie anywhere.
    """
    dtype = _TYPES.get(x.dtype)
    _require(x.is_cuda and dtype is not None and x.ndim == 2 and (x.stride(1) == 1 or x.shape[1] <= 1),
             "x is a float16, bfloat16 or float32 matrix on a HIP device with adjacent columns")
    m, k = x.shape
    if gated:
        _require(k % 2 == 0, "a gated x has two halves of equal width")
        k //= 2
    device, n, index = x.device, m, 0
    if rows is not None:
        _on_device(rows, device, "rows")
        _require(rows.dtype == torch.int32 and rows.ndim == 1 and rows.is_contiguous(), "rows are contiguous int32 indices")
        n, index = rows.shape[0], rows.data_ptr()
    kb = -(-k // BLOCK)
    codes = _new((n, kb * BLOCK), torch.uint8, device, stream)
    scales = _new((kb, n), torch.float32, device, stream)
    if n and k:
        _call(device, L.lib().aeisu_quantize_rows, x.data_ptr(), dtype, m, x.stride(0), k, gated, index, n, codes.data_ptr(),
              kb * BLOCK, scales.data_ptr(), n, _stream(device, stream))
    return QuantRows(codes, scales, k)


def quantize_weight(w: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> QuantWeight:
    """[n, k] or [experts, n, k] float16 / bfloat16 / float32 -> E4M3 weights with a scale for each 128 x 128 tile,
    by the rule of ``quantize_rows``."""
    dtype = _TYPES.get(w.dtype)
    _require(w.is_cuda and dtype is not None and w.ndim in (2, 3) and (w.stride(-1) == 1 or w.shape[-1] <= 1),
             "w is a float16, bfloat16 or float32 [n, k] or [experts, n, k] on a HIP device with adjacent columns")
    n, k = w.shape[-2:]
    e = w.shape[0] if w.ndim == 3 else 1
    lead = w.shape[:-2]
    codes = _new((*lead, n, _blocks(k) * BLOCK), torch.uint8, w.device, stream)
    scales = _new((*lead, _blocks(n), _blocks(k)), torch.float32, w.device, stream)
    if codes.numel():
        _call(w.device, L.lib().aeisu_quantize_weight, w.data_ptr(), dtype, e, n, k, w.stride(0) if w.ndim == 3 else 0,
              w.stride(-2), codes.data_ptr(), scales.data_ptr(), _stream(w.device, stream))
    return QuantWeight(codes, scales, k)


def _product(x, w, offsets, bias, slope, out_dtype, out, stream) -> torch.Tensor:
    grouped = offsets is not None
    device = x.device
    if isinstance(x, QuantRows):
        _require(isinstance(w, QuantWeight), "quantised rows are multiplied by a QuantWeight")
        kind, xt, wt, k, wk = L.TYPE_E4M3, x.codes, w.codes, x.cols, w.cols
        x_scales, x_scales_stride, w_scales = x.scales.data_ptr(), x.scales.stride(0), w.scales.data_ptr()
        _require((x.scales.stride(1) == 1 or x.scales.shape[1] <= 1) and xt.stride(1) == 1 and wt.stride(-1) == 1,
                 "the columns of codes and the rows of scales have to be adjacent")
    else:
        _require(isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor) and x.dtype == w.dtype
                 and x.dtype in (torch.float16, torch.bfloat16) and x.ndim == 2,
                 "x and w are QuantRows and QuantWeight, or float16 / bfloat16 tensors of one type")
        kind, xt, wt, k, wk = _TYPES[x.dtype], x, w, x.shape[1], w.shape[-1]
        x_scales = x_scales_stride = w_scales = 0
        _require((x.stride(1) == 1 or k <= 1) and (w.stride(-1) == 1 or wk <= 1), "the columns of x and w have to be adjacent")
    _require(wt.ndim == (3 if grouped else 2), "w is [experts, n, k]" if grouped else "w is [n, k]")
    m, n = xt.shape[0], wt.shape[-2]
    _require(k == wk, f"x has {k} columns, w has {wk}")
    _require(xt.is_cuda and wt.device == device, "x and w lie on one HIP device")
    if out is None:
        out_dtype = out_dtype or (torch.float16 if kind == L.TYPE_E4M3 else x.dtype)
        _require(out_dtype in _TYPES, "results are float16, bfloat16 or float32")
        out = _new((m, n), out_dtype, device, stream)
    else:
        _on_device(out, device, "out")
        _require(out.shape == (m, n) and out.dtype in _TYPES and out_dtype in (None, out.dtype)
                 and (out.stride(1) == 1 or n <= 1) and (out.stride(0) >= n or m <= 1),
                 f"out is a [{m}, {n}] matrix of the result's type with adjacent columns")
    bp = 0
    if bias is not None:
        _on_device(bias, device, "bias")
        _require(bias.dtype == torch.float32 and bias.shape == wt.shape[:-1] and bias.is_contiguous(),
                 f"bias is contiguous float32 {tuple(wt.shape[:-1])}")
        bp = bias.data_ptr()
    _require(slope is None or 0 <= slope < float("inf"), "slope is a finite number, at least 0")
    if grouped:
        _on_device(offsets, device, "offsets")
        _require(offsets.dtype == torch.int32 and offsets.is_contiguous() and offsets.shape == (wt.shape[0] + 1,),
                 f"offsets are {wt.shape[0] + 1} contiguous int32 numbers")
        _require(wt.shape[0] >= 1, "there is at least one expert")
    if m == 0 or n == 0:
        return out
    p = L.Product(kind, _TYPES[out.dtype], m, n, k, xt.data_ptr(), xt.stride(0), x_scales, x_scales_stride, wt.data_ptr(),
                  wt.stride(-2), wt.stride(0) if grouped else 0, w_scales, bp, 1.0 if slope is None else slope,
                  out.data_ptr(), out.stride(0))
    if grouped:
        _call(device, L.lib().aeisu_grouped_matmul, ctypes.byref(p), offsets.data_ptr(), wt.shape[0], _stream(device, stream))
    else:
        _call(device, L.lib().aeisu_matmul, ctypes.byref(p), _stream(device, stream))
    return out


def matmul(x: QuantRows, w: QuantWeight, bias: Optional[torch.Tensor] = None, slope: Optional[float] = None,
           out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
           stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """act(x w^T + bias): [m, k] x [n, k] -> [m, n] in ``out_dtype`` (float16 unless given, or ``out``'s).

    ``bias`` float32 [n]; ``slope``: LeakyReLU of that slope.
    """
    _require(isinstance(x, QuantRows) and isinstance(w, QuantWeight), "x and w are a QuantRows and a QuantWeight")
    return _product(x, w, None, bias, slope, out_dtype, out, stream)


def grouped_matmul(x: Union[QuantRows, torch.Tensor], w: Union[QuantWeight, torch.Tensor], offsets: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, slope: Optional[float] = None,
                   out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                   stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Rows sorted by expert times each expert's weight: row m of expert e gives act(x[m] w[e]^T + bias[e]).

    Expert e has the rows offsets[e] <= m < offsets[e + 1]; ``offsets`` (int32 [experts + 1], on the device, not
    decreasing) is read by the kernel, so nothing waits for the host.  Rows of no expert give zeros.  ``x`` and ``w``
    are a ``QuantRows`` and a ``QuantWeight`` [experts, n, k], or float16 / bfloat16 tensors; ``bias`` float32
    [experts, n].  The result has ``out_dtype`` (unless given: ``out``'s, else float16 for E4M3 operands and theirs for others).
    """
    _require(isinstance(offsets, torch.Tensor), "offsets are an int32 tensor")
    return _product(x, w, offsets, bias, slope, out_dtype, out, stream)
