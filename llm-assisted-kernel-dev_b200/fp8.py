"""Linear layers in 8-bit floating point with a scale for each block of 128, on B200.

A matrix is e4m3 codes and fp32 scales: activations have one scale for each row and 128 columns,
weights one for each 128 x 128 block (the format of the reference's experts,
moe/moe_fibench_ref.py:20-33).  ``fp8_linear`` quantises fp16 / bf16 activations and multiplies
them with a quantised weight; ``fp8_gemm`` takes both operands quantised.  The arithmetic runs in
libb200nvfp4.so (csrc/fp8_blocks.cuh, csrc/fp8_gemm_kernels.cuh); there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib

E4M3 = torch.float8_e4m3fn
BLOCK = 128
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _raw_stream(device_index: int) -> int:
    """cudaStream_t of the device's current stream."""
    return torch._C._cuda_getCurrentRawStream(device_index)


def _dtype_code(dtype: torch.dtype, name: str) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{name} must be float16 or bfloat16, got {dtype}")
    return code


def _check_activations(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise ValueError(f"{what} needs a CUDA tensor (there is no CPU path)")
    if x.dim() != 2 or x.shape[1] == 0 or (x.stride(1) != 1 and x.shape[1] > 1):
        raise ValueError(f"{what}: expected a matrix [rows, k >= 1] with unit stride along k")


def _row_pitch(t: torch.Tensor) -> int:
    """Row pitch in elements; the stride of a single row means nothing."""
    return t.stride(0) if t.shape[0] > 1 else _padded(t.shape[1], 16)


def _padded(n: int, to: int) -> int:
    return (n + to - 1) // to * to


def empty_rows(rows: int, k: int, device):
    """Uninitialised ``(q, sf)`` of a row-quantised [rows, k] matrix: code rows on 16-byte
    boundaries, scales stored block by block (the scales of one 128-wide block of consecutive
    rows are neighbours), seen as [rows, ceil(k / 128)]."""
    q = torch.empty((rows, _padded(k, 16)), dtype=torch.uint8, device=device)[:, :k].view(E4M3)
    sf = torch.empty((-(-k // BLOCK), rows), dtype=torch.float32, device=device).t()
    return q, sf


def quantize_fp8(x: torch.Tensor, *, pow2: bool = False):
    """x [rows, k] (fp16 or bf16, unit stride along k, any rows >= 0, k >= 1) -> ``(q, sf)``: ``q``
    [rows, k] e4m3 (row pitch padded to 16 bytes) and ``sf`` [rows, ceil(k / 128)] float32.

    With a = max(max |x|, 2^-100) of a row's 128 columns: ``sf = a / 448`` and ``q = e4m3(448 x / a)``;
    ``pow2=True``: ``sf`` the smallest power of two with ``a <= 448 sf`` and ``q = e4m3(x / sf)``."""
    _check_activations(x, "quantize_fp8")
    dtype = _dtype_code(x.dtype, "x")
    rows, k = x.shape
    q, sf = empty_rows(rows, k, x.device)
    if rows == 0:
        return q, sf
    code = _lib.load().b200_fp8_quantize_rows(x.data_ptr(), dtype, rows, k, _row_pitch(x), q.data_ptr(), _row_pitch(q),
                                              sf.data_ptr(), 1, rows, 1 if pow2 else 0,
                                              _raw_stream(x.device.index), x.device.index)
    _lib.check(code)
    return q, sf


def quantize_fp8_weight(w: torch.Tensor):
    """w [n, k] (fp16 or bf16, unit stride along k) -> ``(q, sf)``: ``q`` [n, k] e4m3 (row pitch
    padded to 16 bytes) and ``sf`` [ceil(n / 128), ceil(k / 128)] float32, one scale for each
    128 x 128 block by the first rule of ``quantize_fp8``."""
    _check_activations(w, "quantize_fp8_weight")
    dtype = _dtype_code(w.dtype, "w")
    n, k = w.shape
    if n == 0:
        raise ValueError("quantize_fp8_weight: a weight needs at least one row")
    q = torch.empty((n, _padded(k, 16)), dtype=torch.uint8, device=w.device)[:, :k].view(E4M3)
    sf = torch.empty((-(-n // BLOCK), -(-k // BLOCK)), dtype=torch.float32, device=w.device)
    code = _lib.load().b200_fp8_quantize_blocks(w.data_ptr(), dtype, n, k, _row_pitch(w), q.data_ptr(), _row_pitch(q),
                                                sf.data_ptr(), sf.stride(0), sf.stride(1),
                                                _raw_stream(w.device.index), w.device.index)
    _lib.check(code)
    return q, sf


def dequantize_fp8(q: torch.Tensor, sf: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Values of a row-quantised matrix, rounded to ``dtype`` (exact for ``pow2`` scales whose values it holds)."""
    _check_quantized(q, sf, q.shape[0], "q", "dequantize_fp8")
    rows, k = q.shape
    out = torch.empty((rows, k), dtype=dtype, device=q.device)
    code = _dtype_code(dtype, "dtype")
    if rows:
        _lib.check(_lib.load().b200_fp8_dequantize_rows(q.data_ptr(), _row_pitch(q), sf.data_ptr(), sf.stride(0), sf.stride(1),
                                                        rows, k, code, out.data_ptr(), k,
                                                        _raw_stream(q.device.index), q.device.index))
    return out


def _check_quantized(q, sf, sf_rows: int, name: str, what: str) -> None:
    if not q.is_cuda:
        raise ValueError(f"{what} needs CUDA tensors (there is no CPU path)")
    if q.dtype != E4M3:
        raise ValueError(f"{what}: {name} must be float8_e4m3fn, got {q.dtype}")
    if q.dim() != 2 or q.shape[1] == 0 or (q.shape[1] > 1 and q.stride(1) != 1):
        raise ValueError(f"{what}: {name} must be a matrix [rows, k >= 1] with unit stride along k")
    if sf.dtype != torch.float32 or sf.device != q.device:
        raise ValueError(f"{what}: the scales of {name} must be float32 on the same device")
    if tuple(sf.shape) != (sf_rows, -(-q.shape[1] // BLOCK)):
        raise ValueError(f"{what}: the scales of {name} must be {(sf_rows, -(-q.shape[1] // BLOCK))}, got {tuple(sf.shape)}")


def _check_weight(wq, wsf, k: int, device, what: str) -> None:
    _check_quantized(wq, wsf, -(-wq.shape[0] // BLOCK), "the weight", what)
    if wq.shape[1] != k:
        raise ValueError(f"{what}: the weight has k={wq.shape[1]}, the activations k={k}")
    if wq.device != device:
        raise ValueError(f"{what}: all tensors must live on the same CUDA device")


def _check_out(out, m: int, n: int, device, what: str) -> None:
    if tuple(out.shape) != (m, n) or out.stride(1) != 1 or out.device != device:
        raise ValueError(f"{what}: out must be [{m}, {n}] with unit stride along n on the activations' device")


def fp8_gemm(a: torch.Tensor, sfa: torch.Tensor, b: torch.Tensor, sfb: torch.Tensor, *, out: torch.Tensor | None = None,
             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``C [m, n] = values(a) @ values(b).T``.

    a, sfa   [m, k] e4m3 and [m, ceil(k / 128)] float32 (``quantize_fp8``); any strides of ``sfa``
    b, sfb   [n, k] e4m3 and [ceil(n / 128), ceil(k / 128)] float32 (``quantize_fp8_weight``)
    out      optional [m, n] fp16 / bf16, row pitch a multiple of 8; else allocated as ``out_dtype``

    Row pitches of ``a`` and ``b`` are multiples of 16, n of 8; m and k are free.  fp32 accumulation,
    one rounding.  Runs on the current stream, no synchronisation."""
    _check_quantized(a, sfa, a.shape[0], "a", "fp8_gemm")
    m, k = a.shape
    n = b.shape[0]
    _check_weight(b, sfb, k, a.device, "fp8_gemm")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    else:
        _check_out(out, m, n, a.device, "fp8_gemm")
    dtype = _dtype_code(out.dtype, "out")
    if m == 0:
        return out
    code = _lib.load().b200_fp8_gemm(a.data_ptr(), _row_pitch(a), sfa.data_ptr(), sfa.stride(0), sfa.stride(1), b.data_ptr(),
                                     _row_pitch(b), sfb.data_ptr(), sfb.stride(0), sfb.stride(1), out.data_ptr(),
                                     _row_pitch(out), dtype, m, n, k, _raw_stream(a.device.index),
                                     a.device.index, None)
    _lib.check(code)
    return out


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_sf: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``values(quantize_fp8(x)) @ values(weight).T`` in the type of ``x``.

    x                   [..., k] fp16 / bf16
    weight, weight_sf   [n, k] e4m3 and its 128 x 128 scales (``quantize_fp8_weight``)
    out                 optional [..., n] contiguous result

    A quantised weight is not trained: there is no gradient, and a call that would need one is refused."""
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("fp8_linear has no backward pass: call it under torch.no_grad() or with a detached input")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("fp8_linear: x must be [..., k] with k >= 1")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    m, k = x2.shape
    dtype, device = _DTYPES.get(x.dtype), x.device
    # a short call's time is the host's: one expression where everything is as it should be, the checks that say what is not otherwise
    if not (dtype is not None and x2.is_cuda and x2.stride(1) == 1 and weight.dtype is E4M3 and weight.dim() == 2
            and weight.shape[1] == k and weight.stride(1) == 1 and weight.device == device and weight_sf.dtype is torch.float32
            and weight_sf.device == device and weight_sf.shape == (-(-weight.shape[0] // BLOCK), -(-k // BLOCK))):
        _check_activations(x2, "fp8_linear")
        dtype = _dtype_code(x.dtype, "x")
        _check_weight(weight, weight_sf, k, device, "fp8_linear")
    n = weight.shape[0]
    if out is None:
        y = x2.new_empty((m, n))
    else:
        y = out if out.dim() == 2 else out.view(-1, out.shape[-1])
        _check_out(y, m, n, device, "fp8_linear")
        if out.dtype != x.dtype:
            raise ValueError(f"fp8_linear: out must be {x.dtype}, got {out.dtype}")
    if m:
        # up to 16 rows are quantised inside the product's kernel; scratch in elements of x's two bytes
        nbytes = m * ((k + 15) // 16 * 16) + 4 * m * -(-k // BLOCK) if m > 16 else 0
        scratch = x2.new_empty(nbytes // 2) if nbytes else None
        index = device.index
        code = _lib.load().b200_fp8_linear(x2.data_ptr(), x2.stride(0) if m > 1 else k, dtype, weight.data_ptr(), _row_pitch(weight),
                                           weight_sf.data_ptr(), weight_sf.stride(0), weight_sf.stride(1), y.data_ptr(),
                                           y.stride(0) if m > 1 else (n + 7) // 8 * 8, m, n, k,
                                           scratch.data_ptr() if nbytes else None, nbytes, _raw_stream(index), index, None)
        if code:
            _lib.check(code)
    if out is not None:
        return out
    return y if x.dim() == 2 else y.view(*x.shape[:-1], n)
