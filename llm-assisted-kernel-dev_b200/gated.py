"""Gated feed-forward block ``h = act(x @ w1.T) * (x @ w2.T)`` in fp16 / bf16 on B200, with its
backward pass: the trainable sibling of ``dual_gemm`` (same formula, dual_gemm/submission.py:596-611,
on unquantised operands).

``gated_ffn`` is differentiable.  Between the passes it keeps either nothing but its inputs and
forms the two projections again (``keep="inputs"``), or 8-bit copies of the input and of both
projections (``keep="fp8"``: 2 n + k bytes per row instead of the 4 n + 2 k of 16-bit copies; a
power-of-two scale for each row and 128 columns, see ``fp8.quantize_fp8``).  The arithmetic runs in
libb200nvfp4.so (csrc/gated_kernels.cuh); there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib, fp8

ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
KEEP = ("inputs", "fp8")


def _matrix(t: torch.Tensor) -> torch.Tensor:
    """A matrix the kernels can read in place (unit column stride, rows on 16-byte boundaries), copied if it is not."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] == 1 or t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _check(x, w1, w2, activation, keep="inputs"):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if keep not in KEEP:
        raise ValueError(f"keep must be one of {KEEP}, got {keep!r}")
    if not x.is_cuda:
        raise ValueError("the gated block needs CUDA tensors (there is no CPU path)")
    fp8._dtype_code(x.dtype, "x")
    if x.dim() < 1 or w1.dim() != 2 or w1.shape != w2.shape or x.shape[-1] != w1.shape[1]:
        raise ValueError(f"expected x [..., k], w1 [n, k], w2 [n, k]; got {tuple(x.shape)}, {tuple(w1.shape)}, {tuple(w2.shape)}")
    if w1.shape[0] % 8 or w1.shape[1] % 8 or w1.numel() == 0:
        raise ValueError(f"n={w1.shape[0]} and k={w1.shape[1]} must be positive multiples of 8")
    for t in (w1, w2):
        if t.dtype != x.dtype or t.device != x.device:
            raise ValueError("x, w1 and w2 must have one type and live on one device")


def _stream(t: torch.Tensor):
    index = t.device.index
    return fp8._raw_stream(index), index


def _mat(t: torch.Tensor):
    return t.data_ptr(), fp8._row_pitch(t)


def _forward(x, w1, w2, act: int, kept):
    """h of matrices; ``kept`` None or (qg, sg, qu, su) to be filled."""
    m, k = x.shape
    n = w1.shape[0]
    h = torch.empty((m, n), dtype=x.dtype, device=x.device)
    if m == 0:
        return h
    if kept is None:
        tail = (None, None, 0, None, None, 0, 0)
    else:
        qg, sg, qu, su = kept
        tail = (qg.data_ptr(), qu.data_ptr(), fp8._row_pitch(qg), sg.data_ptr(), su.data_ptr(), sg.stride(0), sg.stride(1))
    _lib.check(_lib.load().b200_gated_forward(*_mat(x), *_mat(w1), *_mat(w2), fp8._dtype_code(x.dtype, "x"), act, h.data_ptr(), n,
                                              *tail, m, n, k, *_stream(x), None))
    return h


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w2, act, keep):
        ctx.act, ctx.keep = act, keep
        if keep == "inputs":
            ctx.save_for_backward(x, w1, w2)
            return _forward(x, w1, w2, act, None)
        kept = (*fp8.empty_rows(x.shape[0], w1.shape[0], x.device), *fp8.empty_rows(x.shape[0], w1.shape[0], x.device))
        h = _forward(x, w1, w2, act, kept)
        qx, sx = fp8.quantize_fp8(x, pow2=True) if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else (None, None)
        ctx.save_for_backward(w1, w2, *kept, qx, sx)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        lib = _lib.load()
        dh = _matrix(dh)
        m, n = dh.shape
        dtype = fp8._dtype_code(dh.dtype, "dh")
        if ctx.keep == "inputs":
            x, w1, w2 = ctx.saved_tensors
        else:
            w1, w2, qg, sg, qu, su, qx, sx = ctx.saved_tensors
        k = w1.shape[1]
        need_x, need_w1, need_w2 = ctx.needs_input_grad[:3]
        if m == 0:
            return (dh.new_empty((0, k)) if need_x else None, torch.zeros_like(w1) if need_w1 else None,
                    torch.zeros_like(w2) if need_w2 else None, None, None)
        dg, du = torch.empty((m, n), dtype=dh.dtype, device=dh.device), torch.empty((m, n), dtype=dh.dtype, device=dh.device)
        if ctx.keep == "inputs":
            _lib.check(lib.b200_gated_grad_hidden(*_mat(x), *_mat(w1), *_mat(w2), dtype, ctx.act, *_mat(dh), dg.data_ptr(),
                                                  du.data_ptr(), n, m, n, k, *_stream(dh), None))
        else:
            _lib.check(lib.b200_gated_grad_hidden_kept(qg.data_ptr(), qu.data_ptr(), fp8._row_pitch(qg), sg.data_ptr(),
                                                       su.data_ptr(), sg.stride(0), sg.stride(1), dtype, ctx.act, *_mat(dh),
                                                       dg.data_ptr(), du.data_ptr(), n, m, n, *_stream(dh)))
        dx = dw1 = dw2 = None
        if need_x:
            dx = torch.empty((m, k), dtype=dh.dtype, device=dh.device)
            _lib.check(lib.b200_gated_grad_input(dg.data_ptr(), du.data_ptr(), n, *_mat(w1), *_mat(w2), dtype, dx.data_ptr(), k,
                                                 m, n, k, *_stream(dh), None))
        if need_w1 or need_w2:
            if ctx.keep == "fp8":
                x = fp8.dequantize_fp8(qx, sx, dh.dtype)
            dw1 = torch.empty((n, k), dtype=dh.dtype, device=dh.device)
            dw2 = torch.empty((n, k), dtype=dh.dtype, device=dh.device)
            _lib.check(lib.b200_gated_grad_weight(dg.data_ptr(), du.data_ptr(), n, *_mat(x), dtype, dw1.data_ptr(),
                                                  dw2.data_ptr(), k, m, n, k, *_stream(dh), None))
        return dx, dw1 if need_w1 else None, dw2 if need_w2 else None, None, None


def gated_ffn(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, *, activation: str = "silu", keep: str = "inputs") -> torch.Tensor:
    """``act(x @ w1.T) * (x @ w2.T)``, differentiable in x, w1 and w2.

    x           [..., k] fp16 / bf16
    w1, w2      [n, k], the gate's and the other projection's weights; n and k multiples of 8
    activation  "silu" or "gelu" (tanh form)
    keep        what the backward pass works from: "inputs" (x and the weights; the projections are
                formed again) or "fp8" (8-bit copies of x and of both projections)

    fp32 accumulation and gate, one rounding for each of h, dx, dw1, dw2 and for the gradients of the
    two projections, which are operands of the last three.  Runs on the current stream, no synchronisation."""
    _check(x, w1, w2, activation, keep)
    lead = x.shape[:-1]
    x2 = _matrix(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    w1, w2 = _matrix(w1), _matrix(w2)
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or w1.requires_grad or w2.requires_grad):
        h = _GatedFfn.apply(x2, w1, w2, act, keep)
    else:
        h = _forward(x2, w1, w2, act, None)
    return h if x.dim() == 2 else h.view(*lead, w1.shape[0])
