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


def _kept_bytes(m: int, n: int, k: int, keep_x: bool) -> int:
    rows = 2 * fp8._padded(n, 16) + 4 * 2 * -(-n // fp8.BLOCK)
    if keep_x:
        rows += fp8._padded(k, 16) + 4 * -(-k // fp8.BLOCK)
    return m * rows


def kept_copies(kept: torch.Tensor, m: int, n: int, k: int):
    """``(g, g_sf, u, u_sf, x, x_sf)``: the quantised matrices inside the buffer that ``keep="fp8"`` saves (``x`` and
    ``x_sf`` None if the weights need no gradient), in the form ``fp8.dequantize_fp8`` takes."""
    keep_x = kept.numel() != _kept_bytes(m, n, k, False)
    widths = (n, n, k) if keep_x else (n, n)
    codes, scales, at = [], [], 0
    for w in widths:
        pitch = fp8._padded(w, 16)
        codes.append(kept[at:at + m * pitch].view(m, pitch)[:, :w].view(fp8.E4M3))
        at += m * pitch
    for w in widths:
        blocks = -(-w // fp8.BLOCK)
        scales.append(kept[at:at + 4 * m * blocks].view(torch.float32).view(blocks, m).t())
        at += 4 * m * blocks
    out = [t for pair in zip(codes, scales) for t in pair]
    return tuple(out) if keep_x else (*out, None, None)


def _forward(x, w1, w2, act: int, kept, keep_x: bool):
    """h of matrices; ``kept`` None or the buffer to be filled."""
    m, k = x.shape
    n = w1.shape[0]
    device = x.device
    h = x.new_empty((m, n))
    if m == 0:
        return h
    pitch = fp8._row_pitch
    code = _lib.load().b200_gated_forward(x.data_ptr(), pitch(x), w1.data_ptr(), pitch(w1), w2.data_ptr(), pitch(w2),
                                          fp8._DTYPES[x.dtype], act, h.data_ptr(), n, None if kept is None else kept.data_ptr(),
                                          0 if kept is None else kept.numel(), keep_x, m, n, k, fp8._raw_stream(device.index),
                                          device.index, None)
    if code:
        _lib.check(code)
    return h


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w2, act, keep):
        ctx.act, ctx.keep = act, keep
        if keep == "inputs":
            ctx.save_for_backward(w1, w2, x)
            return _forward(x, w1, w2, act, None, False)
        m, k = x.shape
        keep_x = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        kept = torch.empty(_kept_bytes(m, w1.shape[0], k, keep_x), dtype=torch.uint8, device=x.device)
        ctx.save_for_backward(w1, w2, kept)
        return _forward(x, w1, w2, act, kept, keep_x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        w1, w2, saved = ctx.saved_tensors
        need_x, need_w1, need_w2 = ctx.needs_input_grad[:3]
        dh = _matrix(dh)
        m, n = dh.shape
        k = w1.shape[1]
        device = dh.device
        if m == 0:
            return (dh.new_empty((0, k)) if need_x else None, torch.zeros_like(w1) if need_w1 else None,
                    torch.zeros_like(w2) if need_w2 else None, None, None)
        dx = dh.new_empty((m, k)) if need_x else None
        dw1 = dh.new_empty((n, k)) if need_w1 else None
        dw2 = dh.new_empty((n, k)) if need_w2 else None
        address = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        pitch = fp8._row_pitch
        if ctx.keep == "inputs":
            source = (saved.data_ptr(), pitch(saved), None, 0, 0)
            nbytes = 4 * m * n
        else:
            source = (None, 0, saved.data_ptr(), saved.numel(), saved.numel() != _kept_bytes(m, n, k, False))
            nbytes = 4 * m * n + 2 * m * k
        scratch = dh.new_empty(nbytes // 2)
        code = _lib.load().b200_gated_backward(*source, w1.data_ptr(), pitch(w1), w2.data_ptr(), pitch(w2), fp8._DTYPES[dh.dtype],
                                               ctx.act, dh.data_ptr(), pitch(dh), address(dx), k, address(dw1), address(dw2), k,
                                               m, n, k, scratch.data_ptr(), nbytes, fp8._raw_stream(device.index),
                                               device.index, None)
        if code:
            _lib.check(code)
        return dx, dw1, dw2, None, None


def gated_ffn(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, *, activation: str = "silu", keep: str = "inputs") -> torch.Tensor:
    """``act(x @ w1.T) * (x @ w2.T)``, differentiable in x, w1 and w2.

    x           [..., k] fp16 / bf16
    w1, w2      [n, k], the gate's and the other projection's weights; n and k multiples of 8
    activation  "silu" or "gelu" (tanh form)
    keep        what the backward pass works from: "inputs" (x and the weights; the projections are
                formed again) or "fp8" (8-bit copies of x and of both projections)

    To capture a training step in a CUDA graph, let every eager graph of the same leaves go first and make one call
    outside the capture (autograd refuses to cross streams inside one, and the library sets itself up on its first call).

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
        h = _forward(x2, w1, w2, act, None, False)
    return h if x.dim() == 2 else h.view(*lead, w1.shape[0])
