"""64-bit oracle of the fp8 block-128 linear layer and of the gated feed-forward block.

TEST INFRASTRUCTURE ONLY: imported by tests/ and nothing else.  Works on the device of its inputs."""
from __future__ import annotations

import math

import torch

BLOCK = 128
AMAX_FLOOR = 2.0 ** -100
GELU_A, GELU_B = math.sqrt(2.0 / math.pi), 0.044715


def e4m3_round(v: torch.Tensor) -> torch.Tensor:
    """v (float64) to the nearest e4m3 value, ties to even, saturating at 448 (no infinities)."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp_min(-9))     # four significant bits; 2^-9 below 2^-6
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def pow2_scale(amax: torch.Tensor) -> torch.Tensor:
    """Smallest power of two s with amax <= 448 s."""
    f, e = torch.frexp(amax / 448.0)
    return torch.ldexp(torch.ones_like(amax), torch.where(f == 0.5, e - 1, e))


def quantize_rows(x: torch.Tensor, pow2: bool):
    """(codes [rows, k] float64, scales [rows, blocks] float64; linear scales rounded to fp32 once)."""
    rows, k = x.shape
    nb = -(-k // BLOCK)
    p = torch.zeros((rows, nb * BLOCK), dtype=torch.float64, device=x.device)
    p[:, :k] = x
    p = p.view(rows, nb, BLOCK)
    a = p.abs().amax(dim=2, keepdim=True).clamp_min(AMAX_FLOOR)
    if pow2:
        s = pow2_scale(a)
        codes = e4m3_round(p / s)
    else:
        s = (a / 448.0).float().double()
        codes = e4m3_round(p * 448.0 / a)
    return codes.view(rows, -1)[:, :k], s.view(rows, nb)


def quantize_blocks(w: torch.Tensor):
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    p = torch.zeros((nb * BLOCK, kb * BLOCK), dtype=torch.float64, device=w.device)
    p[:n, :k] = w
    p = p.view(nb, BLOCK, kb, BLOCK)
    a = p.abs().amax(dim=(1, 3), keepdim=True).clamp_min(AMAX_FLOOR)
    codes = e4m3_round(p * 448.0 / a)
    return codes.view(nb * BLOCK, kb * BLOCK)[:n, :k], (a / 448.0).float().double().view(nb, kb)


def row_values(codes, s):
    k = codes.shape[1]
    return codes.double() * s.double().repeat_interleave(BLOCK, 1)[:, :k]


def block_values(codes, s):
    n, k = codes.shape
    return codes.double() * s.double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def gate(z: torch.Tensor, name: str):
    """act(z) and act'(z)."""
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1.0 + z * (1.0 - s))
    t = torch.tanh(GELU_A * (z + GELU_B * z ** 3))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_A * (1.0 + 3.0 * GELU_B * z * z)


def gated(x, w1, w2, name):
    return gate(x.double() @ w1.double().t(), name)[0] * (x.double() @ w2.double().t())


def gated_hidden_grads(g, u, dh, name):
    a, da = gate(g, name)
    return dh.double() * u * da, dh.double() * a
