"""Cases, plain forms and 64-bit definitions of the fp8 block-128 linear layer and of the gated
feed-forward block with its backward pass (inputs kept, or activations kept in 8 bits).

    fp8      y = (q_x . s_x) (q_w . s_w)^T   x is quantised on the way: one fp32 scale for each row and
             128 columns; the weight holds e4m3 codes with one scale for each 128 x 128 block
    gated    h = act(x w1^T) * (x w2^T)
    train    h and, for a given dh, dx, dw1, dw2.  keep = "inputs": the two projections are formed again;
             keep = "fp8": x and both projections are kept as e4m3 with a power-of-two scale for each row
             and 128 columns, and the backward pass works on the values that these stand for
"""
import importlib
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100      # a block of zeros gets this in place of its largest magnitude
GELU_A = math.sqrt(2.0 / math.pi)
GELU_B = 0.044715


def _pkg():
    return importlib.import_module("llm-assisted-kernel-dev_b200")


def listed():
    return [
        # one token of a decoding sequence, quantised projection: the weight's bytes are all there is
        {"name": "fp8 m1 n4096 k7168", "op": "fp8", "type": "bf16", "m": 1, "n": 4096, "k": 7168},
        # a decoding batch of 48 sequences on a smaller projection
        {"name": "fp8 m48 n7168 k2048 fp16", "op": "fp8", "type": "fp16", "m": 48, "n": 7168, "k": 2048},
        # a short prompt: the shape of the dual GEMM's skinny benchmark
        {"name": "fp8 m256 n4096 k7168", "op": "fp8", "type": "bf16", "m": 256, "n": 4096, "k": 7168},
        # a ragged batch of prompts, no size a multiple of a tile, the last block of k not full
        {"name": "fp8 m1999 n5000 k2120 fp16", "op": "fp8", "type": "fp16", "m": 1999, "n": 5000, "k": 2120},
        # a long prompt through the feed-forward projection of the headline benchmark
        {"name": "fp8 m8192 n14336 k4096", "op": "fp8", "type": "bf16", "m": 8192, "n": 14336, "k": 4096},
        # one token through the gated block
        {"name": "gated m1 n14336 k4096", "op": "gated", "type": "bf16", "act": "silu", "m": 1, "n": 14336, "k": 4096},
        # a decoding batch through the gated block
        {"name": "gated m100 n4096 k7168 fp16", "op": "gated", "type": "fp16", "act": "gelu", "m": 100, "n": 4096, "k": 7168},
        # a long prompt through the gated block
        {"name": "gated m8192 n14336 k4096", "op": "gated", "type": "bf16", "act": "silu", "m": 8192, "n": 14336, "k": 4096},
        # training on a short batch, nothing but the inputs kept
        {"name": "train m512 n4096 k7168", "op": "train", "type": "bf16", "act": "silu", "keep": "inputs",
         "m": 512, "n": 4096, "k": 7168},
        # training on a packed batch of odd length, ragged widths
        {"name": "train m1237 n2056 k1544 fp16", "op": "train", "type": "fp16", "act": "gelu", "keep": "inputs",
         "m": 1237, "n": 2056, "k": 1544},
        # training with the activations kept in 8 bits, an ordinary and a large step
        {"name": "train8 m2048 n4096 k7168", "op": "train", "type": "bf16", "act": "silu", "keep": "fp8",
         "m": 2048, "n": 4096, "k": 7168},
        {"name": "train8 m8192 n14336 k4096", "op": "train", "type": "bf16", "act": "silu", "keep": "fp8",
         "m": 8192, "n": 14336, "k": 4096},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["fp8", "fp8", "gated", "train", "train"])
    m = _spread(rng, 1 if op != "train" else 64, 8192)
    n = max(8, _spread(rng, 512, 14336) // 8 * 8)
    k = max(8, _spread(rng, 512, 7168) // 8 * 8)
    if rng.random() < 0.4:                     # widths in whole blocks, as most models have them
        n, k = max(BLOCK, n // BLOCK * BLOCK), max(BLOCK, k // BLOCK * BLOCK)
    while m * n * k > 8192 * 14336 * 4096:
        m //= 2
    case = {"op": op, "type": rng.choice(["bf16", "bf16", "fp16"]), "m": m, "n": n, "k": k}
    if op != "fp8":
        case["act"] = rng.choice(["silu", "silu", "gelu"])
    if op == "train":
        case["keep"] = rng.choice(["inputs", "fp8"])
    return case


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def _blocks(t, rows, cols):
    """t [r, c] -> [r/rows, rows, c/cols, cols], zeros behind the last row and column."""
    r, c = t.shape
    t = torch.nn.functional.pad(t, (0, -c % cols, 0, -r % rows))
    return t.reshape(t.shape[0] // rows, rows, t.shape[1] // cols, cols)


def _codes(b, amax):
    """448 b / amax as e4m3.  Both factors are exact, so that a quotient half way between two codes is met exactly."""
    return ((b * (E4M3_MAX / 512.0)) / (amax / 512.0)).to(torch.float8_e4m3fn)


def _quantized_weight(w):
    """e4m3 codes [n, k] (rows start on 16-byte boundaries) and fp32 scales [n/128, k/128] of w [n, k]."""
    n, k = w.shape
    b = _blocks(w.float(), BLOCK, BLOCK)
    amax = b.abs().amax(dim=(1, 3)).clamp_min(AMAX_FLOOR)
    codes = _codes(b, amax[:, None, :, None]).reshape(b.shape[0] * BLOCK, b.shape[2] * BLOCK)[:n]
    out = torch.empty((n, (k + 15) // 16 * 16), dtype=torch.float8_e4m3fn, device=w.device)
    out[:, :k] = codes[:, :k]
    return out[:, :k], amax / E4M3_MAX


def _inputs(case, seed):
    dev = "cuda"
    dtype = TYPES[case["type"]]
    m, n, k = case["m"], case["n"], case["k"]
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    # activations behind a norm: unit variance, a few channels much larger than the rest
    channel = torch.ones(k, device=dev)
    channel[torch.randint(0, k, (max(1, k // 256),), generator=gen, device=dev)] = 8.0
    x = (torch.randn((m, k), generator=gen, device=dev) * channel).to(dtype)
    w1 = (torch.randn((n, k), generator=gen, device=dev) * k ** -0.5).to(dtype)
    if case["op"] == "fp8":
        return x, w1
    w2 = (torch.randn((n, k), generator=gen, device=dev) * k ** -0.5).to(dtype)
    if case["op"] == "gated":
        return x, w1, w2
    dh = (torch.randn((m, n), generator=gen, device=dev) * n ** -0.5).to(dtype)
    return x, w1, w2, dh


def prepare(case, seed):
    given = _inputs(case, seed)
    state = {"case": case, "x": given[0]}
    if case["op"] == "fp8":
        state["wq"], state["ws"] = _quantized_weight(given[1])
        return state
    state["w1"], state["w2"] = given[1], given[2]
    if case["op"] == "train":
        state["dh"] = given[3]
        for name in ("x", "w1", "w2"):
            state[name].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------
def _fp8_values(x):
    """What x [m, k] stands for as e4m3 with one scale for each row and 128 columns."""
    m, k = x.shape
    b = _blocks(x.float(), 1, BLOCK)
    amax = b.abs().amax(dim=3, keepdim=True).clamp_min(AMAX_FLOOR)
    values = _codes(b, amax).float() * (amax / E4M3_MAX)
    return values.reshape(m, -1)[:, :k]


def _kept_values(x):
    """The same with the smallest power of two that brings the block's largest magnitude to 448 or below."""
    m, k = x.shape
    b = _blocks(x.float(), 1, BLOCK)
    amax = b.abs().amax(dim=3, keepdim=True).clamp_min(AMAX_FLOOR)
    fraction, exponent = torch.frexp(amax)                 # amax = fraction 2^exponent, 1/2 <= fraction < 1
    exponent = exponent - 9 + (fraction > 0.875).int()     # 448 = 0.875 * 2^9
    scale = torch.ldexp(torch.ones_like(amax), exponent)
    values = (b / scale).to(torch.float8_e4m3fn).float() * scale
    return values.reshape(m, -1)[:, :k]


def _act(g, name):
    """act(g) and its derivative."""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    t = torch.tanh(GELU_A * (g + GELU_B * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * GELU_A * (1.0 + 3.0 * GELU_B * g * g)


def _plain_fp8(s):
    k = s["x"].shape[1]
    n = s["wq"].shape[0]
    scale = s["ws"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return (_fp8_values(s["x"]) @ (s["wq"].float() * scale).t()).to(s["x"].dtype)


def _plain_gated(s):
    x = s["x"].float()
    a, _ = _act(x @ s["w1"].float().t(), s["case"]["act"])
    return (a * (x @ s["w2"].float().t())).to(s["x"].dtype)


def _plain_train(s):
    dtype, act = s["x"].dtype, s["case"]["act"]
    x, w1, w2, dh = (s[name].detach().float() for name in ("x", "w1", "w2", "dh"))
    g, u = x @ w1.t(), x @ w2.t()
    h = _act(g, act)[0] * u
    if s["case"]["keep"] == "fp8":
        x, g, u = _kept_values(x), _kept_values(g), _kept_values(u)
    a, da = _act(g, act)
    dg, du = dh * u * da, dh * a
    return {"h": h.to(dtype), "dx": (dg @ w1 + du @ w2).to(dtype), "dw1": (dg.t() @ x).to(dtype),
            "dw2": (du.t() @ x).to(dtype)}


def run(state):
    case = state["case"]
    if case["op"] == "fp8":
        if own:
            return _pkg().fp8.fp8_linear(state["x"], state["wq"], state["ws"])
        return _plain_fp8(state)
    if case["op"] == "gated":
        if own:
            return _pkg().gated.gated_ffn(state["x"], state["w1"], state["w2"], activation=case["act"])
        return _plain_gated(state)
    if own:
        leaves = (state["x"], state["w1"], state["w2"])
        h = _pkg().gated.gated_ffn(*leaves, activation=case["act"], keep=case["keep"])
        dx, dw1, dw2 = torch.autograd.grad(h, leaves, state["dh"])
        return {"h": h.detach(), "dx": dx, "dw1": dw1, "dw2": dw2}
    return _plain_train(state)


def work(case):
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "fp8":
        scales = 4 * -(-n // BLOCK) * -(-k // BLOCK)
        return {"bytes": 2 * m * k + n * k + scales + 2 * m * n, "flops": 2 * m * n * k}
    if case["op"] == "gated":
        return {"bytes": 2 * (m * k + 2 * n * k + m * n), "flops": 4 * m * n * k}
    # x, w1, w2, dh in; h, dx, dw1, dw2 out; two products forward, two for dx, one for each weight
    return {"bytes": 2 * (2 * m * k + 4 * n * k + 2 * m * n), "flops": 12 * m * n * k}


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _e4m3_64(v):
    """v (float64, |v| <= 448 (1 + 2^-20)) rounded to the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(v)                                  # |v| in [2^(e-1), 2^e): four significant bits
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp_min(-9))
    return torch.round(v / step) * step


def _quantized_64(x, power_of_two):
    m, k = x.shape
    columns = -(-k // BLOCK) * BLOCK
    padded = torch.zeros((m, columns), dtype=torch.float64, device=x.device)
    padded[:, :k] = x
    padded = padded.view(m, columns // BLOCK, BLOCK)
    top = padded.abs().max(dim=2).values.clamp_min(AMAX_FLOOR)[:, :, None]
    if power_of_two:
        f, e = torch.frexp(top / E4M3_MAX)                 # in (2^(e-1), 2^e], or a power of two itself
        scale = torch.where(f == 0.5, torch.ldexp(torch.ones_like(f), e - 1), torch.ldexp(torch.ones_like(f), e))
        values = _e4m3_64(padded / scale) * scale
    else:
        values = _e4m3_64(padded * E4M3_MAX / top) * (top / E4M3_MAX)
    return values.view(m, columns)[:, :k]


def exact(case, seed):
    with torch.no_grad():
        given = [t.detach() for t in _inputs(case, seed)]
        x = given[0].double()
        if case["op"] == "fp8":
            wq, ws = _quantized_weight(given[1])
            w = wq.double()
            n, k = w.shape
            rows = torch.arange(n, device=w.device) // BLOCK
            cols = torch.arange(k, device=w.device) // BLOCK
            return _quantized_64(x, False) @ (w * ws.double()[rows][:, cols]).t()
        w1, w2 = given[1].double(), given[2].double()
        g, u = torch.mm(x, w1.t()), torch.mm(x, w2.t())

        def gate(v):
            """value and slope of the activation"""
            if case["act"] == "silu":
                p = torch.sigmoid(v)
                return v * p, p + v * p * (1.0 - p)
            inner = GELU_A * (v + GELU_B * v ** 3)
            th = torch.tanh(inner)
            return 0.5 * v * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * v * (1.0 - th ** 2) * GELU_A * (1.0 + 3.0 * GELU_B * v ** 2)

        h = gate(g)[0] * u
        if case["op"] == "gated":
            return h
        dh = given[3].double()
        if case["keep"] == "fp8":
            x, g, u = _quantized_64(x, True), _quantized_64(g, True), _quantized_64(u, True)
        value, slope = gate(g)
        dg, du = dh * u * slope, dh * value
        return {"h": h, "dx": torch.mm(dg, w1) + torch.mm(du, w2), "dw1": torch.mm(dg.t(), x), "dw2": torch.mm(du.t(), x)}
