"""fp8 block-128 quantisers and GEMM on the GPU against a 64-bit implementation.

Tolerances.  Codes and scales are compared bit for bit: the scale is one correctly rounded fp32 division, and
a quotient 448 x / a of 16-bit x and a is either half way between two codes exactly or at least 2^-16 of itself
away, far more than fp32 arithmetic errs.  For the GEMM, with S = sum |a_i b_i| over the whole row: a block of
128 is four fp32 accumulations of 32 exact products (each off by at most 2^-22 S: two bits below fp32's 24 for
the alignment of 32 addends), the factor s_A s_B one rounding, the sum over b blocks b + 1 fused multiply-adds:
(4 * 2^-22 + (b + 2) 2^-24) S; then half a step of the result's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def dense():
    from oracle import dense_oracle
    return dense_oracle


def _rand(shape, dtype, seed, spread=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    if spread:
        x = x * torch.exp2(spread * torch.randn((shape[0], 1), generator=g, device="cuda"))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 1000), (64, 4096), (257, 264), (1000, 8)])
def test_quantize_rows_bit_for_bit(pkg, dense, dtype, pow2, rows, k):
    x = _rand((rows, k), dtype, rows * 7 + k, spread=3.0)
    x[0, 0] = 0.0
    q, sf = pkg.fp8.quantize_fp8(x, pow2=pow2)
    codes, s = dense.quantize_rows(x, pow2)
    assert q.dtype == E4M3 and q.shape == (rows, k) and sf.shape == s.shape
    assert torch.equal(sf.double(), s)
    assert torch.equal(q.double(), codes)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_quantize_every_mantissa_against_every_maximum(pkg, dense, dtype):
    # all pairs of a maximum's mantissa (rows) and an element's mantissa: every tie that the type can form
    bits = 7 if dtype == BF16 else 10
    top = (1.0 + torch.arange(2 ** bits, device="cuda") / 2 ** bits) * 2
    el = 1.0 + torch.arange(2 ** bits, device="cuda") / 2 ** bits
    cols = 127
    for start in range(0, 2 ** bits, cols):
        part = el[start:start + cols]
        x = torch.cat([top[:, None], part[None, :].expand(len(top), -1)], dim=1).to(dtype)
        for scale in (1.0, 0.125):       # two places on the code grid
            y = x.clone()
            y[:, 1:] *= scale
            for pow2 in (False, True):
                q, sf = pkg.fp8.quantize_fp8(y, pow2=pow2)
                codes, s = dense.quantize_rows(y, pow2)
                assert torch.equal(sf.double(), s) and torch.equal(q.double(), codes)


@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_zeros_tiny_huge_and_not_finite(pkg, dense, pow2):
    x = torch.zeros((8, 256), dtype=BF16, device="cuda")
    x[1] = 2.0 ** -130                                  # below the floor: codes are zero
    x[2, :128] = 3.0e38
    x[2, 5] = -1.0e38
    x[3, 7] = float("nan")
    x[3, 8] = 2.0
    x[4, 9] = float("inf")
    x[4, 10] = 1.0
    x[5, 200] = 2.0 ** -100
    q, sf = pkg.fp8.quantize_fp8(x, pow2=pow2)
    codes, s = dense.quantize_rows(x[[0, 1, 2, 5, 6, 7]], pow2)
    assert torch.equal(q.double()[[0, 1, 2, 5, 6, 7]], codes) and torch.equal(sf.double()[[0, 1, 2, 5, 6, 7]], s)
    v = dense.row_values(q.float(), sf).float()
    assert torch.isnan(v[3, 7]) and v[3, 8] == 2.0 and torch.isfinite(v[3, 128:]).all()
    assert not torch.isfinite(v[4, 9]) and torch.isfinite(v[4, 128:]).all()
    if pow2:
        assert torch.isinf(v[4, 9])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 260), (1000, 72), (257, 1001)])
def test_quantize_weight_bit_for_bit(pkg, dense, dtype, n, k):
    w = _rand((n, k), dtype, n + k, spread=2.0)
    q, sf = pkg.fp8.quantize_fp8_weight(w)
    codes, s = dense.quantize_blocks(w)
    assert torch.equal(sf.double(), s) and torch.equal(q.double(), codes)


def test_quantize_strided_and_misaligned_inputs(pkg, dense):
    base = _rand((40, 777), BF16, 5)
    for x in (base[:, 8:400], base[::2, 3:260], base[:, :1]):
        for pow2 in (False, True):
            q, sf = pkg.fp8.quantize_fp8(x, pow2=pow2)
            codes, s = dense.quantize_rows(x, pow2)
            assert torch.equal(q.double(), codes) and torch.equal(sf.double(), s)
        q, sf = pkg.fp8.quantize_fp8_weight(x)
        codes, s = dense.quantize_blocks(x)
        assert torch.equal(q.double(), codes) and torch.equal(sf.double(), s)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_pow2_values_come_back_exactly(pkg, dense, dtype):
    x = _rand((33, 300), dtype, 9)
    q, sf = pkg.fp8.quantize_fp8(x, pow2=True)
    assert torch.equal(pkg.fp8.dequantize_fp8(q, sf, dtype).double(), dense.row_values(q.float(), sf))
    assert pkg.fp8.dequantize_fp8(q[:0], sf[:0], dtype).shape == (0, 300)


def _operands(pkg, m, n, k, seed, spread=1.0):
    a, sfa = pkg.fp8.quantize_fp8(_rand((m, k), BF16, seed, spread))
    b, sfb = pkg.fp8.quantize_fp8_weight(_rand((n, k), BF16, seed + 1, spread))
    return a, sfa, b, sfb


def _check_gemm(dense, got, a, sfa, b, sfb):
    av, bv = dense.row_values(a.float(), sfa), dense.block_values(b.float(), sfb)
    want, total = av @ bv.t(), av.abs() @ bv.abs().t()
    blocks = sfa.shape[1]
    tol = (4 * 2.0 ** -22 + (blocks + 2) * 2.0 ** -24) * total
    tol = tol + torch.finfo(got.dtype).eps / 2 * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), (got.double() - want).abs().max().item())


GEMM_SIZES = [(1, 8, 1), (1, 128, 128), (1, 4096, 2048), (2, 136, 130), (3, 264, 4000), (16, 512, 512), (17, 1032, 700),
              (31, 128, 7168), (33, 1024, 96), (64, 2048, 1000), (65, 384, 640), (100, 776, 1024), (127, 256, 255),
              (128, 640, 2048), (129, 136, 512), (200, 1000, 333), (256, 256, 128), (257, 264, 136), (300, 520, 2120),
              (511, 768, 1536), (700, 2056, 520), (1025, 512, 384), (2000, 1288, 264), (1100, 8200, 300), (2300, 2056, 1100),
              (600, 2600, 1300), (4500, 4104, 130)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", GEMM_SIZES)
def test_gemm(pkg, dense, dtype, m, n, k):
    a, sfa, b, sfb = _operands(pkg, m, n, k, m + n + k)
    out = torch.full((m + 2, n), 7.0, dtype=dtype, device="cuda")       # rows behind the last one stay as they were
    got = pkg.fp8.fp8_gemm(a, sfa, b, sfb, out=out[:m])
    _check_gemm(dense, got, a, sfa, b, sfb)
    assert (out[m:] == 7.0).all()
    assert torch.equal(pkg.fp8.fp8_gemm(a, sfa, b, sfb, out_dtype=dtype), got)
    assert pkg._lib.read_status(0) == 0


def test_gemm_strides_of_scales_operands_and_result(pkg, dense):
    m, n, k = 70, 264, 400
    a, sfa, b, sfb = _operands(pkg, m, n, k, 3)
    want = pkg.fp8.fp8_gemm(a, sfa, b, sfb)
    wide_a = torch.zeros((m, 512), dtype=torch.uint8, device="cuda")
    wide_a[:, 64:64 + k] = a.view(torch.uint8)
    wide_b = torch.zeros((2 * n, 448), dtype=torch.uint8, device="cuda")
    wide_b[::2, :k] = b.view(torch.uint8)
    out = torch.zeros((m, 2 * n), dtype=BF16, device="cuda")
    got = pkg.fp8.fp8_gemm(wide_a.view(E4M3)[:, 64:64 + k], sfa.contiguous(), wide_b.view(E4M3)[::2, :k],
                           torch.cat([sfb, sfb], 1)[:, :sfb.shape[1]], out=out[:, n:])
    assert torch.equal(got, want) and (out[:, :n] == 0).all()


def test_gemm_codes_and_scales_that_make_large_and_small_sums(pkg, dense):
    # blocks of very different scale: the sum over blocks must not lose the small ones where the large are zero
    m, n, k = 40, 256, 512
    x = _rand((m, k), BF16, 1)
    x[:, :128] *= 2.0 ** 40
    x[::2, :128] = 0
    a, sfa = pkg.fp8.quantize_fp8(x)
    b, sfb = pkg.fp8.quantize_fp8_weight(_rand((n, k), BF16, 2))
    _check_gemm(dense, pkg.fp8.fp8_gemm(a, sfa, b, sfb), a, sfa, b, sfb)


@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("m", [10, 50, 140, 700])
def test_what_is_not_finite_stays_in_its_row(pkg, m, bad):
    x = _rand((m, 384), BF16, 1)
    x[7, 200] = float(bad)
    b, sfb = pkg.fp8.quantize_fp8_weight(_rand((1032, 384), BF16, 2))
    y = pkg.fp8.fp8_linear(x, b, sfb)
    assert torch.isnan(y[7]).all() and torch.isfinite(y[[i for i in range(m) if i != 7]]).all()


def test_first_call_under_capture_is_refused():
    """In a process of its own: the set-up of a device cannot be captured, and says so before it touches the capture."""
    import subprocess
    import sys
    code = """
import importlib, torch
pkg = importlib.import_module("llm-assisted-kernel-dev_b200")
x = torch.ones((4, 128), dtype=torch.bfloat16, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    try:
        pkg.fp8.quantize_fp8(x)
        said = None
    except ValueError as e:
        said = e.code
    y = x + 1
assert said == pkg._lib.E_CAPTURE, said
g.replay()
q, sf = pkg.fp8.quantize_fp8(x)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    q, sf = pkg.fp8.quantize_fp8(x)
g.replay()
torch.cuda.synchronize()
assert (y == 2).all() and (pkg.fp8.dequantize_fp8(q, sf).float() - 1).abs().max() < 2 ** -8
print("fine")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("m", [1, 9, 130])
def test_linear_is_quantise_then_gemm(pkg, dense, m):
    x = _rand((m, 520), FP16, m)
    b, sfb = pkg.fp8.quantize_fp8_weight(_rand((264, 520), FP16, 2))
    q, sf = pkg.fp8.quantize_fp8(x)
    want = pkg.fp8.fp8_gemm(q, sf, b, sfb, out_dtype=FP16)
    assert torch.equal(pkg.fp8.fp8_linear(x, b, sfb), want)
    assert torch.equal(pkg.fp8.fp8_linear(x.view(1, m, 520), b, sfb), want.view(1, m, 264))
    out = torch.empty((m, 264), dtype=FP16, device="cuda")
    assert pkg.fp8.fp8_linear(x, b, sfb, out=out) is out and torch.equal(out, want)
    assert pkg.fp8.fp8_linear(x[:0], b, sfb).shape == (0, 264)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_on_another_stream_and_in_a_graph(pkg, m):
    x = _rand((m, 1024), BF16, 4)
    b, sfb = pkg.fp8.quantize_fp8_weight(_rand((512, 1024), BF16, 2))
    want = pkg.fp8.fp8_linear(x, b, sfb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = pkg.fp8.fp8_linear(x, b, sfb)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two captured graphs of the same layer, replayed on two streams at once
    graphs, inputs, outs = [], [], []
    for i in range(2):
        xi = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = pkg.fp8.fp8_linear(xi, b, sfb)
        graphs.append(g), inputs.append(xi), outs.append(y)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    other = _rand((m, 1024), BF16, 99)
    inputs[1].copy_(other)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], pkg.fp8.fp8_linear(other, b, sfb))
    assert pkg._lib.read_status(0) == 0


def test_same_bits_every_time(pkg):
    for m in (1, 33, 200, 900):
        x = _rand((m, 2048), BF16, m)
        b, sfb = pkg.fp8.quantize_fp8_weight(_rand((1032, 2048), BF16, 2))
        first = pkg.fp8.fp8_linear(x, b, sfb)
        for _ in range(5):
            assert torch.equal(pkg.fp8.fp8_linear(x, b, sfb), first)


def test_offsets_past_32_bits(pkg, dense):
    """2.2e9 elements: the last rows of codes, scales and product are those of the last rows alone."""
    m, k, n = 270_000, 8192, 128
    x = torch.empty((m, k), dtype=BF16, device="cuda")
    x[:-300] = 1.0
    x[-300:] = _rand((300, k), BF16, 1)
    q, sf = pkg.fp8.quantize_fp8(x)
    q1, sf1 = pkg.fp8.quantize_fp8(x[-300:].clone())
    assert torch.equal(q[-300:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(sf[-300:], sf1)
    b, sfb = pkg.fp8.quantize_fp8_weight(_rand((n, k), BF16, 2))
    y = pkg.fp8.fp8_gemm(q, sf, b, sfb)
    _check_gemm(dense, y[-300:], q1, sf1, b, sfb)
    assert torch.equal(y[0].expand(200, n), y[:200]) and torch.equal(y[0], y[-301])
    back = pkg.fp8.dequantize_fp8(q, sf)
    assert torch.equal(back[-300:], pkg.fp8.dequantize_fp8(q1, sf1)) and pkg._lib.read_status(0) == 0


def test_two_streams_at_once(pkg):
    b, sfb = pkg.fp8.quantize_fp8_weight(_rand((1032, 2048), BF16, 2))
    for m in (3, 60, 400):
        xs = [_rand((m, 2048), BF16, i) for i in range(2)]
        want = [pkg.fp8.fp8_linear(x, b, sfb) for x in xs]
        streams = [torch.cuda.Stream() for _ in xs]
        torch.cuda.synchronize()
        for _ in range(30):
            got = []
            for x, s in zip(xs, streams):
                with torch.cuda.stream(s):
                    got.append(pkg.fp8.fp8_linear(x, b, sfb))
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))


def test_refusals(pkg):
    x = _rand((8, 256), BF16, 1)
    b, sfb = pkg.fp8.quantize_fp8_weight(_rand((136, 256), BF16, 2))
    q, sf = pkg.fp8.quantize_fp8(x)
    bad = [
        (lambda: pkg.fp8.quantize_fp8(x.float()), "float16 or bfloat16"),
        (lambda: pkg.fp8.quantize_fp8(x[0]), "matrix"),
        (lambda: pkg.fp8.quantize_fp8(x.t()), "unit stride"),
        (lambda: pkg.fp8.quantize_fp8(x[:1].expand(8, 256)), "ldx=0"),
        (lambda: pkg.fp8.quantize_fp8_weight(x[:0]), "at least one row"),
        (lambda: pkg.fp8.fp8_gemm(q.float(), sf, b, sfb), "float8_e4m3fn"),
        (lambda: pkg.fp8.fp8_gemm(q, sf[:4], b, sfb), "scales of a"),
        (lambda: pkg.fp8.fp8_gemm(q, sf.half(), b, sfb), "float32"),
        (lambda: pkg.fp8.fp8_gemm(q, sf, b, sfb[:1]), "scales of the weight"),
        (lambda: pkg.fp8.fp8_gemm(q[:, :128], sf[:, :1], b, sfb), "k=256"),
        (lambda: pkg.fp8.fp8_gemm(q, sf, b[:132], sfb), "n=132"),
        (lambda: pkg.fp8.fp8_gemm(q, sf, b, sfb, out_dtype=torch.float32), "out must be"),
        (lambda: pkg.fp8.fp8_gemm(q, sf, b, sfb, out=torch.empty((8, 128), dtype=BF16, device="cuda")), "out must be"),
        (lambda: pkg.fp8.fp8_gemm(q, sf, b, sfb, out=torch.empty((8, 140), dtype=BF16, device="cuda")[:, 4:]), "16-byte"),
        (lambda: pkg.fp8.fp8_linear(x.requires_grad_(), b, sfb), "no backward pass"),
        (lambda: pkg.fp8.fp8_linear(x.detach()[:, :0], b, sfb), "k >= 1"),
        (lambda: pkg.fp8.fp8_linear(x.detach(), b, sfb, out=torch.empty((8, 136), dtype=FP16, device="cuda")), "out must be"),
    ]
    for call, needle in bad:
        with pytest.raises(ValueError, match=needle):
            call()
    with torch.no_grad():
        assert pkg.fp8.fp8_linear(x, b, sfb).shape == (8, 136)
    assert pkg.fp8.fp8_linear(x.detach()[0], b, sfb).shape == (136,)
