"""The fp8 block-128 GEMM and the gated feed-forward block without a GPU: bad arguments are rejected on the host
before any CUDA work, and the 64-bit oracle agrees with torch's own e4m3 and with its autograd."""
import pytest
import torch

FAKE = 0x7F0000000000  # 16-byte aligned fake device address; never dereferenced on the host
NULL, SHAPE, ALIGN, VARIANT, LIMIT = -1, -2, -3, -5, -7


@pytest.fixture(scope="module")
def dense():
    from oracle import dense_oracle
    return dense_oracle


@pytest.fixture()
def lib(pkg):
    return pkg._lib.load()


def _rejected(lib, rc, code, needle):
    assert rc == code and needle in lib.b200_last_error().decode(), (rc, lib.b200_last_error())


@pytest.mark.parametrize("kw,code,needle", [
    (dict(x=None), NULL, "NULL"), (dict(sf=None), NULL, "NULL"), (dict(q=None), NULL, "q is NULL"), (dict(dtype=2), VARIANT, "dtype 2"),
    (dict(rows=0), SHAPE, "positive"), (dict(k=0), SHAPE, "positive"), (dict(rows=-4), SHAPE, "positive"), (dict(ldx=255), ALIGN, "ldx=255"),
    (dict(q=FAKE + 8), ALIGN, "16-byte"), (dict(ldq=264), ALIGN, "pitch 264"), (dict(ldq=240), ALIGN, "pitch 240"),
])
def test_quantize_rows_refusals(lib, kw, code, needle):
    a = dict(x=FAKE, dtype=1, rows=4, k=256, ldx=256, q=FAKE + 4096, ldq=256, sf=FAKE + 8192)
    a.update(kw)
    _rejected(lib, lib.b200_fp8_quantize_rows(a["x"], a["dtype"], a["rows"], a["k"], a["ldx"], a["q"], a["ldq"], a["sf"], 1, 4, 0, None, 0),
              code, needle)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(w=None), NULL, "NULL"), (dict(dtype=-1), VARIANT, "dtype -1"), (dict(n=0), SHAPE, "positive"), (dict(ldw=100), ALIGN, "ldw=100"),
    (dict(ldq=248), ALIGN, "pitch 248"), (dict(n=65536 * 128), LIMIT, "more than"),
])
def test_quantize_blocks_refusals(lib, kw, code, needle):
    a = dict(w=FAKE, dtype=1, n=128, k=256, ldw=256, q=FAKE + 4096, ldq=256, sf=FAKE + 8192)
    a.update(kw)
    _rejected(lib, lib.b200_fp8_quantize_blocks(a["w"], a["dtype"], a["n"], a["k"], a["ldw"], a["q"], a["ldq"], a["sf"], 2, 1, None, 0),
              code, needle)


def test_dequantize_refusals(lib):
    f = lambda q=FAKE, ldq=256, sf=FAKE, rows=4, k=256, dtype=1, out=FAKE, ldo=256: lib.b200_fp8_dequantize_rows(  # noqa: E731
        q, ldq, sf, 1, 4, rows, k, dtype, out, ldo, None, 0)
    _rejected(lib, f(q=None), NULL, "q is NULL")
    _rejected(lib, f(out=None), NULL, "NULL")
    _rejected(lib, f(dtype=7), VARIANT, "dtype 7")
    _rejected(lib, f(rows=0), SHAPE, "positive")
    _rejected(lib, f(ldo=255), ALIGN, "ldo=255")
    _rejected(lib, f(q=FAKE + 1), ALIGN, "16-byte")


@pytest.mark.parametrize("kw,code,needle", [
    (dict(a=None), NULL, "a is NULL"), (dict(b=None), NULL, "b is NULL"), (dict(c=None), NULL, "c is NULL"),
    (dict(sfa=None), NULL, "scale"), (dict(sfb=None), NULL, "scale"), (dict(dtype=3), VARIANT, "dtype 3"),
    (dict(m=0), SHAPE, "positive"), (dict(n=0), SHAPE, "positive"), (dict(k=-1), SHAPE, "positive"), (dict(n=132, ldc=136), SHAPE, "n=132"),
    (dict(lda=250), ALIGN, "of a"), (dict(lda=264), ALIGN, "of a"), (dict(ldb=264), ALIGN, "of b"), (dict(ldc=120), ALIGN, "of c"),
    (dict(ldc=132), ALIGN, "of c"), (dict(a=FAKE + 4), ALIGN, "a must be 16-byte"), (dict(c=FAKE + 2), ALIGN, "c must be 16-byte"),
])
def test_gemm_refusals(lib, kw, code, needle):
    v = dict(a=FAKE, lda=256, sfa=FAKE, b=FAKE + 4096, ldb=256, sfb=FAKE, c=FAKE + 8192, ldc=128, dtype=1, m=4, n=128, k=256)
    v.update(kw)
    _rejected(lib, lib.b200_fp8_gemm(v["a"], v["lda"], v["sfa"], 1, 4, v["b"], v["ldb"], v["sfb"], 2, 1, v["c"], v["ldc"], v["dtype"],
                                     v["m"], v["n"], v["k"], None, 0, None), code, needle)


GATED_BAD = [
    (dict(x=None), NULL, "x is NULL"), (dict(w1=None), NULL, "w1 is NULL"), (dict(w2=None), NULL, "w2 is NULL"), (dict(dtype=4), VARIANT, "dtype 4"),
    (dict(act=2), VARIANT, "activation 2"), (dict(m=0), SHAPE, "positive"), (dict(n=0), SHAPE, "positive"), (dict(n=100), SHAPE, "n=100"),
    (dict(k=68), SHAPE, "k=68"), (dict(ldx=60), ALIGN, "of x"), (dict(ldx=68), ALIGN, "of x"), (dict(ldw=68), ALIGN, "of w1"),
    (dict(x=FAKE + 2), ALIGN, "x must be"), (dict(out=None), NULL, "NULL"), (dict(ld_out=100), ALIGN, "pitch 100"),
]


def _gated_args(kw):
    v = dict(x=FAKE, ldx=64, w1=FAKE + 4096, w2=FAKE + 8192, ldw=64, dtype=1, act=0, out=FAKE + 65536, ld_out=128, m=4, n=128, k=64)
    v.update(kw)
    return v


@pytest.mark.parametrize("kw,code,needle", GATED_BAD)
def test_gated_forward_refusals(lib, kw, code, needle):
    v = _gated_args(kw)
    _rejected(lib, lib.b200_gated_forward(v["x"], v["ldx"], v["w1"], v["ldw"], v["w2"], v["ldw"], v["dtype"], v["act"], v["out"], v["ld_out"],
                                          None, None, 0, None, None, 0, 0, v["m"], v["n"], v["k"], None, 0, None), code, needle)


def test_gated_forward_kept_copies_refusals(lib):
    def f(qg=FAKE, qu=FAKE, ldq=128, sg=FAKE, su=FAKE):
        return lib.b200_gated_forward(FAKE, 64, FAKE, 64, FAKE, 64, 1, 0, FAKE, 128, qg, qu, ldq, sg, su, 1, 4, 4, 128, 64, None, 0, None)
    _rejected(lib, f(qu=None), NULL, "qu is NULL")
    _rejected(lib, f(sg=None), NULL, "scales")
    _rejected(lib, f(ldq=136), ALIGN, "qg")
    _rejected(lib, f(qg=FAKE + 8), ALIGN, "qg must be")


@pytest.mark.parametrize("kw,code,needle", GATED_BAD)
def test_gated_grad_hidden_refusals(lib, kw, code, needle):
    v = _gated_args(kw)
    _rejected(lib, lib.b200_gated_grad_hidden(v["x"], v["ldx"], v["w1"], v["ldw"], v["w2"], v["ldw"], v["dtype"], v["act"], FAKE, 128,
                                              v["out"], v["out"], v["ld_out"], v["m"], v["n"], v["k"], None, 0, None), code, needle)


def test_gated_other_gradient_refusals(lib):
    kept = lambda qg=FAKE, ldq=128, sg=FAKE, act=0, dh=FAKE, ld=128, n=128, m=4: lib.b200_gated_grad_hidden_kept(  # noqa: E731
        qg, FAKE, ldq, sg, FAKE, 1, 4, 1, act, dh, ld, FAKE, FAKE, 128, m, n, None, 0)
    _rejected(lib, kept(qg=None), NULL, "qg is NULL")
    _rejected(lib, kept(sg=None), NULL, "scale")
    _rejected(lib, kept(act=5), VARIANT, "activation 5")
    _rejected(lib, kept(n=100), SHAPE, "n=100")
    _rejected(lib, kept(m=0), SHAPE, "positive")
    _rejected(lib, kept(ldq=120), ALIGN, "of qg")
    _rejected(lib, kept(ld=100), ALIGN, "of dh")
    dx = lambda dg=FAKE, ld=128, ldw=64, out=FAKE, ldo=64, m=4, n=128, k=64, dtype=1: lib.b200_gated_grad_input(  # noqa: E731
        dg, FAKE, ld, FAKE, ldw, FAKE, ldw, dtype, out, ldo, m, n, k, None, 0, None)
    dw = lambda dg=FAKE, ld=128, ldw=64, out=FAKE, ldo=64, m=4, n=128, k=64, dtype=1: lib.b200_gated_grad_weight(  # noqa: E731
        dg, FAKE, ld, FAKE, ldw, dtype, out, FAKE, ldo, m, n, k, None, 0, None)
    for f in (dx, dw):
        _rejected(lib, f(dg=None), NULL, "dg is NULL")
        _rejected(lib, f(out=None), NULL, "is NULL")
        _rejected(lib, f(ld=100), ALIGN, "of dg")
        _rejected(lib, f(ldw=60), ALIGN, "pitch 60")
        _rejected(lib, f(ldo=60), ALIGN, "pitch 60")
        _rejected(lib, f(m=0), SHAPE, "positive")
        _rejected(lib, f(n=12), SHAPE, "n=12")
        _rejected(lib, f(dtype=9), VARIANT, "dtype 9")


def test_no_cpu_path(pkg):
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(128, 64, dtype=torch.bfloat16)
    for call in (lambda: pkg.fp8.quantize_fp8(x), lambda: pkg.fp8.quantize_fp8_weight(w), lambda: pkg.gated.gated_ffn(x, w, w)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    q, s = torch.zeros(4, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(4, 1)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.fp8.fp8_gemm(q, s, q, s[:1])
    with pytest.raises(ValueError, match="CUDA"):
        pkg.fp8.fp8_linear(x, q, s[:1])
    with pytest.raises(ValueError, match="CUDA"):
        pkg.fp8.dequantize_fp8(q, s)


def test_gated_argument_names_are_checked_first(pkg):
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(128, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="activation"):
        pkg.gated.gated_ffn(x, w, w, activation="relu")
    with pytest.raises(ValueError, match="keep"):
        pkg.gated.gated_ffn(x, w, w, keep="bf16")


def test_oracle_rounds_like_torchs_e4m3(dense):
    v = torch.cat([torch.linspace(-448, 448, 40001), torch.linspace(-0.05, 0.05, 20001)]).float()
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    codes = codes[torch.isfinite(codes)].sort().values
    v = torch.cat([v, codes, (codes[1:] + codes[:-1]) / 2])         # every code and every half-way point
    assert torch.equal(dense.e4m3_round(v.double()), v.to(torch.float8_e4m3fn).double())


def test_oracle_scales(dense):
    a = torch.tensor([448.0, 448.5, 447.0, 224.0, 225.0, 1.75, 1.76, 2.0 ** -100, 3.0e38], dtype=torch.float64)
    s = dense.pow2_scale(a)
    assert (a <= 448 * s).all() and (a > 224 * s).all() and torch.equal(torch.frexp(s)[0], torch.full_like(a, 0.5))
    x = torch.randn(9, 300, dtype=torch.float64)
    codes, sf = dense.quantize_rows(x, False)
    assert codes.abs().amax() == 448 and ((dense.row_values(codes, sf) - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -9 * sf.max()).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_oracle_gate_slope_is_autograds(dense, act):
    z = torch.linspace(-30, 30, 2001, dtype=torch.float64, requires_grad=True)
    value, slope = dense.gate(z, act)
    want = torch.nn.functional.silu(z) if act == "silu" else torch.nn.functional.gelu(z, approximate="tanh")
    assert torch.allclose(value, want, rtol=1e-12, atol=1e-14)
    assert torch.allclose(slope, torch.autograd.grad(want.sum(), z)[0], rtol=1e-9, atol=1e-12)
