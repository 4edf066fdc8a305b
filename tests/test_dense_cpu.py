"""The fp8 block-128 GEMM and the gated feed-forward block without a GPU: bad arguments are rejected on the host
before any CUDA work, and the 64-bit oracle agrees with torch's own e4m3 and with its autograd."""
import pytest
import torch

FAKE = 0x7F0000000000  # 16-byte aligned fake device address; never dereferenced on the host
NULL, SHAPE, ALIGN, WORKSPACE, VARIANT, LIMIT = -1, -2, -3, -4, -5, -7


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
                                          None, 0, 0, v["m"], v["n"], v["k"], None, 0, None), code, needle)


def test_gated_kept_buffer(lib, pkg):
    size = lib.b200_gated_kept_bytes
    for m, n, k in ((4, 128, 64), (7, 136, 200), (1, 8, 8)):
        for keep_x in (0, 1):
            assert size(m, n, k, keep_x) == pkg.gated._kept_bytes(m, n, k, bool(keep_x))
        assert size(m, n, k, 1) > size(m, n, k, 0)
    assert size(0, 128, 64, 1) == 0
    f = lambda kept, nbytes, keep_x: lib.b200_gated_forward(FAKE, 64, FAKE, 64, FAKE, 64, 1, 0, FAKE, 128, kept, nbytes, keep_x,  # noqa: E731
                                                            4, 128, 64, None, 0, None)
    _rejected(lib, f(FAKE, size(4, 128, 64, 1) - 1, 1), WORKSPACE, str(size(4, 128, 64, 1)))
    _rejected(lib, f(FAKE, size(4, 128, 64, 0) - 1, 0), WORKSPACE, str(size(4, 128, 64, 0)))
    _rejected(lib, f(FAKE + 8, 1 << 20, 1), WORKSPACE, "aligned")


def _backward(lib, **kw):
    v = dict(x=FAKE, ldx=64, kept=None, kept_bytes=0, keep_x=0, w1=FAKE, w2=FAKE, ldw=64, dtype=1, act=0, dh=FAKE, ld_dh=128, dx=FAKE, ld_dx=64,
             dw1=FAKE, dw2=FAKE, ld_dw=64, m=4, n=128, k=64, scratch=FAKE, nbytes=1 << 20)
    v.update(kw)
    return lib.b200_gated_backward(v["x"], v["ldx"], v["kept"], v["kept_bytes"], v["keep_x"], v["w1"], v["ldw"], v["w2"], v["ldw"], v["dtype"],
                                   v["act"], v["dh"], v["ld_dh"], v["dx"], v["ld_dx"], v["dw1"], v["dw2"], v["ld_dw"], v["m"], v["n"],
                                   v["k"], v["scratch"], v["nbytes"], None, 0, None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(x=None), NULL, "x is NULL"), (dict(w1=None), NULL, "w1 is NULL"), (dict(w2=None), NULL, "w2 is NULL"), (dict(dh=None), NULL, "dh is NULL"),
    (dict(dx=None, dw1=None, dw2=None), NULL, "no gradient"), (dict(dtype=4), VARIANT, "dtype 4"), (dict(act=2), VARIANT, "activation 2"),
    (dict(m=0), SHAPE, "positive"), (dict(n=100), SHAPE, "n=100"), (dict(k=68), SHAPE, "k=68"), (dict(ldx=60), ALIGN, "of x"),
    (dict(ldw=68), ALIGN, "of w1"), (dict(ld_dh=100), ALIGN, "of dh"), (dict(ld_dx=60), ALIGN, "of dx"), (dict(ld_dw=60), ALIGN, "of dw1"),
    (dict(dw1=None, ld_dw=60), ALIGN, "of dw2"), (dict(dh=FAKE + 2), ALIGN, "dh must be"), (dict(scratch=None), WORKSPACE, "scratch"),
    (dict(scratch=FAKE + 4), WORKSPACE, "aligned"), (dict(nbytes=4 * 4 * 128 - 1), WORKSPACE, "2048"),
    (dict(kept=FAKE, kept_bytes=16, keep_x=1), WORKSPACE, "8-bit copies"), (dict(kept=FAKE, kept_bytes=1 << 20, keep_x=0), VARIANT, "keep_x"),
    (dict(kept=FAKE, kept_bytes=1 << 20, keep_x=1, nbytes=4 * 4 * 128 + 2 * 4 * 64 - 1), WORKSPACE, "2560"),
])
def test_gated_backward_refusals(lib, kw, code, needle):
    _rejected(lib, _backward(lib, **kw), code, needle)


def test_fp8_linear_scratch(lib):
    assert lib.b200_fp8_linear_scratch_bytes(16, 4096) == 0 and lib.b200_fp8_linear_scratch_bytes(0, 64) == 0
    need = lib.b200_fp8_linear_scratch_bytes(17, 200)
    assert need == 17 * 208 + 17 * 2 * 4
    f = lambda m=17, x=FAKE, w=FAKE, sf=FAKE, y=FAKE, n=128, scratch=FAKE, nbytes=1 << 20, ldx=200, dtype=0: lib.b200_fp8_linear(  # noqa: E731
        x, ldx, dtype, w, 208, sf, 2, 1, y, 128, m, n, 200, scratch, nbytes, None, 0, None)
    _rejected(lib, f(nbytes=need - 1), WORKSPACE, str(need))
    _rejected(lib, f(scratch=None), WORKSPACE, "scratch")
    _rejected(lib, f(scratch=FAKE + 8), WORKSPACE, "aligned")
    _rejected(lib, f(x=None), NULL, "NULL")
    _rejected(lib, f(w=None), NULL, "w is NULL")
    _rejected(lib, f(y=None), NULL, "y is NULL")
    _rejected(lib, f(sf=None), NULL, "NULL")
    _rejected(lib, f(n=4), SHAPE, "n=4")
    _rejected(lib, f(m=0), SHAPE, "positive")
    _rejected(lib, f(ldx=199), ALIGN, "ldx=199")
    _rejected(lib, f(dtype=5), VARIANT, "dtype 5")


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
