"""Gated feed-forward block on the GPU, forward and backward, against a 64-bit implementation.

Tolerances, with e = half a step of the type (bf16 2^-8, fp16 2^-11 relative) and S_y = the sum of magnitudes behind
a sum y.  A projection of length k is ceil(k / 16) fp32 accumulations of 16 exact products, each off by at most 2^-22 of
S (two bits below fp32's 24 for the alignment of the addends): d_g = ceil(k / 16) 2^-22 S_g.  act is 1.13-Lipschitz and its
fp32 evaluation is good to 2^-18 of |act| (exp's argument carries |c| 2^-24, |c| < 40 where sigma is not negligible);
act' is 1.7-Lipschitz, good to 2^-18.  So, to first order,
    h    e |h| + |u| (1.13 d_g + 2^-18 |act|) + |act| d_u
    dg   e |dg| + |dh| (|act'| d_u + |u| (1.7 d_g + 2^-18 (1 + |g|))),  du likewise
    dx   e |dx| + the errors of dg and du carried through |w| + (2 n / 16 + 2) 2^-22 S_dx,  dw likewise."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
ALL = ("x", "w1", "w2")


@pytest.fixture(scope="module")
def dense():
    from oracle import dense_oracle
    return dense_oracle


def _inputs(m, n, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m * 3 + n * 5 + k * 7)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, w1, w2 = r(m, k), r(n, k) * k ** -0.5, r(n, k) * k ** -0.5
    return x.to(dtype), w1.to(dtype), w2.to(dtype), r(m, n).to(dtype)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _within(got, want, tol, what):
    assert got.shape == want.shape, what
    d = (got.double() - want).abs()
    assert not (d > tol).any(), (what, int((d > tol).sum()), d.max().item(), (d / tol).max().item())


def _projections(x, w):
    y = x.double() @ w.double().t()
    return y, -(-x.shape[1] // 16) * 2.0 ** -22 * (x.double().abs() @ w.double().abs().t())


def _forward_bound(dense, x, w1, w2, act):
    g, dg = _projections(x, w1)
    u, du = _projections(x, w2)
    a, _ = dense.gate(g, act)
    h = a * u
    err = u.abs() * (1.13 * dg + 2.0 ** -18 * a.abs()) + (a.abs() + 1.13 * dg) * du
    return h, err + _half_step(x.dtype) * (h.abs() + err) + _floor(x.dtype)


def _hidden_bound(dense, g, d_g, u, d_u, dh, act, dtype):
    a, da = dense.gate(g, act)
    dh = dh.double()
    dg, du = dh * u * da, dh * a
    eg = dh.abs() * (da.abs() * d_u + (u.abs() + d_u) * (1.7 * d_g + 2.0 ** -18 * (1 + g.abs())))
    eu = dh.abs() * (1.13 * d_g + 2.0 ** -18 * a.abs())
    e = _half_step(dtype)
    return dg, eg + e * (dg.abs() + eg) + _floor(dtype), du, eu + e * (du.abs() + eu) + _floor(dtype)


def _grads_bound(dg, eg, du, eu, x, w1, w2, dtype):
    x, w1, w2 = x.double(), w1.double(), w2.double()
    m, n = dg.shape
    e = _half_step(dtype)

    def close(y, carried, total, steps):
        t = carried + (steps + 2) * 2.0 ** -22 * total
        return y, t + e * (y.abs() + t) + _floor(dtype)

    dx = close(dg @ w1 + du @ w2, eg @ w1.abs() + eu @ w2.abs(), (dg.abs() + eg) @ w1.abs() + (du.abs() + eu) @ w2.abs(), n / 8)
    dw1 = close(dg.t() @ x, eg.t() @ x.abs(), (dg.abs() + eg).t() @ x.abs(), m / 16)
    dw2 = close(du.t() @ x, eu.t() @ x.abs(), (du.abs() + eu).t() @ x.abs(), m / 16)
    return {"x": dx, "w1": dw1, "w2": dw2}


SIZES = [(1, 8, 8), (1, 128, 256), (1, 1000, 2048), (2, 264, 72), (5, 136, 1000), (16, 512, 512), (33, 72, 136), (64, 1032, 264),
         (100, 640, 1032), (128, 128, 64), (129, 136, 200), (256, 256, 128), (257, 392, 520), (300, 1024, 88), (520, 264, 776),
         (1100, 520, 136), (1300, 2600, 200), (600, 1288, 2200)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward(pkg, dense, m, n, k, dtype, act):
    x, w1, w2, _ = _inputs(m, n, k, dtype)
    got = pkg.gated.gated_ffn(x, w1, w2, activation=act)
    _within(got, *_forward_bound(dense, x, w1, w2, act), "h")
    assert torch.equal(got, pkg.gated.gated_ffn(x, w1, w2, activation=act))
    assert pkg._lib.read_status(0) == 0


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_backward_from_the_inputs(pkg, dense, m, n, k, dtype, act):
    x, w1, w2, dh = _inputs(m, n, k, dtype)
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    h = pkg.gated.gated_ffn(*leaves, activation=act)
    grads = torch.autograd.grad(h, leaves, dh)
    with torch.no_grad():
        _within(h, *_forward_bound(dense, x, w1, w2, act), "h")
        g, d_g = _projections(x, w1)
        u, d_u = _projections(x, w2)
        hidden = _hidden_bound(dense, g, d_g, u, d_u, dh, act, dtype)
        want = _grads_bound(*hidden, x, w1, w2, dtype)
        for name, got in zip(ALL, grads):
            _within(got, *want[name], name)
    assert pkg._lib.read_status(0) == 0


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_kept_copies_and_the_backward_pass_from_them(pkg, dense, m, n, k, dtype, act):
    x, w1, w2, dh = _inputs(m, n, k, dtype)
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    h = pkg.gated.gated_ffn(*leaves, activation=act, keep="fp8")
    qg, sg, qu, su, qx, sx = pkg.gated.kept_copies(h.grad_fn.saved_tensors[2], m, n, k)
    grads = torch.autograd.grad(h, leaves, dh)
    with torch.no_grad():
        _within(h, *_forward_bound(dense, x, w1, w2, act), "h")
        values = []
        for q, s, w in ((qg, sg, w1), (qu, su, w2)):
            y, d = _projections(x, w)
            v = dense.row_values(q.float(), s)
            steps = s.double().repeat_interleave(128, 1)[:, :n]
            # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale near zero), and the projection's own error
            _within(v, y, 2.0 ** -4 * (y.abs() + d) + 2.0 ** -10 * steps + d, "kept values")
            amax = torch.nn.functional.pad(y.abs() , (0, -n % 128)).view(m, -1, 128).amax(2)
            slack = torch.nn.functional.pad(d, (0, -n % 128)).view(m, -1, 128).amax(2)
            low, high = dense.pow2_scale((amax - slack).clamp_min(2.0 ** -100)), dense.pow2_scale((amax + slack).clamp_min(2.0 ** -100))
            assert ((s.double() >= low) & (s.double() <= high)).all()
            values.append(v)
        codes, s = dense.quantize_rows(x, True)
        assert torch.equal(qx.double(), codes) and torch.equal(sx.double(), s)
        zero = torch.zeros_like(values[0])
        hidden = _hidden_bound(dense, values[0], zero, values[1], zero, dh, act, dtype)
        want = _grads_bound(*hidden, dense.row_values(qx.float(), sx), w1, w2, dtype)
        for name, got in zip(ALL, grads):
            _within(got, *want[name], name)
    assert pkg._lib.read_status(0) == 0


@pytest.mark.parametrize("m,n,k", [(5, 16, 24), (130, 72, 264), (300, 520, 200), (700, 2600, 2200), (2600, 1288, 520)])
def test_gradients_are_exact_on_integers(pkg, m, n, k):
    """g is an integer of at least 24 (a column of ones in x, 32 in w1): sigma(g) is 1 in fp32, act(g) = g and act' = 1, so dg = dh u
    and du = dh g are integers below 2^8 and every sum behind dx and dw is exact in fp32: any difference is a mistake."""
    r = torch.Generator(device="cuda").manual_seed(m)

    def ints(*s):
        some = torch.rand(s, generator=r, device="cuda") < 0.02
        return (torch.randint(-1, 2, s, generator=r, device="cuda") * some).to(BF16)

    x, w1, w2 = ints(m, k), ints(n, k), ints(n, k)
    x[:, 0], w1[:, 0], w2[:, 0] = 1, 32, 2
    dh = torch.randint(-3, 4, (m, n), generator=r, device="cuda").to(BF16)
    g, u = x.double() @ w1.double().t(), x.double() @ w2.double().t()
    assert g.min() >= 24 and g.max() < 64 and u.abs().max() < 64
    dg, du = dh.double() * u, dh.double() * g
    want = (dg @ w1.double() + du @ w2.double(), dg.t() @ x.double(), du.t() @ x.double())
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    for got, y in zip(torch.autograd.grad(pkg.gated.gated_ffn(*leaves), leaves, dh), want):
        assert y.abs().max() < 2 ** 24 and torch.equal(got, y.float().to(BF16))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_against_differences(pkg, dense, act):
    """<dx, v> against (L(x + t v) - L(x - t v)) / 2t of the 64-bit forward: the quotient is off by t^2 / 6 times a
    third derivative (t = 1e-4: below 1e-6 here), the gradient by its tolerance."""
    m, n, k = 37, 136, 72
    x, w1, w2, dh = _inputs(m, n, k, FP16)
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    grads = torch.autograd.grad(pkg.gated.gated_ffn(*leaves, activation=act), leaves, dh)
    with torch.no_grad():
        g, d_g = _projections(x, w1)
        u, d_u = _projections(x, w2)
        want = _grads_bound(*_hidden_bound(dense, g, d_g, u, d_u, dh, act, FP16), x, w1, w2, FP16)
        at = [t.detach().double() for t in leaves]
        for i, (name, got) in enumerate(zip(ALL, grads)):
            v = torch.randn(at[i].shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").double()
            def loss(t):
                p = list(at)
                p[i] = at[i] + t * v
                return (dense.gated(*p, act) * dh.double()).sum()
            quotient = (loss(1e-4) - loss(-1e-4)) / 2e-4
            assert abs((got.double() * v).sum() - quotient) <= (want[name][1] * v.abs()).sum() + 1e-4 * quotient.abs() + 1e-4


@pytest.mark.parametrize("keep", ["inputs", "fp8"])
def test_only_what_is_asked_for(pkg, keep):
    x, w1, w2, dh = _inputs(70, 136, 200, BF16)
    full = [t.clone().requires_grad_() for t in (x, w1, w2)]
    want = torch.autograd.grad(pkg.gated.gated_ffn(*full, keep=keep), full, dh)
    for mask in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)):
        leaves = [t.clone().requires_grad_(bool(f)) for t, f in zip((x, w1, w2), mask)]
        got = torch.autograd.grad(pkg.gated.gated_ffn(*leaves, keep=keep), [t for t in leaves if t.requires_grad], dh)
        for a, b in zip(got, [w for w, f in zip(want, mask) if f]):
            assert torch.equal(a, b)
        # the same gradients out of a block that could have given all
        h = pkg.gated.gated_ffn(*full, keep=keep)
        got = torch.autograd.grad(h, [t for t, f in zip(full, mask) if f], dh)
        for a, b in zip(got, [w for w, f in zip(want, mask) if f]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("keep", ["inputs", "fp8"])
def test_layouts_of_inputs_and_gradients(pkg, keep):
    x, w1, w2, dh = _inputs(60, 136, 200, BF16)
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    h = pkg.gated.gated_ffn(*leaves, keep=keep)
    want = torch.autograd.grad(h, leaves, dh)
    # leading dimensions; an input that is a slice of a wider buffer, one at an odd address, one transposed
    wide = torch.zeros((60, 264), dtype=BF16, device="cuda")
    wide[:, 8:208] = x
    odd = torch.zeros(60 * 200 + 1, dtype=BF16, device="cuda")[1:].view(60, 200)
    odd.copy_(x)
    for xin in (x.view(3, 20, 200), wide[:, 8:208], odd, x.t().contiguous().t()):
        xin = xin.detach().requires_grad_()
        hh = pkg.gated.gated_ffn(xin, leaves[1], leaves[2], keep=keep)
        assert hh.shape == (*xin.shape[:-1], 136) and torch.equal(hh.reshape(60, 136), h)
        got = torch.autograd.grad(hh, (xin, leaves[1], leaves[2]), dh.view(hh.shape))
        assert torch.equal(got[0].reshape(60, 200), want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    # a gradient that is one number seen through zero strides, and one that is transposed
    ones = torch.autograd.grad(pkg.gated.gated_ffn(*leaves, keep=keep), leaves, torch.ones_like(h))
    summed = torch.autograd.grad(pkg.gated.gated_ffn(*leaves, keep=keep).sum(), leaves)
    turned = torch.autograd.grad(pkg.gated.gated_ffn(*leaves, keep=keep), leaves, dh.t().contiguous().t())
    for a, b in list(zip(ones, summed)) + list(zip(turned, want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("keep", ["inputs", "fp8"])
def test_no_rows_and_rows_of_zeros(pkg, keep):
    x, w1, w2, dh = _inputs(4, 136, 72, BF16)
    leaves = [t.clone().requires_grad_() for t in (x[:0], w1, w2)]
    h = pkg.gated.gated_ffn(*leaves, keep=keep)
    dx, dw1, dw2 = torch.autograd.grad(h, leaves, dh[:0])
    assert h.shape == (0, 136) and dx.shape == (0, 72) and not dw1.any() and not dw2.any()
    # padded tokens: rows of zeros give zeros and add nothing to the weights' gradients
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    padded = torch.zeros((300, 72), dtype=BF16, device="cuda")
    padded[:4] = x
    more = [padded.requires_grad_(), leaves[1], leaves[2]]
    want = torch.autograd.grad(pkg.gated.gated_ffn(*leaves, keep=keep), leaves, dh)
    dh_more = torch.ones((300, 136), dtype=BF16, device="cuda")
    dh_more[:4] = dh
    h = pkg.gated.gated_ffn(*more, keep=keep)
    got = torch.autograd.grad(h, more, dh_more)
    assert not h[4:].any() and torch.equal(got[0][:4], want[0])
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("keep", ["inputs", "fp8"])
def test_training_step_on_a_side_stream_and_in_a_graph(pkg, keep):
    x, w1, w2, dh = _inputs(130, 264, 200, BF16)
    leaves = [t.requires_grad_() for t in (x, w1, w2)]

    def step():
        h = pkg.gated.gated_ffn(*leaves, keep=keep)
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for t in outs:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    with torch.no_grad():
        x.copy_(_inputs(130, 264, 200, BF16, seed=9)[0])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, step()))
    del graph


def test_kept_memory(pkg):
    """keep="fp8" holds 2 n + k bytes per row and one scale for each 128 of them; keep="inputs" nothing new."""
    m, n, k = 256, 1024, 512
    x, w1, w2, _ = _inputs(m, n, k, BF16)
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    own = {t.data_ptr() for t in leaves}
    size = lambda h: sum(t.numel() * t.element_size() for t in h.grad_fn.saved_tensors if t.data_ptr() not in own)  # noqa: E731
    assert size(pkg.gated.gated_ffn(*leaves)) == 0
    assert size(pkg.gated.gated_ffn(*leaves, keep="fp8")) == m * (2 * n + k) + 4 * m * (2 * n + k) // 128


def test_block_then_quantised_projection(pkg, dense):
    """The two operators in a row, as a serving layer runs them: gated block, then the fp8 down projection."""
    x, w1, w2, _ = _inputs(150, 520, 264, BF16)
    down, down_sf = pkg.fp8.quantize_fp8_weight(_inputs(1, 264, 520, BF16)[1])
    y = pkg.fp8.fp8_linear(pkg.gated.gated_ffn(x, w1, w2), down, down_sf)
    h = pkg.gated.gated_ffn(x, w1, w2)
    codes, s = dense.quantize_rows(h, False)
    av, bv = dense.row_values(codes, s), dense.block_values(down.float(), down_sf)
    want, total = av @ bv.t(), av.abs() @ bv.abs().t()
    tol = (4 * 2.0 ** -22 + (s.shape[1] + 2) * 2.0 ** -24) * total
    _within(y, want, tol + _half_step(BF16) * (want.abs() + tol), "y")


def test_offsets_past_32_bits(pkg):
    """2.2e9 hidden elements: the last rows' results are those of the last rows alone, rows of zeros in between."""
    m, n, k = 130_000, 16896, 64
    x = torch.zeros((m, k), dtype=BF16, device="cuda")
    part, w1, w2, dh_part = _inputs(300, n, k, BF16)
    x[-300:] = part
    dh = torch.zeros((m, n), dtype=BF16, device="cuda")
    dh[-300:] = dh_part
    for keep in ("inputs", "fp8"):
        small = [t.clone().requires_grad_() for t in (part, w1, w2)]
        hs = pkg.gated.gated_ffn(*small, keep=keep)
        want = torch.autograd.grad(hs, small, dh_part)
        large = [t.detach().requires_grad_() for t in (x, w1, w2)]
        h = pkg.gated.gated_ffn(*large, keep=keep)
        assert torch.allclose(h[-300:].float(), hs.float(), rtol=2 ** -7, atol=1e-5) and not h[0].any() and not h[-301].any()
        dx, dw1, dw2 = torch.autograd.grad(h, large, dh)
        for got, ref in ((dx[-300:], want[0]), (dw1, want[1]), (dw2, want[2])):
            assert (got.double() - ref.double()).norm() <= 2 ** -6 * ref.double().norm()
        assert not dx[0].any() and not dx[-301].any()
        del h, hs, dx
    assert pkg._lib.read_status(0) == 0


def test_two_streams_at_once(pkg):
    for m in (5, 100, 400):
        sets = [[t.requires_grad_() if i < 3 else t for i, t in enumerate(_inputs(m, 264, 520, BF16, seed))] for seed in (1, 2)]
        want = [torch.autograd.grad(pkg.gated.gated_ffn(*s[:3], keep="fp8"), s[:3], s[3]) for s in sets]
        streams = [torch.cuda.Stream() for _ in sets]
        torch.cuda.synchronize()
        for _ in range(10):
            got = []
            for s, st in zip(sets, streams):
                with torch.cuda.stream(st):
                    got.append(torch.autograd.grad(pkg.gated.gated_ffn(*s[:3], keep="fp8"), s[:3], s[3]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_shared_and_broadcast_inputs(pkg):
    """One weight in both places gets the sum of its two gradients; an input seen through zero strides the sum over its rows."""
    x, w1, w2, dh = _inputs(40, 136, 72, FP16)
    two = [x.clone().requires_grad_(), w1.clone().requires_grad_(), w1.clone().requires_grad_()]
    g = torch.autograd.grad(pkg.gated.gated_ffn(*two), two, dh)
    w = w1.clone().requires_grad_()
    both, = torch.autograd.grad(pkg.gated.gated_ffn(x, w, w), (w,), dh)
    assert torch.equal(both, g[1] + g[2])
    row = x[:1].clone().requires_grad_()
    spread = x[:1].expand(40, 72).contiguous().requires_grad_()
    a, = torch.autograd.grad(pkg.gated.gated_ffn(row.expand(40, 72), w1, w2), (row,), dh)
    b, = torch.autograd.grad(pkg.gated.gated_ffn(spread, w1, w2), (spread,), dh)
    assert torch.equal(a, b.sum(0, keepdim=True))
    assert pkg.gated.gated_ffn(x[0], w1, w2).shape == (136,)


def test_refusals(pkg):
    x, w1, w2, _ = _inputs(8, 136, 72, BF16)
    bad = [
        (lambda: pkg.gated.gated_ffn(x.float(), w1.float(), w2.float()), "float16 or bfloat16"),
        (lambda: pkg.gated.gated_ffn(x, w1.half(), w2), "one type"),
        (lambda: pkg.gated.gated_ffn(x, w1, w2[:128]), "expected x"),
        (lambda: pkg.gated.gated_ffn(x[:, :64], w1, w2), "expected x"),
        (lambda: pkg.gated.gated_ffn(x, w1[:132], w2[:132]), "multiples of 8"),
        (lambda: pkg.gated.gated_ffn(x[:, :68], w1[:, :68], w2[:, :68]), "multiples of 8"),
        (lambda: pkg.gated.gated_ffn(x, w1.cpu(), w2), "one device"),
    ]
    for call, needle in bad:
        with pytest.raises(ValueError, match=needle):
            call()
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    h = pkg.gated.gated_ffn(*leaves)
    g, = torch.autograd.grad(h, (x,), torch.ones_like(h).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):            # there is no second derivative
        torch.autograd.grad(g.sum(), (x,))
