"""MXFP4 kernels against fp64: the quantiser exactly, products within their accumulation error."""
import pytest
import torch

from firefly_b200 import (
    MXFP4Linear,
    MXFP4SwiGLU,
    MXFP4Tensor,
    _capi,
    mxfp4_linear,
    mxfp4_matmul,
    mxfp4_swiglu,
    quantize_fp_to_mxfp4,
    quantize_fp_to_mxfp4_dual,
)
from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(r, c, seed, dtype=torch.bfloat16, scale=1.0):
    g = _gen(seed)
    x = torch.randn(r, c, device=DEV, generator=g) * scale
    x *= torch.exp2(torch.randint(-6, 7, (r, 1), device=DEV, generator=g).float())  # rows of several magnitudes
    return x.to(dtype)


def _check_values(q, x):
    assert torch.equal(q.scale_bytes(), O.scale_exponents(x))
    torch.testing.assert_close(q.dequantize(torch.float32).double(), O.values(x), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,c", [(1, 1), (1, 32), (3, 31), (1, 4096), (17, 4095), (128, 128), (129, 160), (257, 33),
                                 (300, 1000), (31, 257)])
def test_quantiser_is_exact_along_both_axes(r, c, dtype):
    x = _randn(r, c, r * 7 + c, dtype)
    _check_values(quantize_fp_to_mxfp4(x), x)
    q, qt = quantize_fp_to_mxfp4_dual(x)
    _check_values(q, x)
    _check_values(qt, x.t())
    assert qt.shape == (c, r)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_rounds_every_border_to_even(dtype):
    """Every midpoint between two codes, its neighbours in the type, and both ends, in both signs."""
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.5, 0.125, 4.0], dtype=torch.float64)
    mids = base.to(dtype)
    up = torch.nextafter(mids.float(), torch.full((12,), 100.0)) if dtype == torch.float32 else \
        (mids.view(torch.int16) + 1).view(dtype)
    down = torch.nextafter(mids.float(), torch.zeros(12)) if dtype == torch.float32 else \
        (mids.view(torch.int16) - 1).view(dtype)
    row = torch.cat([mids, up.to(dtype), down.to(dtype)])
    x = torch.zeros(64, 32, dtype=dtype)
    for i in range(36):
        x[i, 0] = 4.0  # the block's scale stays 1 (or 2^0 for the values up to 7.99)
        x[i, 1 + i % 31] = row[i]
    x[36:] = -x[:28]
    x = x.to(DEV)
    q, qt = quantize_fp_to_mxfp4_dual(x)
    _check_values(q, x)
    _check_values(qt, x.t())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_of_zeros_subnormals_and_the_largest_values(dtype):
    info = torch.finfo(dtype)
    x = torch.zeros(6, 96, dtype=dtype)
    x[1, 5] = info.smallest_normal
    x[2, 40] = info.smallest_normal * info.eps * 3  # subnormal
    x[3] = info.max
    x[4, ::3] = -info.max
    x[5, 64:] = -0.0
    x = x.to(DEV)
    q, qt = quantize_fp_to_mxfp4_dual(x)
    _check_values(q, x)
    _check_values(qt, x.t())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_non_finite_value_makes_its_block_nan(dtype, bad):
    x = _randn(70, 100, 5, dtype)
    x[3, 50] = bad
    q, qt = quantize_fp_to_mxfp4_dual(x)
    _check_values(q, x)
    _check_values(qt, x.t())
    y = mxfp4_matmul(q, quantize_fp_to_mxfp4(_randn(40, 100, 6)), out_dtype=torch.float32)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[:3]).all() and torch.isfinite(y[4:]).all()


def test_quantiser_of_strided_and_unaligned_views():
    big = _randn(200, 515, 3)
    for x in (big[:, :300], big[:, 1:258], big[5:105, 3:200], big.t()[7:90], big[::2], big[:, ::3]):
        q, qt = quantize_fp_to_mxfp4_dual(x)
        _check_values(q, x.contiguous())
        _check_values(qt, x.t().contiguous())


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantize_types(dtype):
    x = _randn(33, 77, 9, scale=0.1)
    got = quantize_fp_to_mxfp4(x).dequantize(dtype)
    assert got.dtype == dtype
    torch.testing.assert_close(got, O.values(x).to(dtype), rtol=0, atol=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,c,ld", [(1, 1, 1), (5, 264, 264), (9, 4095, 4095), (31, 257, 300), (300, 1001, 1001),
                                    (130, 2056, 2056), (67, 520, 523)])
def test_dequantize_writes_its_columns_only(r, c, ld, dtype):
    """Rows of any alignment, through the C entry: what lies between and behind them stays."""
    x = _randn(r, c, 21, scale=0.1)
    q = quantize_fp_to_mxfp4(x)
    buf = torch.full((r * ld + 40,), 7.0, dtype=dtype, device=DEV)
    for skip in (0, 1):
        buf.fill_(7.0)
        codes, scales = q._pair()
        _capi._call("ff_mxfp4_dequant", _capi._addr(codes), codes.shape[1], _capi._addr(scales), r, c,
                    buf.data_ptr() + skip * buf.element_size(), _capi._dtype_code(dtype), ld, _capi._raw_stream(x.device))
        view = buf[skip:skip + r * ld].view(r, ld)
        torch.testing.assert_close(view[:, :c], O.values(x).to(dtype), rtol=0, atol=0)
        assert bool((view[:, c:] == 7).all()) and bool((buf[:skip] == 7).all()) and bool((buf[skip + r * ld:] == 7).all())


def _tolerance(v, mag, K, dtype):
    """fp32 accumulation of ceil(K / 32) scaled block sums, each step off by at most 2^-23 of the sum of
    magnitudes (a truncating adder), then one rounding of the output."""
    tol = ((K + 31) // 32 + 2) * 2.0 ** -23 * mag
    return tol if dtype == torch.float32 else tol + 2.0 ** -8 * (v.abs() + tol)


def _check_product(got, a, b, bias=None):
    v, mag = O.product(a, b)
    if bias is not None:
        v, mag = v + bias.double(), mag + bias.double().abs()
    tol = _tolerance(v, mag, a.shape[1], got.dtype)
    off = (got.double() - v).abs()
    assert bool((off <= tol).all()), f"off by {float((off / tol.clamp(min=1e-300)).max())} of the tolerance"


SHAPES = [(1, 1, 1), (1, 128, 256), (1, 4096, 4096), (2, 130, 64), (16, 256, 512), (17, 1000, 100), (32, 96, 4096),
          (33, 300, 777), (64, 128, 2000), (65, 129, 257), (128, 384, 1024), (129, 65, 320), (200, 500, 300),
          (255, 257, 288), (256, 256, 256), (257, 513, 1100), (512, 768, 2048), (700, 1300, 96), (1000, 3000, 640),
          (4096, 300, 128), (300, 5000, 31),
          (1500, 3300, 1100), (2500, 1999, 288), (2304, 2560, 4096), (130, 20000, 512),
          (200, 512, 11008), (300, 130, 8200), (96, 3000, 2048), (50, 9000, 1056)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_product_against_fp64(M, N, K, out):
    a, b = _randn(M, K, 1), _randn(N, K, 2, scale=0.02)
    bias = torch.randn(N, device=DEV, generator=_gen(3)) if M % 2 else None
    got = mxfp4_matmul(quantize_fp_to_mxfp4(a), quantize_fp_to_mxfp4(b), bias, out_dtype=out)
    assert got.shape == (M, N) and got.dtype == out
    _check_product(got, O.values(a), O.values(b), bias)
    assert _capi.device_status() == 0


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K,ld", [(300, 400, 512, 400), (300, 401, 512, 401), (700, 1025, 256, 1030), (1500, 2047, 288, 2048)])
def test_product_writes_its_columns_only(M, N, K, ld, out):
    a, b = _randn(M, K, 1), _randn(N, K, 2, scale=0.02)
    qa, qb = quantize_fp_to_mxfp4(a), quantize_fp_to_mxfp4(b)
    want = mxfp4_matmul(qa, qb, None, out_dtype=out)
    _check_product(want, O.values(a), O.values(b))
    for skip in (0, 1):
        buf = torch.full((M * ld + 40,), 7.0, dtype=out, device=DEV)
        (ca, sa), (cb, sb) = qa._pair(), qb._pair()
        _capi._call("ff_mxfp4_gemm", ca.data_ptr(), ca.shape[1], sa.data_ptr(), cb.data_ptr(), cb.shape[1], sb.data_ptr(),
                    None, buf.data_ptr() + skip * buf.element_size(), ld,
                    _capi.FF_OUT_F32 if out == torch.float32 else _capi.FF_OUT_BF16, M, N, K, _capi._raw_stream(a.device))
        view = buf[skip:skip + M * ld].view(M, ld)
        assert torch.equal(view[:, :N], want)
        assert bool((view[:, N:] == 7).all()) and bool((buf[:skip] == 7).all()) and bool((buf[skip + M * ld:] == 7).all())
    assert _capi.device_status() == 0


@pytest.mark.parametrize("M,N,K", [(5, 200, 512), (300, 400, 512), (700, 900, 1024), (1500, 3300, 1024)])
def test_product_of_whole_numbers_is_exact(M, N, K):
    """Codes times powers of two whose sums stay below 2^24: every order of addition is exact."""
    g = _gen(11)
    lev = torch.tensor([0, 1, 2, 3, 4, 6], device=DEV, dtype=torch.float32)
    def mk(r):
        x = lev[torch.randint(0, 6, (r, K), device=DEV, generator=g)] * (torch.randint(0, 2, (r, K), device=DEV, generator=g) * 2 - 1)
        x[:, ::32] = 6.0  # every block's scale is 1
        return x * torch.exp2(torch.randint(0, 3, (r, 1), device=DEV, generator=g).float())
    a, b = mk(M), mk(N)
    got = mxfp4_matmul(quantize_fp_to_mxfp4(a), quantize_fp_to_mxfp4(b), out_dtype=torch.float32)
    torch.testing.assert_close(got.double(), a.double() @ b.double().t(), rtol=0, atol=0)


def test_product_uses_every_scale():
    """One value per block, every block with its own scale on both sides: a scale taken from a
    neighbouring row or block changes the result."""
    g = _gen(12)
    for M, N, K in ((40, 300, 1024), (400, 600, 1024), (1500, 3300, 1792)):
        a = torch.zeros(M, K, device=DEV)
        b = torch.zeros(N, K, device=DEV)
        a[:, ::32] = torch.exp2(torch.randint(-5, 6, (M, K // 32), device=DEV, generator=g).float())
        b[:, ::32] = torch.exp2(torch.randint(-5, 6, (N, K // 32), device=DEV, generator=g).float())
        got = mxfp4_matmul(quantize_fp_to_mxfp4(a), quantize_fp_to_mxfp4(b), out_dtype=torch.float32)
        torch.testing.assert_close(got.double(), a.double() @ b.double().t(), rtol=0, atol=0)


def test_product_is_the_same_every_time():
    for M, N, K in ((1, 4096, 4096), (20, 1000, 11008), (600, 900, 2048), (2000, 4100, 2048)):
        a, b = quantize_fp_to_mxfp4(_randn(M, K, 1)), quantize_fp_to_mxfp4(_randn(N, K, 2))
        first = mxfp4_matmul(a, b, out_dtype=torch.float32)
        for _ in range(4):
            assert torch.equal(first, mxfp4_matmul(a, b, out_dtype=torch.float32))


# ---------------------------------------------------------------------------
# linear layer
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T,K,N", [(1, 64, 40), (7, 100, 130), (33, 256, 96), (300, 520, 260), (1030, 96, 700)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_forward_and_gradients(T, K, N, dtype, bias):
    x = _randn(T, K, 1, dtype).requires_grad_(True)
    w = (_randn(N, K, 2, scale=0.02)).to(dtype).requires_grad_(True)
    b = torch.randn(N, device=DEV, generator=_gen(3)).to(dtype).requires_grad_(True) if bias else None
    dy = _randn(T, N, 4, torch.bfloat16, 1e-2)
    y = mxfp4_linear(x, w, b)
    assert y.dtype == torch.bfloat16
    y.backward(dy)
    _check_product(y, O.values(x.detach()), O.values(w.detach()), None if b is None else b.detach())
    for got, p, q in ((x.grad, dy, w.detach().t()), (w.grad, dy.t(), x.detach().t())):
        assert got.dtype == dtype
        v, mag = O.product(O.values(p), O.values(q))
        eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # half a subnormal step is below this
        tol = _tolerance(v, mag, p.shape[1], torch.float32)
        tol = tol + eps * (v.abs() + tol) + tiny
        assert bool(((got.double() - v).abs() <= tol).all())
    if bias:
        want = dy.double().sum(0)
        # T additions in fp32 (each half a step of the running sum of magnitudes), then the bias's type
        tol = T * 2.0 ** -24 * dy.double().abs().sum(0)
        if dtype != torch.float32:
            tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + torch.finfo(dtype).smallest_normal
        assert bool(((b.grad.double() - want).abs() <= tol).all())


def test_gradients_are_those_of_the_quantised_operands():
    """dx and dw against differences: the product is linear in each quantised operand, so moving an operand by
    one code step changes the sum of y * dy by that step times the gradient of the other operand's values."""
    T, K, N = 64, 64, 64
    lev = torch.tensor([-4.0, -2.0, -1.0, 1.0, 2.0, 4.0], device=DEV)
    g = _gen(8)
    mk = lambda r, c: lev[torch.randint(0, 6, (r, c), device=DEV, generator=g)]
    x, w, dy = mk(T, K), mk(N, K), mk(T, N)
    for t in (x, w, dy):  # every block along either axis has the largest code, so the values are exact
        t[::32, :] = 4.0
        t[:, ::32] = 4.0
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    mxfp4_linear(xg, wg).backward(dy.bfloat16())
    f = lambda x_, w_: (O.values(x_) @ O.values(w_).t() * dy.double()).sum()
    for (i, j) in ((1, 5), (33, 40), (63, 63)):
        for t, grad in ((x, xg.grad), (w, wg.grad)):
            moved = t.clone()
            moved[i, j] = 3.0 if float(t[i, j]) != 3.0 else 2.0
            args = (moved, w) if t is x else (x, moved)
            diff = (f(*args) - f(x, w)) / float(moved[i, j] - t[i, j])
            assert float(diff) == float(grad[i, j])


def test_linear_through_a_held_weight():
    T, K, N = 50, 300, 200
    w = _randn(N, K, 2, scale=0.02)
    x = _randn(T, K, 1).requires_grad_(True)
    dy = _randn(T, N, 4)
    ref = mxfp4_linear(x, w)
    (gref,) = torch.autograd.grad(ref, x, dy)
    held = quantize_fp_to_mxfp4(w, transposed=True)
    y = mxfp4_linear(x, held)
    (g,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(y, ref) and torch.equal(g, gref)
    with torch.no_grad():
        assert torch.equal(mxfp4_linear(x, quantize_fp_to_mxfp4(w)), ref)
    with pytest.raises(ValueError, match="transposed"):
        mxfp4_linear(x, quantize_fp_to_mxfp4(w))
    lin = MXFP4Linear(w, input_grad=True)
    assert torch.equal(lin(x.view(5, 10, K)).view(T, N), ref)
    other = MXFP4Linear(torch.zeros_like(w), input_grad=True)
    other.load_state_dict(lin.state_dict())
    assert torch.equal(other(x), ref)


def test_linear_of_no_rows():
    w = _randn(40, 64, 2).requires_grad_(True)
    b = torch.zeros(40, device=DEV, requires_grad=True)
    x = torch.zeros(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = mxfp4_linear(x, w, b)
    assert y.shape == (0, 40)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and not w.grad.any() and not b.grad.any()
    assert mxfp4_swiglu(x, _randn(128, 64, 1), _randn(8, 64, 2)).shape == (0, 8)


# ---------------------------------------------------------------------------
# gated block
# ---------------------------------------------------------------------------
def _flip_tolerance(v, mag, K, dtype, left, right):
    """A bf16 value between two products may round the other way (its fp32 sum is off by the accumulation
    error), and its MXFP4 code may then move by one step, at most a third of the block's largest value.  That
    many terms are few; the allowance is eight such terms of the largest size."""
    return _tolerance(v, mag, K, dtype) + 8 * left.abs().amax(1, keepdim=True) / 3 * right.abs().amax(1)[None]


@pytest.mark.parametrize("T,K,F,N", [(1, 64, 128, 96), (3, 256, 32, 40), (16, 512, 384, 512), (40, 100, 160, 77),
                                     (130, 256, 256, 300), (300, 320, 640, 256), (513, 512, 128, 260), (1300, 512, 1152, 640), (2200, 256, 640, 300),
                                     (100, 4096, 128, 64), (128, 8192, 256, 64), (20, 700, 1408, 90)])
def test_gated_block_forward_and_gradients(T, K, F, N):
    x = _randn(T, K, 1).requires_grad_(True)
    wgu = _randn(2 * F, K, 2, scale=0.05).requires_grad_(True)
    wd = _randn(N, F, 3, scale=0.05).requires_grad_(True)
    dy = _randn(T, N, 4, scale=1e-2)
    y = mxfp4_swiglu(x, wgu, wd)
    y.backward(dy)
    with torch.no_grad():
        y0 = mxfp4_swiglu(x, quantize_fp_to_mxfp4(wgu), quantize_fp_to_mxfp4(wd))
    # the chain in fp64 on the kernels' own bf16 activations (their products are checked above)
    gu = mxfp4_matmul(quantize_fp_to_mxfp4(x), quantize_fp_to_mxfp4(wgu)).double()
    g, u = gu[:, :F], gu[:, F:]
    h = O.bf16(O.swiglu(g, u))
    hv, wv = O.values(h), O.values(wd.detach())
    v, mag = O.product(hv, wv)
    tol = _flip_tolerance(v, mag, F, torch.bfloat16, hv, wv)
    for got in (y, y0):
        assert bool(((got.double() - v).abs() <= tol).all())
    dh = mxfp4_matmul(quantize_fp_to_mxfp4(dy), quantize_fp_to_mxfp4(wd.detach().t())).double()
    dgu = torch.cat([O.bf16(t) for t in O.swiglu_grad(dh, g, u)], 1)
    for got, p, q in ((x.grad, dgu, wgu.detach().t()), (wgu.grad, dgu.t(), x.detach().t()),
                      (wd.grad, dy.t().double(), h.t())):
        pv, qv = O.values(p), O.values(q)
        v, mag = O.product(pv, qv)
        tol = _flip_tolerance(v, mag, p.shape[1], torch.bfloat16, pv, qv)
        if got is wd.grad:
            tol = tol + 8 * pv.abs().amax(1, keepdim=True) * qv.abs().amax(1)[None] / 3
        assert bool(((got.double() - v).abs() <= tol).all())
    assert _capi.device_status() == 0


@pytest.mark.parametrize("T,F", [(1, 32), (5, 96), (130, 160), (257, 256)])
def test_activation_quantisers(T, F):
    """h and [dg | du] quantised without being written: the codes are those of the bf16 values up to roundings
    that the fp32 sigmoid (a few steps of 2^-23) moves across a border: few, and by one code."""
    gu = _randn(T, 2 * F, 1)
    dh = _randn(T, F, 2)
    g, u = gu[:, :F].double(), gu[:, F:].double()
    h = O.bf16(O.swiglu(g, u))
    d = torch.cat([O.bf16(t) for t in O.swiglu_grad(dh.double(), g, u)], 1)
    rows, cols = _capi.mxfp4_swiglu_quant(gu, cols=True)
    brow, bcol = _capi.mxfp4_swiglu_bwd_quant(dh, gu)
    for pair, want in ((rows, h), (cols, h.t()), (brow, d), (bcol, d.t())):
        q = MXFP4Tensor(*pair, tuple(want.shape))
        got, ref = q.dequantize(torch.float32).double(), O.values(want)
        blk = torch.nn.functional.pad(want, (0, (-want.shape[1]) % 32)).reshape(want.shape[0], -1, 32).abs().amax(2)
        step = blk.repeat_interleave(32, 1)[:, :want.shape[1]]
        assert bool(((got - ref).abs() <= step / 2).all())
        assert float((got != ref).double().mean()) < 2e-3


def test_held_gated_block_equals_the_training_forward():
    T, K, F, N = 70, 256, 256, 128
    x, wgu, wd = _randn(T, K, 1).requires_grad_(True), _randn(2 * F, K, 2, scale=0.05), _randn(N, F, 3, scale=0.05)
    dy = _randn(T, N, 4)
    blk = MXFP4SwiGLU(wgu, wd, input_grad=True)
    y = blk(x)
    ref = mxfp4_swiglu(x, wgu, wd)
    assert torch.equal(y, ref)
    assert torch.equal(*(torch.autograd.grad(t, x, dy)[0] for t in (y, ref)))


# ---------------------------------------------------------------------------
# streams, graphs, several at once
# ---------------------------------------------------------------------------
def test_captured_and_replayed():
    x, w = _randn(9, 512, 1), quantize_fp_to_mxfp4(_randn(300, 512, 2))
    gu, dn = quantize_fp_to_mxfp4(_randn(512, 512, 3)), quantize_fp_to_mxfp4(_randn(512, 256, 4))
    side = torch.cuda.Stream()
    graphs = []
    with torch.no_grad():
        with torch.cuda.stream(side):
            mxfp4_linear(mxfp4_swiglu(x, gu, dn), w)
        torch.cuda.synchronize()
        for _ in range(2):
            xin = x.clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = mxfp4_linear(mxfp4_swiglu(xin, gu, dn), w)
            graphs.append((g, xin, out))
        wants = []
        for k, (g, xin, out) in enumerate(graphs):
            xin.copy_(x * (k + 2))
            wants.append(mxfp4_linear(mxfp4_swiglu(xin, gu, dn), w))
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        for _ in range(3):  # both graphs at once, on two streams
            graphs[0][0].replay()
            with torch.cuda.stream(other):
                graphs[1][0].replay()
        torch.cuda.synchronize()
        for (g, xin, out), want in zip(graphs, wants):
            assert torch.equal(out, want)


def test_two_streams_at_once():
    ws = [quantize_fp_to_mxfp4(_randn(1500, 2048, s)) for s in (1, 2)]
    xs = [_randn(30, 2048, s) for s in (3, 4)]
    wants = [mxfp4_linear(x, w) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ws]
    outs = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[k].append(mxfp4_linear(xs[k], ws[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for o in outs[k]:
            assert torch.equal(o, wants[k])


def test_serving_calls_equal_their_parts():
    """The fused calls against quantiser and products one by one, few and many rows, with odd widths."""
    for T, K, F, N in ((1, 4096, 2048, 300), (15, 100, 128, 77), (40, 1000, 384, 260), (700, 512, 1280, 640)):
        x = _randn(T, K, 1)
        wgu, wd = quantize_fp_to_mxfp4(_randn(2 * F, K, 2, scale=0.05)), quantize_fp_to_mxfp4(_randn(N, F, 3, scale=0.05))
        b = torch.randn(2 * F, device=DEV, generator=_gen(4))
        assert torch.equal(mxfp4_linear(x, wgu, b), mxfp4_matmul(quantize_fp_to_mxfp4(x), wgu, b))
        qx = quantize_fp_to_mxfp4(x)
        h = MXFP4Tensor(*_capi.mxfp4_swiglu_quant(mxfp4_matmul(qx, wgu))[0], (T, F))
        hq = MXFP4Tensor(*_capi.mxfp4_swiglu_gemm(qx._pair(), wgu._pair(), T, F, K), (T, F))
        assert torch.equal(h.codes, hq.codes) and torch.equal(h.scale_bytes(), hq.scale_bytes())
        assert torch.equal(mxfp4_swiglu(x, wgu, wd), mxfp4_matmul(h, wd))
    assert _capi.device_status() == 0


def test_a_weight_quantised_just_before_the_call():
    """The serving kernels start early and ask for the weight first: it has to be there all the same."""
    x = _randn(1, 4096, 1)
    for s in range(6):
        w = _randn(4096, 4096, 10 + s)
        want = mxfp4_linear(x, quantize_fp_to_mxfp4(w))
        torch.cuda.synchronize()
        held = quantize_fp_to_mxfp4(torch.zeros_like(w))
        torch.cuda.synchronize()
        q = quantize_fp_to_mxfp4(w)
        held.codes.copy_(q.codes)
        held.scales.copy_(q.scales)
        assert torch.equal(mxfp4_linear(x, held), want)


def test_rows_of_nothing():
    q = quantize_fp_to_mxfp4(torch.zeros(0, 64, device=DEV))
    assert q.dequantize().shape == (0, 64) and q.scale_bytes().shape == (0, 2)
    assert mxfp4_matmul(q, quantize_fp_to_mxfp4(_randn(5, 64, 1))).shape == (0, 5)


def test_teacher_in_four_bits_distils_a_student():
    """The operators as they are used together: a held MXFP4 teacher, its top logits, the distillation loss of an
    MXFP4 student and the gradients of its weights, against the same chain in fp64 on the kernels' logits."""
    from firefly_b200 import distillation_loss
    from oracle import distill_oracle as D

    d, f, V, T, k = 128, 256, 500, 40, 12
    x = _randn(T, d, 1)
    teacher = MXFP4SwiGLU(_randn(2 * f, d, 2, scale=0.05), _randn(d, f, 3, scale=0.05))
    head_t = MXFP4Linear(_randn(V, d, 4, scale=0.2))
    with torch.no_grad():
        tl = head_t(teacher(x)).float()
    top = tl.topk(k, dim=1)
    lse = torch.logsumexp(tl / 2, 1)
    wgu, wd, head = (_randn(*s, scale=c).requires_grad_(True)
                     for s, c in (((2 * f, d, 5), 0.05), ((d, f, 6), 0.05), ((V, d, 7), 0.2)))
    labels = torch.randint(0, V, (T,), device=DEV, generator=_gen(8))
    hidden = mxfp4_swiglu(x, wgu, wd)
    logits = mxfp4_linear(hidden, head)
    logits.retain_grad()
    hidden.retain_grad()
    loss = distillation_loss(logits, top.indices, top.values, labels, teacher_lse=lse, temperature=2.0, alpha=0.5)
    loss.backward()
    s64 = logits.detach().double().requires_grad_(True)
    rows, _, scale = D.losses(s64, top.indices, top.values, labels, lse, 2.0, 0.5)
    assert abs(float(loss.detach()) - float(rows.detach().mean())) <= 2.0 ** -19 * (4 * (4 + float(scale.max())) + 16)
    rows.mean().backward()
    assert float((logits.grad.double() - s64.grad).abs().max()) <= 2.0 ** -8 * float(s64.grad.abs().max())
    v, mag = O.product(O.values(logits.grad.t()), O.values(hidden.detach().t()))
    assert bool(((head.grad.double() - v).abs() <= _tolerance(v, mag, T, torch.bfloat16)).all())
    v, mag = O.product(O.values(logits.grad), O.values(head.detach().t()))
    assert bool(((hidden.grad.double() - v).abs() <= _tolerance(v, mag, V, torch.bfloat16)).all())
    for w in (wgu, wd):
        assert torch.isfinite(w.grad).all() and bool(w.grad.any())


def test_more_than_2_31_elements():
    """Offsets past 32 bits: the last rows of large matrices against the same rows by themselves."""
    x = torch.empty(540000, 4096, device=DEV, dtype=torch.bfloat16)
    x.normal_(generator=_gen(1))
    q, qt = quantize_fp_to_mxfp4_dual(x)
    _check_values(quantize_fp_to_mxfp4(x[-130:]), x[-130:])
    assert torch.equal(q.codes[-130:], quantize_fp_to_mxfp4(x[-130:]).codes)
    tail = x[-256:].t().contiguous()  # 540000 is a multiple of 32: the last 256 rows are whole blocks
    assert torch.equal(qt.codes[:, -128:], quantize_fp_to_mxfp4(tail).codes)
    back = q.dequantize()
    assert torch.equal(back[-130:].double(), O.values(x[-130:]))
    del back, qt, q, x
    a, b = _randn(70000, 64, 2), _randn(33000, 64, 3)
    y = mxfp4_matmul(quantize_fp_to_mxfp4(a), quantize_fp_to_mxfp4(b))
    assert y.numel() > 2 ** 31
    _check_product(y[-70:], O.values(a)[-70:], O.values(b))
    _check_product(y[35000:35070], O.values(a)[35000:35070], O.values(b))


def test_the_smallest_products():
    for M, N, K in ((1, 1, 1), (1, 1, 33), (2, 3, 5), (300, 1, 1), (1, 300, 2)):
        a, b = _randn(M, K, 1), _randn(N, K, 2)
        _check_product(mxfp4_matmul(quantize_fp_to_mxfp4(a), quantize_fp_to_mxfp4(b), out_dtype=torch.float32), O.values(a),
                       O.values(b))


def test_gradients_through_a_broadcast_and_a_reused_input():
    """One input in two layers, its gradient the sum; an expanded upstream gradient (stride 0)."""
    x = _randn(40, 128, 1).requires_grad_(True)
    w1, w2 = _randn(64, 128, 2), _randn(64, 128, 3)
    (mxfp4_linear(x, w1) + mxfp4_linear(x, w2)).sum().backward()
    ones = torch.ones(40, 64, device=DEV, dtype=torch.bfloat16)
    got = x.grad.clone()
    parts = []
    for w in (w1, w2):
        y = x.detach().clone().requires_grad_(True)
        mxfp4_linear(y, w).backward(ones)
        parts.append(y.grad)
    assert torch.equal(got, parts[0] + parts[1]) or torch.equal(got, parts[1] + parts[0])


def test_training_step_captured_and_replayed():
    x = _randn(64, 256, 1).requires_grad_(True)
    wgu, wd = _randn(512, 256, 2, scale=0.05).requires_grad_(True), _randn(128, 256, 3, scale=0.05).requires_grad_(True)
    dy = _randn(64, 128, 4)

    def step():
        y = mxfp4_swiglu(x, wgu, wd)
        return (y.detach(), *torch.autograd.grad(y, [x, wgu, wd], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in (1, 2):
        with torch.no_grad():
            x.mul_(1.5)
            wgu.add_(0.01 * k)
            dy.mul_(0.75)
        g.replay()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_forward_mode_is_refused_as_by_the_other_layers():
    """There is no forward-mode derivative: a tangent is refused and not lost, on held weights too."""
    from torch.autograd import forward_ad

    x, w, wgu, wd = _randn(3, 64, 1), _randn(8, 64, 2), _randn(256, 64, 3), _randn(8, 128, 4)
    held = [quantize_fp_to_mxfp4(v) for v in (w, wgu, wd)]
    want = mxfp4_linear(x, held[0]), mxfp4_swiglu(x, *held[1:])
    bias = torch.zeros(8, device=DEV)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        b = forward_ad.make_dual(bias, torch.ones_like(bias))
        for call in (lambda: mxfp4_linear(d, held[0]), lambda: mxfp4_swiglu(d, *held[1:]), lambda: mxfp4_linear(d, w),
                     lambda: mxfp4_swiglu(d, wgu, wd), lambda: mxfp4_linear(x, held[0], b)):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        assert torch.equal(mxfp4_linear(x, held[0]), want[0]) and torch.equal(mxfp4_swiglu(x, *held[1:]), want[1])


# ---------------------------------------------------------------------------
# the one-call training passes against their parts
# ---------------------------------------------------------------------------
def _tensor(pair, shape):
    return MXFP4Tensor(*pair, shape)


def _within(got, a, b, dtype):
    """Whether got is the product of two value matrices within the accumulation error."""
    v, mag = O.product(a, b)
    return bool(((got.double() - v).abs() <= _tolerance(v, mag, a.shape[1], dtype)).all())


@pytest.mark.parametrize("T,K,F,N", [(1, 64, 128, 96), (3, 256, 32, 40), (16, 512, 384, 512), (40, 100, 160, 77),
                                     (130, 256, 256, 300), (300, 320, 640, 256), (513, 512, 128, 260), (1300, 512, 1152, 640),
                                     (100, 4096, 128, 64), (20, 700, 1408, 90)])
def test_gated_training_step_equals_its_parts(T, K, F, N):
    """The block's forward and backward bit for bit from the quantisers and the product, each product against fp64 on the codes
    that went into it; the same bound refuses a gradient of zeros and one with gate and up exchanged."""
    x, dy = _randn(T, K, 1).requires_grad_(True), _randn(T, N, 4, scale=1e-2)
    wgu, wd = _randn(2 * F, K, 2, scale=0.05).requires_grad_(True), _randn(N, F, 3, scale=0.05).requires_grad_(True)
    y = mxfp4_swiglu(x, wgu, wd)
    y.backward(dy)
    (qx, qxt), (qgu, qgut), (qd, qdt), (qy, qyt) = (quantize_fp_to_mxfp4_dual(m.detach()) for m in (x, wgu, wd, dy))
    gu = mxfp4_matmul(qx, qgu)
    rows, cols = _capi.mxfp4_swiglu_quant(gu, cols=True)
    h, ht = _tensor(rows, (T, F)), _tensor(cols, (F, T))
    dh = mxfp4_matmul(qy, qdt)
    rows, cols = _capi.mxfp4_swiglu_bwd_quant(dh, gu)
    p, pt = _tensor(rows, (T, 2 * F)), _tensor(cols, (2 * F, T))
    assert torch.equal(y, mxfp4_matmul(h, qd))
    for got, a, b in ((x.grad, p, qgut), (wgu.grad, pt, qxt), (wd.grad, qyt, ht)):
        assert torch.equal(got, mxfp4_matmul(a, b))
        av, bv = a.dequantize(torch.float32).double(), b.dequantize(torch.float32).double()
        assert _within(got, av, bv, torch.bfloat16)
        assert not _within(torch.zeros_like(got), av, bv, torch.bfloat16)
    swapped = p.dequantize(torch.float32).double()
    swapped = torch.cat([swapped[:, F:], swapped[:, :F]], 1)
    back = qgut.dequantize(torch.float32).double()
    assert not _within(x.grad, swapped, back, torch.bfloat16)
    assert not _within(wgu.grad, swapped.t(), qxt.dequantize(torch.float32).double(), torch.bfloat16)
    assert _capi.device_status() == 0


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (1, 0, 1)])
def test_gradients_of_some_inputs_equal_those_of_all(need):
    T, K, F, N = 70, 256, 192, 130
    args = [_randn(T, K, 1), _randn(2 * F, K, 2, scale=0.05), _randn(N, F, 3, scale=0.05)]
    dy = _randn(T, N, 4)
    leaves = [a.clone().requires_grad_(True) for a in args]
    every = torch.autograd.grad(mxfp4_swiglu(*leaves), leaves, dy)
    some = [a.clone().requires_grad_(bool(k)) for a, k in zip(args, need)]
    got = torch.autograd.grad(mxfp4_swiglu(*some), [a for a, k in zip(some, need) if k], dy)
    for a, b in zip(got, [g for g, k in zip(every, need) if k]):
        assert torch.equal(a, b)
    lin = [args[0], args[1], torch.randn(2 * F, device=DEV, generator=_gen(5))]
    dy = _randn(T, 2 * F, 6)
    leaves = [a.clone().requires_grad_(True) for a in lin]
    every = torch.autograd.grad(mxfp4_linear(*leaves), leaves, dy)
    some = [a.clone().requires_grad_(bool(k)) for a, k in zip(lin, need)]
    got = torch.autograd.grad(mxfp4_linear(*some), [a for a, k in zip(some, need) if k], dy)
    for a, b in zip(got, [g for g, k in zip(every, need) if k]):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# layers made from trained ones
# ---------------------------------------------------------------------------
def test_layers_from_trained_int8_layers():
    from firefly_b200 import BitLinear
    from firefly_b200.swiglu import SwiGLUMLP

    lin = BitLinear(96, 40, bias=True).to(DEV)
    with torch.no_grad():
        lin.bias.normal_(generator=_gen(1))
    x, dy = _randn(9, 96, 2).requires_grad_(True), _randn(9, 40, 3)
    w = lin.int_weight.float() * lin.weight_scale[:, None]
    held = MXFP4Linear.from_bitlinear(lin, input_grad=True)
    want = mxfp4_linear(x, w, lin.bias.detach())
    assert torch.equal(held(x), want)
    assert torch.equal(*(torch.autograd.grad(y, x, dy)[0] for y in (held(x), want)))
    with torch.no_grad():
        lin.bias.add_(1.0)  # the held layer has its own
    assert torch.equal(held(x), want) and not list(held.parameters())
    with pytest.raises(ValueError, match="transposed"):
        MXFP4Linear.from_bitlinear(lin)(x)
    mlp = SwiGLUMLP(64, 96).to(DEV)
    blk = MXFP4SwiGLU.from_swiglu_mlp(mlp, input_grad=True)
    x, dy = _randn(2, 5 * 64, 4).view(2, 5, 64).requires_grad_(True), _randn(2, 5 * 64, 5).view(2, 5, 64)
    ws = [m.int_weight.float() * m.weight_scale[:, None] for m in (mlp.gate_up, mlp.down)]
    want = mxfp4_swiglu(x, *ws)
    assert torch.equal(blk(x), want)
    assert torch.equal(*(torch.autograd.grad(y, x, dy)[0] for y in (blk(x), want)))
    mlp.down = BitLinear(96, 64, bias=True).to(DEV)
    with pytest.raises(ValueError, match="bias"):
        MXFP4SwiGLU.from_swiglu_mlp(mlp)


def test_a_trained_decoder_runs_in_four_bits():
    """MXFP4 layers in the places of a decoder's (and a SwiGLU block's) int8 layers, all of them or one: the fused int8
    operators step aside, and the result is that of the layers one after another."""
    from firefly_b200.decoder import DecoderConfig, build_decoder
    from firefly_b200.swiglu import SwiGLUMLP
    from torch.nn import functional as F

    cfg = DecoderConfig(vocab=96, d_model=64, heads=2, ffn=128, layers=2, max_seq=16)
    model = build_decoder(cfg, DEV, seed=1)
    ids = torch.randint(0, cfg.vocab, (2, 16), device=DEV, generator=_gen(2))
    with torch.no_grad():
        before = model(ids)
    for names in (("up",), ("down",), ("qkv", "proj", "up", "down")):
        model = build_decoder(cfg, DEV, seed=1)
        for layer in model.layers:
            for name in names:
                setattr(layer, name, MXFP4Linear.from_bitlinear(getattr(layer, name), input_grad=True))
        got = model(ids)
        assert got.shape == before.shape and torch.isfinite(got).all()
        layer = model.layers[0]
        x = _randn(2, 16 * 64, 3, scale=0.1).view(2, 16, 64).requires_grad_(True)
        y = layer.mlp(x)
        ref = layer.down(F.gelu(layer.up(x), approximate="tanh"))
        assert torch.equal(y, ref)
        dy = _randn(2, 16 * 64, 4).view(2, 16, 64)
        assert torch.equal(*(torch.autograd.grad(t, x, dy)[0] for t in (y, ref)))
    model.lm_head = MXFP4Linear.from_bitlinear(model.lm_head)
    with torch.no_grad():
        top = model(ids).float().topk(8, dim=-1)
    student = build_decoder(cfg, DEV, seed=3)
    student.distill_loss(ids, ids, top.indices, top.values).backward()
    for lin in student.bit_modules():
        assert lin.consume_weight_grad() is not None
    mlp = SwiGLUMLP(64, 128).to(DEV)
    x = _randn(5, 64, 5)
    for name in ("gate_up", "down"):
        setattr(mlp, name, MXFP4Linear.from_bitlinear(getattr(mlp, name)))
        with torch.no_grad():
            g, u = mlp.gate_up(x).chunk(2, dim=-1)
            assert torch.equal(mlp(x), mlp.down(F.silu(g) * u))


def test_no_outputs():
    """Weights without rows: empty results, gradients of zeros."""
    x = _randn(7, 64, 1).requires_grad_(True)
    w, b = _randn(5, 64, 2)[:0].requires_grad_(True), torch.zeros(0, device=DEV, requires_grad=True)
    y = mxfp4_linear(x, w, b)
    assert y.shape == (7, 0)
    dx, dw, db = torch.autograd.grad(y.sum(), [x, w, b])
    assert dx.shape == (7, 64) and not dx.any() and dw.shape == (0, 64) and db.shape == (0,)
    wgu, wd = _randn(64, 64, 3).requires_grad_(True), _randn(5, 32, 4)[:0].requires_grad_(True)
    y = mxfp4_swiglu(x, wgu, wd)
    assert y.shape == (7, 0)
    dx, dgu, dd = torch.autograd.grad(y.sum(), [x, wgu, wd])
    assert dx.shape == (7, 64) and not dx.any() and dgu.shape == (64, 64) and not dgu.any() and dd.shape == (0, 32)
