"""The 4-bit operators on the GPU against float64.

Quantisation is exact: codes and scales are compared bit by bit.  In a product every term is exact; the fp32 sum of K
terms is off by at most K steps of 2^-23 of sum |a w| (a step each if the adder truncates), the result is rounded once
(half a step: 2^-11 of it in fp16, 2^-24 in fp32), and the activations pass an error on with a slope of at most 1.13.
Their own errors: GELU in fp32 1e-5 of the value; its tanh in fp16 and 4-bit results is the hardware's, documented as
2^-11 relative, so 0.5 |x| 2^-11; tanhf 2^-22.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_oracle as X
from effective_transformer_b200 import _capi, mxfp4

pytestmark = pytest.mark.gpu
NP = {torch.float16: np.float16, torch.float32: np.float32}
DTYPES = [torch.float16, torch.float32]
DT = {torch.float16: _capi.ET_FP16, torch.float32: _capi.ET_FP32}


def route(rows, n, k, dtype=1):
    m, t, one = C.c_int(), C.c_int(), C.c_int()
    assert _capi.load().et_mxfp4_route(dtype, rows, n, k, C.byref(m), C.byref(t), C.byref(one)) == 0
    return m.value, t.value, one.value


def rows_of(rng, rows, k, dtype, spread=True):
    x = rng.randn(rows, k)
    if spread:
        x *= np.exp2(rng.randint(-6, 7, size=(rows, max(1, k // 32)))).repeat(32, axis=1)[:, :k]
    return x.astype(NP[dtype])


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def count(n):
    return torch.full((1,), n, dtype=torch.int32, device="cuda")


def same_parts(mx, x):
    codes, scales = X.mx_parts(x)
    got_codes, got_scales = X.mx_unpack(mx.data.cpu().numpy(), x.shape[0], x.shape[1])
    assert np.array_equal(got_scales, scales)
    assert np.array_equal(got_codes, codes)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 1024), (7, 96), (33, 256), (128, 288), (129, 768), (300, 2080),
                                    (1000, 1024)])
def test_quantize(dtype, rows, k):
    x = rows_of(np.random.RandomState(rows + k), rows, k, dtype)
    mx = mxfp4.quantize(cuda(x))
    same_parts(mx, x)
    back = mxfp4.dequantize(mx, torch.float32).cpu().numpy()
    assert np.array_equal(back, X.mx_values(x).astype(np.float32))
    assert np.array_equal(mxfp4.dequantize(mx, torch.float16).cpu().numpy(), X.mx_values(x).astype(np.float16))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties_ranges_and_specials(dtype):
    t = NP[dtype]
    x = np.zeros((12, 64), t)
    x[0] = np.arange(64) / 8                                  # ties and saturation, scale 1 and 1
    x[1] = -x[0]
    x[2] = np.finfo(t).max
    x[3] = np.finfo(t).smallest_subnormal
    x[4, ::2] = np.finfo(t).tiny
    x[5, 5] = np.inf
    x[6, 40] = -np.inf
    x[7, 63] = np.nan
    x[8, :32] = np.linspace(-7.9, 7.9, 32)
    x[9] = -0.0
    x[10, 0], x[10, 1:32] = 4096, np.linspace(1, 600, 31)     # a value that dwarfs its block
    x[11] = np.float64(np.finfo(t).smallest_subnormal) * np.arange(64)
    mx = mxfp4.quantize(cuda(x))
    same_parts(mx, x)
    want = X.mx_values(x)
    got = mxfp4.dequantize(mx, torch.float32).cpu().numpy()
    assert np.array_equal(got, want.astype(np.float32), equal_nan=True)
    assert np.isnan(got[5, :32]).all() and not np.isnan(got[5, 32:]).any()


def test_every_code_at_every_scale_comes_back():
    """Both directions are exact in fp32; in fp16 the one rounding of a value (2^-24 steps below 2^-14, infinity above)."""
    codes = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
    block = np.concatenate([codes, -codes, -codes, codes])
    x = (block[None, :] * 2.0 ** np.arange(-127, 126)[:, None]).astype(np.float32)
    mx = mxfp4.quantize(cuda(x))
    same_parts(mx, x)
    assert np.array_equal(mxfp4.dequantize(mx, torch.float32).cpu().numpy(), x)
    with np.errstate(over="ignore"):
        want = x.astype(np.float16)
    got = mxfp4.dequantize(mx, torch.float16).cpu().numpy()
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strided_rows_and_rows_past_the_count(dtype):
    rng = np.random.RandomState(3)
    wide = cuda(rows_of(rng, 200, 3 * 96, dtype))
    x = wide[:, 96:192]                                        # a head group of a fused projection's rows
    mx = mxfp4.empty(200, 96)
    mx.data.fill_(0xAB)
    mxfp4.quantize(x, valid_rows=count(133), out=mx)
    codes, scales = X.mx_unpack(mx.data.cpu().numpy(), 200, 96)
    want_codes, want_scales = X.mx_parts(x[:133].cpu().numpy())
    assert np.array_equal(codes[:133], want_codes) and np.array_equal(scales[:133], want_scales)
    assert (scales[133:] == 0xAB).all() and (codes[133:, 0::2] == 0xB).all() and (codes[133:, 1::2] == 0xA).all()
    out = torch.full((200, 96), 7.0, dtype=dtype, device="cuda")
    mxfp4.dequantize(mx, dtype, valid_rows=count(100), out=out)
    assert torch.equal(out[:100].cpu().double(), torch.from_numpy(X.mx_values(x[:100].cpu().numpy())))
    assert (out[100:] == 7.0).all()
    for n in (0, -5):
        mx.data.fill_(0xAB)
        mxfp4.quantize(x, valid_rows=count(n), out=mx)
        assert (mx.data == 0xAB).all()
    mxfp4.quantize(x, valid_rows=count(10 ** 6), out=mx)       # a count past the capacity is the capacity
    same_parts(mx, x.cpu().numpy())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(32, 32), (96, 160), (768, 128), (800, 2304)])
def test_pack_weight(dtype, k, n):
    w = rows_of(np.random.RandomState(k + n), n, k, dtype).T.copy()
    mx = mxfp4.pack_weight(cuda(w))
    assert (mx.rows, mx.cols) == (n, k)
    same_parts(mx, np.ascontiguousarray(w.T))


def reference(x, kernel, bias, act, residual, dtype, rough=False):
    """(result, bound on |error|) in float64, on the GPU."""
    a, w = cuda(X.mx_values(x)), cuda(X.mx_values(np.ascontiguousarray(kernel.T)))
    k = x.shape[1]
    y = a @ w.t()
    err = (k + 8) * 2.0 ** -23 * (a.abs() @ w.abs().t())
    if bias is not None:
        y = y + bias.double()
        err = err + 2.0 ** -24 * y.abs()
    if act == "gelu":
        u = y
        y = X.gelu(u)
        err = 1.13 * err + 1e-5 * y.abs() + (0.5 * u.abs() * 2.0 ** -11 if rough or dtype == torch.float16 else 0)
    elif act == "tanh":
        y = y.tanh()
        err = err + 2.0 ** -22
    if residual is not None:
        y = y + residual.double()
        err = err + 2.0 ** -24 * y.abs()
    half_step = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    return y, err + half_step * (y.abs() + err) + 2.0 ** -25  # (half a step of fp16 subnormals)


def product_case(seed, m, k, n, dtype, act, with_bias, with_residual, spread=False):
    rng = np.random.RandomState(seed)
    x = rows_of(rng, m, k, dtype, spread)
    kernel = (rng.randn(k, n) * 0.05).astype(NP[dtype])
    bias = cuda((rng.randn(n) * 0.3).astype(NP[dtype])) if with_bias else None
    residual = cuda(rng.randn(m, n).astype(NP[dtype])) if with_residual else None
    return x, kernel, bias, residual, reference(x, kernel, bias, act, residual, dtype)


SHAPES = [(1, 32, 32), (1, 1024, 1024), (3, 64, 64), (37, 96, 160), (64, 768, 2304), (128, 256, 128), (129, 800, 96),
          (200, 1056, 288), (513, 128, 4096), (1000, 2048, 512)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product(dtype, m, k, n):
    x, kernel, bias, _, (want, bound) = product_case(m + k + n, m, k, n, dtype, None, True, False)
    a, w = mxfp4.quantize(cuda(x)), mxfp4.pack_weight(cuda(kernel))
    got = mxfp4.gemm(a, w, bias=bias)
    assert got.dtype == dtype and got.shape == (m, n)
    assert ((got.double() - want).abs() <= bound).all()
    assert mxfp4.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 32, 32), (1, 1024, 4096), (2, 1536, 96), (32, 800, 160), (128, 96, 1024),
                                   (42, 768, 2304), (25, 1056, 288)])
def test_few_rows_in_one_kernel(dtype, m, k, n):
    """The product that quantises its rows itself: the same bits as quantisation and product, at any stride, with rows past
    the count left alone, into fp16, fp32 and 4 bits."""
    assert route(m, n, k, DT[dtype])[2] == 1
    x, kernel, bias, residual, (want, bound) = product_case(m + k, m, k, n, dtype, "gelu", True, True, True)
    w, xt = mxfp4.pack_weight(cuda(kernel)), cuda(x)
    got = mxfp4.linear(xt, w, bias=bias, activation="gelu", residual=residual)
    assert ((got.double() - want).abs() <= bound).all()
    a = mxfp4.quantize(xt)
    assert torch.equal(got, mxfp4.gemm(a, w, bias=bias, activation="gelu", residual=residual))
    wide = torch.full((m, k + 32), float("nan"), dtype=dtype, device="cuda")
    wide[:, 16:k + 16] = xt
    out = torch.full((m, n), 3.0, dtype=dtype, device="cuda")
    for valid in {0, 1, m // 2, m, m + 5}:
        t = min(valid, m)
        out.fill_(3.0)
        mxfp4.linear(wide[:, 16:k + 16], w, bias=bias, activation="gelu", residual=residual, valid_rows=count(valid), out=out)
        assert torch.equal(out[:t], got[:t]) and (out[t:] == 3.0).all()
    if n % 64 == 0:
        in4, two = mxfp4.linear(xt, w, bias=bias, out=mxfp4.empty(m, n)), mxfp4.gemm(a, w, bias=bias, out=mxfp4.empty(m, n))
        assert torch.equal(mxfp4.dequantize(in4, torch.float32), mxfp4.dequantize(two, torch.float32))
    assert mxfp4.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "gelu", "tanh"])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("m,k,n", [(5, 128, 96), (300, 512, 640)])
def test_epilogues(dtype, act, with_residual, m, k, n):
    x, kernel, bias, residual, (want, bound) = product_case(17, m, k, n, dtype, act, True, with_residual, True)
    w = mxfp4.pack_weight(cuda(kernel))
    got = mxfp4.linear(cuda(x), w, bias=bias, activation=act, residual=residual)
    assert ((got.double() - want).abs() <= bound).all()
    if residual is not None:                                    # in place on the residual
        same = mxfp4.linear(cuda(x), w, bias=bias, activation=act, residual=residual, out=residual)
        assert same is residual and torch.equal(residual, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n,act,with_residual", [
    (4100, 256, 2048, None, False), (8200, 800, 1088, "gelu", False), (6000, 96, 1440, None, True),
    (20011, 1312, 1024, "tanh", True), (33000, 64, 288, "gelu", True), (4097, 2592, 2080, None, False),
    (4100, 2048, 1216, "gelu", False), (6000, 2080, 1440, None, True), (9001, 2336, 1024, "tanh", True),
    (33000, 2144, 288, "gelu", True), (38000, 2048, 32, None, False), (20011, 800, 480, "gelu", True)])
def test_large_products(dtype, m, k, n, act, with_residual):
    """Many tiles to a CTA; from K = 2048 on the kernel of CTA pairs: last tiles of 64, 128 and 192 columns that begin at
    the start or in the middle of a row block of W, k-tiles with one to four steps, a row block too many."""
    if k >= 2048:
        assert route(m, n, k) == (256, 192, 0) and (m * n < 3 * 148 * 2**14 or route(m, n, k, 0) == (256, 192, 0))
    x, kernel, bias, residual, (want, bound) = product_case(m, m, k, n, dtype, act, True, with_residual)
    got = mxfp4.linear(cuda(x), mxfp4.pack_weight(cuda(kernel)), bias=bias, activation=act, residual=residual)
    assert ((got.double() - want).abs() <= bound).all()
    valid = m - 300
    out = torch.full((m, n), 3.0, dtype=dtype, device="cuda")
    mxfp4.linear(cuda(x), mxfp4.pack_weight(cuda(kernel)), bias=bias, activation=act, residual=residual,
                 valid_rows=count(valid), out=out)
    assert torch.equal(out[:valid], got[:valid]) and (out[valid:] == 3.0).all()
    assert mxfp4.device_status() == 0


@pytest.mark.parametrize("m,k,n", [(1, 512, 256), (130, 1024, 512), (700, 320, 1024), (9000, 1024, 1152)])
def test_products_of_small_numbers_are_exact(m, k, n):
    """Operands of one scale: sums of multiples of 2^-2 below 2^16 fit 24 bits, whatever the order."""
    rng = np.random.RandomState(m)
    x = rng.choice(np.concatenate([X.GRID, -X.GRID]), size=(m, k)).astype(np.float32)
    kernel = rng.choice(np.concatenate([X.GRID, -X.GRID]), size=(k, n)).astype(np.float32)
    x[:, ::32], kernel[::32] = 6.0, -6.0                        # every block has scale 1
    got = mxfp4.gemm(mxfp4.quantize(cuda(x)), mxfp4.pack_weight(cuda(kernel)), dtype=torch.float32)
    assert torch.equal(got.double(), cuda(x).double() @ cuda(kernel).double())


@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (77, 768, 320), (300, 512, 1024), (5001, 288, 1856),
                                   (5001, 2080, 1856)])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_product_in_4_bits(m, k, n, act):
    """c_mx is the quantised form of the fp32 result: scales and codes agree except where the fp32 result lies within
    its bound of a border, and there they are off by one code."""
    x, kernel, bias, _, _ = product_case(5, m, k, n, torch.float16, None, True, False)
    a, w = mxfp4.quantize(cuda(x)), mxfp4.pack_weight(cuda(kernel))
    out = mxfp4.gemm(a, w, bias=bias, activation=act, out=mxfp4.empty(m, n))
    want, bound = reference(x, kernel, bias, act, None, torch.float32, rough=True)
    got = mxfp4.dequantize(out, torch.float32).cpu().numpy()
    lo, hi = (want - bound).cpu().numpy(), (want + bound).cpu().numpy()
    top_lo = np.abs(want.cpu().numpy()).reshape(m, -1, 32).max(-1) - bound.cpu().numpy().reshape(m, -1, 32).max(-1)
    top_hi = np.abs(want.cpu().numpy()).reshape(m, -1, 32).max(-1) + bound.cpu().numpy().reshape(m, -1, 32).max(-1)
    _, scales = X.mx_unpack(out.data.cpu().numpy(), m, n)
    e = scales.astype(np.float64) - 127 + 2
    assert (np.floor(np.log2(np.maximum(top_lo, 1e-30))) <= e).all() and (e <= np.floor(np.log2(top_hi))).all()

    def code_values(v):                                         # rounded on the scales that came back
        s = np.exp2(scales.astype(np.float64) - 127).repeat(32, axis=1)
        q = np.abs(v) / s
        c = np.zeros(q.shape, int)
        for i in range(7):
            mid = (X.GRID[i] + X.GRID[i + 1]) / 2
            c += (q > mid) if i % 2 == 0 else (q >= mid)
        return np.copysign(X.GRID[c], v) * s

    assert (got >= code_values(lo)).all() and (got <= code_values(hi)).all()


# From few rows to CTA pairs: one kernel, tiles of 128 x 128, tiles of 256 x 192 (k >= 768 and three rounds of tiles).
GELU_SHAPES = [(3, 64, 1), (300, 64, 0), (8000, 768, 0)]


def gelu_bias(n, dtype, low, high):
    """Pre-activations: rows of zeros leave the bias alone."""
    return torch.linspace(low, high, n, dtype=torch.float64, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,one", GELU_SHAPES)
def test_gelu_holds_its_precision_in_the_negative_tail(dtype, m, k, one):
    """Relative to the result, not to x: for negative x the two terms of 0.5 x (1 + tanh u) cancel.

    The product is exactly zero, so the pre-activation is the bias.  x / (1 + exp(-2u)) in fp32: the argument of the
    exponential is below 37 for |x| <= 6 (as a power of two) and rounded four times, each 2^-24 of it, times ln 2; the
    exponential, the reciprocal and two products add less than eight steps of 2^-23 between them: 7.1e-6 in all."""
    n = 1024
    assert route(m, n, k, DT[dtype])[2] == one and (m != 8000 or route(m, n, k, DT[dtype])[0] == 256)
    bias = gelu_bias(n, dtype, -6.0, 6.0)
    x = torch.zeros(m, k, dtype=dtype, device="cuda")
    got = mxfp4.linear(x, mxfp4.pack_weight(torch.ones(k, n, dtype=dtype, device="cuda")), bias=bias, activation="gelu")
    want = X.gelu(bias.double()).expand(m, n)
    half_step = (2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24) * want.abs()
    subnormal = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert ((got.double() - want).abs() <= (half_step + 7.5e-6 * want.abs()).clamp(min=subnormal) * (1 + 1e-5)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,one", GELU_SHAPES)
def test_gelu_in_4_bits_in_the_negative_tail(dtype, m, k, one):
    """Whole scale blocks of negative pre-activations: codes and scales of the float64 values, but where a value is
    within the fp32 error above of a border."""
    n = 1024
    bias = gelu_bias(n, dtype, -6.0, -0.05)
    x = torch.zeros(m, k, dtype=dtype, device="cuda")
    w = mxfp4.pack_weight(torch.ones(k, n, dtype=dtype, device="cuda"))
    out = mxfp4.linear(x, w, bias=bias, activation="gelu", out=mxfp4.empty(m, n))
    want = X.gelu(bias.double())[None, :].cpu().numpy()
    lo, hi = (X.mx_values(want * (1 + s * 7.5e-6)) for s in (1, -1))     # (negative: the larger magnitude is lower)
    got = mxfp4.dequantize(out, torch.float32).double().cpu().numpy()
    assert (got >= lo).all() and (got <= hi).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_far_out(dtype):
    """Nothing is left of large negative values, all of large positive ones."""
    far = torch.tensor([-65000.0, -1000.0, -40.0, -20.0, 20.0, 40.0, 1000.0, 65000.0], device="cuda")
    if dtype == torch.float32:
        far = torch.cat([far, torch.tensor([-3e38, -1e20, 1e20, 3e38], device="cuda")])
    bias = torch.zeros(64, dtype=dtype, device="cuda")
    bias[:len(far)] = far.to(dtype)
    x = torch.zeros(5, 64, dtype=dtype, device="cuda")
    w = mxfp4.pack_weight(torch.ones(64, 64, dtype=dtype, device="cuda"))
    got = mxfp4.linear(x, w, bias=bias, activation="gelu")
    assert torch.equal(got, torch.where(bias > 0, bias, torch.zeros_like(bias)).expand(5, 64))


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("m,k,n", [(77, 768, 320), (300, 512, 1024), (5001, 2080, 1856), (9001, 1024, 1088)])
def test_product_in_4_bits_of_an_fp32_program(m, k, n, act):
    """test_product_in_4_bits with bias and rows in fp32: on the last two sizes the CTA-pair kernel that the first
    feed-forward projection of an fp32 handle runs on a full batch."""
    if m > 5000:
        assert route(m, n, k) == (256, 192, 0)
    x, kernel, bias, _, _ = product_case(6, m, k, n, torch.float32, None, True, False)
    w = mxfp4.pack_weight(cuda(kernel))
    out = mxfp4.gemm(mxfp4.quantize(cuda(x)), w, bias=bias, activation=act, out=mxfp4.empty(m, n))
    want, bound = reference(x, kernel, bias, act, None, torch.float32, rough=True)
    X.check_codes(out, want, bound)
    same = mxfp4.linear(cuda(x), w, bias=bias, activation=act, out=mxfp4.empty(m, n))
    assert torch.equal(mxfp4.dequantize(same, torch.float32), mxfp4.dequantize(out, torch.float32))
    valid = m - 70
    part = mxfp4.empty(m, n)
    part.data.fill_(0xCD)
    mxfp4.linear(cuda(x), w, bias=bias, activation=act, valid_rows=count(valid), out=part)
    assert torch.equal(mxfp4.dequantize(part, torch.float32)[:valid], mxfp4.dequantize(out, torch.float32)[:valid])
    codes, scales = X.mx_unpack(part.data.cpu().numpy(), m, n)
    assert (scales[valid:] == 0xCD).all() and (codes[valid:, 0::2] == 0xD).all() and (codes[valid:, 1::2] == 0xC).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_past_the_count_are_left_alone(dtype):
    x, kernel, bias, _, (want, bound) = product_case(23, 400, 288, 224, dtype, None, True, False)
    w = mxfp4.pack_weight(cuda(kernel))
    for valid in (0, 1, 127, 128, 129, 399, 400, 1000):
        xt = cuda(x)
        xt[valid:] = float("nan")
        out = torch.full((400, 224), 3.0, dtype=dtype, device="cuda")
        mxfp4.linear(xt, w, bias=bias, valid_rows=count(valid), out=out)
        t = min(valid, 400)
        assert ((out[:t].double() - want[:t]).abs() <= bound[:t]).all()
        assert (out[t:] == 3.0).all()
    small = mxfp4.empty(400, 64)
    small.data.fill_(0xCD)
    w64 = mxfp4.pack_weight(cuda(kernel[:, :64].copy()))
    mxfp4.linear(cuda(x), w64, valid_rows=count(250), out=small)
    codes, scales = X.mx_unpack(small.data.cpu().numpy(), 400, 64)
    assert (scales[250:] == 0xCD).all() and (codes[250:, 0::2] == 0xD).all() and (codes[250:, 1::2] == 0xC).all()


def test_non_finite_rows_stay_in_their_rows():
    x, kernel, bias, _, (want, bound) = product_case(29, 140, 512, 160, torch.float16, None, True, False)
    x[3, 100], x[130, 0] = np.inf, np.nan
    got = mxfp4.linear(cuda(x), mxfp4.pack_weight(cuda(kernel)), bias=bias)
    bad = torch.zeros(140, dtype=torch.bool, device="cuda")
    bad[[3, 130]] = True
    assert got[bad].isnan().all()
    assert ((got[~bad].double() - want[~bad]).abs() <= bound[~bad]).all()
    kernel[7, 5] = np.nan                                       # and in the column of a weight
    got = mxfp4.linear(cuda(x), mxfp4.pack_weight(cuda(kernel)), bias=bias)
    assert got[:, 5].isnan().all() and not got[~bad][:, [4, 6]].isnan().any()


def test_results_repeat_bit_by_bit():
    x, kernel, bias, _, _ = product_case(31, 300, 1024, 256, torch.float16, None, True, False)
    w = mxfp4.pack_weight(cuda(kernel))
    first = mxfp4.linear(cuda(x), w, bias=bias)
    for _ in range(3):
        assert torch.equal(mxfp4.linear(cuda(x), w, bias=bias), first)


def test_other_streams_and_capture():
    x, kernel, bias, _, (want, bound) = product_case(37, 90, 768, 256, torch.float16, "gelu", True, False)
    w, xt = mxfp4.pack_weight(cuda(kernel)), cuda(x)
    mxfp4.device_status()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mxfp4.linear(xt, w, bias=bias, activation="gelu")
    torch.cuda.current_stream().wait_stream(side)
    assert ((got.double() - want).abs() <= bound).all()
    ws, out, valid = mxfp4.empty(90, 768), torch.zeros(90, 256, dtype=torch.float16, device="cuda"), count(90)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mxfp4.linear(xt, w, bias=bias, activation="gelu", valid_rows=valid, workspace=ws, out=out)
    for rows in (90, 11, 64):
        out.zero_()
        valid.fill_(rows)
        graph.replay()
        assert ((out[:rows].double() - want[:rows]).abs() <= bound[:rows]).all() and (out[rows:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 32, 200])
def test_linear_in_place(dtype, rows):
    """out = x (and residual = x): every row has been quantised before a result is written."""
    assert route(rows, 768, 768, DT[dtype])[2] == (rows < 100)
    rng = np.random.RandomState(rows)
    x, kernel = cuda(rows_of(rng, rows, 768, dtype)), cuda(rows_of(rng, 768, 768, dtype))
    w = mxfp4.pack_weight(kernel)
    for residual in (False, True):
        want = mxfp4.linear(x, w, residual=x if residual else None)
        y = x.clone()
        got = mxfp4.linear(y, w, residual=y if residual else None, out=y)
        assert got is y and torch.equal(got, want)


def test_calls_on_two_streams_at_once():
    """Products of all three kernels, rows and norms on two streams, each with its own buffers: what one call alone gives.
    (They share the weights, the status word and the SMs' tensor memory.)"""
    rng = np.random.RandomState(8)
    shapes = [(5000, 768, 2304), (300, 768, 768), (9, 256, 512), (2, 1024, 1024), (4200, 2048, 1088)]
    jobs = []
    for m, k, n in shapes:
        x = cuda(rows_of(rng, m, k, torch.float16))
        w = mxfp4.pack_weight(cuda(rows_of(rng, k, n, torch.float16)))
        jobs.append((x, w, mxfp4.linear(x, w)))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    torch.cuda.synchronize()
    for turn in range(6):
        for s, stream in enumerate(side):
            with torch.cuda.stream(stream):
                x, w, _ = jobs[(turn + 2 * s) % len(jobs)]
                got[s].append(((turn + 2 * s) % len(jobs), mxfp4.linear(x, w), mxfp4.dequantize(mxfp4.quantize(x), x.dtype)))
    torch.cuda.synchronize()
    for results in got:
        for i, y, back in results:
            x, _, want = jobs[i]
            assert torch.equal(y, want)
            assert torch.equal(back, mxfp4.dequantize(mxfp4.quantize(x), x.dtype))
    assert mxfp4.device_status() == 0


def test_capture_needs_a_status_word_first():
    word = mxfp4._status.pop(torch.cuda.current_device(), None)
    try:
        a = mxfp4.empty(4, 64)
        w = mxfp4.empty(64, 64)
        out = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            torch.zeros(1, device="cuda")
            with pytest.raises(ValueError, match="captured"):
                mxfp4.gemm(a, w, out=out)
    finally:
        if word is not None:
            mxfp4._status[torch.cuda.current_device()] = word


def test_python_refusals_on_the_gpu():
    x = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    w = mxfp4.pack_weight(torch.zeros(64, 96, dtype=torch.float16, device="cuda"))
    b = torch.zeros(96, dtype=torch.float16, device="cuda")
    a = mxfp4.quantize(x)
    for call in (lambda: mxfp4.quantize(x[:, :33]), lambda: mxfp4.quantize(x.t()), lambda: mxfp4.quantize(x.double()),
                 lambda: mxfp4.quantize(x, out=mxfp4.empty(3, 64)), lambda: mxfp4.quantize(x, out=mxfp4.empty(4, 96)),
                 lambda: mxfp4.quantize(x, valid_rows=torch.ones(1, device="cuda")),
                 lambda: mxfp4.quantize(x, valid_rows=torch.ones(1, dtype=torch.int32)),
                 lambda: mxfp4.linear(x, w, activation="gelu"), lambda: mxfp4.linear(x, w, bias=b, activation="relu"),
                 lambda: mxfp4.linear(x, w, bias=b.float()), lambda: mxfp4.linear(x, w, bias=b[:64]),
                 lambda: mxfp4.linear(x, w, residual=x), lambda: mxfp4.linear(x, w, out=mxfp4.empty(4, 96)),
                 lambda: mxfp4.linear(x, w, out=torch.zeros(4, 96, device="cuda")),
                 lambda: mxfp4.gemm(a, w, out=torch.zeros(5, 96, dtype=torch.float16, device="cuda")),
                 lambda: mxfp4.gemm(a, mxfp4.pack_weight(torch.zeros(96, 64, dtype=torch.float16, device="cuda"))),
                 lambda: mxfp4.dequantize(a, torch.float16, out=torch.zeros(5, 64, dtype=torch.float16, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_capi.EtError):                          # rows that start between two 16-byte boundaries
        mxfp4.quantize(torch.zeros(4 * 64 + 4, dtype=torch.float16, device="cuda")[4:].view(4, 64))


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batches(dtype):
    x, b = torch.zeros(0, 64, dtype=dtype, device="cuda"), torch.zeros(128, dtype=dtype, device="cuda")
    w = mxfp4.pack_weight(torch.zeros(64, 128, dtype=dtype, device="cuda"))
    a = mxfp4.quantize(x)
    assert (a.rows, a.cols) == (0, 64) and mxfp4.dequantize(a, dtype).shape == (0, 64)
    for y in (mxfp4.gemm(a, w, dtype=dtype), mxfp4.gemm(a, w, bias=b, activation="gelu", residual=x.new_zeros(0, 128)),
              mxfp4.linear(x, w), mxfp4.linear(x, w, bias=b, activation="tanh", valid_rows=count(0))):
        assert y.shape == (0, 128) and y.dtype == dtype
    out = mxfp4.empty(0, 128)
    assert mxfp4.gemm(a, w, bias=b, out=out) is out and mxfp4.linear(x, w, out=out) is out


def test_gradients_are_not_lost_silently():
    x = torch.randn(4, 64, device="cuda").half()
    w = mxfp4.pack_weight(torch.nn.Parameter(torch.randn(64, 64, device="cuda").half()))
    b = torch.nn.Parameter(torch.zeros(64, device="cuda").half())
    leaf = x.clone().requires_grad_()
    want = mxfp4.linear(x, w, bias=b.detach(), residual=x)
    a = mxfp4.quantize(x)
    for call in (lambda: mxfp4.linear(x, w, bias=b, residual=x), lambda: mxfp4.gemm(a, w, bias=b, residual=x),
                 lambda: mxfp4.linear(leaf, w, bias=b.detach(), residual=x),
                 lambda: mxfp4.gemm(a, w, bias=b.detach(), residual=leaf)):
        y = call()
        assert torch.equal(y, want) and y.requires_grad
        with pytest.raises(NotImplementedError, match="no backward"):
            (y.float().sum() + leaf.float().sum()).backward()
        with torch.no_grad():
            assert torch.equal(call(), want) and not call().requires_grad
    assert not want.requires_grad
    out = torch.empty_like(x)
    for call in (lambda: mxfp4.linear(leaf, w, out=out), lambda: mxfp4.gemm(a, w, bias=b, out=out),
                 lambda: mxfp4.quantize(leaf), lambda: mxfp4.linear(x, w, bias=b, out=mxfp4.empty(4, 64))):
        with pytest.raises(ValueError, match="no backward"):
            call()
        with torch.no_grad():
            call()
