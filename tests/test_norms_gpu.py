"""norms.gated_residual_norm against float64.

One rounding per output: 2^-11 (fp16) or 2^-24 (fp32) of the value.  In front of it the fp32 arithmetic: a mean of n
terms and a mean of squares summed in groups of at most 32 * 4 * 8 / 32 terms per lane and 8 more levels carry less than
64 steps of 2^-24, a row with |mean| = 60 sigma loses 60 of them to the difference, rsqrtf 2 steps, and the two norms
follow one another: 1e-5 relative to the row's largest |h| (gamma and the gate are of order one) bounds all of it.
"""
import numpy as np
import pytest
import torch

import mx_oracle as X
from effective_transformer_b200 import mxfp4, norms

pytestmark = pytest.mark.gpu
HALF = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DTYPES = [torch.float16, torch.float32]


def make(seed, rows, n, dtype, seqs=0, mean=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, centre=0.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + centre).to(dtype)

    a = dict(x=normal(rows, n, centre=mean), bias=normal(n, scale=0.1), residual=normal(rows, n),
             post_gamma=normal(n, scale=0.1, centre=1.0), post_beta=normal(n, scale=0.1),
             pre_gamma=normal(n, scale=0.1, centre=1.0), pre_beta=normal(n, scale=0.1))
    if seqs:
        a["gate"] = normal(seqs, n, scale=0.5)
        a["batch_idx"] = torch.sort(torch.randint(0, seqs, (rows,), generator=gen, device="cuda", dtype=torch.int32))[0]
    return a


def want_of(a, post, pre, scale=1.0, eps=1e-6):
    return X.gated_norm(a["x"], a.get("bias"), a.get("residual"), scale, a.get("gate"), a.get("batch_idx"), post,
                        a["post_gamma"], a["post_beta"], pre, a["pre_gamma"], a["pre_beta"], eps)


def close(got, want, h, dtype):
    """h: the row whose size scales the fp32 error."""
    size = torch.maximum(want.abs(), h.abs()).amax(-1, keepdim=True) + 1.0
    assert ((got.double() - want).abs() <= HALF[dtype] * want.abs() + 1e-5 * size + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(1, 8), (1, 768), (5, 136), (33, 1024), (9, 2080), (300, 256), (17, 4096)])
@pytest.mark.parametrize("post,pre", [("none", "layer"), ("layer", "rms"), ("rms", "layer"), ("rms", "none"), ("layer", "layer")])
def test_norms(dtype, rows, n, post, pre):
    a = make(rows + n, rows, n, dtype, seqs=3)
    h, y = norms.gated_residual_norm(**a, post_norm=post, pre_norm=pre, residual_scale=0.75)
    wh, wy = want_of(a, post, pre, 0.75)
    close(h, wh, wh, dtype)
    close(y, wy, wh, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(601, 96), (400, 512), (301, 760), (333, 1024), (299, 1000), (301, 1536), (310, 2048),
                                    (170, 2600), (160, 4096)])
def test_norms_of_many_rows(dtype, rows, n):
    """More rows than one to a CTA: two rows at a time or two vectors a lane, rounds of the grid, rows past the count."""
    a = make(rows + n, rows, n, dtype, seqs=7)
    h, y = torch.full_like(a["x"], 3.0), torch.full_like(a["x"], 3.0)
    valid = torch.full((1,), rows - 5, dtype=torch.int32, device="cuda")
    norms.gated_residual_norm(**a, post_norm="layer", pre_norm="rms", residual_scale=0.75, valid_rows=valid, h_out=h,
                              y_out=y)
    wh, wy = want_of(a, "layer", "rms", 0.75)
    close(h[:-5], wh[:-5], wh[:-5], dtype)
    close(y[:-5], wy[:-5], wh[:-5], dtype)
    assert (h[-5:] == 3.0).all() and (y[-5:] == 3.0).all()


# (dtype, rows, width, rows of one round of the grid at the most: SMs x CTAs that 64 K registers hold x rows of a CTA)
F16, F32 = DTYPES
ROUNDS = [(F16, 12003, 96, 148 * 4 * 8), (F16, 12003, 256, 148 * 4 * 8), (F16, 7001, 512, 148 * 4 * 4),
          (F16, 4099, 760, 148 * 5 * 2), (F16, 5003, 1024, 148 * 4 * 2), (F16, 3001, 1536, 148 * 2 * 2),
          (F16, 2999, 1000, 148 * 4 * 2), (F16, 1501, 4096, 148 * 1 * 2), (F16, 1203, 4608, 148 * 2), (F16, 1203, 5120, 148 * 2),
          (F16, 701, 5768, 148), (F16, 701, 8192, 148),
          (F32, 12003, 96, 148 * 4 * 8), (F32, 7001, 256, 148 * 4 * 4), (F32, 4099, 640, 148 * 3 * 2),
          (F32, 4099, 896, 148 * 2 * 2), (F32, 5003, 1024, 148 * 4), (F32, 3001, 1280, 148 * 4), (F32, 3001, 1536, 148 * 3),
          (F32, 3001, 1792, 148 * 3), (F32, 3001, 1184, 148 * 4), (F32, 3001, 1408, 148 * 3), (F32, 3001, 1664, 148 * 3), (F32, 2001, 2048, 148 * 2), (F32, 2001, 2080, 148 * 2), (F32, 2001, 2560, 148 * 2),
          (F32, 1003, 2688, 148), (F32, 1003, 4096, 148)]


@pytest.mark.parametrize("dtype,rows,n,one_round", ROUNDS)
def test_rounds_of_the_grid(dtype, rows, n, one_round):
    """More rows than the grid holds at once, several times over: what a lane fetches ahead for its next rows, the last
    round's rows of which one or none is there, and every number of warps to a row, with the gate found through
    batch_idx two rounds ahead."""
    assert rows > 2 * one_round and rows % 2 == 1
    a = make(rows + n, rows, n, dtype, seqs=37)
    a["batch_idx"] = a["batch_idx"][torch.randperm(rows, device="cuda")].contiguous()
    valid_rows = rows - 6
    valid = torch.full((1,), valid_rows, dtype=torch.int32, device="cuda")
    wh, wy = want_of(a, "layer", "rms", 0.75)
    h, y = torch.full_like(a["x"], 3.0), torch.full_like(a["x"], 3.0)
    norms.gated_residual_norm(**a, post_norm="layer", pre_norm="rms", residual_scale=0.75, valid_rows=valid, h_out=h,
                              y_out=y)
    close(h[:valid_rows], wh[:valid_rows], wh[:valid_rows], dtype)
    close(y[:valid_rows], wy[:valid_rows], wh[:valid_rows], dtype)
    assert (h[valid_rows:] == 3.0).all() and (y[valid_rows:] == 3.0).all()
    # over its own inputs: what is fetched ahead is not what has just been written
    norms.gated_residual_norm(**a, post_norm="layer", pre_norm="rms", residual_scale=0.75, h_out=a["x"],
                              y_out=a["residual"])
    assert torch.equal(a["x"][:valid_rows], h[:valid_rows]) and torch.equal(a["residual"][:valid_rows], y[:valid_rows])
    close(a["x"], wh, wh, dtype)
    close(a["residual"], wy, wh, dtype)


@pytest.mark.parametrize("dtype,rows,n", [
    (F16, 700, 96), (F16, 333, 1024), (F16, 301, 1536), (F16, 12003, 96), (F16, 5003, 1024), (F16, 1501, 4096),
    (F16, 1203, 5120), (F16, 701, 8192), (F32, 700, 96), (F32, 333, 1024), (F32, 301, 1536), (F32, 4099, 608),
    (F32, 5003, 1024), (F32, 2001, 2080), (F32, 1003, 4096)])
def test_quantized_rows_of_a_batch(dtype, rows, n):
    """y in 4 bits of many rows against the codes of float64: they agree but where a value lies within the fp32 error
    (1e-5 of the row's size, as above) of a border."""
    a = make(rows + n, rows, n, dtype, seqs=5)
    valid_rows = rows - 3
    valid = torch.full((1,), valid_rows, dtype=torch.int32, device="cuda")
    mx = mxfp4.empty(rows, n)
    mx.data.fill_(0xEE)
    y_out = torch.full_like(a["x"], 3.0)
    h, _ = norms.gated_residual_norm(**a, post_norm="rms", pre_norm="layer", valid_rows=valid, y_out=y_out, mx_out=mx)
    wh, wy = want_of(a, "rms", "layer")
    close(h[:valid_rows], wh[:valid_rows], wh[:valid_rows], dtype)
    close(y_out[:valid_rows], wy[:valid_rows], wh[:valid_rows], dtype)
    size = torch.maximum(wy.abs(), wh.abs()).amax(-1, keepdim=True) + 1.0
    X.check_codes(mx, wy[:valid_rows], (1e-5 * size).expand_as(wy)[:valid_rows])
    codes, scales = X.mx_unpack(mx.data.cpu().numpy(), rows, n)
    assert (scales[valid_rows:] == 0xEE).all() and (codes[valid_rows:] == 0xE).all() and (y_out[valid_rows:] == 3.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_and_product_repeat_bit_by_bit(dtype):
    """The rows that a norm leaves in 4 bits and the product behind it, over and over on buffers full of other values."""
    a = make(77, 5003, 1024, dtype)
    w = mxfp4.pack_weight(torch.randn(1024, 1088, device="cuda").to(dtype))
    mx, out = mxfp4.empty(5003, 1024), torch.empty(5003, 1088, dtype=dtype, device="cuda")
    first = None
    for turn in range(12):
        mx.data.fill_(0x11 * turn)
        out.fill_(float("nan"))
        h, _ = norms.gated_residual_norm(**a, post_norm="none", pre_norm="layer", mx_out=mx)
        mxfp4.gemm(mx, w, out=out)
        got = (h, mxfp4.dequantize(mx, torch.float32), out.clone())
        first = first or got
        assert all(torch.equal(u, v) for u, v in zip(got, first))


def test_norms_on_two_streams_at_once():
    """Norms, their 4-bit rows and the products behind them on two streams, each with its own buffers: what one call
    alone gives."""
    shapes = [(5003, 1024), (40, 768), (1501, 4096), (2, 1024)]
    jobs = []
    for rows, n in shapes:
        a = make(rows + n, rows, n, torch.float16, seqs=3)
        w = mxfp4.pack_weight(torch.randn(n, 576, device="cuda").half())

        def chain(a=a, w=w, rows=rows, n=n):
            mx = mxfp4.empty(rows, n)
            h, _ = norms.gated_residual_norm(**a, post_norm="layer", mx_out=mx)
            return h, mxfp4.gemm(mx, w)

        jobs.append((chain, chain()))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for turn in range(8):
        for s, stream in enumerate(side):
            with torch.cuda.stream(stream):
                i = (turn + s) % len(jobs)
                got.append((i, jobs[i][0]()))
    torch.cuda.synchronize()
    for i, results in got:
        assert all(torch.equal(u, v) for u, v in zip(results, jobs[i][1]))
    assert mxfp4.device_status() == 0


@pytest.mark.parametrize("n", [8192, 5000, 8184])
def test_widest_fp16_rows(n):
    a = make(n, 6, n, torch.float16)
    h, y = norms.gated_residual_norm(**a, post_norm="layer", pre_norm="rms")
    wh, wy = want_of(a, "layer", "rms")
    close(h, wh, wh, torch.float16)
    close(y, wy, wh, torch.float16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("drop", ["bias", "residual", "gate", "all"])
def test_absent_terms(dtype, drop):
    a = make(3, 40, 384, dtype, seqs=4)
    for k in ("bias", "residual", "gate", "batch_idx"):
        if drop in (k, "all") or (drop == "gate" and k == "batch_idx"):
            a[k] = None
    h, y = norms.gated_residual_norm(**a, post_norm="rms", pre_norm="layer", residual_scale=2.0)
    wh, wy = want_of(a, "rms", "layer", 2.0)
    close(h, wh, wh, dtype)
    close(y, wy, wh, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gates(dtype):
    a = make(4, 64, 256, dtype)
    for gate in (torch.randn(256, device="cuda").to(dtype), torch.randn(1, 256, device="cuda").to(dtype)):
        a["gate"] = gate
        h, _ = norms.gated_residual_norm(**a, post_norm="layer")
        wh, _ = want_of(a, "layer", "layer")
        close(h, wh, wh, dtype)
    a = make(5, 64, 256, dtype, seqs=7)
    a["batch_idx"] = torch.randint(0, 7, (64,), device="cuda", dtype=torch.int32)
    a["batch_idx"][[3, 9, 63]] = torch.tensor([-1, 7, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    a["x"][9] = float("inf")                                    # a closed gate lets nothing through
    h, y = norms.gated_residual_norm(**a, pre_norm="rms", residual_scale=0.5)
    assert torch.equal(h[[3, 9, 63]].double(), (a["residual"][[3, 9, 63]].double() * 0.5).to(dtype).double())
    wh, wy = want_of(a, "none", "rms", 0.5)
    close(h, wh, wh, dtype)
    close(y, wy, wh, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_rows_and_large_means(dtype):
    """A constant row has no spread: LayerNorm gives beta.  |mean| = 60 sigma loses no more than the bound says."""
    a = make(6, 8, 1024, dtype, mean=60.0)
    a["x"][2], a["bias"], a["residual"] = 5.0, None, None
    h, y = norms.gated_residual_norm(**a, post_norm="none", pre_norm="layer")
    wh, wy = want_of(a, "none", "layer")
    assert torch.equal(y[2], a["pre_beta"])
    close(h, wh, wh, dtype)
    close(y, wy, wh, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_rows_stay_in_their_rows(dtype):
    a = make(7, 12, 512, dtype)
    a["x"][4, 7], a["x"][5, 0] = float("nan"), float("inf")
    h, y = norms.gated_residual_norm(**a, post_norm="layer", pre_norm="layer")
    keep = [i for i in range(12) if i not in (4, 5)]
    wh, wy = want_of(a, "layer", "layer")
    assert y[4].isnan().all() and y[5].isnan().all()
    close(h[keep], wh[keep], wh[keep], dtype)
    close(y[keep], wy[keep], wh[keep], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_and_rows_past_the_count(dtype):
    a = make(8, 100, 640, dtype, seqs=5)
    wh, wy = want_of(a, "layer", "rms")
    for valid in (0, 1, 57, 100, 1000):
        b = {k: (v.clone() if v is not None else None) for k, v in a.items()}
        t = min(valid, 100)
        n = torch.full((1,), valid, dtype=torch.int32, device="cuda")
        h, y = norms.gated_residual_norm(**b, post_norm="layer", pre_norm="rms", valid_rows=n, h_out=b["residual"],
                                         y_out=b["x"])
        assert h is b["residual"] and y is b["x"]
        close(h[:t], wh[:t], wh[:t], dtype)
        close(y[:t], wy[:t], wh[:t], dtype)
        assert torch.equal(h[t:], a["residual"][t:]) and torch.equal(y[t:], a["x"][t:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [(1, 32), (70, 96), (131, 1024), (40, 2080), (3, 4096), (5, 416)])
def test_quantized_output_is_the_quantised_y(dtype, rows, n):
    """y in 4 bits next to y itself: what fp32 y rounds to, up to the rounding of y as it is returned (a code's border
    may lie between); with fp32 rows they are equal bit by bit."""
    a = make(rows + n, rows, n, dtype)
    mx = mxfp4.empty(rows, n)
    mx.data.fill_(0xEE)
    y_out = torch.empty_like(a["x"])
    h, y = norms.gated_residual_norm(**a, post_norm="none", pre_norm="layer", y_out=y_out, mx_out=mx)
    got = X.mx_unpack(mx.data.cpu().numpy(), rows, n)
    if dtype == torch.float32:
        codes, scales = X.mx_parts(y.cpu().numpy())
        assert np.array_equal(got[0], codes) and np.array_equal(got[1], scales)
    else:
        yv = y.double().cpu().numpy()
        back = mxfp4.dequantize(mx, torch.float32).cpu().numpy()
        step = np.exp2(got[1].astype(np.float64) - 127).repeat(32, axis=1) * np.where(
            np.abs(back) >= 4 * np.exp2(got[1].astype(np.float64) - 127).repeat(32, axis=1), 2.0, 1.0)
        assert (np.abs(back - yv) <= step * (1 + 2.0 ** -10)).all()
    # the block between an odd width / 32 and a multiple of 64 is zero: the product reads it
    kernel = torch.randn(n, 64, device="cuda").to(dtype)
    c = mxfp4.gemm(mx, mxfp4.pack_weight(kernel), dtype=torch.float32)
    v = mxfp4.dequantize(mx, torch.float32).double() @ mxfp4.dequantize(mxfp4.pack_weight(kernel), torch.float32).double().t()
    assert ((c.double() - v).abs() <= 1e-4 * v.abs().max() + 1e-6).all()
    only, none = norms.gated_residual_norm(**a, post_norm="none", pre_norm="layer", mx_out=mxfp4.empty(rows, n))
    assert none is None and torch.equal(only, h)


def test_refusals():
    x = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    g = torch.ones(64, dtype=torch.float16, device="cuda")
    ok = dict(pre_gamma=g, pre_beta=g)
    for kw in (dict(), dict(pre_gamma=g), dict(ok, post_norm="layer"), dict(ok, post_norm="batch"),
               dict(ok, gate=torch.zeros(3, 64, dtype=torch.float16, device="cuda")), dict(ok, gate=g[:32]),
               dict(ok, residual=x[:2]), dict(ok, bias=g.float()), dict(ok, h_out=x, y_out=x),
               dict(ok, mx_out=mxfp4.empty(3, 64)), dict(pre_gamma=g, pre_beta=g.cpu()),
               dict(ok, gate=torch.zeros(3, 64, dtype=torch.float16, device="cuda"),
                    batch_idx=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            norms.gated_residual_norm(x, **kw)
    with pytest.raises(ValueError):
        norms.gated_residual_norm(x.t(), **ok)


def test_streams_and_capture():
    a = make(9, 50, 768, torch.float16)
    wh, wy = want_of(a, "layer", "layer")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h, y = norms.gated_residual_norm(**a, post_norm="layer")
    torch.cuda.current_stream().wait_stream(side)
    close(y, wy, wh, torch.float16)
    h2, y2 = torch.zeros_like(a["x"]), torch.zeros_like(a["x"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms.gated_residual_norm(**a, post_norm="layer", h_out=h2, y_out=y2)
    graph.replay()
    assert torch.equal(h2, h) and torch.equal(y2, y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batches(dtype):
    a = make(10, 4, 64, dtype, seqs=3)
    for k in ("x", "residual", "batch_idx"):
        a[k] = a[k][:0]
    h, y = norms.gated_residual_norm(**a, post_norm="rms")
    assert h.shape == y.shape == (0, 64) and h.dtype == dtype
    mx = mxfp4.empty(0, 64)
    h, y = norms.gated_residual_norm(**a, post_norm="rms", mx_out=mx, valid_rows=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert h.shape == (0, 64) and y is None


@pytest.mark.parametrize("name", ["x", "bias", "residual", "gate", "post_gamma", "post_beta", "pre_gamma", "pre_beta"])
def test_gradients_are_not_lost_silently(name):
    a = make(11, 4, 64, torch.float16, seqs=2)
    want = norms.gated_residual_norm(**a, post_norm="layer")
    a[name] = a[name].clone().requires_grad_()
    got = norms.gated_residual_norm(**a, post_norm="layer")
    assert all(torch.equal(u, v) and u.requires_grad for u, v in zip(got, want))
    for u in got:
        with pytest.raises(NotImplementedError, match="no backward"):
            u.float().sum().backward(retain_graph=True)
    for kw in (dict(h_out=torch.empty_like(a["x"])), dict(y_out=torch.empty_like(a["x"])), dict(mx_out=mxfp4.empty(4, 64))):
        with pytest.raises(ValueError, match="no backward"):
            norms.gated_residual_norm(**a, post_norm="layer", **kw)
        with torch.no_grad():
            norms.gated_residual_norm(**a, post_norm="layer", **kw)
