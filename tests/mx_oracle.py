"""MXFP4 and the gated norm in float64, written from the definitions; shared by the CPU and GPU tests."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
KIND = {"none": 0, "layer": 1, "rms": 2}


def mx_parts(x):
    """(codes [rows, k], scale bytes [rows, k / 32]) of x (fp16 or fp32 numpy)."""
    rows, k = x.shape
    b = x.astype(np.float64).reshape(rows, k // 32, 32)
    finite = np.isfinite(b).all(-1)
    top = np.abs(np.where(finite[..., None], b, 0.0)).max(-1) if k else np.zeros((rows, 0))
    with np.errstate(divide="ignore"):
        e = np.where(top > 0, np.frexp(top)[1] - 1, -1000) - 2
    e = np.clip(e, -127, 125)
    a = np.abs(b) / np.exp2(e)[..., None]
    codes = np.zeros(a.shape, np.uint8)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        codes += (a > mid) if i % 2 == 0 else (a >= mid)
    codes |= (np.signbit(b).astype(np.uint8) << 3)
    codes[~finite] = 0
    return codes.reshape(rows, k), np.where(finite, e + 127, 255).astype(np.uint8)


def mx_values(x):
    """The values that the MXFP4 form of x stands for, float64."""
    codes, scales = mx_parts(x)
    rows, k = x.shape
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(rows, k // 32, 32) * s[..., None]).reshape(rows, k)


def mx_bytes(rows, k):
    return -(-rows // 128) * -(-k // 256) * 17408


def mx_unpack(data, rows, k):
    """(codes, scale bytes) read out of the buffer of an MXFP4 tensor, by the layout's formula."""
    tiles = data.reshape(-(-rows // 128), -(-k // 256), 17408)
    r, c = np.arange(rows)[:, None], np.arange(k)[None, :]
    p = (r & ~0x1e) | ((r & 0x18) >> 2) | ((r & 0x06) << 2)     # where a row stands: bits 1-2 and 3-4 change places
    b = (c % 256) // 32
    pos = (p % 128) * 128 + ((b ^ (p % 8)) * 16) + (c % 32) // 2
    byte = tiles[r // 128, c // 256, pos]
    codes = np.where(c % 2 == 0, byte & 15, byte >> 4).astype(np.uint8)
    cb = np.arange(k // 32)[None, :]
    bb = cb % 8
    spos = 16384 + (bb // 4) * 512 + (p % 32) * 16 + ((p % 128) // 32) * 4 + bb % 4
    return codes, tiles[r // 128, cb // 8, spos]


def gelu(x):
    return x / (1 + torch.exp(-2 * 0.7978845608028654 * (x + 0.044715 * x ** 3)))


def norm(x, kind, gamma, beta, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double() + beta.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double()


def gated_norm(x, bias, residual, scale, gate, batch_idx, post, post_gamma, post_beta, pre, pre_gamma, pre_beta, eps):
    """(h, y) in float64."""
    p = x.double() if bias is None else x.double() + bias.double()
    p = norm(p, post, post_gamma, post_beta, eps)
    if gate is not None:
        g = gate.double()
        if g.dim() == 2 and g.shape[0] > 1:
            idx = batch_idx.long()
            inside = (idx >= 0) & (idx < g.shape[0])
            g = g[torch.where(inside, idx, 0)]
            p = torch.where(inside[:, None], p * g, torch.zeros_like(p))
        else:
            p = p * g.reshape(-1)
    h = p if residual is None else p + scale * residual.double()
    return h, norm(h, pre, pre_gamma, pre_beta, eps)


def code_values(v, scales):
    """v [rows, k] rounded to codes on given scale bytes [rows, k / 32], as values."""
    s = np.exp2(scales.astype(np.float64) - 127).repeat(32, axis=1)
    q = np.abs(v) / s
    c = np.zeros(q.shape, np.int8)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        c += (q > mid) if i % 2 == 0 else (q >= mid)
    return np.copysign(GRID[c], v) * s


def check_codes(mx, want, bound):
    """The first rows of mx (an MxTensor on a GPU) hold the quantised form of values within `bound` of `want` (float64,
    on the GPU): scales and codes agree with those of `want` but where a border lies in between."""
    rows, k = want.shape
    codes, scales = (part[:rows] for part in mx_unpack(mx.data.cpu().numpy(), mx.rows, k))
    got = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0) * np.exp2(scales.astype(np.float64) - 127).repeat(32, axis=1)
    want, bound = want.cpu().numpy(), bound.cpu().numpy()
    lo, hi = want - bound, want + bound
    size = np.abs(want)
    top_lo = np.maximum(size - bound, 1e-30).reshape(rows, -1, 32).max(-1)
    top_hi = (size + bound).reshape(rows, -1, 32).max(-1)
    e = scales.astype(np.float64) - 127 + 2
    assert (np.floor(np.log2(top_lo)) <= e).all() and (e <= np.floor(np.log2(top_hi))).all()
    assert (got >= code_values(lo, scales)).all() and (got <= code_values(hi, scales)).all()
