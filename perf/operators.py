"""The 4-bit projections of an encoder layer and the norms between them, as cases that can be timed.

Three operators that a user calls on packed token rows (effective_transformer_b200.mxfp4 and .norms):

  quantize   rows to microscaled 4-bit floating point (MXFP4: e2m1 codes, one power-of-two scale per 32
             values of a row) and back: what an activation becomes in front of a 4-bit projection
  linear     act(x W + bias) (+ residual) with x quantised in the call and W quantised once, when it is loaded
  norm       p = post(x + bias), h = residual_scale * residual + gate * p, y = pre(h): the norm behind a block,
             its gate and residual scale, and the norm in front of the next block; with "quantized" the
             normalised rows go straight into a 4-bit projection

`own` is set from outside: False computes the operators from elementary torch operations, True makes the
framework's calls.
"""
import math

import torch

own = False

BLOCK = 32  # values that share a scale


def listed():
    def quantize(name, dtype, rows, valid, k):
        return dict(name=name, op="quantize", dtype=dtype, rows=rows, valid=valid, k=k)

    def linear(name, dtype, rows, valid, k, n, act, residual=False):
        return dict(name=name, op="linear", dtype=dtype, rows=rows, valid=valid, k=k, n=n, act=act, residual=residual)

    def norm(name, dtype, rows, valid, k, post, pre, gate, seqs, scale, n=0):
        return dict(name=name, op="norm", dtype=dtype, rows=rows, valid=valid, k=k, post=post, pre=pre, gate=gate,
                    seqs=seqs, scale=scale, n=n)

    return [
        # the first-token row of one request on its way into the pooler's projection
        quantize("quantize_fp16_one_token", "fp16", 1, 1, 1024),
        # a ragged fp32 batch of an odd width: half a scale group is left over at the end of a row
        quantize("quantize_fp32_ragged", "fp32", 4099, 3001, 800),
        # the feed-forward activations of a full batch: 62 % of the positions hold tokens
        quantize("quantize_fp16_full_batch", "fp16", 64000, 39778, 4096),
        # one token through the first feed-forward projection: latency and the weights' bytes
        linear("linear_one_token_gelu", "fp16", 1, 1, 1024, 4096, "gelu"),
        # a small online batch through a fused query / key / value projection
        linear("linear_small_batch_qkv", "fp16", 256, 133, 768, 2304, "bias"),
        # a medium batch through the second feed-forward projection with its residual
        linear("linear_medium_residual", "fp16", 3200, 2000, 4096, 1024, "bias", True),
        # fp32 rows in, fp32 rows out, odd count: users who keep activations in 32 bits
        linear("linear_fp32_odd_rows", "fp32", 20011, 20011, 1024, 1024, "none"),
        # the first feed-forward projection of a full batch, the largest product
        linear("linear_full_batch_gelu", "fp16", 64000, 39778, 1024, 4096, "gelu"),
        # one token behind an attention block: post-norm encoder, residual added and normalised
        norm("norm_one_token", "fp16", 1, 1, 768, "none", "layer", "none", 1, 1.0),
        # fp32 rows of a wide model, RMS norms on both sides, one gate per channel, scaled residual
        norm("norm_fp32_rms_channel_gate", "fp32", 4099, 4099, 2080, "rms", "rms", "channel", 1, 0.70710678),
        # the largest: layer norms on both sides of the residual stream, one gate row per sequence
        norm("norm_fp16_full_batch", "fp16", 64000, 39778, 1024, "layer", "layer", "sequence", 1000, 1.25),
        # norm in front of a 4-bit projection: the normalised rows are quantised where they are made
        norm("norm_quantized_projection", "fp16", 16000, 11003, 1024, "none", "layer", "none", 1, 1.0, n=1024),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: 1 to 64000 rows with 40 to 100 % of them valid, widths of 64 to 4096 in steps of a scale block."""
    op = rng.choice(["quantize", "linear", "linear", "norm", "norm"])
    dtype = rng.choice(["fp16", "fp16", "fp32"])
    width = lambda: BLOCK * _log_int(rng, 2, 128)  # noqa: E731
    rows = _log_int(rng, 1, 64000)
    valid = max(1, int(rows * rng.uniform(0.4, 1.0)))
    k = width()
    if op == "quantize":
        while rows * k > 64000 * 2048:
            rows, valid = rows // 2, max(1, valid // 2)
        return dict(op=op, dtype=dtype, rows=rows, valid=valid, k=k)
    if op == "linear":
        n = width()
        while rows * k * n > 64000 * 1024 * 2048 or rows * max(k, n) > 64000 * 2048:
            rows, valid = rows // 2, max(1, valid // 2)
        return dict(op=op, dtype=dtype, rows=rows, valid=valid, k=k, n=n,
                    act=rng.choice(["none", "bias", "gelu", "tanh"]), residual=rng.random() < 0.3)
    while rows * k > 64000 * 512:
        rows, valid = rows // 2, max(1, valid // 2)
    # (a handful of rows would make one value next to a border of the 4-bit grid visible in the product)
    n = width() if rng.random() < 0.3 and valid >= 3000 else 0
    while n and rows * n > 64000 * 1024:
        n = BLOCK * max(1, n // BLOCK // 2)
    pre = rng.choice(["layer", "rms"]) if n else rng.choice(["layer", "rms", "none"])
    return dict(op=op, dtype=dtype, rows=rows, valid=valid, k=k, post=rng.choice(["none", "layer", "rms"]), pre=pre,
                gate=rng.choice(["none", "channel", "sequence"]), seqs=max(1, min(valid, _log_int(rng, 1, 2000))),
                scale=rng.choice([1.0, 0.5, 1.25]), n=n)


def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.float32


# ---- plain forms ------------------------------------------------------------------------------------

def _mx_values(x):
    """The values that the rows of x stand for in MXFP4, in fp32: per block of 32 the scale is 2 to the exponent
    of the largest magnitude, less the two that the largest code carries; values are rounded to the nearest of
    0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale, ties to the even code, and saturate."""
    b = x.float().reshape(x.shape[0], -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1)
    e = torch.where(top > 0, e - 3, torch.full_like(e, -127)).clamp(-127, 125)
    r = torch.ldexp(b, -e)
    a = r.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return torch.ldexp(torch.copysign(q, r), e).reshape(x.shape)


def _act(y, act):
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return torch.tanh(y) if act == "tanh" else y


def _normed(x, kind, gamma, beta, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.float() + beta.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.float()


def _plain(s):
    c, t = s["case"], s["case"]["valid"]
    dtype = _dtype(c)
    if c["op"] == "quantize":
        return _mx_values(s["x"][:t]).to(dtype)
    if c["op"] == "linear":
        y = _mx_values(s["x"][:t]) @ s["weight"].t()
        if c["act"] != "none":
            y = y + s["bias"].float()
        y = _act(y, c["act"])
        if c["residual"]:
            y = y + s["residual"][:t].float()
        return y.to(dtype)
    p = _normed(s["x"][:t].float() + s["bias"].float(), c["post"], s["post_gamma"], s["post_beta"], s["eps"])
    if c["gate"] == "channel":
        p = p * s["gate"].float()
    elif c["gate"] == "sequence":
        p = p * s["gate"].float()[s["batch_idx"][:t].long()]
    h = s["residual"][:t].float() * c["scale"] + p
    y = _normed(h, c["pre"], s["pre_gamma"], s["pre_beta"], s["eps"])
    if c["n"]:
        return h.to(dtype), (_mx_values(y) @ s["weight"].t()).to(dtype)
    return h.to(dtype), y.to(dtype)


# ---- inputs -----------------------------------------------------------------------------------------

def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, k, n = _dtype(case), case["rows"], case["k"], case.get("n", 0)

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).add_(mean).to(dtype)

    # activations as a normalised stream has them: unit variance, a few channels that stand out
    x = torch.randn(rows, k, generator=gen, device="cuda")
    x[:, torch.randperm(k, generator=gen, device="cuda")[:max(1, k // 128)]] *= 6.0
    s = dict(case=case, x=x.to(dtype), eps=1e-6,
             valid=torch.full((1,), case["valid"], dtype=torch.int32, device="cuda"))
    if n:
        s["kernel"] = normal(k, n, scale=0.02)
    if case["op"] == "linear":
        s["bias"] = normal(n, scale=0.02)
        s["residual"] = normal(rows, n) if case["residual"] else None
    if case["op"] == "norm":
        s["bias"], s["residual"] = normal(k, scale=0.02), normal(rows, k)
        s["post_gamma"], s["post_beta"] = normal(k, scale=0.1, mean=1.0), normal(k, scale=0.1)
        s["pre_gamma"], s["pre_beta"] = normal(k, scale=0.1, mean=1.0), normal(k, scale=0.1)
        if case["gate"] == "channel":
            s["gate"] = normal(k, scale=0.3)
        elif case["gate"] == "sequence":
            s["gate"] = normal(case["seqs"], k, scale=0.3)
            # rows of one sequence stand together, in batch order
            s["batch_idx"] = torch.sort(torch.randint(0, case["seqs"], (rows,), generator=gen, device="cuda",
                                                      dtype=torch.int32))[0]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    rows, k, n, dtype = case["rows"], case["k"], case.get("n", 0), _dtype(case)
    if not own:
        if n:
            s["weight"] = _mx_values(s.pop("kernel").t().contiguous())
        return s
    from effective_transformer_b200 import mxfp4

    # weights are quantised when they are loaded; results go into buffers that the program keeps
    if n:
        s["weight"] = mxfp4.pack_weight(s.pop("kernel"))
    if case["op"] != "norm" or n:
        s["mx"] = mxfp4.empty(rows, k)
    if case["op"] == "quantize":
        s["out"] = torch.zeros(rows, k, dtype=dtype, device="cuda")
    elif n:
        s["out"] = torch.zeros(rows, n, dtype=dtype, device="cuda")
    if case["op"] == "norm":
        s["h"] = torch.zeros(rows, k, dtype=dtype, device="cuda")
        s["y"] = None if n else torch.zeros(rows, k, dtype=dtype, device="cuda")
    return s


def run(s):
    if not own:
        return _plain(s)
    from effective_transformer_b200 import mxfp4, norms

    c, t = s["case"], s["case"]["valid"]
    if c["op"] == "quantize":
        q = mxfp4.quantize(s["x"], valid_rows=s["valid"], out=s["mx"])
        return mxfp4.dequantize(q, s["out"].dtype, valid_rows=s["valid"], out=s["out"])[:t]
    if c["op"] == "linear":
        return mxfp4.linear(s["x"], s["weight"], bias=None if c["act"] == "none" else s["bias"],
                            activation=c["act"] if c["act"] in ("gelu", "tanh") else None, residual=s["residual"],
                            valid_rows=s["valid"], workspace=s["mx"], out=s["out"])[:t]
    norms.gated_residual_norm(
        s["x"], bias=s["bias"], residual=s["residual"], residual_scale=c["scale"], gate=s.get("gate"),
        batch_idx=s.get("batch_idx"), post_norm=c["post"], post_gamma=s["post_gamma"], post_beta=s["post_beta"],
        pre_norm=c["pre"], pre_gamma=s["pre_gamma"], pre_beta=s["pre_beta"], eps=s["eps"], valid_rows=s["valid"],
        h_out=s["h"], y_out=s["y"], mx_out=s["mx"] if c["n"] else None)
    if c["n"]:
        return s["h"][:t], mxfp4.gemm(s["mx"], s["weight"], valid_rows=s["valid"], out=s["out"])[:t]
    return s["h"][:t], s["y"][:t]


def work(case):
    """Bytes: every input read once and every output written once; a 4-bit block of 32 values is 17 bytes."""
    e, t, k, n = (2 if case["dtype"] == "fp16" else 4), case["valid"], case["k"], case.get("n", 0)
    mx = lambda r, c: r * c * 17 / 32  # noqa: E731
    if case["op"] == "quantize":  # to 4 bits and back: the 4-bit rows are written and read
        return {"bytes": 2 * t * k * e + 2 * mx(t, k), "flops": 4 * t * k}
    if case["op"] == "linear":
        return {"bytes": t * k * e + mx(n, k) + t * n * e * (2 if case["residual"] else 1), "flops": 2 * t * n * k}
    seqs = case["seqs"] if case["gate"] == "sequence" else 1
    moved = 3 * t * k * e + seqs * k * e + 5 * k * e
    if n:
        return {"bytes": moved + mx(n, k) + t * n * e, "flops": 2 * t * n * k + 20 * t * k}
    return {"bytes": moved + t * k * e, "flops": 20 * t * k}


# ---- the definition in 64 bits ----------------------------------------------------------------------

_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx_exact(x):
    """Counts the midpoints between neighbouring magnitudes that a value is past; a tie belongs to the even code."""
    b = x.double().reshape(x.shape[0], -1, BLOCK)
    top = b.abs().amax(-1)
    e = torch.full_like(top, -127.0)
    e[top > 0] = torch.floor(torch.log2(top[top > 0])) - 2
    e = torch.where(top >= torch.exp2(e + 3), e + 1, torch.where((top > 0) & (top < torch.exp2(e + 2)), e - 1, e))
    scale = torch.exp2(e.clamp(-127, 125)).unsqueeze(-1)
    a = b.abs() / scale
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i in range(7):
        mid = (_MAGNITUDES[i] + _MAGNITUDES[i + 1]) / 2
        code += (a > mid) if i % 2 == 0 else (a >= mid)
    table = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=x.device)
    return (table[code.long()] * scale * torch.sign(b)).reshape(x.shape)


def _norm_exact(x, kind, gamma, beta, eps):
    if kind == "none":
        return x
    centre = x.mean(1) if kind == "layer" else torch.zeros_like(x[:, 0])
    second = (x * x).mean(1) - centre * centre  # (64 bits: nothing is lost to the difference here)
    y = (x - centre[:, None]) / torch.sqrt(second + eps)[:, None] * gamma.double()
    return y + beta.double() if kind == "layer" else y


def exact(case, seed):
    s, t = _inputs(case, seed), case["valid"]
    x = s["x"][:t]
    if case["op"] == "quantize":
        return _mx_exact(x)
    w = _mx_exact(s["kernel"].t().contiguous()) if case.get("n") else None
    if case["op"] == "linear":
        y = torch.matmul(_mx_exact(x), w.t())
        if case["act"] != "none":
            y += s["bias"].double()
        if case["act"] == "gelu":  # x / (1 + exp(-2u)) is 0.5 x (1 + tanh u)
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        elif case["act"] == "tanh":
            y = y.tanh()
        return y + s["residual"][:t].double() if case["residual"] else y
    p = _norm_exact(x.double() + s["bias"].double(), case["post"], s["post_gamma"], s["post_beta"], s["eps"])
    if case["gate"] != "none":
        g = s["gate"].double()
        p = p * (g[s["batch_idx"][:t].long()] if case["gate"] == "sequence" else g)
    h = case["scale"] * s["residual"][:t].double() + p
    y = _norm_exact(h, case["pre"], s["pre_gamma"], s["pre_beta"], s["eps"])
    return (h, torch.matmul(_mx_exact(y), w.t())) if case["n"] else (h, y)
