"""The 4-bit operators without a GPU: the oracle against a search over all codes, sizes, and every refusal."""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_oracle as X
from effective_transformer_b200 import _capi, mxfp4, norms

LIB = _capi.load()
BAD = _capi.ET_INVALID_ARGUMENT
P = 1 << 20  # an aligned address that no refused call reads


def nearest(x, scale):
    """Code of |x| by search: the nearest grid value, of two equally near ones the even code."""
    d = np.abs(abs(x) / scale - X.GRID)
    best = np.flatnonzero(d == d.min())
    return int(best[0] if len(best) == 1 else best[best % 2 == 0][0])


def test_oracle_rounds_to_the_nearest_code():
    rng = np.random.RandomState(0)
    x = rng.randn(3, 64).astype(np.float32)
    x[1, :32] = np.arange(32) / 4            # 0.25 steps up to 7.75: every tie, and saturation
    x[2] = 0.0
    codes, scales = X.mx_parts(x)
    for r in range(3):
        for b in range(2):
            block = x[r, b * 32:b * 32 + 32]
            top = np.abs(block).max()
            e = np.floor(np.log2(top)) - 2 if top > 0 else -127
            assert scales[r, b] == e + 127
            assert [c & 7 for c in codes[r, b * 32:b * 32 + 32]] == [nearest(v, 2.0 ** e) for v in block]


def test_bytes():
    for rows, k in ((0, 32), (1, 32), (128, 256), (129, 256), (128, 288), (40000, 4096), (2 ** 31 - 1, 65536)):
        assert LIB.et_mxfp4_bytes(rows, k) == X.mx_bytes(rows, k)
    for rows, k in ((-1, 32), (1, 0), (1, 16), (1, -32), (1, 33)):
        assert LIB.et_mxfp4_bytes(rows, k) == 0


def refused(rc, text):
    assert rc == BAD
    assert text in LIB.et_last_error(None).decode()


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype"), (dict(k=0), "multiple of 32"), (dict(k=48), "multiple of 32"), (dict(m=-1), "negative"),
    (dict(stride=32), "row_stride"), (dict(stride=68), "row_stride"), (dict(x=None), "null"), (dict(mx=None), "null"),
    (dict(x=P + 8), "aligned"), (dict(mx=P + 4), "aligned")])
def test_quantize_refusals(change, text):
    a = dict(dtype=1, x=P, stride=64, m=5, k=64, mx=P)
    a.update(change)
    refused(LIB.et_mxfp4_quantize(a["dtype"], a["x"], a["stride"], None, a["m"], a["k"], a["mx"], None), text)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=-1), "dtype"), (dict(k=31), "multiple of 32"), (dict(m=-1), "negative"), (dict(out=None), "null"),
    (dict(mx=None), "null"), (dict(out=P + 2), "aligned")])
def test_dequantize_refusals(change, text):
    a = dict(dtype=0, mx=P, m=5, k=64, out=P)
    a.update(change)
    refused(LIB.et_mxfp4_dequantize(a["dtype"], a["mx"], None, a["m"], a["k"], a["out"], None), text)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "dtype"), (dict(k=40), "multiple of 32"), (dict(n=0), "n must"), (dict(n=40), "n must"),
    (dict(w=None), "null"), (dict(mx=None), "null"), (dict(mx=P + 1), "aligned")])
def test_pack_weight_refusals(change, text):
    a = dict(dtype=1, w=P, mx=P, k=64, n=64)
    a.update(change)
    refused(LIB.et_mxfp4_pack_weight(a["dtype"], a["w"], a["mx"], a["k"], a["n"], None), text)


GEMM_BAD = [
    (dict(dtype=5), "dtype"), (dict(k=0), "multiple of 32"), (dict(k=72), "multiple of 32"), (dict(n=48), "n a"),
    (dict(n=0), "n a"), (dict(m=-3), "negative"), (dict(epi=4), "epilogue"), (dict(epi=-1), "epilogue"),
    (dict(c=None), "exactly one"), (dict(c_mx=P), "exactly one"), (dict(c=None, c_mx=P, n=96), "multiple of 64"),
    (dict(c=None, c_mx=P, residual=P), "no residual"), (dict(a=None), "null"), (dict(w=None), "null"),
    (dict(epi=2, bias=None), "null"), (dict(a=P + 8), "aligned"), (dict(w=P + 16), "aligned"), (dict(c=None, c_mx=P + 64), "aligned"), (dict(c=P + 2), "aligned"),
    (dict(bias=P + 2, epi=1), "aligned"), (dict(residual=P + 2), "aligned")]


@pytest.mark.parametrize("change,text", GEMM_BAD)
def test_gemm_refusals(change, text):
    a = dict(dtype=1, a=P, w=P, bias=None, residual=None, c=P, c_mx=None, m=3, n=64, k=64, epi=0)
    a.update(change)
    refused(LIB.et_mxfp4_gemm(a["dtype"], a["a"], a["w"], a["bias"], a["residual"], a["c"], a["c_mx"], None, a["m"],
                              a["n"], a["k"], a["epi"], None, None), text)


@pytest.mark.parametrize("change,text", GEMM_BAD + [
    (dict(stride=32), "row_stride"), (dict(stride=67), "row_stride"), (dict(x_mx=None), "x_mx"), (dict(x_mx=P + 8), "x_mx")])
def test_linear_refusals(change, text):
    a = dict(dtype=1, a=P, stride=64, x_mx=P, w=P, bias=None, residual=None, c=P, c_mx=None, m=3, n=64, k=64, epi=0)
    a.update(change)
    refused(LIB.et_mxfp4_linear(a["dtype"], a["a"], a["stride"], a["x_mx"], a["w"], a["bias"], a["residual"], a["c"],
                                a["c_mx"], None, a["m"], a["n"], a["k"], a["epi"], None, None), text)


NORM_BAD = [
    (dict(max_m=-1), "negative"), (dict(n=0), "16 bytes"), (dict(n=12), "16 bytes"), (dict(n=8200), "limited"),
    (dict(post_norm=3), "post_norm"), (dict(pre_norm=-1), "pre_norm"), (dict(post_norm=1), "gamma"),
    (dict(post_norm=1, post_gamma=P), "gamma"), (dict(post_norm=2), "gamma"), (dict(pre_norm=1), "gamma"),
    (dict(h_out=None), "at least one"), (dict(y_mx=P, n=48), "multiple of 32"), (dict(gate=P, gate_rows=0), "gate"),
    (dict(gate=P, gate_rows=2), "gate"), (dict(x=None), "null"), (dict(x=P + 8), "aligned"),
    (dict(residual=P + 4), "aligned"), (dict(gate=P + 2, gate_rows=1), "aligned"), (dict(y_out=P + 2), "aligned"), (dict(y_mx=P + 16), "aligned")]


@pytest.mark.parametrize("change,text", NORM_BAD)
def test_norm_refusals(change, text):
    p = _capi.GatedNormParam()
    p.x, p.h_out, p.max_m, p.n, p.residual_scale = P, P, 4, 64, 1.0
    for k, v in change.items():
        setattr(p, k, v)
    refused(LIB.et_gated_residual_norm(1, C.byref(p), None), text)


def test_norm_parameters_as_bytes():
    values = list(range(1, 14)) + [-3, 5, 7, 1, 2, 0.5, 1e-5]
    p = _capi.GatedNormParam(*values)
    assert norms._PARAM.pack(*values) == bytes(p) and norms._PARAM.size == C.sizeof(p)
    refused(LIB.et_gated_residual_norm(1, norms._PARAM.pack(*([P] * 13 + [-1, 64, 0, 0, 0, 1.0, 0.0])), None), "negative")


def test_norm_refuses_types_and_null():
    p = _capi.GatedNormParam()
    refused(LIB.et_gated_residual_norm(9, C.byref(p), None), "dtype")
    refused(LIB.et_gated_residual_norm(1, None, None), "null")
    p.x, p.h_out, p.max_m, p.n = P, P, 4, 4100
    refused(LIB.et_gated_residual_norm(0, C.byref(p), None), "limited")


FAR = P + (1 << 30)


@pytest.mark.parametrize("change", [
    dict(c=None, c_mx=P), dict(c=P + 17408 - 16), dict(c=FAR + 16), dict(residual=FAR + (1 << 20) + 16, c=FAR + (1 << 20)),
    dict(bias=FAR + (1 << 20) + 128, c=FAR + (1 << 20), epi=1), dict(c=None, c_mx=FAR)])
def test_products_refuse_results_that_overlap_an_operand(change):
    a = dict(dtype=1, a=P, w=FAR, bias=None, residual=None, c=FAR + (1 << 20), c_mx=None, m=3, n=64, k=64, epi=0)
    a.update(change)
    tail = (a["w"], a["bias"], a["residual"], a["c"], a["c_mx"], None, a["m"], a["n"], a["k"], a["epi"], None, None)
    refused(LIB.et_mxfp4_gemm(a["dtype"], a["a"], *tail), "overlap")
    refused(LIB.et_mxfp4_linear(a["dtype"], P + (1 << 20), 64, a["a"], *tail), "overlap")


def test_rows_and_their_mxfp4_tensor_do_not_overlap():
    refused(LIB.et_mxfp4_quantize(1, P, 96, None, 3, 64, P + 256, None), "overlap")          # (the third row's end)
    refused(LIB.et_mxfp4_dequantize(0, P, None, 3, 64, P + 17408 - 16, None), "overlap")
    refused(LIB.et_mxfp4_pack_weight(1, P, P, 64, 64, None), "overlap")
    for x, w, bias, residual in ((P + 512, FAR, None, None), (FAR, P, None, None), (FAR, FAR, P, None),
                                 (FAR, FAR, None, P)):
        refused(LIB.et_mxfp4_linear(1, x, 64, P, w, bias, residual, FAR + (1 << 20), None, None, 3, 64, 64,
                                    0 if bias is None else 1, None, None), "overlap")


@pytest.mark.parametrize("change", [
    dict(y_out=P), dict(h_out=P + 128), dict(y_out=P + 128), dict(y_mx=P), dict(y_mx=FAR, y_out=FAR),
    dict(residual=FAR, h_out=FAR + 16), dict(bias=P + 16), dict(gate=P, gate_rows=1),
    dict(gate=FAR, gate_rows=3, batch_idx=P), dict(pre_gamma=P, pre_beta=FAR, pre_norm=1)])
def test_norm_refuses_outputs_that_overlap(change):
    p = _capi.GatedNormParam()
    p.x, p.h_out, p.max_m, p.n, p.residual_scale = P, P, 4, 64, 1.0
    for k, v in change.items():
        setattr(p, k, v)
    refused(LIB.et_gated_residual_norm(1, C.byref(p), None), "overlap")


def test_an_mxtensor_holds_what_it_says():
    data = torch.zeros(17408, dtype=torch.uint8)
    assert mxfp4.MxTensor(data, 128, 256).ptr == data.data_ptr()
    for args in ((data, 129, 256), (data, 1, 288), (data, 1, 40), (data, -1, 64), (data.int(), 1, 64), (None, 1, 64),
                 (torch.zeros(2 * 17408, dtype=torch.uint8)[::2], 1, 64)):
        with pytest.raises(ValueError):
            mxfp4.MxTensor(*args)


def test_empty_batches_are_fine():
    assert LIB.et_mxfp4_quantize(1, None, 64, None, 0, 64, None, None) == 0
    assert LIB.et_mxfp4_dequantize(1, None, None, 0, 64, None, None) == 0
    assert LIB.et_mxfp4_gemm(1, P, P, None, None, P, None, None, 0, 64, 64, 0, None, None) == 0
    p = _capi.GatedNormParam()
    p.h_out, p.n = P, 64
    assert LIB.et_gated_residual_norm(1, C.byref(p), None) == 0


def test_pointers_that_their_type_does_not_allow_are_refused():
    """A row count, a status word or gate rows between two words, a weight between two elements: faults on the GPU."""
    text = "4-byte aligned"
    refused(LIB.et_mxfp4_quantize(1, P, 64, P + 2, 3, 64, FAR, None), text)
    refused(LIB.et_mxfp4_dequantize(1, P, P + 1, 3, 64, FAR, None), text)
    for dtype, off in ((1, 1), (0, 2)):
        refused(LIB.et_mxfp4_pack_weight(dtype, FAR + off, P, 64, 64, None), text)
    for m_ptr, status in ((P + 2, None), (None, P + 1)):
        tail = (FAR, None, None, FAR + (1 << 20), None, m_ptr, 3, 64, 64, 0, status, None)
        refused(LIB.et_mxfp4_gemm(1, P, *tail), text)
        refused(LIB.et_mxfp4_linear(1, P + (1 << 20), 64, P, *tail), text)
    for change in (dict(m_ptr=FAR + 2), dict(gate=FAR, gate_rows=3, batch_idx=FAR + 4098)):
        p = _capi.GatedNormParam()
        p.x, p.h_out, p.max_m, p.n, p.residual_scale = P, P, 4, 64, 1.0
        for k, v in change.items():
            setattr(p, k, v)
        refused(LIB.et_gated_residual_norm(1, C.byref(p), None), text)


def test_threads_share_one_status_word(monkeypatch):
    """Two threads whose first product on a device comes at the same time: a second word would take the first one's place
    and free memory that a kernel may write to."""
    import contextlib
    import threading
    import time
    made, words, entered = [], [], []

    def zeros(*_, **__):
        made.append(torch.empty(1, dtype=torch.int32))
        time.sleep(0.2)                                         # (the other thread comes in meanwhile)
        return made[-1]

    @contextlib.contextmanager
    def on(device):
        entered.append(device)
        yield

    class Stream:
        def synchronize(self):
            pass

    monkeypatch.setattr(mxfp4, "_status", {})
    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: Stream())
    threads = [threading.Thread(target=lambda: words.append(mxfp4._status_word(3))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and words == [made[0].data_ptr()] * 4
    assert set(entered) == {3}                                  # (a capture on that device's stream is what is asked about)


def test_empty_tensors_have_no_address():
    """A torch tensor without rows has a null pointer; sizes are checked all the same."""
    for mx in (None, P):
        assert LIB.et_mxfp4_gemm(1, None, P, P, None, None, mx, None, 0, 64, 64, 1, None, None) == 0
        assert LIB.et_mxfp4_linear(0, None, 64, None, P, P, None, None, mx, None, 0, 64, 64, 2, None, None) == 0
    refused(LIB.et_mxfp4_gemm(1, None, P, None, None, None, None, None, 0, 64, 40, 0, None, None), "multiple of 32")
    refused(LIB.et_mxfp4_linear(1, None, 64, None, P, None, None, None, None, None, 0, 48, 64, 0, None, None), "n a")
    refused(LIB.et_mxfp4_linear(1, None, 32, None, P, None, None, None, None, None, 0, 64, 64, 0, None, None), "row_stride")
    p = _capi.GatedNormParam()
    p.n, p.gate, p.gate_rows, p.pre_norm, p.pre_gamma, p.pre_beta = 64, P, 3, 1, P, P
    assert LIB.et_gated_residual_norm(1, C.byref(p), None) == 0
    p.pre_beta = None
    refused(LIB.et_gated_residual_norm(1, C.byref(p), None), "beta")


def test_python_refuses_before_any_launch():
    x = torch.zeros(4, 64, dtype=torch.float16)
    w = mxfp4.MxTensor(torch.zeros(17408, dtype=torch.uint8), 64, 64)
    for call in (lambda: mxfp4.quantize(x), lambda: mxfp4.linear(x, w), lambda: mxfp4.pack_weight(x),
                 lambda: norms.gated_residual_norm(x), lambda: mxfp4.dequantize(w, torch.bfloat16),
                 lambda: mxfp4.dequantize(x, torch.float16), lambda: mxfp4.gemm(x, w), lambda: mxfp4.gemm(w, x),
                 lambda: mxfp4.empty(-1, 64, "cpu"), lambda: mxfp4.empty(1, 40, "cpu"),
                 lambda: mxfp4.gemm(w, mxfp4.MxTensor(w.data, 64, 96))):
        with pytest.raises(ValueError):
            call()
    assert mxfp4.empty(129, 288, "cpu").data.numel() == X.mx_bytes(129, 288)


def test_the_ring_of_the_products_is_drained():
    """What tests/test_kernel_sources_cpu.py asks of the other rings: the producer waits for its stages once inside the
    loop and once behind it, since commits arrive asynchronously; copies in flight land behind a wait that ran out."""
    from test_kernel_sources_cpu import kernels, read
    bodies = {k: b for k, _, b in kernels(read("gemm_mxfp4.cu"))}
    assert len(bodies) == 3
    for name, body in bodies.items():
        # (the kernel of few rows uses each stage once)
        assert body.count("mbar_wait(free_bar(") == (0 if name == "gemm_mxfp4_rows_kernel" else 2)
        assert body.count("mbar_drain(full_bar(") == 1 and body.count("mbar_drain(drain_bar") == 1


def route(rows, n, k, dtype=1):
    m, t, one = C.c_int(), C.c_int(), C.c_int()
    assert LIB.et_mxfp4_route(dtype, rows, n, k, C.byref(m), C.byref(t), C.byref(one)) == 0
    return m.value, t.value, one.value


def test_routes():
    assert route(1, 4096, 1024) == (128, 128, 1) and route(42, 2304, 768) == (128, 128, 1)
    assert route(43, 2304, 768) == (128, 128, 0) and route(1, 4096, 2048) == (128, 128, 0)
    assert route(128, 96, 256)[2] == 1 and route(129, 96, 32)[2] == 0
    assert route(1, 148 * 64, 768)[2] == 1 and route(1, 149 * 64, 768)[2] == 0
    pair = (256, 192, 0)
    assert route(40000, 4096, 1024) == route(40000, 1024, 4096) == route(128 * 445, 32, 768) == pair
    assert route(128 * 444, 32, 768) == route(128 * 445, 32, 736) == (128, 128, 0)
    assert route(128 * 18, 1024, 2048) == (128, 128, 0) and route(128 * 19, 1024, 2048) == pair
    assert route(128 * 19, 1024, 2016) == route(128 * 55, 1024, 4096, 0) == (128, 128, 0)
    assert route(128 * 56, 1024, 768, 0) == pair
    a = C.c_int()
    for rows, n, k in ((0, 32, 32), (1, 16, 32), (1, 32, 16), (1, 0, 32)):
        assert LIB.et_mxfp4_route(1, rows, n, k, C.byref(a), C.byref(a), C.byref(a)) == BAD
    assert LIB.et_mxfp4_route(2, 1, 32, 32, C.byref(a), C.byref(a), C.byref(a)) == BAD
    assert LIB.et_mxfp4_route(1, 1, 32, 32, None, C.byref(a), C.byref(a)) == BAD


def test_the_attention_of_a_4_bit_layer_starts_with_the_rows_that_came_last():
    """Products, rows and norms in 4 bits only run first-to-last, so the attention behind them always runs last-to-first;
    left to the flag that the attention itself flips, its order would depend on the calls before."""
    import os
    import re
    with open(os.path.join(os.path.dirname(_capi.__file__), "csrc", "encoder.cu")) as f:
        body = re.search(r"\nint run_layer_mx\(.*?\n\}\n", f.read(), re.S).group(0)
    steps = re.findall(r"ET_PROF_\w+|run_attention|prev_ascending = true", body)
    assert steps == ["ET_PROF_GEMM_QKV"] * 2 + ["prev_ascending = true", "run_attention", "ET_PROF_GEMM_ATTN_OUT",
                                                "ET_PROF_LAYERNORM", "ET_PROF_GEMM_FFN1", "ET_PROF_GEMM_FFN2",
                                                "ET_PROF_LAYERNORM", "prev_ascending = true"]


def test_products_take_tensor_memory_behind_their_wait():
    """A CTA that holds tensor memory while it waits for the kernel in front can leave none for a CTA of that kernel which
    has yet to allocate: both would wait for good.  (The attention's CTAs release their dependents before they allocate, and
    one of them fits an SM beside a CTA of the pair kernel, which takes all 512 columns.)  And dependents are released
    behind the allocation, for the same reason the other way round."""
    import re
    from test_kernel_sources_cpu import kernels, read
    text = read("gemm_mxfp4.cu")
    take = re.search(r"uint32_t take_tmem\(.*?\n\}", text, re.S).group(0)
    assert take.index("alloc();") < take.index("pdl_trigger();")
    for name, _, body in kernels(text):
        wait = body.index("else pdl_wait();")
        alloc = [m.start() for m in re.finditer(r"tmem_alloc(_pair)?\(", body)]
        assert len(alloc) == 1 and wait < body.index("take_tmem(") < alloc[0], name
        assert "pdl_trigger" not in body, name
