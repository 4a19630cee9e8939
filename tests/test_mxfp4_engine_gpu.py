"""A handle with 4-bit projections: its pass is the public operators in a row (bit by bit), every call of the handle
runs it, weights set later are quantised too, and a handle that is switched back gives what it gave before."""
import numpy as np
import pytest
import torch

import effective_transformer_b200 as et
from effective_transformer_b200 import mxfp4, norms
from effective_transformer_b200 import workloads as W
from util import DT, iptr, lib, ok, padding_offsets, status_word, stream

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.float32]


def make(dtype, batch, seq, layers=2, heads=4, ffn=640, seed=0):
    spec = W.tiny_spec(dtype="fp16" if dtype == torch.float16 else "fp32", layers=layers, heads=heads, ffn=ffn,
                       batch=batch, max_seq_len=seq, seed=seed)
    wl = W.make_workload(spec, random_gamma_beta=True)
    eng = et.EffectiveTransformer(layers, heads, 64, ffn, batch, seq, dtype=dtype)
    eng.set_weights(wl.weights)
    x = torch.from_numpy(np.asarray(wl.from_tensor)).to(dtype).cuda()
    mask = torch.from_numpy(np.asarray(wl.mask)).to(torch.int32).cuda()
    return eng, wl, x, mask


def attention(dtype, qkv, idx, batch, seq, heads):
    """The attention entry the handle's pass uses, on [rows, 3 H] -> [rows, H]."""
    rows, h3 = qkv.shape
    h = h3 // 3
    ctx = torch.zeros(rows, h, dtype=dtype, device="cuda")
    st = status_word()
    q, k, v = qkv.data_ptr(), qkv.data_ptr() + h * qkv.element_size(), qkv.data_ptr() + 2 * h * qkv.element_size()
    if dtype == torch.float16 and seq <= 128:
        plan = torch.zeros(lib().et_attention_plan_ints(batch, rows), dtype=torch.int32, device="cuda")
        ok(lib().et_attention_plan(iptr(idx["cu_seqlens"]), batch, rows, iptr(plan), stream()))
        ok(lib().et_attention_tiles(q, k, v, h3, 64, iptr(ctx), iptr(plan), batch, seq, rows, heads, 64, iptr(st), stream()))
    else:
        ok(lib().et_attention(DT[dtype], q, k, v, h3, 64, iptr(ctx), iptr(idx["cu_seqlens"]), batch, seq, rows, heads, 64,
                              0, iptr(st), stream()))
    return ctx


def by_operators(wl, x, mask, dtype, heads, layers):
    """The same pass from the public operators, packed rows [batch * seq, H]."""
    b, s, h = x.shape
    idx = padding_offsets(mask)
    t = idx["valid_word_num"]
    packed = torch.zeros(b * s, h, dtype=dtype, device="cuda")
    ok(lib().et_remove_padding(DT[dtype], iptr(x), iptr(idx["batch_idx"]), iptr(idx["word_idx"]), iptr(t), iptr(packed),
                               b, s, h, stream()))
    packed_mx = mxfp4.quantize(packed, valid_rows=t)
    for l in range(layers):
        w = [torch.from_numpy(np.asarray(a)).to(dtype).cuda() for a in wl.weights[16 * l:16 * l + 16]]
        qkv_w = mxfp4.pack_weight(torch.cat([w[0], w[2], w[4]], 1).contiguous())
        qkv = mxfp4.gemm(packed_mx, qkv_w, bias=torch.cat([w[1], w[3], w[5]]), valid_rows=t)
        ctx = attention(dtype, qkv, idx, b, s, heads)
        att = mxfp4.linear(ctx, mxfp4.pack_weight(w[6]), valid_rows=t)
        y, mx = torch.zeros_like(att), mxfp4.empty(b * s, h)
        norms.gated_residual_norm(att, bias=w[7], residual=packed, pre_gamma=w[9], pre_beta=w[8], valid_rows=t, y_out=y,
                                  mx_out=mx)
        f = mxfp4.gemm(mx, mxfp4.pack_weight(w[10]), bias=w[11], activation="gelu", valid_rows=t,
                       out=mxfp4.empty(b * s, w[10].shape[1]))
        o = mxfp4.gemm(f, mxfp4.pack_weight(w[12]), valid_rows=t, dtype=dtype)
        # the next layer reads the norm's own 4-bit rows, quantised from fp32, not these fp16 or fp32 rows again
        packed, packed_mx = torch.zeros_like(att), mxfp4.empty(b * s, h)
        norms.gated_residual_norm(o, bias=w[13], residual=y, pre_gamma=w[15], pre_beta=w[14], valid_rows=t, y_out=packed,
                                  mx_out=packed_mx)
    out = torch.zeros_like(x)
    ok(lib().et_restore_padding(DT[dtype], iptr(packed), iptr(idx["batch_idx"]), iptr(idx["word_idx"]), iptr(t), iptr(out),
                                b, s, h, stream()))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,seq", [(1, 7), (9, 40), (3, 200), (60, 96)])
def test_the_pass_is_the_operators_in_a_row(dtype, batch, seq):
    eng, wl, x, mask = make(dtype, batch, seq, seed=batch)
    plain = eng.forward(x, mask)
    eng.set_mxfp4_projections(True)
    got = eng.forward(x, mask)
    assert torch.equal(got, by_operators(wl, x, mask, dtype, 4, 2))
    assert eng.device_status() == 0 and mxfp4.device_status() == 0
    # 4 bits cost something, but it is the same model: LayerNorm rows of unit size, two layers of products whose
    # operands are off by an eighth at the most
    off = (got.double() - plain.double()).norm() / plain.double().norm()
    assert 0 < off < 0.5
    assert (got[mask == 0] == 0).all()
    eng.set_mxfp4_projections(False)
    assert torch.equal(eng.forward(x, mask), plain)
    eng.close()


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_call_of_the_handle(dtype):
    eng, wl, x, mask = make(dtype, 12, 32, seed=5)
    eng.set_mxfp4_projections(True)
    want = eng.forward(x, mask)
    # op by op: the layer op returns fp16 / fp32 rows, which the next one quantises again.  A value within half a step of
    # fp16 (2^-11) of one of the borders (seven a sign, an eighth to a whole scale apart) takes the next code: at most
    # 2^-11 * 14 = 0.7 % of them, off by half at the most, so sqrt(0.007) / 2 = 4 % of a projection's result in norm
    cur, valid, bidx, widx = eng.effective_transformer_input(x, mask)
    for l in range(2):
        cur = eng.effective_transformer(l, cur, cur, None, valid, bidx, widx)
    ops = eng.effective_transformer_output(cur, valid, bidx, widx)
    assert (ops.double() - want.double()).norm() <= 0.05 * want.double().norm()
    one = et.EffectiveTransformer(1, 4, 64, 640, 12, 32, dtype=dtype)
    one.set_weights(wl.weights[:16])
    one.set_mxfp4_projections(True)
    first = one.forward(x, mask)
    cur, valid, bidx, widx = one.effective_transformer_input(x, mask)
    cur = one.effective_transformer(0, cur, cur, None, valid, bidx, widx)
    assert torch.equal(one.effective_transformer_output(cur, valid, bidx, widx), first)
    # recorded, with host buffers, and under a general mask that allows what the key-only mask allows
    out = torch.zeros_like(x)
    eng.capture(x, mask, out)
    out.zero_()
    eng.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    host, t = eng.forward_host(x.cpu().numpy(), mask.cpu().numpy())
    assert t == int(mask.sum()) and np.array_equal(host, want.cpu().numpy())
    for _ in range(3):                                          # (the replayed form of the host-buffer call)
        host, _ = eng.forward_host(x.cpu().numpy(), mask.cpu().numpy())
    assert np.array_equal(host, want.cpu().numpy())
    full = torch.ones(12, 32, 32, dtype=dtype, device="cuda")
    ones = torch.ones_like(mask)
    assert (eng.forward_general_mask(x, ones, full).double() - eng.forward(x, ones).double()).abs().max() < 0.5
    eng.set_debug_simt(True)
    eng.set_mxfp4_projections(False)
    simt = eng.forward(x, mask)
    eng.set_mxfp4_projections(True)
    assert torch.equal(eng.forward(x, mask), simt)              # the CUDA-core path takes precedence
    eng.close()
    one.close()


def test_weights_set_later_follow():
    eng, wl, x, mask = make(torch.float16, 5, 24, seed=7)
    eng.set_mxfp4_projections(True)
    before = eng.forward(x, mask)
    other = [np.asarray(w) for w in wl.weights]
    changed = list(other)
    changed[16] = other[16] * 1.5
    eng.set_layer_weights(1, changed[16:32])
    after = eng.forward(x, mask)
    assert not torch.equal(after, before)
    fresh = et.EffectiveTransformer(2, 4, 64, 640, 5, 24, dtype=torch.float16)
    fresh.set_mxfp4_projections(True)                           # switched on before it has weights
    fresh.set_weights(changed)
    assert torch.equal(fresh.forward(x, mask), after)
    eng.set_layer_weights(1, other[16:32])
    assert torch.equal(eng.forward(x, mask), before)
    eng.close()
    fresh.close()


def test_toggling_drops_recorded_graphs():
    eng, _, x, mask = make(torch.float16, 3, 16, seed=9)
    out = torch.zeros_like(x)
    eng.capture(x, mask, out)
    eng.set_mxfp4_projections(True)
    with pytest.raises(et.EtError):
        eng.replay()
    eng.close()


@pytest.mark.parametrize("dtype", DTYPES)
def test_chunks_of_a_host_call_run_the_whole_batchs_kernels(dtype):
    """A chunk has few rows where the batch has many: neither a product nor a norm may take another order of sums."""
    eng, _, x, mask = make(dtype, 16, 24, layers=1, heads=16, ffn=256, seed=11)
    eng.set_mxfp4_projections(True)
    want = eng.forward(x, mask).cpu().numpy()
    for _ in range(3):
        host, t = eng.forward_host(x.cpu().numpy(), mask.cpu().numpy())
        assert t == int(mask.sum()) and np.array_equal(host, want)
    eng.close()
