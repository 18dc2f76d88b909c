"""The operators of a decoder layer together, as the segment driver runs them, through the host-buffer calls, and refused."""
import math

import numpy as np
import pytest

import bfuse_project_b200 as bf
from bfuse_project_b200 import segment as sg

pytestmark = pytest.mark.gpu


def layer_reference(torch, b, lens, heads, kv_heads):
    """float64, with the roundings to bf16 of the buffers between the operators"""
    f = {n: t.double() for n, t in b.buf.items()}
    r = lambda t: t.to(torch.bfloat16).double()
    tokens, hidden = f["x"].shape
    d = hidden // heads
    norm = lambda t, w: t / (t.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * w
    xn = r(norm(f["x"], f["wn1"]))
    q, k, v = (r(xn @ f["w" + n].T) for n in "qkv")
    ang = torch.arange(tokens, device=q.device, dtype=torch.float64)[:, None] * f["inv_freq"][None]

    def rope(t, h):
        t = t.view(tokens, h, d)
        a, c = t[..., :d // 2], t[..., d // 2:]
        cs, sn = ang.cos()[:, None], ang.sin()[:, None]
        return r(torch.cat([a * cs - c * sn, c * cs + a * sn], -1))

    q, k, v = rope(q, heads), rope(k, kv_heads), v.view(tokens, kv_heads, d)
    ctx, at = torch.zeros_like(q), 0
    for n in lens:
        s = torch.einsum("qhd,khd->hqk", q[at:at + n], k[at:at + n].repeat_interleave(heads // kv_heads, 1)) * d ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf)
        ctx[at:at + n] = torch.einsum("hqk,khd->qhd", s.softmax(-1), v[at:at + n].repeat_interleave(heads // kv_heads, 1))
        at += n
    attn = r(r(ctx).reshape(tokens, hidden) @ f["wo"].T)
    h = f["x"] + attn
    hn = r(norm(h, f["wn2"]))
    gate = hn @ f["wgate"].T
    act = r(gate * gate.sigmoid() * r(hn @ f["wup"].T))
    return r(act @ f["wdown"].T + r(h))


@pytest.mark.parametrize("lens", [(150,), (1, 77, 200, 3)])
def test_decoder_layer(lens):
    import torch
    rt = bf.Runtime(0)
    heads, kv_heads = 8, 2
    b, ops = sg.llama_layer(rt, torch, lens=lens, hidden=512, heads=heads, kv_heads=kv_heads, ffn=1536, seed=3)
    seg = sg.Segment(rt, ops)
    assert seg.launches_fused < seg.launches_sequential == 12
    stream = torch.cuda.current_stream().cuda_stream
    want = layer_reference(torch, b, lens, heads, kv_heads)
    outs = {}
    for name, program in (("alone", seg.run_sequential), ("unfused", seg.run_unfused), ("fused", seg.run_fused)):
        for n in sorted({w for o in ops for w in o.writes}):
            b.buf[n].zero_()
        program(stream)
        assert rt.read_status() == 0
        outs[name] = b.buf["out"].clone()
    assert torch.equal(outs["fused"], outs["unfused"])
    for got in outs.values():
        # the buffers between the operators are rounded as in the reference, but a value next to a border may fall to its other
        # side (one step, 2^-7): over 1536 terms of the last product such steps add up to well below two of the output's
        err = (got.double() - want).abs()
        assert float(err.pow(2).mean().sqrt()) <= 2.0 ** -8 * float(want.pow(2).mean().sqrt()) and float(err.max()) <= 2.0 ** -5 * float(want.abs().max())
    # captured once, replayed on other inputs
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        seg.run_fused(torch.cuda.current_stream().cuda_stream)
    b.buf["x"].copy_(b.buf["x"].flip(0))
    want = layer_reference(torch, b, lens, heads, kv_heads)
    graph.replay()
    assert rt.read_status() == 0
    err = (b.buf["out"].double() - want).abs()
    assert float(err.pow(2).mean().sqrt()) <= 2.0 ** -8 * float(want.pow(2).mean().sqrt())
    rt.close()


def bits(torch, t):
    return t.view(torch.int16).cpu().numpy()


def test_host_buffer_calls():
    """run_kernel: inputs in, launch, outputs out; arguments that an operator may do without are not copied."""
    import torch
    rt = bf.Runtime(0)
    rng = np.random.default_rng(0)
    dev = lambda *s, dt=None: torch.zeros(s, device="cuda", dtype=dt or torch.bfloat16)
    host = lambda *s: bits(torch, torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(torch.bfloat16))
    val = lambda a: torch.from_numpy(a.astype(np.int16)).view(torch.bfloat16).double()
    # norm without r, without gate
    x, blk, w, y = dev(6, 64), dev(6, 64), dev(1, 64), dev(6, 64)
    h = rt.register_kernel(rt.describe("n", bf.OP_RESIDUAL_NORM_BF16, (6, 64, bf.NORM_BEFORE), [x.data_ptr(), blk.data_ptr(), None, w.data_ptr(), None, y.data_ptr()],
                                       fparam=(1e-5, 1.0)))
    hx, hb, hw, hy = host(6, 64), host(6, 64), host(1, 64), np.zeros((6, 64), np.int16)
    rt.run_kernel(h, [hx, hb, None, hw, None, hy])
    r = val(hx) + val(hb)
    want = r / (r.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * val(hw)
    assert ((val(hy) - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4).all()
    # product with a residual
    a, wt, o, res = dev(5, 64), dev(16, 64), dev(5, 16), dev(5, 16)
    h = rt.register_kernel(rt.describe("g", bf.OP_GEMM_ACT_BF16, (1, 5, 16, 64), [a.data_ptr(), wt.data_ptr(), None, res.data_ptr(), o.data_ptr()]))
    ha, hwt, hr, ho = host(5, 64), host(16, 64), host(5, 16), np.zeros((5, 16), np.int16)
    rt.run_kernel(h, [ha, hwt, None, hr, ho])
    want = val(ha) @ val(hwt).T + val(hr)
    assert ((val(ho) - want).abs() <= 2.0 ** -8 * want.abs() + 1e-3).all()
    # attention, and offsets that leave the tensors
    q, k, v, out, cu = dev(9, 4, 64), dev(9, 2, 64), dev(9, 2, 64), dev(9, 4, 64), dev(3, dt=torch.int32)
    h = rt.register_kernel(rt.describe("a", bf.OP_ATTENTION_BF16, (2, 9, 9, 4, 2, 64), [t.data_ptr() for t in (q, k, v, cu)] + [None, out.data_ptr()], fparam=(0.125,)))
    hq, hk, hv, ho = host(9, 4, 64), host(9, 2, 64), host(9, 2, 64), np.zeros((9, 4, 64), np.int16)
    rt.run_kernel(h, [hq, hk, hv, np.array([0, 2, 9], np.int32), None, ho])
    for lo, hi in ((0, 2), (2, 9)):
        s = torch.einsum("qhd,khd->hqk", val(hq)[lo:hi], val(hk)[lo:hi].repeat_interleave(2, 1)) * 0.125
        want = torch.einsum("hqk,khd->qhd", s.softmax(-1), val(hv)[lo:hi].repeat_interleave(2, 1))
        assert ((val(ho)[lo:hi] - want).abs() <= 2.0 ** -7 * val(hv).abs().max()).all()
    with pytest.raises(bf.BfuseError) as e:
        rt.run_kernel(h, [hq, hk, hv, np.array([0, 2, 10], np.int32), None, ho])
    assert e.value.code == 1
    rt.run_kernel(h, [hq, hk, hv, np.array([0, 2, 9], np.int32), None, ho])      # the context goes on
    rt.close()


def test_registration_refusals():
    import torch
    rt = bf.Runtime(0)
    p = torch.zeros(1 << 16, device="cuda", dtype=torch.bfloat16).data_ptr()

    def refused(code, op, shape, args, **kw):
        fields = {k: kw.pop(k) for k in ("grid", "block", "smem") if k in kw}
        with pytest.raises(bf.BfuseError) as e:
            rt.register_kernel(rt.describe("k", op, shape, args, **kw, **fields))
        assert e.value.code == code

    gemm, norm, attn = bf.OP_GEMM_ACT_BF16, bf.OP_RESIDUAL_NORM_BF16, bf.OP_ATTENTION_BF16
    refused(1, gemm, (1, 8, 8, 8), [p, p, 0, 0, 0])                                        # no output
    refused(1, gemm, (1, 8, 8, 8), [p, p, 0, 0, p + 2])                                    # not 16-byte aligned
    refused(1, gemm, (1, 8, 8, 8), [p, p, 0, 0, p], flags=bf.FLAG_MUL)                     # nothing to multiply by
    refused(1, gemm, (1, 8, 8, 8), [p, p, 0, 0, p], flags=bf.flag_act(9))
    refused(1, gemm, (1, 8, 8, 8), [p, p, 0, 0, p], flags=bf.FLAG_CAUSAL)
    refused(2, gemm, (1, 8, 12, 8), [p, p, 0, 0, p])                                       # rows that are no 16-byte multiples
    refused(2, gemm, (1, 8, 8, 12), [p, p, 0, 0, p])
    refused(2, gemm, (1, 8, 8, 8, 128, 1, 16), [p, p, 0, 0, p], grid=(2, 1, 1))
    refused(2, gemm, (1, 8, 8, 8, 256, 1, 256, 2), [p, p, 0, 0, p], grid=(3, 1, 1))        # half a pair
    refused(2, gemm, (1, 8, 8, 8, 256, 1, 256, 2), [p, p, 0, 0, p], grid=(4, 1, 1))        # more pairs than tiles
    refused(2, gemm, (1, 8, 8, 8, 256, 1, 256, 2), [p, p, 0, 0, p], smem=100 * 1024)
    refused(1, norm, (4, 64, 3), [p, p, 0, 0, p, p], fparam=(1e-5, 1.0))                   # norms without weights
    refused(1, norm, (4, 64, 2), [p, p, 0, p, p, 0], fparam=(1e-5, 1.0))                   # a norm without its output
    refused(1, norm, (4, 64, 1), [p, p, 0, p, p, p], fparam=(1e-5, 1.0))                   # an output without its norm
    refused(1, norm, (4, 64, 0), [p, p, 0, 0, 0, 0], fparam=(1e-5, 1.0))                   # no output
    refused(2, norm, (4, 4096, 3), [p, p, 0, p, p, p], fparam=(1e-5, 1.0), block=(96, 2, 1))
    refused(2, norm, (4, 4096, 3), [p, p, 0, p, p, p], fparam=(1e-5, 1.0), block=(64, 1, 1))
    refused(2, norm, (4, 4096, 3), [p, p, 0, p, p, p], fparam=(1e-5, 1.0), grid=(3, 1, 1))
    refused(2, norm, (4, 4096, 3), [p, p, 0, p, p, p], fparam=(1e-5, 1.0), smem=0)
    refused(1, attn, (1, 8, 8, 4, 4, 64), [p, p, p, 0, p, p], fparam=(0.1,))               # no offsets
    refused(2, attn, (1, 8, 8, 4, 4, 64), [p, p, p, p, p, p], fparam=(0.1,), grid=(4, 2, 1))
    refused(2, attn, (1, 8, 8, 4, 4, 64), [p, p, p, p, p, p], fparam=(0.1,), block=(128, 1, 1))
    refused(2, attn, (1, 8, 8, 4, 4, 64), [p, p, p, p, p, p], fparam=(0.1,), smem=32 * 1024)
    refused(2, attn, (1, 8, 8, 4, 4, 64), [p, p, p, p, p, p], fparam=(0.0,))
    assert rt.read_status() == 0
    rt.close()


def test_overlapping_buffers_are_refused():
    import torch
    rt = bf.Runtime(0)
    p = torch.zeros(1 << 16, device="cuda", dtype=torch.bfloat16).data_ptr()
    at = lambda i: p + 8192 * i
    gemm, norm, attn = bf.OP_GEMM_ACT_BF16, bf.OP_RESIDUAL_NORM_BF16, bf.OP_ATTENTION_BF16

    def describe(op, shape, args, **kw):
        return rt.describe("k", op, shape, args, **kw)

    def refused(*a, **kw):
        with pytest.raises(bf.BfuseError) as e:
            rt.register_kernel(describe(*a, **kw))
        assert e.value.code == 1 and "overlap" in str(e.value)

    def taken(*a, **kw):
        rt.unregister_kernel(rt.register_kernel(describe(*a, **kw)))

    size = (1, 8, 8, 8)                                                                  # 128 bytes each
    for i in range(3):                                                                   # out over A, W, bias; a part of the residual
        args = [at(0), at(1), at(2), at(3), at(4)]
        args[4] = args[i] + 16
        refused(gemm, size, args)
    refused(gemm, size, [at(0), at(1), at(2), at(3), at(3) + 64])
    taken(gemm, size, [at(0), at(1), at(2), at(3), at(3)])
    taken(gemm, size, [at(0), at(1), at(2), at(3), at(0) + 128])                          # behind A
    size, kw = (4, 64, 3, 2), dict(fparam=(1e-5, 1.0))                                   # 512 bytes
    refused(norm, size, [at(0), at(1), at(2), at(3), at(2), at(5)], **kw)                # the gate
    refused(norm, size, [at(0), at(1), at(2), at(3), at(4), at(3) + 128], **kw)          # the weights
    refused(norm, size, [at(0), at(1), at(2), at(3), at(4), at(4)], **kw)                # both outputs
    refused(norm, size, [at(0), at(1), at(2), at(3), at(0) + 128, at(5)], **kw)          # other rows of the stream
    taken(norm, size, [at(0), at(1), at(2), at(3), at(0), at(1)], **kw)
    size, kw = (1, 8, 8, 1, 1, 64), dict(fparam=(0.1,))                                  # 1 KB
    for i in range(5):
        args = [at(0), at(1), at(2), at(3), at(4), at(5)]
        args[5] = args[i]
        refused(attn, size, args, **kw)
    taken(attn, size, [at(0), at(1), at(2), at(3), at(4), at(0) + 1024], **kw)
    assert rt.read_status() == 0
    rt.close()
