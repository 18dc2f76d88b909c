"""Edges of the language-model operators on the GPU: what a call may ask for that their other tests leave out."""
import math

import numpy as np
import pytest

import bfuse_project_b200 as bf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return bf.Runtime(0)


def normal(torch, seed, *shape, mean=0.0, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(shape, device="cuda", dtype=torch.bfloat16).normal_(mean, std, generator=g)


def offsets(torch, lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def attention(rt, q, k, v, cu_q, cu_kv, out, causal=True):
    shape = (cu_q.numel() - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2])
    d = rt.describe("attention", bf.OP_ATTENTION_BF16, shape, [q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_kv.data_ptr(), out.data_ptr()],
                    fparam=(q.shape[2] ** -0.5,), flags=bf.flag_share(1) | (bf.FLAG_CAUSAL if causal else 0))
    return d, rt.register_kernel(d)


@pytest.mark.parametrize("dim", [64, 128])
def test_first_tile_of_a_pair_without_keys_is_zero(rt, dim):
    # two query tiles of 128 positions a CTA.  Where 232, 128 or 200 of a pair's 256 positions come before the first query that
    # sees a key, its first tile is all behind the mask and its second one is not.  Every launch, every head: exact zeros.
    import torch
    kv_lens = [2200, 2100, 2300]
    q_lens = [kv + n for kv, n in zip(kv_lens, (2 * 256 + 232, 4 * 256 + 128, 6 * 256 + 200))]
    heads = 24
    q, k, v = normal(torch, 1, sum(q_lens), heads, dim), normal(torch, 2, sum(kv_lens), heads, dim), normal(torch, 3, sum(kv_lens), heads, dim)
    cu_q, cu_kv, out = offsets(torch, q_lens), offsets(torch, kv_lens), torch.empty_like(q)
    d, h = attention(rt, q, k, v, cu_q, cu_kv, out)
    assert d.shape[9] == 2
    for _ in range(20):
        out.fill_(7.0)
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        assert rt.read_status() == 0
        q0 = 0
        for a, b in zip(q_lens, kv_lens):
            assert (out[q0:q0 + a - b] == 0).all()
            q0 += a
    q0 = k0 = 0
    for a, b in zip(q_lens, kv_lens):       # the first rows with keys, against the definition (tolerance: see the attention tests)
        n = 200
        for head in (0, heads - 1):
            s = q[q0 + a - b:q0 + a - b + n, head].double() @ k[k0:k0 + n, head].double().T * dim ** -0.5
            p = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf).softmax(-1)
            vv = v[k0:k0 + n, head].double()
            want, mag = p @ vv, p @ vv.abs()
            off = (out[q0 + a - b:q0 + a - b + n, head].double() - want).abs() / (2.0 ** -8 * (mag + want.abs()) + 2.0 ** -14 * mag)
            assert float(off.max()) <= 1.0, float(off.max())
        q0, k0 = q0 + a, k0 + b
    rt.unregister_kernel(h)


@pytest.mark.parametrize("dim,lens", [(64, [100] * 90), (128, [300, 40, 0, 700, 1] * 8)])
def test_work_queue_runs_tile_after_tile_of_attention(rt, dim, lens):
    # more tiles than resident CTAs: a CTA's next tile loads its queries where the last one's rows were staged
    import torch
    stream = torch.cuda.current_stream().cuda_stream
    cu, heads = offsets(torch, lens), 12
    sets = []
    for seed in (1, 5):
        q, k, v = (normal(torch, seed + i, sum(lens), heads, dim) for i in range(3))
        sets.append((q, k, v, torch.zeros_like(q)))
    handles = []
    for (q, k, v, out), causal in zip(sets, (True, False)):
        shape = (len(lens), sum(lens), sum(lens), heads, heads, dim)
        d = rt.describe("attention", bf.OP_ATTENTION_BF16, shape, [t.data_ptr() for t in (q, k, v, cu, cu, out)], fparam=(dim ** -0.5,),
                        flags=bf.FLAG_CAUSAL if causal else 0)
        handles.append(rt.register_kernel(d))
    f = rt.register_fusion(handles[0], handles[1], bf.WORK_QUEUE, 1, 1)
    rt.launch_sequential(f, stream)
    assert rt.read_status() == 0
    want = [s[3].clone() for s in sets]
    assert all(bool(w.any()) for w in want)
    for _ in range(10):
        for s in sets:
            s[3].fill_(7.0)
        rt.launch_fused(f, stream)
        assert rt.read_status() == 0
        assert all(torch.equal(s[3], w) for s, w in zip(sets, want))
    rt.unregister_fusion(f)


@pytest.mark.parametrize("rows,cols", [(1, 8), (300, 264), (700, 1000), (130, 4096), (3, 8192)])
@pytest.mark.parametrize("norms", [0, 1, 2, 3])
def test_norms_in_place_give_the_same_bits(rt, rows, cols, norms):
    # r over x, over the block, y over the other one: rows whose neighbours share their sectors (cols of 8 modulo 16) among them
    import torch
    stream = torch.cuda.current_stream().cuda_stream
    x, b, gate = normal(torch, 1, rows, cols), normal(torch, 2, rows, cols), normal(torch, 3, rows, cols)
    w = normal(torch, 4, max(1, bin(norms).count("1")), cols, mean=1.0)

    def launched(r, y, px, pb):
        d = rt.describe("residual_norm", bf.OP_RESIDUAL_NORM_BF16, (rows, cols, norms, 1),
                        [t.data_ptr() for t in (px, pb, gate)] + [w.data_ptr() if norms else None, r.data_ptr(), y.data_ptr() if y is not None else None],
                        fparam=(1e-5, 0.5))
        h = rt.register_kernel(d)
        rt.launch_kernel(h, stream)
        assert rt.read_status() == 0
        rt.unregister_kernel(h)
        return r, y

    second = norms & bf.NORM_BEFORE
    r, y = launched(torch.zeros_like(x), torch.zeros_like(x) if second else None, x, b)
    assert bool(r.any()) and (not second or bool(y.any()))
    for swap in (False, True):
        px, pb = x.clone(), b.clone()
        gr, gy = launched(pb if swap else px, (px if swap else pb) if second else None, px, pb)
        assert torch.equal(gr, r) and (not second or torch.equal(gy, y))


def product(rt, torch, m, n, k, tiling=(0, 0, 0, 0), act=bf.ACT_NONE, other=False, seed=0):
    a, w, o = normal(torch, seed, m, k), normal(torch, seed + 1, n, k, std=k ** -0.5), normal(torch, seed + 2, m, n) if other else None
    out = torch.full((m, n), 7.0, device="cuda", dtype=torch.bfloat16)
    d = rt.describe("gemm_act", bf.OP_GEMM_ACT_BF16, (1, m, n, k) + tuple(tiling), [a.data_ptr(), w.data_ptr(), None, o.data_ptr() if other else None, out.data_ptr()],
                    flags=bf.flag_share(1) | bf.flag_act(act))
    h = rt.register_kernel(d)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    # the product in fp32 (K 2^-23 of the terms at worst), one rounding
    z, mag = a.double() @ w.double().T, a.double().abs() @ w.double().abs().T
    want = z + (o.double() if other else 0)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + k * 2.0 ** -23 * mag).all()
    return d, h, (a, w, o, out)


@pytest.mark.parametrize("split", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("m", [1, 4, 32])
def test_few_rows_in_any_number_of_k_slices(rt, split, m):
    import torch
    if split in (6, 7):      # what so many slices of 128 rows exchange is more than a window, for any number of rows: refused
        for rows in (m, 33):
            with pytest.raises(bf.BfuseError, match="shared memory"):
                product(rt, torch, rows, 264, 4096, (0, split), other=True)
        return
    d, h, _ = product(rt, torch, m, 264, 4096, (0, split), other=True)
    assert d.shape[5] == split and d.shape[6] == (128 if split in (3, 5) else 16 if m <= 16 else 32)
    rt.unregister_kernel(h)


def test_pairs_of_ctas_asked_for_with_few_rows(rt):
    import torch
    for m in (1, 32):
        d, h, _ = product(rt, torch, m, 264, 1096, (0, 0, 0, 2), other=True)
        assert d.shape[6] == 256 and d.shape[7] == 2
        rt.unregister_kernel(h)


def test_timeline_of_a_form_that_records_none_is_refused(rt):
    import torch
    for tiling in ((0, 0, 16), (0, 0, 0, 2)):
        _, h, buffers = product(rt, torch, 16, 264, 1096, tiling)
        with pytest.raises(bf.BfuseError, match="timeline"):
            rt.gemm_timeline(h)
        rt.unregister_kernel(h)
    _, h, buffers = product(rt, torch, 16, 264, 1096, (128, 1, 128))
    marks = rt.gemm_timeline(h)
    assert marks["end"] >= marks["acc_ready"] >= marks["setup_done"] >= 0 and marks["end"] > 0
    rt.unregister_kernel(h)


def activation(torch, act, z):
    if act == bf.ACT_GELU:
        return z * torch.special.log_ndtr(z).exp()
    if act == bf.ACT_GELU_TANH:
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z)


@pytest.mark.parametrize("form", [(128, 1, 128, 1), (128, 1, 16, 1), (256, 1, 256, 2)])
@pytest.mark.parametrize("act,lowest", [(bf.ACT_GELU, -14.0), (bf.ACT_GELU_TANH, -10.5), (bf.ACT_SILU, -95.0)])
def test_tails_of_the_activations(rt, act, lowest, form):
    # The product is 0, so the bias alone is activated: as it is, in fp32.  Against 64 bits, relative to the value: the activation
    # within 2^-16 (a few 2^-24 of the exponent, which is 126 / log2(e) at most: 2^-17; the rest 2^-20), half a step of bf16 (2^-8), and
    # nothing finer than the smallest normal value (2^-126).
    import torch
    n, k = 8192, 64
    z = torch.cat([torch.linspace(lowest, 0, n // 2, device="cuda"), torch.linspace(0, -lowest, n // 2, device="cuda")]).contiguous()
    for m in (1, 16):
        a, w = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16), normal(torch, 1, n, k)
        out = torch.full((m, n), 7.0, device="cuda", dtype=torch.bfloat16)
        d = rt.describe("gemm_act", bf.OP_GEMM_ACT_BF16, (1, m, n, k) + form, [a.data_ptr(), w.data_ptr(), z.data_ptr(), None, out.data_ptr()],
                        flags=bf.flag_share(1) | bf.flag_act(act))
        h = rt.register_kernel(d)
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        assert rt.read_status() == 0
        want = activation(torch, act, z.double())
        off = (out.double() - want).abs() / ((2.0 ** -8 + 2.0 ** -16) * want.abs() + 2.0 ** -126)
        assert float(off.max()) <= 1.0, (float(off.max()), float(z[off.max(0).values.argmax()]))
        rt.unregister_kernel(h)


@pytest.mark.parametrize("act", [bf.ACT_RELU, bf.ACT_GELU, bf.ACT_GELU_TANH, bf.ACT_SILU])
def test_activations_of_huge_values_and_nan(rt, act):
    import torch
    z = torch.tensor([math.inf, 3e38, 1e30, 100.0, -100.0, -1e30, -3e38, math.nan], device="cuda")
    for form in ((128, 1, 128, 1), (128, 1, 16, 1)):
        a, w = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16), normal(torch, 1, 8, 64)
        out = torch.full((2, 8), 7.0, device="cuda", dtype=torch.bfloat16)
        h = rt.register_kernel(rt.describe("gemm_act", bf.OP_GEMM_ACT_BF16, (1, 2, 8, 64) + form, [a.data_ptr(), w.data_ptr(), z.data_ptr(), None, out.data_ptr()],
                                           flags=bf.flag_share(1) | bf.flag_act(act)))
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        assert rt.read_status() == 0
        for row in out.float():
            assert torch.equal(row[:4], z[:4].to(torch.bfloat16).float()) and (row[4:7] == 0).all() and bool(row[7].isnan())
        rt.unregister_kernel(h)


@pytest.mark.parametrize("form", [(64, 1, 128, 1), (128, 4, 128, 1), (256, 1, 256, 1), (128, 1, 16, 1), (128, 8, 32, 1), (256, 1, 256, 2), (128, 1, 256, 2)])
@pytest.mark.parametrize("mul", [False, True])
def test_products_in_place_give_the_same_bits(rt, form, mul):
    # the residual (or the factor) is the output, in every form of the product
    import torch
    m, n, k = 300, 520, 1096
    a, w, other = normal(torch, 1, 2, m, k), normal(torch, 2, 2, n, k, std=k ** -0.5), normal(torch, 3, 2, m, n)
    outs = []
    for src, dst in ((other, torch.zeros_like(other)), (other.clone(), None)):
        dst = src if dst is None else dst
        h = rt.register_kernel(rt.describe("gemm_act", bf.OP_GEMM_ACT_BF16, (2, m, n, k) + form, [a.data_ptr(), w.data_ptr(), None, src.data_ptr(), dst.data_ptr()],
                                           flags=bf.flag_share(1) | bf.flag_act(bf.ACT_SILU) | (bf.FLAG_MUL if mul else 0)))
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        assert rt.read_status() == 0
        rt.unregister_kernel(h)
        outs.append(dst)
    assert bool(outs[0].any()) and torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("seqs", [3, 12, 40])
def test_caches_with_room_to_grow(rt, seqs):
    # a sequence without queries owns the room behind each cache; what lies there does not matter, and the offsets move as caches grow
    import torch
    heads, kvh, dim, room = 8, 2, 64, 400
    rng = np.random.default_rng(seqs)
    lens = [int(x) for x in rng.integers(1, room, seqs)]
    q, k, v = normal(torch, 1, seqs, heads, dim), normal(torch, 2, seqs * room, kvh, dim), normal(torch, 3, seqs * room, kvh, dim)
    cu_q = torch.tensor([0] + [i // 2 + 1 for i in range(2 * seqs)], dtype=torch.int32, device="cuda")
    cu_kv, out = torch.zeros(2 * seqs + 1, dtype=torch.int32, device="cuda"), torch.empty_like(q)
    _, h = attention(rt, q, k, v, cu_q, cu_kv, out)
    keep_k, keep_v = k.clone(), v.clone()
    for step in range(3):
        ends = [x for i, n in enumerate(lens) for x in (i * room + n, (i + 1) * room)]
        cu_kv.copy_(torch.tensor([0] + ends, dtype=torch.int32))
        for i, n in enumerate(lens):
            k[i * room:(i + 1) * room], v[i * room:(i + 1) * room] = keep_k[i * room:(i + 1) * room], keep_v[i * room:(i + 1) * room]
            k[i * room + n:(i + 1) * room], v[i * room + n:(i + 1) * room] = math.nan, math.inf
        out.fill_(7.0)
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        assert rt.read_status() == 0
        for i, n in enumerate(lens):
            kk, vv = (t[i * room:i * room + n].double().repeat_interleave(heads // kvh, 1) for t in (keep_k, keep_v))
            p = (torch.einsum("hd,khd->hk", q[i].double(), kk) * dim ** -0.5).softmax(-1)
            want, mag = torch.einsum("hk,khd->hd", p, vv), torch.einsum("hk,khd->hd", p, vv.abs())
            off = (out[i].double() - want).abs() / (2.0 ** -8 * (mag + want.abs()) + 2.0 ** -14 * mag)
            assert float(off.max()) <= 1.0, float(off.max())
        lens = [min(room, n + 1) for n in lens]
    rt.unregister_kernel(h)


def test_offsets_that_pass_32_bits(rt):
    # 2.3e9 elements of keys, of values, of queries and of the output: bytes and elements past 32 and 31 bits
    import torch
    kvh, dim, tokens = 8, 128, 2_250_000
    k, v = (torch.empty(tokens, kvh, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    k[-700:], v[-700:] = normal(torch, 1, 700, kvh, dim), normal(torch, 2, 700, kvh, dim)
    q = normal(torch, 3, 2, 4 * kvh, dim)
    cu_q, cu_kv = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), torch.tensor([tokens - 700, tokens - 300, tokens], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def check(got, qq, kk, vv):
        kk, vv = (t.double().repeat_interleave(qq.shape[0] // t.shape[1], 1) for t in (kk, vv))
        p = (torch.einsum("hd,khd->hk", qq.double(), kk) * dim ** -0.5).softmax(-1)
        want, mag = torch.einsum("hk,khd->hd", p, vv), torch.einsum("hk,khd->hd", p, vv.abs())
        assert ((got.double() - want).abs() <= 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -14 * mag).all()

    _, h = attention(rt, q, k, v, cu_q, cu_kv, out)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    check(out[0], q[0], k[-700:-300], v[-700:-300])
    check(out[1], q[1], k[-300:], v[-300:])
    rt.unregister_kernel(h)
    # the same buffers as queries and output: one key for all but the last three positions
    q, out, keys, values = k, v, normal(torch, 4, 4, kvh, dim), normal(torch, 5, 4, kvh, dim)
    q[-3:] = normal(torch, 6, 3, kvh, dim)
    q[:-3].zero_()
    cu_q, cu_kv = torch.tensor([0, tokens - 3, tokens], dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 4], dtype=torch.int32, device="cuda")
    out.fill_(7.0)
    _, h = attention(rt, q, keys, values, cu_q, cu_kv, out, causal=False)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    for i in (-3, -2, -1):
        check(out[i], q[i], keys[1:], values[1:])
    assert torch.equal(out[:-3:100_000], values[:1].expand_as(out[:-3:100_000])) and torch.equal(out[-5], values[0])
    rt.unregister_kernel(h)


@pytest.mark.parametrize("pattern", [bf.ZIGZAG, bf.PROPORTIONAL, bf.SM_STRIPED, bf.THREAD_SPLIT, bf.RANGE_SPLIT, bf.WORK_QUEUE])
def test_fused_norms_against_the_definition(rt, pattern):
    # (two roundings of 2^-8 at most: r's, and y's; fp32 adds less than 2^-16 of the terms)
    import torch
    stream, eps, scale = torch.cuda.current_stream().cuda_stream, 1e-5, 0.5
    sets, handles = [], []
    for seed, (rows, cols) in enumerate(((700, 4096), (333, 768))):
        x, b, w = normal(torch, 10 * seed, rows, cols), normal(torch, 10 * seed + 1, rows, cols), normal(torch, 10 * seed + 2, 2, cols, mean=1.0)
        r, y = torch.zeros_like(x), torch.zeros_like(x)
        d = rt.describe("residual_norm", bf.OP_RESIDUAL_NORM_BF16, (rows, cols, bf.NORM_AFTER | bf.NORM_BEFORE, 0),
                        [x.data_ptr(), b.data_ptr(), None, w.data_ptr(), r.data_ptr(), y.data_ptr()], fparam=(eps, scale))
        handles.append(rt.register_kernel(d))
        sets.append((x, b, w, r, y))
    f = rt.register_fusion(handles[0], handles[1], pattern, 1, 1)
    for launch in (rt.launch_sequential, rt.launch_fused):
        for *_, r, y in sets:
            r.zero_(), y.zero_()
        launch(f, stream)
        assert rt.read_status() == 0
        for x, b, w, r, y in sets:
            x, b, w = x.double(), b.double(), w.double()
            n = scale * b / (b.pow(2).mean(1, keepdim=True) + eps).sqrt() * w[0]
            want, mag = x + n, x.abs() + n.abs()
            inv = 1 / (want.pow(2).mean(1, keepdim=True) + eps).sqrt()
            assert ((r.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * mag).all()
            y_want = want * inv * w[1]
            assert ((y.double() - y_want).abs() <= 2.0 ** -8 * y_want.abs() + 2.0 ** -16 * (mag * inv * w[1].abs() + y_want.abs())).all()
    rt.unregister_fusion(f)


@pytest.mark.parametrize("rows,cols", [(3000, 264), (700, 1000), (40, 8)])
def test_in_place_stream_of_layers(rt, rows, cols):
    # a residual stream updated in place and read by the next launch, which starts under this one's tail: rows that share a sector
    import torch
    stream, layers = torch.cuda.current_stream().cuda_stream, 24
    x, b, w = normal(torch, 1, rows, cols), normal(torch, 2, layers, rows, cols), normal(torch, 3, 2, cols, mean=1.0)
    ys = torch.zeros(layers, rows, cols, device="cuda", dtype=torch.bfloat16)

    def layer(i, r):
        return rt.register_kernel(rt.describe("residual_norm", bf.OP_RESIDUAL_NORM_BF16, (rows, cols, bf.NORM_AFTER | bf.NORM_BEFORE, 0),
                                              [x.data_ptr(), b[i].data_ptr(), None, w.data_ptr(), r.data_ptr(), ys[i].data_ptr()], fparam=(1e-5, 0.5)))

    start, other = x.clone(), torch.zeros_like(x)
    for i in range(layers):      # out of place, one launch at a time
        h = layer(i, other)
        rt.launch_kernel(h, stream)
        torch.cuda.synchronize()
        x.copy_(other)
        torch.cuda.synchronize()
        rt.unregister_kernel(h)
    want = x.clone(), ys.clone()
    handles = [layer(i, x) for i in range(layers)]
    for _ in range(10):
        x.copy_(start)
        ys.zero_()
        for h in handles:
            rt.launch_kernel(h, stream)
        assert rt.read_status() == 0
        assert torch.equal(x, want[0]) and torch.equal(ys, want[1])
    for h in handles:
        rt.unregister_kernel(h)
