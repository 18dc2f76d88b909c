"""Packed attention on the GPU against its definition in 64 bits.

The tolerance counts roundings: p is rounded to bf16 before the second product (2^-8 of p at most, so 2^-8 sum p |v| in
all), the output once more (2^-8 |out|); scores, exponentials and sums in fp32 add less than 2^-14 of sum p |v| for scores
below 64."""
import math

import numpy as np
import pytest

import bfuse_project_b200 as bf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    return bf.Runtime(0)


def cumulative(torch, lens, device="cuda"):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=device)


def reference(torch, q, k, v, q_lens, kv_lens, scale, causal):
    """(out, sum p |v|) in float64"""
    total, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(total, heads, dim, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    q0 = k0 = 0
    for a, b in zip(q_lens, kv_lens):
        if a and b:
            kk = k[k0:k0 + b].double().repeat_interleave(group, 1)
            vv = v[k0:k0 + b].double().repeat_interleave(group, 1)
            s = torch.einsum("qhd,khd->hqk", q[q0:q0 + a].double(), kk) * scale
            if causal:
                hidden = torch.arange(b, device=q.device)[None, :] > torch.arange(b - a, b, device=q.device)[:, None]
                s = s.masked_fill(hidden, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            out[q0:q0 + a] = torch.einsum("hqk,khd->qhd", p, vv)
            mag[q0:q0 + a] = torch.einsum("hqk,khd->qhd", p, vv.abs())
        q0, k0 = q0 + a, k0 + b
    return out, mag


def tensors(torch, q_lens, kv_lens, heads, kv_heads, dim, seed=0, extra=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    mk = lambda n, h: torch.empty(n + extra, h, dim, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    return mk(sum(q_lens), heads), mk(sum(kv_lens), kv_heads), mk(sum(kv_lens), kv_heads)


def kernel(rt, q, k, v, cu_q, cu_kv, out, scale, causal=False, slices=0, share=1, q_stride=0, kv_stride=0, kv_heads=None):
    shape = (cu_q.numel() - 1, q.shape[0], k.shape[0], q.shape[1], kv_heads or k.shape[1], q.shape[2], q_stride, kv_stride, slices)
    d = rt.describe("attention", bf.OP_ATTENTION_BF16, shape,
                    [q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), None if cu_kv is None else cu_kv.data_ptr(), out.data_ptr()],
                    fparam=(scale,), flags=bf.flag_share(share) | (bf.FLAG_CAUSAL if causal else 0))
    return rt.register_kernel(d)


def check(torch, got, want, mag):
    tol = 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -14 * mag + 1e-30
    off = (got.double() - want).abs() / tol
    assert torch.isfinite(got.float()).all()
    assert float(off.max()) <= 1.0, float(off.max())


def run(rt, q_lens, kv_lens, heads, kv_heads, dim, causal, slices=0, seed=0, scale=None):
    import torch
    q, k, v = tensors(torch, q_lens, kv_lens, heads, kv_heads, dim, seed)
    out = torch.full_like(q, 7.0)
    cu_q, cu_kv = cumulative(torch, q_lens), cumulative(torch, kv_lens)
    scale = scale or 1.0 / math.sqrt(dim)
    h = kernel(rt, q, k, v, cu_q, cu_kv, out, scale, causal, slices)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    check(torch, out, *reference(torch, q, k, v, q_lens, kv_lens, scale, causal))
    rt.unregister_kernel(h)


@pytest.mark.parametrize("dim", [128, 64, 8, 40, 80, 96])
@pytest.mark.parametrize("causal", [False, True])
def test_one_block(rt, dim, causal):
    run(rt, [128], [128], 1, 1, dim, causal)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (6, 1), (7, 1), (32, 8), (128, 1), (100, 2)])
def test_head_groups(rt, heads, kv_heads):
    run(rt, [50, 1], [70, 33], heads, kv_heads, 64, True)


@pytest.mark.parametrize("n", [1, 2, 31, 127, 129, 255, 300, 1000])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(rt, n, causal):
    run(rt, [n], [n], 4, 2, 128, causal)


@pytest.mark.parametrize("causal", [False, True])
def test_ragged_batch_with_empty_sequences(rt, causal):
    run(rt, [0, 5, 200, 0, 1, 64, 0, 333, 0], [10, 0, 200, 0, 500, 129, 3, 400, 0], 6, 2, 64, causal)


def test_rows_without_keys_are_zero(rt):
    run(rt, [40, 300], [10, 130], 4, 4, 64, True)     # the first 30 and 170 queries see nothing


@pytest.mark.parametrize("slices", [1, 2, 4, 8])
@pytest.mark.parametrize("dim", [64, 128])
def test_key_slices(rt, slices, dim):
    run(rt, [1, 1, 3, 1], [5, 1500, 700, 1], 8, 2, dim, True, slices)
    run(rt, [1, 2, 0], [4000, 129, 7], 32, 4, dim, True, slices)      # 8 and 16 rows
    run(rt, [70], [1030], 8, 2, dim, False, slices)


def test_many_sequences(rt):
    rng = np.random.default_rng(3)
    run(rt, [1] * 700, [int(x) for x in rng.integers(0, 40, 700)], 4, 1, 64, True)


def test_single_tokens_with_more_tiles_than_fit_at_once(rt):
    # loads late and in any order: the products of a block may wait for V longer than the next block's exponentials take
    run(rt, [1] * 48, [2048 + 37 * i for i in range(48)], 32, 8, 128, True)
    run(rt, [2] * 40, [1500] * 40, 32, 4, 64, True)      # 16 rows a tile


@pytest.mark.parametrize("heads,kv_heads,dim,causal,seqs", [(32, 8, 128, True, 60), (12, 12, 64, False, 40), (12, 12, 64, True, 30), (8, 8, 128, False, 50),
                                                            (16, 2, 40, True, 300)])
def test_blocks_take_tile_after_tile(rt, heads, kv_heads, dim, causal, seqs):
    # more tiles than run at once: of few rows and whole, without queries, without keys, of one block and of several
    rng = np.random.default_rng(seqs)
    q_lens = [int(n) for n in rng.choice([0, 1, 1, 2, 31, 128, 200], seqs)]
    kv_lens = [int(n) for n in rng.choice([0, 1, 90, 128, 129, 400, 700], seqs)]
    run(rt, q_lens, kv_lens, heads, kv_heads, dim, causal)
    run(rt, [1] * seqs * 8, [int(n) for n in rng.choice([0, 3, 128, 300], seqs * 8)], heads, kv_heads, dim, causal)


def test_two_launches_take_their_own_tiles(rt):
    import torch
    sets = []
    for seed in (1, 2):
        lens = [int(n) for n in np.random.default_rng(seed).choice([1, 60, 128, 150], 120)]
        q, k, v = tensors(torch, lens, lens, 12, 12, 64, seed)
        out, cu = torch.empty_like(q), cumulative(torch, lens)
        sets.append((lens, q, k, v, out, cu, kernel(rt, q, k, v, cu, None, out, 0.125, True), torch.cuda.Stream()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side = torch.cuda.current_stream()
        for *_, h, stream in sets:
            stream.wait_stream(side)
            rt.launch_kernel(h, stream.cuda_stream)
            rt.launch_kernel(h, stream.cuda_stream)
            side.wait_stream(stream)
    for direct in (True, False):
        for s in sets:
            s[4].zero_()
        torch.cuda.synchronize()
        if direct:
            for *_, h, stream in sets:
                rt.launch_kernel(h, stream.cuda_stream)
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert rt.read_status() == 0
        for lens, q, k, v, out, *_ in sets:
            check(torch, out, *reference(torch, q, k, v, lens, lens, 0.125, True))


def test_pairs_of_tiles_take_pair_after_pair(rt):
    run(rt, [2100, 4300], [2100, 4300], 16, 16, 64, True)
    run(rt, [3000, 300], [4096, 300], 12, 12, 128, False)
    run(rt, [4500, 700], [200, 4200], 16, 16, 128, True)    # most queries without keys


def test_large_scores_and_growing_maximum(rt):
    import torch
    # keys whose scores rise along the sequence: the running maximum moves at every block
    n, dim = 700, 64
    q = torch.ones(n, 1, dim, device="cuda", dtype=torch.bfloat16)
    k = (torch.arange(n, device="cuda", dtype=torch.float32) * (32.0 / n))[:, None, None].expand(n, 1, dim).to(torch.bfloat16).contiguous()
    v = torch.randn(n, 1, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    for order in (k, k.flip(0).contiguous()):
        out = torch.zeros_like(q)
        cu = cumulative(torch, [n])
        h = kernel(rt, q, order, v, cu, None, out, 1.0 / 32, False)
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        assert rt.read_status() == 0
        check(torch, out, *reference(torch, q, order, v, [n], [n], 1.0 / 32, False))


def test_values_outside_the_sequences_do_not_matter(rt):
    import torch
    q_lens, kv_lens = [3, 60], [150, 90]
    q, k, v = tensors(torch, q_lens, kv_lens, 4, 2, 128, 5, extra=300)
    cu_q, cu_kv = cumulative(torch, q_lens), cumulative(torch, kv_lens)
    want = reference(torch, q[:63], k[:240], v[:240], q_lens, kv_lens, 0.1, True)
    for bad in (math.nan, math.inf):
        q[63:], k[240:], v[240:] = bad, bad, bad
        out = torch.full_like(q, 7.0)
        h = kernel(rt, q, k, v, cu_q, cu_kv, out, 0.1, True)
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        assert rt.read_status() == 0
        check(torch, out[:63], *want)
        assert (out[63:] == 7.0).all()        # rows behind the last sequence stay


def test_masked_keys_may_be_nan(rt):
    import torch
    q, k, v = tensors(torch, [100], [100], 2, 1, 64, 6)
    cu = cumulative(torch, [100])
    want, mag = reference(torch, q, k, v, [100], [100], 0.125, True)
    k[60] = math.nan
    out = torch.zeros_like(q)
    h = kernel(rt, q, k, v, cu, None, out, 0.125, True)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    check(torch, out[:60], want[:60], mag[:60])
    assert torch.isnan(out[60:].float()).all()


def test_strided_projection_output(rt):
    import torch
    # q, k and v as slices of one [tokens, (heads + 2 kv_heads) dim] projection
    lens, heads, kvh, dim = [90, 170], 8, 2, 64
    width = (heads + 2 * kvh) * dim
    qkv = torch.randn(260, width, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(torch.bfloat16)
    q = qkv[:, :heads * dim].reshape(260, heads, dim)
    k = qkv[:, heads * dim:(heads + kvh) * dim].reshape(260, kvh, dim)
    v = qkv[:, (heads + kvh) * dim:].reshape(260, kvh, dim)
    out = torch.zeros(260, heads, dim, device="cuda", dtype=torch.bfloat16)
    cu = cumulative(torch, lens)
    base, e = qkv.data_ptr(), 2
    d = rt.describe("attention", bf.OP_ATTENTION_BF16, (2, 260, 260, heads, kvh, dim, width, width),
                    [base, base + heads * dim * e, base + (heads + kvh) * dim * e, cu.data_ptr(), None, out.data_ptr()], fparam=(0.125,),
                    flags=bf.FLAG_CAUSAL)
    h = rt.register_kernel(d)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    check(torch, out, *reference(torch, q, k, v, lens, lens, 0.125, True))


def test_offsets_are_read_at_every_launch_and_by_a_captured_graph(rt):
    import torch
    q, k, v = tensors(torch, [200], [200], 4, 4, 64, 8)
    out = torch.zeros_like(q)
    cu = cumulative(torch, [120, 80])
    h = kernel(rt, q, k, v, cu, None, out, 0.125, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rt.launch_kernel(h, side.cuda_stream)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    for lens in ([120, 80], [1, 199], [200, 0], [64, 136]):
        cu.copy_(cumulative(torch, lens))
        out.zero_()
        graph.replay()
        assert rt.read_status() == 0
        check(torch, out, *reference(torch, q, k, v, lens, lens, 0.125, True))


def test_bad_offsets_are_reported_and_their_sequence_left_out(rt):
    import torch
    q, k, v = tensors(torch, [100], [100], 2, 2, 64, 9)
    good = torch.zeros_like(q)
    want = reference(torch, q, k, v, [100], [100], 0.125, False)
    for bad_q, bad_kv in (([0, 40, 300], [0, 40, 100]), ([0, 60, 40], [0, 50, 100]), ([0, 40, 100], [0, 40, 1000]), ([0, 40, 100], [-5, 40, 100])):
        cu_q = torch.tensor(bad_q, dtype=torch.int32, device="cuda")
        cu_kv = torch.tensor(bad_kv, dtype=torch.int32, device="cuda")
        out = torch.full_like(q, 3.0)
        h = kernel(rt, q, k, v, cu_q, cu_kv, out, 0.125, False)
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        assert rt.read_status() == bf.STATUS_BAD_OFFSETS
        assert torch.isfinite(out.float()).all()
    cu = cumulative(torch, [100])
    rt.launch_kernel(kernel(rt, q, k, v, cu, None, good, 0.125, False), torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    check(torch, good, *want)


def test_bad_offsets_behind_every_tile_are_reported(rt):
    import torch
    n = 512   # single tokens, a tile each: none is left over for the last sequence, whose offsets leave the tensors
    q, k, v = tensors(torch, [n], [n], 1, 1, 64, 10)
    out = torch.full_like(q, 3.0)
    cu = torch.tensor(list(range(n + 1)) + [9999], dtype=torch.int32, device="cuda")
    rt.launch_kernel(kernel(rt, q, k, v, cu, None, out, 0.125, False), torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == bf.STATUS_BAD_OFFSETS
    check(torch, out, *reference(torch, q, k, v, [1] * n, [1] * n, 0.125, False))


@pytest.mark.parametrize("pattern", [bf.ZIGZAG, bf.PROPORTIONAL, bf.SM_STRIPED, bf.THREAD_SPLIT, bf.RANGE_SPLIT, bf.WORK_QUEUE])
@pytest.mark.parametrize("slices", [1, 4])
def test_fused_with_a_norm_and_with_itself_gives_the_same_bits(rt, pattern, slices):
    import torch
    q, k, v = tensors(torch, [300, 40], [300, 400], 8, 2, 64, 10)
    cu_q, cu_kv = cumulative(torch, [300, 40]), cumulative(torch, [300, 400])
    out, out2 = torch.zeros_like(q), torch.zeros_like(q)
    a = kernel(rt, q, k, v, cu_q, cu_kv, out, 0.125, True, slices, share=2)
    b = kernel(rt, q, k, v, cu_q, cu_kv, out2, 0.125, False, slices, share=2)
    x = torch.randn(600, 512, device="cuda").to(torch.bfloat16)
    w, y = torch.ones(512, device="cuda", dtype=torch.bfloat16), torch.zeros(600, 512, device="cuda", dtype=torch.bfloat16)
    n = rt.register_kernel(rt.describe("rmsnorm", bf.OP_RMSNORM_BF16, (600, 512), [x.data_ptr(), w.data_ptr(), y.data_ptr()], fparam=(1e-5,)))
    stream = torch.cuda.current_stream().cuda_stream
    for k1, k2 in ((a, n), (n, a), (a, b)):
        f = rt.register_fusion(k1, k2, pattern, 1, 1)
        rt.launch_sequential(f, stream)
        assert rt.read_status() == 0
        want = [t.clone() for t in (out, out2, y)]
        for t in (out, out2, y):
            t.zero_()
        rt.launch_fused(f, stream)
        assert rt.read_status() == 0
        for t, u, used in zip((out, out2, y), want, (True, k2 == b, k1 == n or k2 == n)):
            if used:
                assert torch.equal(t, u)
        rt.unregister_fusion(f)
