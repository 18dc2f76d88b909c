"""GEMM with bias, activation and residual / gate in its epilogue, against its definition in 64 bits.

The tolerance counts roundings: the product accumulates K terms in fp32 (K 2^-23 sum |a w|, the accumulator truncating at
worst), the activations change that by a slope of at most 1.13 and add 2^-20 of their value, the output is rounded once (2^-8)."""
import math

import pytest

import bfuse_project_b200 as bf

pytestmark = pytest.mark.gpu
ACTS = {bf.ACT_NONE: lambda t, z: z, bf.ACT_RELU: lambda t, z: t.relu(z), bf.ACT_GELU: lambda t, z: z * t.special.ndtr(z),
        bf.ACT_GELU_TANH: lambda t, z: z * t.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)), bf.ACT_SILU: lambda t, z: z * t.sigmoid(z)}


@pytest.fixture(scope="module")
def rt():
    return bf.Runtime(0)


PAIRS = (256, 1, 256, 2)     # pairs of CTAs that walk 256 x 256 tiles
NARROW = (128, 1, 256, 2)    # 256 x 128


def build(rt, batch, m, n, k, act, bias, other, tiling=(0, 0, 0), seed=0, share=1, std=1.0, grid=None):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    mk = lambda *s, std=1.0: torch.empty(s, device="cuda", dtype=torch.bfloat16).normal_(0, std, generator=g)
    t = {"a": mk(batch, m, k), "w": mk(batch, n, k, std=std / math.sqrt(k)), "bias": torch.randn(n, device="cuda", generator=g) if bias else None,
         "other": mk(batch, m, n) if other else None, "out": torch.full((batch, m, n), 7.0, device="cuda", dtype=torch.bfloat16)}
    d = rt.describe("gemm_act", bf.OP_GEMM_ACT_BF16, (batch, m, n, k) + tuple(tiling),
                    [None if t[x] is None else t[x].data_ptr() for x in ("a", "w", "bias", "other", "out")],
                    flags=bf.flag_share(share) | bf.flag_act(act) | (bf.FLAG_MUL if other == "mul" else 0), grid=grid)
    return t, rt.register_kernel(d)


def check(torch, t, act, other, want_other=None):
    z = torch.bmm(t["a"].double(), t["w"].double().transpose(1, 2))
    mag = torch.bmm(t["a"].double().abs(), t["w"].double().abs().transpose(1, 2))
    if t["bias"] is not None:
        z, mag = z + t["bias"].double(), mag + t["bias"].double().abs()
    y = ACTS[act](torch, z)
    tol = 1.13 * t["a"].shape[2] * 2.0 ** -23 * mag + 2.0 ** -20 * y.abs()
    if other:
        o = (t["other"] if want_other is None else want_other).double()
        y, tol = (y * o, tol * o.abs()) if other == "mul" else (y + o, tol)
    off = (t["out"].double() - y).abs() / (tol + 2.0 ** -8 * y.abs() + 1e-30)
    assert float(off.max()) <= 1.0, float(off.max())


def run(rt, *args, **kw):
    import torch
    t, h = build(rt, *args, **kw)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    check(torch, t, args[4], args[6])
    rt.unregister_kernel(h)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("other", [None, "add", "mul"])
def test_epilogues(rt, act, other):
    run(rt, 1, 200, 136, 72, act, True, other, std=3.0)


@pytest.mark.parametrize("bn,split,bm", [(64, 1, 128), (128, 1, 128), (256, 1, 128), (64, 1, 256), (128, 1, 256), (256, 1, 256), (64, 4, 128), (128, 2, 128),
                                         (256, 2, 128), (128, 3, 128), (256, 4, 128), (128, 5, 128)])
@pytest.mark.parametrize("m,n", [(1, 8), (300, 520), (513, 256)])
def test_tilings(rt, bn, split, bm, m, n):
    run(rt, 2, m, n, 1100 // 8 * 8, bf.ACT_SILU, True, "add", tiling=(bn, split, bm))


@pytest.mark.parametrize("m", [1, 3, 17, 128, 129, 1000])
@pytest.mark.parametrize("n,k", [(8, 8), (1000, 712), (4096, 1024)])
def test_default_tilings(rt, m, n, k):
    run(rt, 1, m, n, k, bf.ACT_GELU_TANH, False, "mul")
    run(rt, 1, m, n, k, bf.ACT_NONE, False, "add")


@pytest.mark.parametrize("m,n,k", [(256, 256, 64), (1, 8, 8), (300, 520, 72), (513, 264, 1096), (129, 2000, 320)])
@pytest.mark.parametrize("other", [None, "add", "mul"])
def test_pairs_of_ctas(rt, m, n, k, other):
    run(rt, 2, m, n, k, bf.ACT_SILU, True, other, tiling=PAIRS)
    run(rt, 2, m, n, k, bf.ACT_NONE, False, other, tiling=PAIRS, grid=(2, 1, 1))      # one pair takes all tiles


@pytest.mark.parametrize("m,n,k", [(256, 128, 64), (1, 8, 8), (300, 520, 72), (513, 264, 1096), (129, 2000, 320)])
@pytest.mark.parametrize("other", [None, "add", "mul"])
def test_pairs_with_narrow_tiles(rt, m, n, k, other):
    run(rt, 2, m, n, k, bf.ACT_GELU_TANH, True, other, tiling=NARROW)
    run(rt, 2, m, n, k, bf.ACT_NONE, False, other, tiling=NARROW, grid=(2, 1, 1))     # one pair takes all tiles


def test_pairs_take_several_tiles(rt):
    run(rt, 1, 2100, 2600, 712, bf.ACT_SILU, True, "mul", tiling=NARROW, grid=(26, 1, 1))   # 189 tiles
    run(rt, 1, 1500, 4096, 520, bf.ACT_NONE, True, "add")                              # the runtime's choice: narrow
    run(rt, 1, 2100, 2600, 712, bf.ACT_GELU, True, "add", tiling=PAIRS)               # 99 tiles
    run(rt, 1, 2100, 2600, 712, bf.ACT_GELU, True, "add", tiling=PAIRS, grid=(26, 1, 1))
    run(rt, 1, 2048, 4096, 1024, bf.ACT_SILU, False, "mul")                            # the runtime's choice


@pytest.mark.parametrize("bm", [16, 32])
@pytest.mark.parametrize("split", [1, 2, 4, 8])
def test_few_rows(rt, bm, split):
    for m in (1, bm - 1, bm, bm + 5):        # the last: two tiles
        run(rt, 2, m, 264, 1096, bf.ACT_GELU, True, "add", tiling=(128, split, bm))
    run(rt, 1, bm, 8, 1096, bf.ACT_SILU, False, "mul", tiling=(128, split, bm))


@pytest.mark.parametrize("m", [1, 16, 17, 32, 33])
def test_few_rows_with_long_k(rt, m):
    run(rt, 1, m, 1024, 8192, bf.ACT_NONE, True, "add")
    run(rt, 1, m, 136, 72, bf.ACT_RELU, True, None)


def test_smallest_ring_reuses_its_buffers(rt):
    import torch
    t, h = build(rt, 1, 500, 512, 256, bf.ACT_RELU, True, "add", tiling=(256, 1, 256))
    rt.unregister_kernel(h)
    d = rt.describe("small", bf.OP_GEMM_ACT_BF16, (1, 500, 512, 256, 256, 1, 128), [t[x].data_ptr() for x in ("a", "w", "bias", "other", "out")],
                    flags=bf.flag_act(bf.ACT_RELU), smem=2048 + 384 * 128)
    h = rt.register_kernel(d)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    check(torch, t, bf.ACT_RELU, "add")


def test_residual_may_be_the_output(rt):
    import torch
    t, h = build(rt, 1, 333, 264, 500 // 8 * 8, bf.ACT_NONE, True, "add")
    other = t["other"].clone()
    rt.set_kernel_args(h, [t[x].data_ptr() for x in ("a", "w", "bias", "other", "other")])
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    t["out"] = t["other"]
    check(torch, t, bf.ACT_NONE, "add", other)


def test_saturated_activations(rt):
    import torch
    t, h = build(rt, 1, 64, 64, 64, bf.ACT_SILU, False, None)
    t["a"].fill_(1.0)
    t["w"].copy_(torch.linspace(-1e36, 1e36, 64, device="cuda")[None, :, None].expand(1, 64, 64))
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    assert rt.read_status() == 0
    z = torch.bmm(t["a"].double(), t["w"].double().transpose(1, 2))
    assert torch.isfinite(t["out"].float()).all()
    assert (t["out"].double() - z.clamp(min=0)).abs().max() <= 2.0 ** -8 * z.max()
    assert (t["out"][z < 0] == 0).all()


@pytest.mark.parametrize("pattern", [bf.ZIGZAG, bf.PROPORTIONAL, bf.SM_STRIPED, bf.THREAD_SPLIT, bf.RANGE_SPLIT, bf.WORK_QUEUE])
def test_fused_launches_give_the_same_bits(rt, pattern):
    import torch
    stream = torch.cuda.current_stream().cuda_stream
    t1, a = build(rt, 1, 300, 512, 1024, bf.ACT_SILU, False, "mul", share=2, seed=1, tiling=(128, 1, 128))
    t2, b = build(rt, 2, 100, 256, 512, bf.ACT_GELU, True, "add", share=2, seed=2, tiling=(128, 1, 128))
    f = rt.register_fusion(a, b, pattern, 1, 1)
    rt.launch_sequential(f, stream)
    assert rt.read_status() == 0
    check(torch, t1, bf.ACT_SILU, "mul")
    check(torch, t2, bf.ACT_GELU, "add")
    want = [t1["out"].clone(), t2["out"].clone()]
    t1["out"].zero_(), t2["out"].zero_()
    rt.launch_fused(f, stream)
    assert rt.read_status() == 0
    assert torch.equal(t1["out"], want[0]) and torch.equal(t2["out"], want[1])


@pytest.mark.parametrize("pattern", [bf.ZIGZAG, bf.THREAD_SPLIT, bf.WORK_QUEUE])
def test_pairs_share_a_launch_in_another_form(rt, pattern):
    import torch
    stream = torch.cuda.current_stream().cuda_stream
    t1, a = build(rt, 1, 600, 512, 1024, bf.ACT_SILU, False, "mul", seed=1, tiling=PAIRS)
    t2, b = build(rt, 1, 100, 256, 512, bf.ACT_NONE, True, "add", seed=2, share=2, tiling=(128, 1, 128))
    f = rt.register_fusion(a, b, pattern, 1, 1)
    assert rt.fusion_info(f)["retiled_unsplit"][0]
    rt.launch_fused(f, stream)
    assert rt.read_status() == 0
    check(torch, t1, bf.ACT_SILU, "mul")
    check(torch, t2, bf.ACT_NONE, "add")
    t1["out"].zero_()
    rt.launch_kernel(a, stream)
    assert rt.read_status() == 0
    check(torch, t1, bf.ACT_SILU, "mul")
    if pattern == bf.ZIGZAG:
        g = rt.register_group([a, b], pattern, 1, 1)
        t1["out"].zero_()
        rt.launch_group(g, stream)
        assert rt.read_status() == 0
        check(torch, t1, bf.ACT_SILU, "mul")


@pytest.mark.parametrize("pattern", [bf.ZIGZAG, bf.PROPORTIONAL, bf.SM_STRIPED, bf.THREAD_SPLIT, bf.RANGE_SPLIT, bf.WORK_QUEUE])
def test_fused_tiles_of_few_rows_give_the_same_bits(rt, pattern):
    import torch
    stream = torch.cuda.current_stream().cuda_stream
    t1, a = build(rt, 1, 5, 1024, 4096, bf.ACT_SILU, False, "mul", share=2, seed=1)
    t2, b = build(rt, 1, 30, 512, 2048, bf.ACT_NONE, True, "add", share=2, seed=2)
    f = rt.register_fusion(a, b, pattern, 1, 1)
    rt.launch_sequential(f, stream)
    assert rt.read_status() == 0
    check(torch, t1, bf.ACT_SILU, "mul")
    check(torch, t2, bf.ACT_NONE, "add")
    want = [t1["out"].clone(), t2["out"].clone()]
    t1["out"].zero_(), t2["out"].zero_()
    rt.launch_fused(f, stream)
    assert rt.read_status() == 0
    assert torch.equal(t1["out"], want[0]) and torch.equal(t2["out"], want[1])
