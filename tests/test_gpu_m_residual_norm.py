"""Norms after and before a block with gate and residual scale, against the definition in 64 bits.

Both outputs are rounded once (2^-8); what fp32 adds over a row of at most 8192 is below 2^-16 of the largest term."""
import pytest

import bfuse_project_b200 as bf

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def rt():
    return bf.Runtime(0)


def build(rt, rows, cols, norms, gate_rows=None, scale=0.5, r=True, seed=0, block=None):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    mk = lambda *s, mean=0.0: torch.empty(s, device="cuda", dtype=torch.bfloat16).normal_(mean, 1.0, generator=g)
    n = bin(norms).count("1")
    t = {"x": mk(rows, cols), "b": mk(rows, cols), "gate": None if gate_rows is None else mk(-(-rows // gate_rows) if gate_rows else 1, cols),
         "w": mk(n, cols, mean=1.0) if n else None, "r": torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16) if r else None,
         "y": torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16) if norms & bf.NORM_BEFORE else None}
    kw = {} if block is None else dict(block=block + (1,), grid=(-(-rows // block[1]), 1, 1))
    d = rt.describe("residual_norm", bf.OP_RESIDUAL_NORM_BF16, (rows, cols, norms, gate_rows or 0),
                    [None if t[k] is None else t[k].data_ptr() for k in ("x", "b", "gate", "w", "r", "y")], fparam=(EPS, scale), **kw)
    return t, rt.register_kernel(d)


def expected(t, norms, gate_rows, scale):
    x, b = t["x"].double(), t["b"].double()
    w = None if t["w"] is None else t["w"].double()
    if norms & bf.NORM_AFTER:
        b = b / (b.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w[0]
    if t["gate"] is not None:
        b = b * t["gate"].double().repeat_interleave(gate_rows or x.shape[0], 0)[:x.shape[0]]
    r = x + scale * b
    y = r / (r.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w[-1] if norms & bf.NORM_BEFORE else None
    return r, y, (x.abs() + (scale * b).abs())


def check(t, norms, gate_rows, scale):
    r, y, mag = expected(t, norms, gate_rows, scale)
    if t["r"] is not None:
        assert ((t["r"].double() - r).abs() <= 2.0 ** -8 * r.abs() + 2.0 ** -16 * mag).all()
    if y is not None:
        slope = (y / r.where(r != 0, r.new_ones(()))).abs() + 1e-30
        assert ((t["y"].double() - y).abs() <= 2.0 ** -8 * y.abs() + 2.0 ** -16 * (mag * slope + y.abs())).all()


@pytest.mark.parametrize("cols", [8, 64, 264, 768, 1000, 2048, 4096, 5120, 8192])
@pytest.mark.parametrize("rows", [1, 3, 130, 700])
def test_sizes(rt, rows, cols):
    import torch
    t, h = build(rt, rows, cols, 3, 0)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    check(t, 3, 0, 0.5)


@pytest.mark.parametrize("norms", [0, 1, 2, 3])
@pytest.mark.parametrize("gate_rows", [None, 0, 1, 7])
def test_forms(rt, norms, gate_rows):
    import torch
    for scale in (1.0, -0.22):
        t, h = build(rt, 40, 520, norms, gate_rows, scale)
        rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        check(t, norms, gate_rows, scale)


def test_only_the_norm_is_kept(rt):
    import torch
    t, h = build(rt, 40, 520, 2, r=False)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    check(t, 2, None, 0.5)


def test_in_place_stream(rt):
    import torch
    t, h = build(rt, 300, 2048, 3, 0)
    r, y, mag = expected(t, 3, 0, 0.5)
    rt.set_kernel_args(h, [t["x"].data_ptr(), t["b"].data_ptr(), t["gate"].data_ptr(), t["w"].data_ptr(), t["x"].data_ptr(), t["b"].data_ptr()])
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert ((t["x"].double() - r).abs() <= 2.0 ** -8 * r.abs() + 2.0 ** -16 * mag).all()
    assert (t["b"].double() - y).abs().max() <= 2.0 ** -7 * y.abs().max()


@pytest.mark.parametrize("block", [(32, 8), (64, 1), (96, 1), (160, 1), (128, 2), (256, 1)])
def test_other_blocks(rt, block):
    import torch
    t, h = build(rt, 77, 1000, 3, 1, block=block)
    rt.launch_kernel(h, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    check(t, 3, 1, 0.5)


@pytest.mark.parametrize("pattern", [bf.ZIGZAG, bf.PROPORTIONAL, bf.SM_STRIPED, bf.THREAD_SPLIT, bf.RANGE_SPLIT, bf.WORK_QUEUE])
def test_fused_launches_give_the_same_bits(rt, pattern):
    import torch
    stream = torch.cuda.current_stream().cuda_stream
    t1, a = build(rt, 700, 4096, 3, 0, seed=1)
    t2, b = build(rt, 333, 768, 2, None, seed=2)
    x = torch.randn(400, 512, device="cuda")
    s = torch.zeros_like(x)
    soft = rt.register_kernel(rt.describe("softmax", bf.OP_SOFTMAX_F32, (400, 512), [x.data_ptr(), s.data_ptr()], fparam=(1.0,)))
    for k1, k2 in ((a, b), (soft, a), (b, soft)):
        f = rt.register_fusion(k1, k2, pattern, 1, 1)
        rt.launch_sequential(f, stream)
        torch.cuda.synchronize()
        outs = [t1["r"], t1["y"], t2["r"], t2["y"], s]
        want = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
        rt.launch_fused(f, stream)
        assert rt.read_status() == 0
        used = [a in (k1, k2)] * 2 + [b in (k1, k2)] * 2 + [soft in (k1, k2)]
        assert all(torch.equal(o, w) for o, w, u in zip(outs, want, used) if u)
        rt.unregister_fusion(f)
    check(t1, 3, 0, 0.5) if t1["r"].any() else None
