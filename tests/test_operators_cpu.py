"""GEMM_ACT_BF16, RESIDUAL_NORM_BF16 and ATTENTION_BF16 without a device: the tilings bfuse_default_launch picks, what it
refuses, argument sizes and the layer that is built of them (context NULL = 148 SMs)."""
import ctypes as C

import pytest

import bfuse_project_b200 as bf
from bfuse_project_b200 import segment as sg


def launch(op, shape, share=2, flags=0, fparam=()):
    d = bf.KernelDesc()
    d.KernelName, d.op, d.flags = b"k", op, flags | bf.flag_share(share)
    for i, v in enumerate(shape):
        d.shape[i] = v
    for i, v in enumerate(fparam):
        d.fparam[i] = v
    return bf.lib().bfuse_default_launch(None, d), d


def arg_bytes(d):
    out = []
    for i in range(d.nargs):
        n, o = C.c_size_t(), C.c_int()
        assert bf.lib().bfuse_arg_info(None, d, i, n, o) == 0
        out.append((n.value, bool(o.value)))
    return out


def test_gemm_act_tilings():
    rc, d = launch(bf.OP_GEMM_ACT_BF16, (1, 4, 4096, 14336), share=1)         # few rows: transposed, K over clusters
    assert rc == 0 and tuple(d.shape[4:8]) == (128, 4, 16, 1) and d.GridDim.tuple() == (4, 32, 1)
    rc, d = launch(bf.OP_GEMM_ACT_BF16, (1, 32, 14336, 4096), share=1)
    assert rc == 0 and tuple(d.shape[4:8]) == (128, 1, 32, 1) and d.GridDim.tuple() == (1, 112, 1)
    rc, d = launch(bf.OP_GEMM_ACT_BF16, (1, 33, 4096, 14336), share=1)
    assert rc == 0 and d.shape[6] == 128
    rc, d = launch(bf.OP_GEMM_ACT_BF16, (1, 4096, 14336, 4096), share=1)      # large and alone: pairs of CTAs
    assert rc == 0 and tuple(d.shape[4:8]) == (256, 1, 256, 2) and d.GridDim.tuple() == (148, 1, 1)
    rc, d = launch(bf.OP_GEMM_ACT_BF16, (1, 512, 4096, 4096), share=1)        # few tiles: narrow ones
    assert rc == 0 and tuple(d.shape[4:8]) == (128, 1, 256, 2) and d.GridDim.tuple() == (128, 1, 1)
    rc, d = launch(bf.OP_GEMM_ACT_BF16, (1, 300, 6000, 2048), share=1)        # a CTA per tile fits the SMs better
    assert rc == 0 and tuple(d.shape[4:8]) == (128, 1, 128, 1)
    assert launch(bf.OP_GEMM_ACT_BF16, (1, 512, 4096, 4096, 64, 1, 256, 2), share=1)[0] == 2
    rc, d = launch(bf.OP_GEMM_ACT_BF16, (1, 4096, 14336, 4096), share=2)      # sharing its launch: a CTA per tile, as GEMM_BF16
    _, g = launch(bf.OP_GEMM_BF16, (1, 4096, 14336, 4096), share=2)
    assert rc == 0 and d.shape[7] == 1 and d.GridDim.tuple() == g.GridDim.tuple() and d.smem_bytes == g.smem_bytes
    assert arg_bytes(launch(bf.OP_GEMM_ACT_BF16, (2, 3, 16, 8))[1]) == [(96, False), (512, False), (64, False), (192, False), (192, True)]


@pytest.mark.parametrize("shape", [(0, 8, 8, 8), (1, 0, 8, 8), (1, 8, -8, 8), (1, 8, 8, 0), (1, 4, 4096, 4096, 128, 3, 16), (1, 4, 4096, 4096, 128, 16, 16),
                                   (1, 300, 512, 512, 48)])
def test_gemm_act_refusals(shape):
    assert launch(bf.OP_GEMM_ACT_BF16, shape)[0] == 2


@pytest.mark.parametrize("rows,cols,block,grid", [(1, 4096, (256, 1, 1), 1), (512, 4096, (256, 1, 1), 512), (12000, 4096, (128, 2, 1), 6000),
                                                  (12007, 5120, (160, 1, 1), 12007), (60000, 768, (32, 8, 1), 7500), (5, 8, (8, 32, 1), 1),
                                                  (3, 8192, (256, 1, 1), 3)])
def test_residual_norm_tilings(rows, cols, block, grid):
    rc, d = launch(bf.OP_RESIDUAL_NORM_BF16, (rows, cols, 3, 0))
    assert rc == 0 and d.BlockDim.tuple() == block and d.GridDim.tuple() == (grid, 1, 1)
    assert d.BlockDim.size() % 32 == 0 and 8 * 4 * block[0] >= cols


def test_residual_norm_arguments_and_refusals():
    d = launch(bf.OP_RESIDUAL_NORM_BF16, (10, 64, bf.NORM_AFTER | bf.NORM_BEFORE, 3))[1]
    assert [n for n, _ in arg_bytes(d)] == [1280, 1280, 512, 256, 1280, 1280]      # a row of the gate for every three rows, two norms
    assert [o for _, o in arg_bytes(d)] == [False] * 4 + [True] * 2
    for shape in ((0, 64), (4, 0), (4, 12), (4, 8200), (4, 64, 4), (4, 64, -1), (4, 64, 3, -1)):
        assert launch(bf.OP_RESIDUAL_NORM_BF16, shape)[0] == 2


def test_attention_tilings():
    rc, d = launch(bf.OP_ATTENTION_BF16, (1, 8192, 8192, 32, 8, 128), share=1, flags=bf.FLAG_CAUSAL, fparam=(0.1,))
    assert rc == 0 and tuple(d.shape[8:10]) == (1, 2) and d.GridDim.tuple() == (8, 128, 1) and d.BlockDim.tuple() == (320, 1, 1)
    rc, d = launch(bf.OP_ATTENTION_BF16, (1, 8192, 8192, 32, 8, 128), share=2, fparam=(0.1,))
    assert rc == 0 and tuple(d.shape[8:10]) == (1, 1) and d.GridDim.tuple() == (8, 256, 1) and d.BlockDim.tuple() == (192, 1, 1)
    rc, d = launch(bf.OP_ATTENTION_BF16, (1, 1, 32768, 32, 8, 128), share=1, fparam=(0.1,))       # few rows, many keys
    assert rc == 0 and tuple(d.shape[8:10]) == (8, 1) and d.GridDim.tuple() == (64, 1, 1)
    rc, d = launch(bf.OP_ATTENTION_BF16, (16, 16, 27849, 32, 8, 128), share=1, fparam=(0.1,))
    assert rc == 0 and d.shape[8] == 1 and d.GridDim.tuple() == (8, 16, 1)
    rc, d = launch(bf.OP_ATTENTION_BF16, (3, 700, 900, 7, 1, 96), fparam=(0.1,))                  # 18 positions a tile
    assert rc == 0 and d.GridDim.tuple() == (1, (700 + 3 * 17) // 18, 1)
    # the number of tiles is enough for any lengths
    for lens in ([700, 0, 0], [1, 1, 698], [19, 19, 662]):
        assert sum(-(-n // 18) for n in lens) <= d.GridDim.Y
    assert [n for n, _ in arg_bytes(d)] == [700 * 7 * 192, 900 * 192, 900 * 192, 16, 16, 700 * 7 * 192]
    d = launch(bf.OP_ATTENTION_BF16, (1, 10, 10, 4, 2, 64, 512, 512), fparam=(0.1,))[1]           # slices of one projection
    assert [n for n, _ in arg_bytes(d)][:3] == [2 * (9 * 512 + 256), 2 * (9 * 512 + 128), 2 * (9 * 512 + 128)]


@pytest.mark.parametrize("shape", [(0, 8, 8, 4, 4, 64), (1, 0, 8, 4, 4, 64), (1, 8, 0, 4, 4, 64), (1, 8, 8, 4, 3, 64), (1, 8, 8, 256, 1, 64), (1, 8, 8, 4, 0, 64),
                                   (1, 8, 8, 4, 4, 136), (1, 8, 8, 4, 4, 60), (1, 8, 8, 4, 4, 64, 255), (1, 8, 8, 4, 4, 64, 128), (1, 8, 8, 4, 4, 64, 0, 260),
                                   (1, 8, 8, 4, 4, 64, 0, 0, 3), (1, 8, 8, 4, 4, 64, 0, 0, 16), (1, 8, 8, 4, 4, 64, 0, 0, 2, 2), (1, 8, 8, 4, 4, 64, 0, 0, 1, 3),
                                   (1, 2 ** 31 - 1, 8, 128, 128, 8)])
def test_attention_refusals(shape):
    assert launch(bf.OP_ATTENTION_BF16, shape, fparam=(0.1,))[0] == 2


@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf")])
def test_attention_scale_is_positive_and_finite(scale):
    assert launch(bf.OP_ATTENTION_BF16, (1, 8, 8, 4, 4, 64), fparam=(scale,))[0] == 2


def test_llama_layer_schedule():
    _, ops = sg.llama_layer(None, None, lens=(100, 28))
    names = [[(kind, [ops[i].name for i in idx]) for kind, idx in step] for step in sg.schedule(ops)]
    assert ("group", ["q_proj", "k_proj", "v_proj"]) in names[1] and ("group", ["rope_q", "rope_k"]) in names[2]
    order = [n for step in names for _, g in step for n in g]
    assert len(order) == len(ops) == 12 and order.index("attention") < order.index("o_proj") < order.index("post_norm") < order.index("up_proj")
    assert order.index("up_proj") < order.index("gate_proj") < order.index("down_proj")
