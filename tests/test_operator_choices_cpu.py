"""What bfuse_default_launch does with tilings that a caller fixes in part (context NULL = 148 SMs; no device)."""
import pytest

import bfuse_project_b200 as bf

SHAPE_ERR = 2


def gemm(*shape, share=1):
    d = bf.KernelDesc()
    d.KernelName, d.op, d.flags = b"k", bf.OP_GEMM_ACT_BF16, bf.flag_share(share)
    for i, v in enumerate(shape):
        d.shape[i] = v
    return bf.lib().bfuse_default_launch(None, d), tuple(d.shape[4:8])


@pytest.mark.parametrize("share", [1, 2])
@pytest.mark.parametrize("split", [1, 2, 3, 4, 5, 6, 7, 8])
def test_k_slices_of_few_rows(split, share):
    # the transposed tiles take 1, 2, 4 or 8 k-slices; any other number runs in tiles of 128 rows, as it does for 33 rows
    rc, tiling = gemm(1, 4, 4096, 4096, 0, split, share=share)
    assert rc == 0 and tiling[1] == split and tiling[2] == (16 if split in (1, 2, 4, 8) else 128) and tiling[3] == 1
    rc, tiling = gemm(1, 33, 4096, 4096, 0, split, share=share)
    assert rc == 0 and tiling[1] == split and tiling[2] == 128


def test_k_slices_that_no_tile_takes():
    assert gemm(1, 4, 4096, 4096, 0, 9)[0] == SHAPE_ERR
    assert gemm(1, 4, 4096, 256, 0, 8)[0] == SHAPE_ERR     # four K blocks
    assert gemm(1, 4, 4096, 4096, 0, 3, 16)[0] == SHAPE_ERR


def test_a_tiling_that_is_asked_for_is_used():
    assert gemm(1, 16, 4096, 4096, 0, 0, 0, 2)[1] == (128, 1, 256, 2)         # pairs of CTAs for few rows, too (32 narrow tiles for 74 pairs)
    assert gemm(1, 16, 4096, 4096, 256, 0, 0, 2)[1] == (256, 1, 256, 2)
    assert gemm(1, 16, 4096, 4096, -1, 0, 0, 2)[1][0] in (128, 256)
    assert gemm(1, 16, 4096, 4096, 0, 0, 0, 1)[1][2:] == (16, 1)
    for tiling in ((256, 1, 256, 2), (128, 1, 256, 2), (128, 4, 16, 1), (128, 1, 32, 1), (64, 2, 128, 1)):   # written back: the same again
        assert gemm(1, 30, 4096, 4096, *tiling) == (0, tiling)


@pytest.mark.parametrize("tiling", [(64, 1, 16), (256, 2, 32), (0, 0, 16, 2), (0, 0, 32, 2), (256, 4, 0, 2), (256, 1, 128, 2), (0, 2, 256, 2), (0, 0, 0, 3),
                                    (0, 0, 0, -1)])
def test_a_tiling_that_no_kernel_runs_is_refused(tiling):
    for m in (4, 32, 300):
        assert gemm(1, m, 4096, 4096, *tiling)[0] == SHAPE_ERR
