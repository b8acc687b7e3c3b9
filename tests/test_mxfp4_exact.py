"""Products with both operands in MXFP4 whose sums f32 holds exactly, in any order: no block of a long row may be missing, doubled or under
another block's scale.  (The allowance for f32 sums of any data grows with the row, to more than a block of the longest ones.)"""
import numpy as np
import pytest

import mxfp4_plain as plain
from test_gpu_parity import fa, to_dev  # noqa: F401 (fa: the module's fixture)

LIMIT = 65568  # columns


def _operands(rows, cols, batch):
    """(codes, scale bytes, their values, activations that are their own quantization).

    Weights are 0, 1/2 or 1 under 2^0, 2^1 or 2^2, activations any code under 2^0 or 2^1 with a 4 or a 6 in every block, which is what its scale
    is made from.  So every product is a multiple of 1/4 and at most 6 * 8, and a sum of LIMIT of them at most 65568 * 48 * 4 quarters,
    which is less than 2^24: every sum of some of them is an f32 number."""
    assert cols <= LIMIT and LIMIT * 48 * 4 < 2 ** 24
    rng = np.random.default_rng(rows + cols + batch)
    blocks = cols // plain.BLOCK
    codes = rng.choice(np.array([0, 1, 2, 9, 10], np.uint8), (rows, cols))
    scales = rng.integers(127, 130, (rows, blocks), dtype=np.uint8)
    x_codes = rng.integers(0, 16, (batch, cols), dtype=np.uint8)
    at = np.arange(blocks) * plain.BLOCK + rng.integers(0, plain.BLOCK, (batch, blocks))
    np.put_along_axis(x_codes, at, rng.choice(np.array([6, 7, 14, 15], np.uint8), (batch, blocks)), 1)
    x_scales = rng.integers(127, 129, (batch, blocks), dtype=np.uint8)
    x = plain.values(x_codes, x_scales).astype(np.float32)
    return codes, scales, plain.values(codes, scales).astype(np.float32), x, x_scales


# both sides of the longest rows that the workgroups quantize for themselves (one, two and four tokens); one and two strips a workgroup, two tiles of
# tokens, tiles whole and in shares; rows that end inside a unit of sixteen blocks and inside a stage of eight
CASES = [(33, 61440, 1), (33, 61472, 1), (33, 65536, 1), (33, 65536, 2), (47, 30688, 2), (47, 30752, 2), (33, 65536, 3), (33, 15360, 4), (33, 15392, 4), (33, 65568, 4),
         (40, 28672, 1), (7201, 15360, 4), (7201, 15392, 4), (7201, 8224, 3), (49, 65568, 9), (33, 65536, 16), (33, 65536, 20), (33, 65568, 32), (33, 65568, 33), (65, 65536, 70),
         (300, 32800, 200), (257, 16416, 300), (2049, 4128, 1100)]


@pytest.mark.parametrize("rows,cols,batch", [(33, 65536, 1), (33, 65568, 4), (40, 28672, 1)])
def test_the_operands_show_every_block(rows, cols, batch):
    """Activations are what their quantization stands for, and every block's sums are other numbers than zero for some output."""
    codes, scales, w, x, x_scales = _operands(rows, cols, batch)
    got_codes, got_scales = plain.quantize(x)
    assert np.array_equal(got_scales, x_scales) and np.array_equal(plain.values(got_codes, got_scales).astype(np.float32), x)
    each = np.matmul(x.reshape(batch, -1, plain.BLOCK).transpose(1, 0, 2), w.reshape(rows, -1, plain.BLOCK).transpose(1, 2, 0))  # [blocks][batch][rows]
    assert (each != 0).any((1, 2)).all()
    assert np.array_equal(each.sum(0, dtype=np.float64), x.astype(np.float64) @ w.T.astype(np.float64))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,batch", CASES)
def test_products_that_are_exact(fa, rows, cols, batch):
    import torch
    print("exact mxfp4 product", rows, cols, batch, flush=True)
    codes, scales, w, x, _ = _operands(rows, cols, batch)
    matrix = fa.Weights.from_device(fa.MXFP4, to_dev(plain.blocks(codes, scales).reshape(-1)), rows, cols)
    want = x @ w.T  # (exact in f32, too)
    xd = to_dev(x)
    assert np.array_equal(matrix.gemm_mxfp4(xd).cpu().numpy(), want)
    assert np.array_equal(matrix.gemm_acts(fa.BatchActs(batch, cols, "mxfp4").quantize(xd)).cpu().numpy(), want)
    # unaligned activations have kernels of their own where the workgroups quantize
    room = torch.zeros(xd.numel() + 1, device="cuda")
    room[1:] = xd.flatten()
    assert np.array_equal(matrix.gemm_mxfp4(room[1:].view(batch, cols)).cpu().numpy(), want)
