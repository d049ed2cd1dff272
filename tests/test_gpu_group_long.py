"""Grouped products and the quantiser on operands whose byte offsets pass 32 bits: rows far down a long C, groups' matrices far apart."""
import numpy as np
import pytest

import maize_amd as mz
from group_util import check, from_f64, random_operand, reference, to_f64
from test_gpu_groups import quantized

pytestmark = pytest.mark.gpu

BF16, E4M3 = mz.IN_BF16, mz.IN_E4M3


@pytest.fixture
def memory(ctx):
    """malloc and upload whose buffers go when the test ends."""
    bufs = []

    def get(x):
        bufs.append(ctx.malloc(x) if isinstance(x, int) else ctx.upload(x))
        return bufs[-1]
    yield get
    ctx.sync()
    for b in bufs:
        b.free()


def test_rows_past_4_gib_of_c(ctx, memory):
    rng = np.random.default_rng(1)
    rows, k, n, period = 1_200_000, 64, 2056, 4096
    block, b = random_operand(rng, (period, k), BF16), random_operand(rng, (2, n, k), BF16)
    a = np.resize(block, (rows, k))
    offsets = np.array([0, 700_001, rows], dtype=np.int32)
    dc = memory(rows * n * 2)
    ctx.gemm_grouped(mz.grouped_desc(mz.Matrix(memory(a), rows, k), mz.Matrix(memory(b), n, k), mz.Matrix(dc, rows, n), memory(offsets), 2, layout=mz.LAYOUT_NT))
    ctx.sync()
    edge = 2 ** 32 // (2 * n)
    for lo in (0, 700_001 - 50, edge - 50, rows - 100):
        got = to_f64(dc.download(np.uint16, 100 * n, lo * n * 2).reshape(100, n), BF16)
        at = np.clip(offsets - lo, 0, 100)
        sums, mag = reference(to_f64(a[lo:lo + 100], BF16), to_f64(b, BF16), at, mz.GROUP_ROWS, True, BF16)
        check(got, sums, mag, k, BF16, label=f"rows from {lo}")


def test_weight_gradients_past_4_gib(ctx, memory):
    rng = np.random.default_rng(2)
    groups, m, n = 600, 2048, 2056
    rows = 2 * groups
    a, b = random_operand(rng, (rows, m), BF16), random_operand(rng, (rows, n), BF16)
    offsets = np.arange(0, rows + 1, 2, dtype=np.int32)
    dc = memory(groups * m * n * 2)
    ctx.gemm_grouped(mz.grouped_desc(mz.Matrix(memory(a), rows, m), mz.Matrix(memory(b), rows, n), mz.Matrix(dc, m, n), memory(offsets), groups, axis=mz.GROUP_DEPTH))
    ctx.sync()
    fa, fb = to_f64(a, BF16), to_f64(b, BF16)
    for g in (0, 2 ** 32 // (2 * m * n), 2 ** 32 // (2 * m * n) + 1, groups - 1):
        got = to_f64(dc.download(np.uint16, m * n, g * m * n * 2).reshape(1, m, n), BF16)
        sums, mag = reference(fa[2 * g:2 * g + 2], fb[2 * g:2 * g + 2], [0, 2], mz.GROUP_DEPTH, False, BF16)
        check(got, sums, mag, 2, BF16, label=f"group {g}")


@pytest.mark.parametrize("in_type", [BF16, E4M3])
@pytest.mark.parametrize("nt", [False, True])
def test_matrices_that_lie_gigabytes_apart(ctx, oracle, memory, in_type, nt):
    rng = np.random.default_rng(3)
    rows, k, n, groups, size = 90, 320, 264, 3, 1 if in_type == E4M3 else 2
    stride = 3_000_000_000 // size + 7
    a, b = random_operand(rng, (rows, k), in_type), random_operand(rng, (groups, n, k) if nt else (groups, k, n), in_type)
    offsets = np.array([0, 20, 50, rows], dtype=np.int32)
    db = memory(((groups - 1) * stride + k * n) * size)
    for g in range(groups):
        db.write(b[g], g * stride * size)
    dc, how, coeff, sa, sb = memory(rows * n * 2), {}, None, None, None
    if in_type == E4M3:
        sa, sb = np.full((3, rows), 0.5, dtype=np.float32), np.ones((groups, 3, 3), dtype=np.float32)
        how, coeff = dict(scale_a=memory(sa), scale_b=memory(sb)), oracle.floor_coeff_f8(k)
    ctx.gemm_grouped(mz.grouped_desc(mz.Matrix(memory(a), rows, k, elem_bytes=size), mz.Matrix(db, *b.shape[1:], elem_bytes=size), mz.Matrix(dc, rows, n), memory(offsets), groups,
                                     layout=mz.LAYOUT_NT if nt else mz.LAYOUT_NN, stride=stride, in_type=in_type, **how))
    ctx.sync()
    got = to_f64(dc.download(np.uint16).reshape(rows, n), BF16)
    sums, mag = reference(to_f64(a, in_type), to_f64(b, in_type), offsets, mz.GROUP_ROWS, nt, in_type, sa, sb)
    check(got, sums, mag, k, in_type, coeff=coeff)


@pytest.mark.parametrize("block", [1, 128])
def test_quantizer_past_4_gib(ctx, memory, block):
    rng = np.random.default_rng(4)
    rows, cols, last = 600_064, 2056, 256
    x = from_f64(rng.standard_normal((last, cols)), mz.IN_F32)
    across = 17
    dx, dq = memory(rows * cols * 4), memory(rows * cols)
    ds = memory(across * (rows if block == 1 else rows // 128) * 4)
    dx.fill(0)
    dx.write(x, (rows - last) * cols * 4)
    ctx.quantize_blocks(mz.quantize_desc(mz.Matrix(dx, rows, cols, elem_bytes=4), mz.Matrix(dq, rows, cols, elem_bytes=1), ds, block, mz.IN_F32))
    ctx.sync()
    want_q, want_scale = quantized(to_f64(x, mz.IN_F32), block)
    assert np.array_equal(dq.download(np.uint8, last * cols, (rows - last) * cols).reshape(last, cols), want_q)
    scale = ds.download(np.float32)
    scale = scale.reshape(across, rows)[:, -last:] if block == 1 else scale.reshape(rows // 128, across)[-last // 128:]
    assert np.array_equal(scale, want_scale) and not dq.download(np.uint8, 4 * cols, 0).any()
