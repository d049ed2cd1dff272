"""Block scales: of a matrix that all groups share, with strides of their own, and of several matrices that are quantised together."""
import numpy as np
import pytest

import maize_amd as mz
from group_util import check, from_f64, launch, random_operand, reference, to_f64
from test_gpu_groups import quantize

E4M3 = mz.IN_E4M3


class Buffer(mz.DeviceBuffer):
    def __init__(self, nbytes):
        super().__init__(None, 0x10000, nbytes)


def desc(scale_b=0x6000, k=200, n=300, groups=5, **how):
    m = mz.GlobalMatrix
    return mz.grouped_desc(m(0x1000, 100, k), m(0x2000, k, n), m(0x3000, 100, n), 0x4000, groups, in_type=E4M3, scale_a=0x5000, scale_b=scale_b, **how)


def test_groups_that_share_a_matrix_share_its_scales():
    assert desc(stride=0).stride_scale_b == 0
    assert desc().stride_scale_b == 2 * 3 and desc(ld_scale_b=7).stride_scale_b == 2 * 7
    assert desc(stride=0, stride_scale_b=6).stride_scale_b == 6           # asked for: scales of each group's own
    assert desc(stride_scale_b=0).stride_scale_b == 0
    mz.validate(desc(stride=0))


def test_one_matrix_of_scales_is_enough_for_a_shared_matrix():
    desc(Buffer(4 * 6), stride=0)
    for buffer, how in ((Buffer(4 * 6 - 1), dict(stride=0)), (Buffer(4 * 30 - 1), dict())):
        with pytest.raises(ValueError):
            desc(buffer, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("nt", [False, True])
@pytest.mark.parametrize("rows", [20, 300])
def test_shared_8bit_matrix(ctx, oracle, rows, nt):
    rng = np.random.default_rng(rows)
    k, n = 300, 264
    a, b = random_operand(rng, (rows, k), E4M3), random_operand(rng, (1, n, k) if nt else (1, k, n), E4M3)
    sa = np.exp(rng.standard_normal((3, rows)) * 0.5).astype(np.float32) / 64
    sb = np.exp(rng.standard_normal((1, -(-b.shape[1] // 128), -(-b.shape[2] // 128))) * 0.5).astype(np.float32) / 64
    offsets = np.array([0, rows // 3, rows // 3, rows - 4, rows], dtype=np.int32)
    got = launch(ctx, a, b, offsets, mz.GROUP_ROWS, nt, E4M3, scale_a=sa, scale_b=sb, shared_b=True)
    sums, mag = reference(to_f64(a, E4M3), np.repeat(to_f64(b, E4M3), 4, axis=0), offsets, mz.GROUP_ROWS, nt, E4M3, sa, np.repeat(sb, 4, axis=0))
    check(got, sums, mag, k, E4M3, coeff=oracle.floor_coeff_f8(k))


@pytest.mark.gpu
@pytest.mark.parametrize("nt", [False, True])
@pytest.mark.parametrize("rows,n", [(20, 264), (300, 264), (4100, 4105)])
def test_scales_with_strides_of_their_own(ctx, rows, n, nt):
    """ld_scale_a, ld_scale_b and stride_scale_b larger than compact, NaN between the scales; 8-bit values whose block sums are exact in fp32, so that
    what is left is a rounding for scale_a * scale_b and two for each block of K."""
    rng = np.random.default_rng(rows + n)
    k, groups = 300, 3
    offsets = np.array([0, rows // 3, rows // 3, rows], dtype=np.int32)
    values = np.array([-3.0, -2.0, -1.5, -1.0, -0.5, 0.0, 0.5, 1.0, 1.5, 2.0, 3.0])
    a, b = (from_f64(rng.choice(values, s), E4M3) for s in ((rows, k), (groups, n, k) if nt else (groups, k, n)))
    down, across = -(-b.shape[1] // 128), -(-b.shape[2] // 128)
    sa = np.full((3, rows + 7), np.nan, dtype=np.float32)
    sa[:, :rows] = np.exp(rng.standard_normal((3, rows)))
    one = down * (across + 3) + 5
    sb = np.full((groups, one), np.nan, dtype=np.float32)
    inner = sb[:, :down * (across + 3)].reshape(groups, down, across + 3)[:, :, :across]
    inner[:] = np.exp(rng.standard_normal(inner.shape))
    bufs = [ctx.upload(x) for x in (a, b, np.zeros((rows, n), dtype=np.float32), offsets, sa, sb)]
    da, db, dc, doff, dsa, dsb = bufs
    try:
        ctx.gemm_grouped(mz.grouped_desc(mz.Matrix(da, rows, k, elem_bytes=1), mz.Matrix(db, *b.shape[1:], elem_bytes=1), mz.Matrix(dc, rows, n, elem_bytes=4), doff, groups,
                                         layout=mz.LAYOUT_NT if nt else mz.LAYOUT_NN, in_type=E4M3, out_type=mz.OUT_F32, scale_a=dsa, scale_b=dsb,
                                         ld_scale_a=rows + 7, ld_scale_b=across + 3, stride_scale_b=one))
        ctx.sync()
        got = dc.download(np.float32).reshape(rows, n).astype(np.float64)
    finally:
        for x in bufs:
            x.free()
    sums, mag = reference(to_f64(a, E4M3), to_f64(b, E4M3), offsets, mz.GROUP_ROWS, nt, E4M3, sa[:, :rows], inner)
    check(got, sums, mag, k, E4M3, mz.OUT_F32, coeff=5 * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("in_type", [mz.IN_BF16, mz.IN_F16, mz.IN_F32])
@pytest.mark.parametrize("block", [1, 128])
def test_quantizer_of_several_matrices(ctx, block, in_type):
    """Three matrices in one call, gaps between them: what each gives by itself, and nothing written in the gaps."""
    rng = np.random.default_rng(block)
    rows, cols, gap = 150, 203, 11
    across, down = 2, 2
    shape = (across, rows) if block == 1 else (down, across)
    x = np.zeros((3, rows * cols + gap), dtype=np.uint32 if in_type == mz.IN_F32 else np.uint16)
    for z in range(3):
        x[z, :rows * cols] = from_f64(rng.standard_normal(rows * cols) * 10.0 ** z, in_type)
    one = shape[0] * shape[1]
    dx, dq, ds = ctx.upload(x), ctx.upload(np.full((3, rows * cols + gap), 0xA5, dtype=np.uint8)), ctx.upload(np.full((3, one + gap), -7.0, dtype=np.float32))
    try:
        ctx.quantize_blocks(mz.quantize_desc(mz.Matrix(dx, rows, cols, elem_bytes=x.itemsize), mz.Matrix(dq, rows, cols, elem_bytes=1), ds, block, in_type, batch=3,
                                             stride_x=rows * cols + gap, stride_q=rows * cols + gap, stride_scale=one + gap))
        ctx.sync()
        q, scale = dq.download(np.uint8).reshape(3, -1), ds.download(np.float32).reshape(3, -1)
    finally:
        for buf in (dx, dq, ds):
            buf.free()
    assert np.all(q[:, rows * cols:] == 0xA5) and np.all(scale[:, one:] == -7.0)
    for z in range(3):
        alone_q, alone_scale = quantize(ctx, x[z, :rows * cols].reshape(rows, cols), in_type, block)
        assert np.array_equal(q[z, :rows * cols].reshape(rows, cols), alone_q) and np.array_equal(scale[z, :one].reshape(shape), alone_scale)
