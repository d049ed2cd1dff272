"""Block scales of a matrix that all groups share: there is one matrix of them, whatever the number of groups."""
import numpy as np
import pytest

import maize_amd as mz
from group_util import check, launch, random_operand, reference, to_f64

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
