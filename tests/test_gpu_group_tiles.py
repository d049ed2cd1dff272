"""Every kernel of the grouped products at its edges, by cases whose plan names it: odd K, N, strides and addresses, empty groups, rows of no group, NaN
next door, and each way to write C, against the definition in 64 bits."""
import os
import re

import numpy as np
import pytest

import maize_amd as mz
from group_tiles import BF16, CASES, E4M3, F16, Case
from group_util import check, from_f64, launch, random_operand, reference, to_f64

HSACO = os.path.join(os.path.dirname(mz.LIB_PATH), "maize_groups_gfx950.hsaco")
EXACT8 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0])


def test_the_cases_reach_every_kernel():
    """Each case is planned on the kernel that it names, in K ranges where it says so; together they name every kernel there is."""
    for c in CASES:
        p = mz.grouped_plan(c.desc())
        assert (p["kernel"], p["ksplit"] > 1) == (c.kernel, c.split), c.label()
    names = set(re.findall(rb"maize_group_\w+", open(HSACO, "rb").read()))
    assert {c.kernel.encode() for c in CASES} == names
    # kernels that can split K: all but the 256 x 256 ones
    assert {c.kernel for c in CASES if c.split} == {c.kernel for c in CASES if "256x256" not in c.kernel}
    # last row panels that are half ones and whole ones, in 16- and 8-bit types, whole and in K ranges
    for c in CASES:
        size, sizes = int(c.kernel.rsplit("_", 1)[1].split("x")[0]), np.diff(c.offsets)
        if c.lay != "tn" and size >= 128 and c.odd:
            rest = sizes[sizes > 0] % size
            assert ((rest > 0) & (rest <= size // 2)).any() and (rest > size // 2).any() and (sizes == 0).any(), c.label()


def operands(c, rng):
    """Bits of A and B, scales, and the numbers that they stand for.  The 8-bit values' products are within the 13 binades that the matrix
    instruction keeps and a block's sums of them are exact in fp32, whatever their order."""
    shape = (c.rows, c.n) if c.lay == "tn" else (c.groups, c.n, c.k) if c.nt else (c.groups, c.k, c.n)
    if c.in_type != E4M3:
        return random_operand(rng, (c.rows, c.k), c.in_type), random_operand(rng, shape, c.in_type, 0.05), None, None
    a, b = (from_f64(rng.choice(EXACT8, s) * rng.choice([-1.0, 1.0], s), E4M3) for s in ((c.rows, c.k), shape))
    sa = np.exp(rng.standard_normal((-(-c.k // 128), c.rows))).astype(np.float32)
    sb = np.exp(rng.standard_normal((c.groups, -(-shape[1] // 128), -(-shape[2] // 128)))).astype(np.float32)
    return a, b, sa, sb


def nan_next_door(c, a, b):
    """NaN where it must not come through -- rows of no group, the matrices of groups without rows, the first and last rows beside a group's --
    and one in each operand where it must."""
    nan = {BF16: 0x7FC0, F16: 0x7E00, E4M3: 0x7F}[c.in_type]
    lo, hi, sizes = c.offsets[0], c.offsets[-1], np.diff(c.offsets)
    a[:lo], a[hi:] = nan, nan
    if c.lay == "tn":
        b[:lo], b[hi:] = nan, nan
    else:
        b[sizes == 0] = nan
    first = int(np.argmax(sizes > 0))                       # a group with rows; its last row, and (rows) the last element of its matrix
    a[c.offsets[first + 1] - 1, c.k - 1] = nan
    if c.lay == "tn":
        b[c.offsets[first], c.n - 1] = nan
    else:
        b[first].reshape(-1)[-1] = nan


@pytest.mark.gpu
@pytest.mark.parametrize("c", CASES, ids=lambda c: c.label())
def test_tile(ctx, c):
    rng = np.random.default_rng(c.rows + c.k + c.n + c.groups)
    a, b, sa, sb = operands(c, rng)
    if c.odd:
        nan_next_door(c, a, b)
    c_type = mz.IN_F32 if c.out_type == mz.OUT_F32 else F16 if (c.in_type == F16 or c.out_type == mz.OUT_F16) else BF16
    shape = (c.groups, c.k, c.n) if c.lay == "tn" else (c.rows, c.n)
    old = to_f64(from_f64(rng.standard_normal(shape, dtype=np.float32), c_type), c_type)
    run = lambda: launch(ctx, a, b, c.offsets, c.axis, c.nt, c.in_type, c.out_type, c.alpha, c.beta, old, scale_a=sa, scale_b=sb, **c.strides())  # noqa: E731
    got = run()
    if c.split:                                             # the ranges are added in order, whoever is last
        assert np.array_equal(got, run(), equal_nan=True)
    lo, hi = c.offsets[0], c.offsets[-1]
    fa, fb = to_f64(a, c.in_type), to_f64(b, c.in_type)
    if c.lay == "tn":
        depth = np.diff(c.offsets)[:, None, None].astype(np.float64)
        sums, mag = reference(fa, fb, c.offsets, c.axis, False, c.in_type)
        check(got, sums, mag, depth, c.in_type, c.out_type, c.alpha, c.beta, old, None, c.label())
        return
    assert np.array_equal(got[:lo], old[:lo]) and np.array_equal(got[hi:], old[hi:]), "rows of no group were written"
    with np.errstate(invalid="ignore"):
        sums, mag = reference(fa, fb, c.offsets, c.axis, c.nt, c.in_type, sa, sb)
    # 8 bits: scale_a * scale_b, and for each block of K a product and a sum (check adds 4 roundings)
    coeff = (-(-c.k // 128) + 2) * 2.0 ** -24 if c.in_type == E4M3 else None
    check(got[lo:hi], sums[lo:hi], mag[lo:hi], c.k, c.in_type, c.out_type, c.alpha, c.beta, old[lo:hi], coeff, c.label())


@pytest.mark.gpu
@pytest.mark.parametrize("offsets", [(5, 3, 4000, 20), (-7, 10, 400, 4090), (0, 4090, 1 << 30, -(1 << 31))])
@pytest.mark.parametrize("in_type,lay,rows,k,n", [(BF16, "nt", 4100, 265, 4105), (E4M3, "nn", 4100, 265, 4105), (F16, "nn", 4100, 2051, 137), (BF16, "tn", 6001, 131, 77)])
def test_a_table_that_is_none_stays_inside_c(ctx, in_type, lay, rows, k, n, offsets):
    """256 x 256 tiles and K ranges on 128 x 128 (rows and depth): whatever the offsets, nothing outside C is written (launch checks that), rows that no pair
    of neighbouring offsets spans keep what they held, and the next call on the same workspace is right."""
    rng = np.random.default_rng(rows + n)
    c = Case("", in_type, lay, rows, k, n, tuple(offsets))
    a, b, sa, sb = operands(c, rng)
    shape = (3, k, n) if lay == "tn" else (rows, n)
    old = rng.integers(-8, 9, shape).astype(np.float64)
    got = launch(ctx, a, b, offsets, c.axis, c.nt, in_type, c_old=old, groups=3, scale_a=sa, scale_b=sb)
    assert np.isfinite(got).all()
    if lay != "tn":
        told = np.zeros(rows, dtype=bool)
        for lo, hi in zip(offsets, offsets[1:]):
            lo = min(max(lo, 0), rows)
            told[lo:min(max(hi, lo), rows)] = True
        assert np.array_equal(got[~told], old[~told])
    table = (0, rows // 3, rows // 3, rows)
    got = launch(ctx, a, b, table, c.axis, c.nt, in_type, mz.OUT_F32, c_old=old, scale_a=sa, scale_b=sb)
    with np.errstate(invalid="ignore"):
        sums, mag = reference(to_f64(a, in_type), to_f64(b, in_type), table, c.axis, c.nt, in_type, sa, sb)
    depth = np.diff(table)[:, None, None].astype(np.float64) if lay == "tn" else k
    check(got, sums, mag, depth, in_type, mz.OUT_F32, coeff=(-(-k // 128) + 2) * 2.0 ** -24 if in_type == E4M3 else None)
