"""Grouped products that reach each kernel by its tile: sizes, offsets and epilogues, each with the kernel that the plan has to name for it."""
from dataclasses import dataclass

import maize_amd as mz

BF16, F16, E4M3 = mz.IN_BF16, mz.IN_F16, mz.IN_E4M3
TAGS = {BF16: "bf16", F16: "f16", E4M3: "e4m3"}


@dataclass(frozen=True)
class Case:
    kernel: str
    in_type: int
    lay: str                       # nt, nn (rows) or tn (depth)
    rows: int
    k: int                         # depth: C is k x n for every group
    n: int
    offsets: tuple
    odd: bool = True               # odd leading dimensions, an element off the allocation, gaps between matrices
    out_type: int = mz.OUT_SAME
    alpha: float = 1.0
    beta: float = 0.0
    split: bool = False            # in K ranges

    @property
    def nt(self):
        return self.lay == "nt"

    @property
    def axis(self):
        return mz.GROUP_DEPTH if self.lay == "tn" else mz.GROUP_ROWS

    @property
    def groups(self):
        return len(self.offsets) - 1

    def strides(self):
        """Leading dimensions and offsets of `group_util.launch`."""
        if not self.odd:
            return {}
        ldb = self.n if self.lay != "nt" else self.k
        return dict(lda=self.k + 5, ldb=ldb + 3, ldc=self.n + 1, shift=1, gap=9)

    def desc(self):
        """The descriptor on addresses that nobody follows."""
        m, scales = mz.GlobalMatrix, dict(scale_a=4096, scale_b=4096) if self.in_type == E4M3 else {}
        s = {x: y for x, y in self.strides().items() if x.startswith("ld")}
        if self.lay == "tn":
            a, b, c = m(4096, self.rows, self.k), m(4096, self.rows, self.n), m(4096, self.k, self.n)
        else:
            a, b, c = m(4096, self.rows, self.k), m(4096, *((self.n, self.k) if self.nt else (self.k, self.n))), m(4096, self.rows, self.n)
        return mz.grouped_desc(a, b, c, 4096, self.groups, axis=self.axis, layout=mz.LAYOUT_NT if self.nt else mz.LAYOUT_NN, in_type=self.in_type,
                               out_type=self.out_type, alpha=self.alpha, beta=self.beta, **s, **scales)

    def label(self):
        more = [f"{self.rows}x{self.k}x{self.n}", f"{self.groups}g"] + (["odd"] if self.odd else []) + (["split"] if self.split else [])
        more += [{mz.OUT_F32: "f32", mz.OUT_F16: "f16"}.get(self.out_type, "same"), f"{self.alpha:g}", f"{self.beta:g}"]
        return self.kernel.replace("maize_group_", "") + "-" + "-".join(more)


def many(rows, groups):
    """Offsets of many groups: every fifth is empty, the others hold one to some two hundred rows; a few rows at both ends are nobody's."""
    sizes, left = [], rows - 5
    for g in range(groups):
        s = 0 if g % 5 == 3 else (g * 53) % 230 + 1
        sizes.append(min(s, left))
        left -= sizes[-1]
    at = [2]
    for s in sizes:
        at.append(at[-1] + s)
    return tuple(at)


# 1000, 0, 1124 and 1971 rows: 4 panels of 256 rows, the last more than half full; 4 and a half one; 8, more than half full.  Of 128 rows: 8 more than
# half full; 9 more than half full; 15 and a half one.
PANELS = (3, 1003, 1003, 2127, 4098)
EPILOGUES = [(mz.OUT_SAME, 1.0, 0.0), (mz.OUT_SAME, -2.0, 0.75), (mz.OUT_F32, 1.5, 1.0)]


def _rows(in_type, lay, tile, epilogues=EPILOGUES, **how):
    for out_type, alpha, beta in epilogues:
        yield Case(f"maize_group_{TAGS[in_type]}_{lay}_{tile}", in_type, lay, out_type=out_type, alpha=alpha, beta=beta, **how)


def cases():
    out = []
    for in_type in (BF16, F16, E4M3):
        half_c = [(mz.OUT_F16, 1.0, 0.0)] if in_type == E4M3 else []
        for lay in ("nt", "nn"):
            few = "32x128" if (in_type, lay) == (E4M3, "nn") else "32x64"
            # odd everything, and extents that divide
            out += _rows(in_type, lay, "256x256", rows=4100, k=265, n=4105, offsets=PANELS)
            out += _rows(in_type, lay, "256x256", half_c or EPILOGUES[:1], rows=4096, k=384, n=4112, offsets=(0, 1024, 2176, 2176, 4096), odd=False)
            # more than 64 groups, in the second sixty-four of them too
            out += _rows(in_type, lay, "128x128", rows=6725, k=201, n=201, offsets=many(6725, 70))
            out += _rows(in_type, lay, few, EPILOGUES[1:2], rows=300, k=201, n=201, offsets=many(300, 70))
            # K ranges
            out += _rows(in_type, lay, "128x128", [*EPILOGUES[:2], (mz.OUT_F32, 1.0, 1.0)], rows=4100, k=2051, n=137, offsets=PANELS, split=True)
            out += _rows(in_type, lay, few, EPILOGUES[2:], rows=40, k=4101, n=137, offsets=(1, 18, 18, 39), split=True)
    # what is left of a 16-byte chunk at the end of K and of N (8-bit operands: of a dword too), on the largest tiles
    for in_type, rests in ((BF16, range(1, 8)), (E4M3, (1, 2, 3, 6, 8, 13, 15))):
        for lay in ("nt", "nn"):
            for rest in rests:
                out += _rows(in_type, lay, "256x256", EPILOGUES[:1], rows=4100, k=(256 if in_type == BF16 else 384) + rest, n=4112 - rest, offsets=PANELS)
    for in_type in (BF16, F16):
        out += _rows(in_type, "tn", "256x256", rows=5000, k=1541, n=2311, offsets=(3, 1703, 1703, 4990))
        out += _rows(in_type, "tn", "256x256", EPILOGUES[:1], rows=4096, k=2048, n=2056, offsets=(0, 1024, 1024, 4096), odd=False)
        out += _rows(in_type, "tn", "128x128", rows=3000, k=131, n=77, offsets=many(3000, 100))
        out += _rows(in_type, "tn", "128x128", rows=6001, k=131, n=77, offsets=(3, 2000, 5990), split=True)
    return out


CASES = cases()
