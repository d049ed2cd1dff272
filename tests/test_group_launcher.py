"""The grouped products' entry point on a model of the HIP runtime (tests/cpu/fake_hip.cpp): what it allocates and launches, eagerly, while a
stream is captured, and where there is no memory.  No device."""
import ctypes as C
import os
import subprocess

import pytest

import maize_amd as mz
from maize_amd import _ffi
from test_launcher_host import CSRC, OTHER, ROOT, STREAM, Device, launches

m = mz.GlobalMatrix


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    so = tmp_path_factory.mktemp("model") / "libmodel.so"
    src = [os.path.join(CSRC, f) for f in ("shim.cpp", "dispatch.cpp", "forms.cpp", "groups.cpp", "group_api.cpp")]
    src += [os.path.join(ROOT, "tests", "cpu", f) for f in ("fake_hip.cpp", "fake_groups.cpp")]
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-Wl,--no-undefined", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-o", str(so)] + src, check=True)
    lib = C.CDLL(str(so))
    lib.fake_log.restype = lib.maize_hip_last_error.restype = C.c_char_p
    lib.fake_memory.argtypes = [C.c_size_t]
    lib.maize_hip_gemm_grouped.argtypes = [C.c_void_p, C.POINTER(_ffi.GroupedDescT), C.c_void_p]
    return lib


@pytest.fixture
def dev(model):
    d = Device(model)
    yield d
    d.close()


def rows_of(rows, groups, k, n, in_type=mz.IN_BF16, nt=True):
    scales = dict(scale_a=4096, scale_b=4096) if in_type == mz.IN_E4M3 else {}
    return mz.grouped_desc(m(16 << 32, rows, k), m(32 << 32, *((n, k) if nt else (k, n))), m(48 << 32, rows, n), 4096, groups,
                           layout=mz.LAYOUT_NT if nt else mz.LAYOUT_NN, in_type=in_type, **scales)


def depth_of(rows, groups, k, n):
    return mz.grouped_desc(m(16 << 32, rows, k), m(32 << 32, rows, n), m(48 << 32, k, n), 4096, groups, axis=mz.GROUP_DEPTH)


# 32 x 64, 32 x 128 and 128 x 128 tiles, rows and depth: each in K ranges
SPLIT = [rows_of(2, 8, 2048, 256), rows_of(40, 2, 4096, 128, nt=False), rows_of(16, 4, 4100, 200, mz.IN_E4M3, False), rows_of(4100, 2, 2050, 136),
         rows_of(4100, 2, 2050, 136, mz.IN_E4M3), depth_of(6001, 2, 131, 77)]


def run(dev, desc, stream=STREAM):
    return dev.lib.maize_hip_gemm_grouped(dev.ctx, C.byref(desc), stream), dev.events()


@pytest.mark.parametrize("desc", SPLIT)
def test_a_product_in_k_ranges_runs_as_planned(dev, desc):
    plan = mz.grouped_plan(desc)
    assert plan["ksplit"] > 1
    rc, ev = run(dev, desc)
    ran, = launches(ev)
    assert rc == 0 and (ran.kernel, ran.grid) == (plan["kernel"], plan["grid"][0])
    assert [e.rest[0] for e in ev if e.what == "malloc"] == [plan["workspace_bytes"] * 3 // 2]


@pytest.mark.parametrize("desc", SPLIT)
@pytest.mark.parametrize("captured", [False, True])
def test_a_product_runs_without_k_ranges_where_there_is_no_memory(dev, model, desc, captured):
    plan = mz.grouped_plan(desc)
    model.fake_memory(0)
    if captured:
        model.fake_capture(OTHER)
    rc, ev = run(dev, desc, OTHER)
    assert not captured or model.fake_end_capture(OTHER) == 1
    ran, = launches(ev)
    assert rc == 0 and ran.grid < plan["grid"][0] and ran.kernel.rsplit("_", 1)[0] == plan["kernel"].rsplit("_", 1)[0]
    assert model.hipGetLastError() == 0
    # with memory again: as planned
    model.fake_memory(1 << 40)
    rc, ev = run(dev, desc, OTHER)
    assert rc == 0 and launches(ev)[0].grid == plan["grid"][0]


def test_a_product_without_k_ranges_allocates_nothing(dev):
    desc = rows_of(4100, 2, 265, 4100)
    assert mz.grouped_plan(desc)["ksplit"] == 1
    rc, ev = run(dev, desc)
    assert rc == 0 and [e.what for e in ev] == ["launch"]
