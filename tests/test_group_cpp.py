"""include/maize_tile.hpp's grouped products and quantiser, compiled and run on the model of the HIP runtime: the descriptors are those of the Python face,
what is launched is what the plan names, and what is refused throws."""
import ctypes as C
import os
import subprocess

import maize_amd as mz
from maize_amd import _ffi
from test_launcher_host import CSRC, ROOT

PROGRAM = r'''
#include <cstdio>
#include "maize_tile.hpp"
using namespace maize;
extern "C" const char* fake_log();
extern "C" void fake_memory(size_t);
template <class T> static void bytes(const T& d) { for (size_t i = 0; i < sizeof d; ++i) std::printf("%02x", ((const unsigned char*)&d)[i]); std::printf("\n"); }
int main() {
    fake_memory((size_t)1 << 40);
    Ctx ctx(0);
    BF16* const p = (BF16*)0x100000000;
    const Matrix x = Matrix::make(p, 100, 200), w = Matrix::make(p, 200, 300), wt = Matrix::make(p, 300, 200), y = Matrix::make(p, 100, 300);
    const int32_t* const offsets = (const int32_t*)0x400000000;
    const float *sa = (const float*)0x500000000, *sb = (const float*)0x600000000;
    maize_gemm_grouped_desc_t shared = grouped_desc(x, w, y, offsets, 5);
    shared.stride = 0;
    const maize_gemm_grouped_desc_t all[] = {grouped_desc(x, w, y, offsets, 5), grouped_desc(x, wt, y, offsets, 5, MAIZE_GROUP_ROWS, Layout::NT, MAIZE_IN_F16, MAIZE_OUT_F32),
                                             grouped_desc(x, y, w, offsets, 5, MAIZE_GROUP_DEPTH), with_block_scales(grouped_desc(x, w, y, offsets, 5), sa, sb),
                                             with_block_scales(shared, sa, sb)};
    for (const auto& d : all) { bytes(d); gemm_grouped(ctx, d, (void*)0x1000); std::printf("%s\n", grouped_plan(d).kernel); }
    maize_quantize_desc_t q = quantize_desc(x, x, (float*)sa, 128, MAIZE_IN_F16);
    bytes(q);
    quantize_blocks(ctx, q);
    int thrown = 0;
    try { gemm_grouped(ctx, grouped_desc(x, wt, y, offsets, 5)); } catch (const Error& e) { thrown += e.code == MAIZE_ERR_SHAPE; }
    try { q.block_rows = 2; quantize_blocks(ctx, q); } catch (const Error& e) { thrown += e.code == MAIZE_ERR_ARG; }
    std::printf("%d\n%s", thrown, fake_log());
}
'''


def test_grouped_products_in_cpp(tmp_path):
    src, exe = tmp_path / "grouped.cpp", tmp_path / "grouped"
    src.write_text(PROGRAM)
    cpp = [os.path.join(CSRC, f) for f in ("shim.cpp", "dispatch.cpp", "forms.cpp", "groups.cpp", "group_api.cpp")]
    cpp += [os.path.join(ROOT, "tests", "cpu", f) for f in ("fake_hip.cpp", "fake_groups.cpp")]
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-o", str(exe), str(src)] + cpp, check=True)
    lines = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    m, p, how = (lambda r, c: mz.GlobalMatrix(1 << 32, r, c)), 4 << 32, dict(in_type=mz.IN_E4M3, scale_a=5 << 32, scale_b=6 << 32)
    x, w, wt, y = m(100, 200), m(200, 300), m(300, 200), m(100, 300)
    want = [mz.grouped_desc(x, w, y, p, 5), mz.grouped_desc(x, wt, y, p, 5, layout=mz.LAYOUT_NT, in_type=mz.IN_F16, out_type=mz.OUT_F32),
            mz.grouped_desc(x, y, w, p, 5, axis=mz.GROUP_DEPTH), mz.grouped_desc(x, w, y, p, 5, **how), mz.grouped_desc(x, w, y, p, 5, stride=0, **how)]
    quant = mz.quantize_desc(x, x, 5 << 32, 128, mz.IN_F16)

    def fields(d):
        return {f: (v.ptr, v.nrows, v.ncols) if isinstance(v := getattr(d, f), _ffi.MatrixT) else v for f, _ in d._fields_ if f != "_pad"}

    def read(line, kind):                                    # (the Python structures have room to spare at their end)
        raw = bytes.fromhex(line)
        return kind.from_buffer_copy(raw + bytes(max(0, C.sizeof(kind) - len(raw))))

    for d, line, kernel in zip(want, lines[0:10:2], lines[1:10:2]):
        assert fields(read(line, _ffi.GroupedDescT)) == fields(d)
        assert kernel == mz.grouped_plan(d)["kernel"]
    assert fields(read(lines[10], _ffi.QuantizeDescT)) == fields(quant)
    assert lines[11] == "2"
    ran = [x.split()[2] for x in lines[12:] if x.startswith("launch")]
    assert ran == lines[1:10:2] + ["maize_quantize_f16_blocks"]
