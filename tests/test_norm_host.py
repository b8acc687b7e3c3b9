"""What norms, MXFP4 quantization and products over quantized activations launch and refuse, on the CPU (host_library.py)."""
import pytest

import host_library

PROGRAM = r"""
#include <cstdio>
#include "frink_amd/csrc/frk_norm.hpp"
#include "include/frink_hip.h"
static float room[64];  // (addresses only: nothing runs)
static void fill(frk_weights &w, int kind, size_t rows, size_t cols) {
    w.kind = kind, w.rows = rows, w.cols = cols, w.dev = (uint8_t *)room;
    if (kind == FRK_KIND_FP8_BLOCK) w.layout = frk::f8_layout(rows, cols, 1, &w.dev_bytes);
    else w.layout = frk::layout_for(kind, cols);
}
static void tell(int rc) {
    size_t most = 0;
    for (const auto &[grid, group] : HipStub::get().shapes) most = std::max(most, (size_t)grid.x * group.x);
    HipStub::get().shapes.clear();
    printf("%d %zu %s | %s\n", rc, most, HipStub::get().take().c_str(), frk_hip_last_error());
}
int main() {  // a call a line; its status, the most threads of a grid's rows, the kernels it launched and its error
    char call[32];
    while (scanf("%31s", call) == 1) {
        const std::string name = call;
        HipStub::get().memory = false;
        if (name == "gemm" || name == "acts") {  // rows, columns, batch
            size_t rows, cols, batch;
            if (scanf("%zu %zu %zu", &rows, &cols, &batch) != 3) return 1;
            frk_weights w;
            fill(w, FRK_KIND_MXFP4, rows, cols);
            if (name == "gemm") {
                tell(frk_hip_gemm_mxfp4_dev(&w, room, batch, room, nullptr));
            } else {
                frk_batch_acts *acts = nullptr;
                int rc = frk_hip_batch_acts_create_form(batch, cols, FRK_ACTS_MXFP4, &acts);
                if (!rc) rc = frk_hip_quantize_batch_acts_dev(acts, room, batch, nullptr);
                if (!rc) rc = frk_hip_gemm_acts_dev(&w, acts, room, nullptr);
                tell(rc);
                if (acts) frk_hip_batch_acts_release(acts);
            }
        } else if (name == "norm") {  // batch, columns, form (-1: plain)
            size_t batch, cols;
            int form;
            if (scanf("%zu %zu %d", &batch, &cols, &form) != 3) return 1;
            frk_batch_acts *acts = nullptr;
            int rc = form < 0 ? 0 : frk_hip_batch_acts_create_form(batch, cols, form, &acts);
            if (!rc) rc = frk_hip_rms_norm_dev(FRK_TYPE_BF16, room, room + 8, FRK_TYPE_F32, room, 1e-5, batch, cols, room + 16, form < 0 ? room + 32 : nullptr, acts, nullptr);
            tell(rc);
            if (acts) frk_hip_batch_acts_release(acts);
        } else if (name == "blocks") {
            size_t n;
            if (scanf("%zu", &n) != 1) return 1;
            tell(frk_hip_quantize_mxfp4_dev(FRK_TYPE_F16, room, n, (uint8_t *)room, nullptr));
            tell(frk_hip_dequantize_mxfp4_dev((uint8_t *)room, n, room, nullptr));
        } else if (name == "elsewhere") {  // objects of device 0, a call on device 1: the first line on device 0
            frk_weights w4, w8;
            fill(w4, FRK_KIND_MXFP4, 64, 128), fill(w8, FRK_KIND_FP8_BLOCK, 64, 128);
            frk_batch_acts *a4 = nullptr, *a8 = nullptr;
            frk_hip_batch_acts_create_form(4, 128, FRK_ACTS_MXFP4, &a4), frk_hip_batch_acts_create_form(4, 128, FRK_ACTS_FP8, &a8);
            frk_hip_quantize_batch_acts_dev(a4, room, 2, nullptr), frk_hip_quantize_batch_acts_dev(a8, room, 2, nullptr);
            tell(frk_hip_gemm_mxfp4_dev(&w4, room, 2, room, nullptr));
            HipStub::get().device = 1;
            tell(frk_hip_gemm_mxfp4_dev(&w4, room, 2, room, nullptr));
            tell(frk_hip_gemm_mxfp4_dev(&w4, room, 200, room, nullptr));
            for (frk_batch_acts *a : {a4, a8}) {
                tell(frk_hip_gemm_acts_dev(a == a4 ? &w4 : &w8, a, room, nullptr));
                tell(frk_hip_batch_acts_values_dev(a, room, nullptr));
                tell(frk_hip_rms_norm_dev(FRK_TYPE_F32, room, nullptr, 0, nullptr, 1e-5, 2, 128, nullptr, nullptr, a, nullptr));
                tell(frk_hip_quantize_batch_acts_dev(a, room, 2, nullptr));
            }
            HipStub::get().device = 0;
            w4.device = 1, w8.device = 1;  // the other way about
            tell(frk_hip_gemm_acts_dev(&w4, a4, room, nullptr));
            tell(frk_hip_gemm_acts_dev(&w8, a8, room, nullptr));
            frk_hip_batch_acts_release(a4), frk_hip_batch_acts_release(a8);
        } else if (name == "kernels") {  // all there are, and those of its calls
            for (const auto &[handle, kernel] : HipStub::get().names)
                for (const char *part : {"mx4_", "rms_norm", "mxfp4_kernel", "acts_values"})
                    if (kernel.find(part) != std::string::npos) {
                        HipStub::get().launched.push_back(kernel);
                        break;
                    }
            tell(0);
            for (const float *x : {room, room + 1})
                for (int type : {(int)FRK_TYPE_F32, (int)FRK_TYPE_BF16, (int)FRK_TYPE_F16}) {
                    const void *p = type == FRK_TYPE_F32 ? (const void *)x : (const void *)((const uint16_t *)room + (x - room));
                    frk_hip_quantize_mxfp4_dev(type, p, 64, (uint8_t *)room, nullptr);
                    frk_hip_dequantize_mxfp4_dev((uint8_t *)room, 64, (float *)x, nullptr);
                    for (size_t cols : {256, 4096, 8192, 32768})
                        for (size_t batch : {1, 20, 400})
                            for (int form : {-1, (int)FRK_ACTS_Q8_K, (int)FRK_ACTS_FP8, (int)FRK_ACTS_MXFP4}) {
                                frk_batch_acts *acts = nullptr;
                                if (form >= 0) frk_hip_batch_acts_create_form(batch, cols, form, &acts);
                                frk_hip_rms_norm_dev(type, p, nullptr, 0, nullptr, 0.0, batch, cols, nullptr, form < 0 ? (void *)p : nullptr, acts, nullptr);
                                if (acts) frk_hip_batch_acts_values_dev(acts, (float *)x, nullptr), frk_hip_batch_acts_release(acts);
                            }
                }
            for (const float *x : {room, room + 1})
                for (size_t rows : {64, 4096, 7168, 14336, 32000})
                    for (size_t cols : {512, 1024, 4096, 16384})
                        for (size_t batch : {1, 4, 8, 20, 40, 64, 100, 300, 1000, 4000}) {
                            frk_weights w;
                            fill(w, FRK_KIND_MXFP4, rows, cols);
                            frk_hip_gemm_mxfp4_dev(&w, x, batch, room, nullptr);
                        }
            tell(0);
        } else {
            return 1;
        }
        HipStub::get().memory = true;
    }
}
"""


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    binary = host_library.build(tmp_path_factory.mktemp("norm"), PROGRAM)

    def of(*calls):
        out = []
        for line in host_library.run(binary, "".join(c + "\n" for c in calls)).splitlines():
            head, error = line.split(" | ") if " | " in line else (line.rstrip(" |"), "")
            rc, most, *names = head.split()
            out.append((int(rc), int(most), names, error))
        return out

    return of


def test_no_kernel_is_built_that_no_call_reaches(said):
    (_, _, built, _), (_, _, launched, _) = said("kernels")
    assert len(built) > 50 and set(built) <= set(launched), set(built) - set(launched)


def test_another_device_is_refused(said):
    here, *elsewhere = said("elsewhere")
    assert here[0] == 0 and here[2] != ["-"] and len(elsewhere) == 12
    for call, (rc, _, names, error) in enumerate(elsewhere):
        assert rc == -4 and names == ["-"] and "device" in error, (call, rc, names, error)


@pytest.mark.parametrize("call", ["norm %d 64 -1" % (1 << 30), "norm 3 %d -1" % (1 << 23), "norm %d 256 0" % (1 << 25), "norm %d 4 1" % (1 << 28), "norm %d 32 2" % (1 << 30),
                                  "gemm 64 32 %d" % (1 << 28), "gemm %d 32 1" % ((1 << 27) - 16), "gemm %d 32 16" % ((1 << 27) - 16), "gemm 64 %d 20" % (1 << 23), "gemm 64 %d 4" % (1 << 23), "acts 4096 4096 %d" % (1 << 22),
                                  "gemm 1 32 %d" % (1 << 30)])
def test_what_grids_hold_is_launched(said, call):
    (rc, most, names, error), = said(call)
    assert rc == 0 and names != ["-"] and 0 < most < 1 << 32, (rc, most, error)


@pytest.mark.parametrize("call", ["norm %d 64 -1" % ((1 << 30) + 1), "norm 1 %d -1" % ((1 << 23) + 1), "norm 4 300 0", "norm 4 48 2", "gemm 64 %d 1" % ((1 << 23) + 32),
                                  "gemm 64 32 %d" % ((1 << 30) + 1), "gemm %d 32 %d" % ((1 << 27) - 16, 1 << 30), "acts %d 32 %d" % ((1 << 27) - 16, 1 << 30), "blocks 0", "blocks 48"])
def test_what_no_launch_holds_is_refused_before_the_first(said, call):
    for rc, _, names, error in said(call):
        assert rc == -3 and not [n for n in names if "quantize" not in n and n != "-"] and error, (rc, names)
        assert call.startswith("acts") or names == ["-"], names


def test_what_each_call_launches(said):
    """One launch where the workgroups quantize for themselves, a quantization in front of more tokens, a sum behind shares of the columns."""
    one, few, tile, shares = said("gemm 4096 4096 1", "gemm 4096 4096 8", "gemm 4096 4096 4096", "gemm 4096 14336 64")
    assert [n.split("<")[0] for n in one[2]] == ["mx4_rows_kernel"] and [n.split("<")[0] for n in few[2]] == ["mx4_quantize_kernel", "mx4_rows_kernel"]
    assert [n.split("<")[0] for n in tile[2]] == ["mx4_quantize_kernel", "mx4_tile_kernel"]
    assert [n.split("<")[0] for n in shares[2]] == ["mx4_quantize_kernel", "mx4_tile_kernel", "sum_parts_kernel"]
    for form in (-1, 0, 1, 2):
        assert [n.split("<")[0] for n in said("norm 100 1024 %d" % form)[0][2]] == ["rms_norm_kernel"]


@pytest.mark.parametrize("name", ["frk_mx4.hip", "frk_mx4_tile.hip", "frk_norm.hip"])
def test_compiled_kernels(tmp_path, name):
    """No MFMA result read across a branch before its time, no LDS read used before its wait, and nothing spilled."""
    import os
    import re
    import subprocess

    import isa_mfma_lint
    import isa_wait_lint
    from frink_amd import build as fb
    out = tmp_path / "kernels.s"
    r = subprocess.run([fb.hipcc()] + fb.HIPCC_FLAGS + ["-x", "hip", "--cuda-device-only", "-S", os.path.join(fb.CSRC, name), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    asm = out.read_text()
    assert ("v_mfma" in asm) == ("mx4" in name) and isa_mfma_lint.violations(asm) == []
    # (only these wait by hand; unaligned activations change the compiler's own loads alone)
    for k in [k for k in isa_wait_lint.kernels(asm) if ("rows_kernel" in k and "ELb1ELb0E" not in k) or "tile_kernel" in k]:
        assert isa_wait_lint.violations(asm, k) == [], k
    scratch = re.findall(r"\.private_segment_fixed_size: (\d+)", asm)
    assert len(scratch) > 3 and set(scratch) == {"0"}, scratch
