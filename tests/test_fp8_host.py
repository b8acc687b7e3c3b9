"""What calls over weights in 8-bit floating point launch and refuse, on the CPU (host_library.py)."""
import pytest

import host_library
import oracle as fo

FP8 = 256
PROGRAM = r"""
#include <cstdio>
#include "frink_amd/csrc/frk_f8.hpp"
#include "include/frink_hip.h"
static float room[64];  // (addresses only: nothing runs)
static void fill(frk_weights &w, int kind, size_t rows, size_t cols, size_t matrices = 1) {
    w.kind = kind, w.rows = rows, w.cols = cols, w.matrices = matrices, w.dev = (uint8_t *)room;
    if (kind == FRK_KIND_FP8_BLOCK) w.layout = frk::f8_layout(rows, cols, matrices, &w.dev_bytes);
    else w.layout = frk::layout_for(kind, cols);
}
static void tell(int rc) {
    printf("%d %s | %s\n", rc, HipStub::get().take().c_str(), frk_hip_last_error());
}
int main() {  // a call a line; its status, the kernels it launched and its error
    char call[32];
    while (scanf("%31s", call) == 1) {
        const std::string name = call;
        if (name == "multi" || name == "ffn") {  // columns, number, kinds
            size_t cols, n;
            if (scanf("%zu %zu", &cols, &n) != 2) return 1;
            std::vector<frk_weights> w(n);
            std::vector<const frk_weights *> ws(n);
            std::vector<float *> ys(n, room);
            for (size_t i = 0; i < n; i++) {
                int kind;
                if (scanf("%d", &kind) != 1) return 1;
                fill(w[i], kind, i < 2 ? 64 : 32, name == "ffn" && i == 2 ? 64 : cols), ws[i] = &w[i];
            }
            tell(name == "ffn" ? frk_hip_ffn_swiglu_dev(ws[0], ws[1], ws[2], room, room, nullptr) : frk_hip_gemv_multi_dev(ws.data(), n, room, ys.data(), nullptr));
        } else if (name == "route") {  // tokens, experts, k; the tokens that its grids hold, and the most threads of one
            size_t batch, n, k;
            if (scanf("%zu %zu %zu", &batch, &n, &k) != 3) return 1;
            frk_route_rule rule{};
            rule.groups = rule.top_groups = rule.group_best = 1;
            const size_t before = HipStub::get().shapes.size();
            const int rc = frk_hip_route_dev(room, batch, n, k, &rule, (int32_t *)room, room, nullptr);
            size_t tokens = 0, most = 0;
            for (size_t i = before; i < HipStub::get().shapes.size(); i++) {
                const auto [grid, group] = HipStub::get().shapes[i];
                tokens += (size_t)grid.x * (group.x / 64), most = std::max(most, (size_t)grid.x * group.x);
            }
            HipStub::get().take();
            printf("%d %zu %zu | %s\n", rc, tokens, most, frk_hip_last_error());
        } else if (name == "kernels") {  // all there are of this kind, and those of its calls at two alignments of x
            for (const auto &[handle, kernel] : HipStub::get().names)
                if (kernel.compare(0, 3, "f8_") == 0 || kernel.find("_f8_") != std::string::npos) HipStub::get().launched.push_back(kernel);
            tell(0);
            std::string all;
            HipStub::get().memory = false;
            for (const float *x : {room, room + 1})
                for (size_t cols : {256, 1028, 8192, 70000}) {
                    frk_weights w, up, down, *fresh = nullptr;
                    fill(w, FRK_KIND_FP8_BLOCK, 4 * 4096, cols, 4), fill(up, FRK_KIND_FP8_BLOCK, 4 * 4096, cols, 4), fill(down, FRK_KIND_FP8_BLOCK, 4 * cols, 4096, 4);
                    for (size_t batch : {1, 3, 8, 16, 24, 40, 64, 100, 300, 4000}) {
                        frk_hip_gemm_dev(&w, x, batch, room, nullptr);
                        frk_hip_gemm_grouped_dev(&w, 4, (int32_t *)room, nullptr, x, batch, batch, room, nullptr);
                        frk_hip_moe_ffn_dev(&w, &up, &down, 4, x, batch, (int32_t *)room, room, 2, room, nullptr);
                    }
                    frk_weights odd, back;
                    fill(odd, FRK_KIND_FP8_BLOCK, 4 * 130, cols, 4), fill(back, FRK_KIND_FP8_BLOCK, 4 * cols, 130, 4);
                    frk_hip_moe_ffn_dev(&odd, &odd, &back, 4, x, 1, (int32_t *)room, room, 2, room, nullptr);
                    frk_weights one;
                    fill(one, FRK_KIND_FP8_BLOCK, 64, cols);
                    for (size_t batch : {20, 40, 64}) frk_hip_gemm_dev(&one, x, batch, room, nullptr);
                    frk_hip_dequant_dev(&w, room, nullptr);
                    frk_hip_weights_from_device_fp8((uint8_t *)room, room, 4, cols, 1, nullptr, &fresh);
                }
            HipStub::get().memory = true;
            tell(0);
        } else if (name == "rows") {  // the largest grid of a one-token product, or what registration says
            size_t rows, matrices;
            if (scanf("%zu %zu", &rows, &matrices) != 2) return 1;
            frk_weights *handle = nullptr;
            HipStub::get().memory = false;
            int rc = frk_hip_weights_from_device_fp8((uint8_t *)room, room, rows, 1, matrices, nullptr, &handle);
            size_t most = 0;
            const std::string error = frk_hip_last_error();
            if (!rc) {
                const size_t before = HipStub::get().shapes.size();
                rc = frk_hip_gemv_dev(handle, room, room, FRK_ACT_F32, nullptr);
                for (size_t i = before; i < HipStub::get().shapes.size(); i++) most = std::max(most, (size_t)HipStub::get().shapes[i].first.x * HipStub::get().shapes[i].second.x);
                frk_hip_weights_release(handle);
            }
            HipStub::get().memory = true;
            HipStub::get().take();
            printf("%d %zu | %s\n", rc, most, error.c_str());
        } else if (name == "gemm" || name == "grouped" || name == "moe") {  // rows, columns, matrices (experts), rows of x (tokens), pairs (top k)
            size_t rows, cols, matrices, x_rows, n;
            if (scanf("%zu %zu %zu %zu %zu", &rows, &cols, &matrices, &x_rows, &n) != 5) return 1;
            frk_weights w, down;
            fill(w, FRK_KIND_FP8_BLOCK, rows * matrices, cols, matrices), fill(down, FRK_KIND_FP8_BLOCK, cols * matrices, rows, matrices);
            int32_t *const ids = (int32_t *)room;
            HipStub::get().memory = false;
            const size_t before = HipStub::get().shapes.size();
            int rc;
            if (name == "gemm") rc = frk_hip_gemm_dev(&w, room, x_rows, room, nullptr);
            else if (name == "grouped") rc = frk_hip_gemm_grouped_dev(&w, matrices, ids, ids, room, x_rows, n, room, nullptr);
            else rc = frk_hip_moe_ffn_dev(&w, &w, &down, matrices, room, x_rows, ids, room, n, room, nullptr);
            HipStub::get().memory = true;
            size_t most = 0;
            for (size_t i = before; i < HipStub::get().shapes.size(); i++) most = std::max(most, (size_t)HipStub::get().shapes[i].first.x * HipStub::get().shapes[i].second.x);
            HipStub::get().take();
            printf("%d %zu %zu | %s\n", rc, HipStub::get().shapes.size() - before, most, frk_hip_last_error());
        } else if (name == "elsewhere") {  // a matrix of device 1, device 0 the current one: every entry point that takes it
            static frk_weights w, q;
            fill(w, FRK_KIND_FP8_BLOCK, 256, 256, 2), fill(q, FRK_KIND_Q4_K, 256, 256);
            w.device = 1;
            int32_t ids[4] = {0, 1, 0, 0};
            float out[1024];
            const frk_weights *const pair[2] = {&q, &w};
            float *const ys[2] = {room, room};
            frk_weights *fresh = nullptr;
            tell(frk_hip_weights_register_fp8((const uint8_t *)out, out, 16, 16, 1, &fresh));
            tell(frk_hip_gemv_dev(&w, room, room, FRK_ACT_F32, nullptr));
            tell(frk_hip_gemm_dev(&w, room, 40, room, nullptr));
            tell(frk_hip_gemm_noalloc_dev(&w, room, 40, room, nullptr));
            tell(frk_hip_gemm_pair_dev(&w, &w, room, 40, room, room, nullptr));
            tell(frk_hip_gemv_multi_dev(pair, 2, room, ys, nullptr));
            tell(frk_hip_ffn_swiglu_dev(&w, &w, &w, room, room, nullptr));
            tell(frk_hip_gemm_grouped_dev(&w, 2, ids, nullptr, room, 4, 4, room, nullptr));
            static frk_weights e[3];
            for (frk_weights &m : e) fill(m, FRK_KIND_FP8_BLOCK, 256, 128, 2);
            e[2].device = 1;
            tell(frk_hip_moe_ffn_dev(&e[0], &e[1], &e[2], 2, room, 2, ids, room, 1, room, nullptr));
            tell(frk_hip_dequant_dev(&w, room, nullptr));
            tell(frk_hip_get_rows_dev(&w, ids, 2, room, nullptr));
            tell(frk_hip_get_rows(&w, ids, 2, out));
            HipStub::get().device = 1;  // the host-buffer entry points' stream is device 0's
            tell(frk_hip_get_rows(&w, ids, 2, out));
            tell(frk_hip_weights_register_fp8((const uint8_t *)out, out, 16, 16, 1, &fresh));
            HipStub::get().device = 0;
        } else {
            return 1;
        }
    }
}
"""


@pytest.fixture(scope="module")
def said(tmp_path_factory):
    binary = host_library.build(tmp_path_factory.mktemp("fp8"), PROGRAM)

    def of(*calls, lines=None):
        count, lines = lines or len(calls), host_library.run(binary, "".join(c + "\n" for c in calls)).splitlines()
        assert len(lines) == count
        split = [(line.split(None, 1)[0], line.split(None, 1)[1].split(" | ") + [""]) for line in lines]
        return [(int(rc), names.split(), error) for rc, (names, error, *_) in split]

    return of


@pytest.mark.parametrize("cols", [28672, 32768])
def test_quantized_rows_of_one_kind_stay_until_their_products(said, cols):
    """Scratch memory that holds Q8_K activations for several products is not written in between."""
    kinds = [[FP8, fo.Q4_K], [fo.Q4_K, FP8, fo.Q6_K], [FP8, fo.Q5_K, fo.Q4_K, FP8], [fo.Q6_K, fo.Q4_K, FP8]]
    calls = ["multi %d %d %s" % (cols, len(k), " ".join(map(str, k))) for k in kinds]
    calls += ["ffn %d 3 %d %d %d" % (cols, a, b, FP8) for a, b in ((FP8, fo.Q4_K), (fo.Q4_K, FP8))]
    for call, (rc, names, error) in zip(calls, said(*calls)):
        assert rc == 0, error
        first = [i for i, n in enumerate(names) if n.startswith("quantize_q8_k")]
        last = max(i for i, n in enumerate(names) if n.startswith("gemv"))
        assert len(first) == 1 and first[0] < last, names
        assert not [n for n in names[first[0]:last] if n.startswith("f8_quantize")], (call, names)


def test_a_matrix_of_another_device_is_refused(said):
    here, *elsewhere = said("elsewhere", lines=14)
    assert here[0] == 0
    for call, (rc, names, error) in enumerate(elsewhere):
        assert rc == -4 and names == ["-"] and "device" in error, (call, rc, names, error)


@pytest.mark.parametrize("batch", [1, 1 << 25, (1 << 25) + 1, (1 << 26) - 4, 1 << 26, (1 << 27) + 5, 1 << 30])
@pytest.mark.parametrize("experts", [1, 70, 1000])
def test_routes_of_any_batch_fit_their_grids(said, batch, experts):
    (rc, (tokens, most), error), = said("route %d %d 1" % (batch, experts))
    assert rc == 0, error
    assert batch <= int(tokens) < batch + 4 * 32 and int(most) < 1 << 32


@pytest.mark.parametrize("rows,matrices", [(1 << 27, 1), ((1 << 27) - 15, 1), (1 << 29, 4), (0x7fffff00, 1)])
def test_matrices_of_more_rows_than_a_grid_holds_are_refused(said, rows, matrices):
    (rc, _, error), = said("rows %d %d" % (rows, matrices))
    assert rc == -3 and "too large" in error


@pytest.mark.parametrize("rows,matrices", [((1 << 27) - 16, 1), (4 * ((1 << 27) - 16), 4), (17, 1)])
def test_the_most_rows_fit_a_grid(said, rows, matrices):
    (rc, (most,), error), = said("rows %d %d" % (rows, matrices))
    assert rc == 0 and 0 < int(most) < 1 << 32, error


@pytest.mark.parametrize("call,needle", [
    ("grouped 1 64 1024 4 %d" % (1 << 30), "grid"), ("grouped 16 4096 8 %d 64" % (1 << 19), "4 GiB"), ("grouped 16 %d 8 %d 600" % (1 << 23, 500), "4 GiB"),
    ("moe 8 4096 16 %d 4" % (1 << 19), "4 GiB"), ("moe 8 4 16 %d 4" % (1 << 24), "2.24 - 1"), ("moe 8 4 16 %d 64" % ((1 << 24) - 1), "top-k|experts"),
    ("moe 300 4 1024 %d 64" % ((1 << 24) - 1), "grid|4 GiB"), ("gemm 1000 8 1 %d 0" % (1 << 30), "grid")])
def test_what_no_launch_can_hold_is_refused_before_the_first(said, call, needle):
    import re
    (rc, (launches, _), error), = said(call)
    assert rc == -3 and launches == "0" and re.search(needle, error), error


@pytest.mark.parametrize("call", ["grouped 1 64 1024 4 %d" % (1 << 29), "grouped 16 4096 8 %d 64" % ((1 << 19) - 1), "grouped 16 4096 64 %d 20" % (1 << 20),
                                  "moe 8 4096 16 %d 4" % ((1 << 19) - 1), "moe 8 4 16 %d 4" % ((1 << 24) - 1), "gemm 1000 8 1 %d 0" % (1 << 22)])
def test_what_a_launch_just_holds_is_launched(said, call):
    (rc, (launches, most), error), = said(call)
    assert rc == 0 and int(launches) and int(most) < 1 << 32, error


def test_no_kernel_is_built_that_no_call_reaches(said):
    (_, built, _), (_, launched, _) = said("kernels", lines=2)
    assert set(built) <= set(launched), set(built) - set(launched)
    # <wavefronts, tiles of tokens, blocks ahead, quantizes itself, mode, how it then reads x>
    rows = [n[len("f8_rows_kernel<"):-1].split(",") for n in built if n.startswith("f8_rows_kernel")]
    assert rows and all(r[5] == "false" for r in rows if r[3] == "false")
