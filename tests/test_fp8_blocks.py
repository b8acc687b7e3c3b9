"""Products with weights in 8-bit floating point, a scale for each block of 128 x 128: against the definition in 64 bits at the
edges of blocks, strips and tiles, dense and grouped; values that are no numbers; refusals."""
import ctypes as C

import numpy as np
import pytest

import fp8_plain as plain
from test_gpu_parity import fa, to_dev  # noqa: F401 (fa: the module's fixture)


def _resident(fa, codes, scales):
    m, rows, cols = codes.shape
    return fa.Weights.from_device_fp8(to_dev(codes), to_dev(scales), m * rows, cols, matrices=m)


def _activations(rng, rows, cols):
    """Rows of different sizes, a few large channels, some zeros."""
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-6, 7, (rows, 1))
    x[:, rng.integers(0, cols, max(1, cols // 64))] *= 30
    x[rng.random((rows, cols)) < 0.05] = 0
    return x.astype(np.float32)


SHAPES = [(1, 1, 1), (15, 127, 2), (16, 128, 1), (17, 129, 3), (129, 255, 16), (128, 640, 17), (300, 1000, 33), (64, 96, 64),
          (257, 2880, 65), (1000, 513, 130), (144, 14336, 5), (576, 2304, 9), (33, 1156, 200), (272, 384, 257), (512, 1152, 300),
          (31, 4100, 1), (768, 2048, 31), (2880, 160, 97), (40, 28672, 1), (33, 32768, 1), (20, 7168, 4), (20, 7300, 4),
          (100, 2500, 8), (4096, 130, 7), (4112, 130, 7), (50, 4096, 5), (50, 4100, 5), (60, 96, 9), (17, 70000, 3), (9, 66000, 20), (9, 132000, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,batch", SHAPES)
def test_product_against_64_bits(fa, rows, cols, batch):
    print("fp8 product", rows, cols, batch, flush=True)
    rng = np.random.default_rng(rows * 7 + cols * 3 + batch)
    codes, scales = plain.random_matrix(rng, rows, cols)
    w = _resident(fa, codes, scales)
    x = _activations(rng, batch, cols)
    want, room = plain.product(codes[0], scales[0], x)
    got = w.gemm(to_dev(x)).cpu().numpy()
    assert (np.abs(got - want) <= room).all()
    assert np.array_equal(got, w.gemm(to_dev(x)).cpu().numpy())  # the same bits again
    assert (w.rows, w.cols, w.kind) == (rows, cols, fa.FP8_BLOCK)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 3, 7, 16, 40, 70, 300])
def test_activations_are_rounded_once_to_the_nearest(fa, batch):
    """A weight row that picks one column returns that activation as quantized, bit for bit: halves between codes, the
    largest value just at and above 448 times a power of two, subnormal codes, the smallest and largest floats."""
    cols = 384
    rng = np.random.default_rng(batch)
    x = (rng.standard_normal((batch, cols)) * 2.0 ** rng.integers(-20, 20, (batch, 1))).astype(np.float32)
    half = (plain.VALUES[:126] + plain.VALUES[1:127]) / 2  # every border between two codes
    for r in range(0, batch, 3):
        scale = 2.0 ** int(rng.integers(-110, 100))
        x[r, :126], x[r, 127] = half * scale, 448 * scale
        x[r, 128:254], x[r, 255] = -np.nextafter(half.astype(np.float32), np.float32(1e9)) * scale, 448 * scale
        x[r, 256:] = 0
        x[r, 300:305] = np.array([1, -2, 3, 5, 449]) * 2.0 ** -149
    for r in range(1, batch, 3):
        x[r, :128] = np.float32(448) * 2.0 ** int(rng.integers(-130, 119)) * rng.choice([1, 0.5, 0.25, -1], 128)
        x[r, 128] = np.nextafter(np.float32(448), np.float32(449)) * np.float32(2.0 ** 10)
        x[r, 256] = np.finfo(np.float32).max
    codes = np.zeros((1, cols, cols), np.uint8)
    codes[0, np.arange(cols), np.arange(cols)] = 0x38  # 1.0
    w = _resident(fa, codes, np.ones((1, 3, 3), np.float32))
    got = w.gemm(to_dev(x)).cpu().numpy()
    assert np.array_equal(got, plain.quantize(x).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 20, 150])
def test_every_code_and_scale(fa, batch):
    """All 256 codes under scales of any size come back by the dequantizer, the row gather and a product with one column."""
    rng = np.random.default_rng(3)
    codes = rng.permutation(np.arange(260 * 300, dtype=np.uint32)).astype(np.uint8).reshape(1, 260, 300)
    scales = (2.0 ** rng.uniform(-30, 30, (1, 3, 3)) * rng.choice([1, -1], (1, 3, 3))).astype(np.float32)
    scales[0, 1, 1] = 0
    w = _resident(fa, codes, scales)
    want = (plain.VALUES[codes[0]].astype(np.float32) * plain.expand(scales[0], 260, 300).astype(np.float32))
    assert np.array_equal(w.dequant().cpu().numpy(), want, equal_nan=True)
    ids = np.array([259, 0, 128, 128, 127], np.int32)
    assert np.array_equal(w.get_rows(to_dev(ids)).cpu().numpy(), want[ids], equal_nan=True)
    assert np.array_equal(w.get_rows_host(ids), want[ids], equal_nan=True)
    codes[0, (codes[0] & 0x7f) == 0x7f] = 0x30
    w = _resident(fa, codes, scales)
    want = (plain.VALUES[codes[0]].astype(np.float32) * plain.expand(scales[0], 260, 300).astype(np.float32))
    x = np.zeros((batch, 300), np.float32)
    at = rng.integers(0, 300, batch)
    x[np.arange(batch), at] = 2.0
    assert np.array_equal(w.gemm(to_dev(x)).cpu().numpy(), want[:, at].T * 2)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 16, 40, 70, 300])
def test_values_that_are_no_numbers_stay_in_their_rows(fa, batch):
    rng = np.random.default_rng(batch)
    rows, cols = 140, 300
    codes, scales = plain.random_matrix(rng, rows, cols)
    codes[0, 7, 130], codes[0, 139, 299] = 0x7f, 0xff
    w = _resident(fa, codes, scales)
    x = _activations(rng, batch, cols)
    bad = rng.choice(batch, max(1, batch // 4), replace=False)
    x[bad, rng.integers(0, cols, bad.size)] = rng.choice([np.inf, -np.inf, np.nan], bad.size)
    want, room = plain.product(codes[0], scales[0], x)
    got = w.gemm(to_dev(x)).cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert fine.sum() == (batch - bad.size) * (rows - 2)
    ok = np.ones(rows, bool)
    ok[[7, 139]] = False
    keep = np.setdiff1d(np.arange(batch), bad)
    a, wd = plain.quantize(x[keep]), plain.dequant(codes[0], scales[0])[ok]
    room = (128 + 3 + 9) * 2.0 ** -24 * (np.abs(a) @ np.abs(wd).T)
    assert (np.abs(got[np.ix_(keep, ok)] - want[np.ix_(keep, ok)]) <= room).all()


@pytest.mark.gpu
def test_zero_rows_and_blocks_give_zero(fa):
    rng = np.random.default_rng(1)
    codes, scales = plain.random_matrix(rng, 50, 260)
    x = _activations(rng, 6, 260)
    x[2] = 0
    x[4, :128] = 0
    got = _resident(fa, codes, scales).gemm(to_dev(x)).cpu().numpy()
    want, room = plain.product(codes[0], scales[0], x)
    assert (got[2] == 0).all() and (np.abs(got - want) <= room).all()


@pytest.mark.gpu
def test_a_stack_is_its_matrices(fa):
    """Matrices whose rows are no whole strips or blocks: one product over the stack is each matrix's own, bit for bit."""
    rng = np.random.default_rng(8)
    codes, scales = plain.random_matrix(rng, 137, 200, matrices=3)
    x = to_dev(_activations(rng, 21, 200))
    whole = _resident(fa, codes, scales).gemm(x).cpu().numpy()
    for m in range(3):
        alone = _resident(fa, codes[m:m + 1], scales[m:m + 1]).gemm(x).cpu().numpy()
        assert np.array_equal(whole[:, 137 * m:137 * (m + 1)], alone)


@pytest.mark.gpu
def test_entry_points_agree(fa):
    """gemv, gemv_multi, gemm_pair, gemm_noalloc and a matrix from host memory: gemm's bits; the FFN its parts' bits."""
    import torch
    rng = np.random.default_rng(11)
    hidden, ffn = 640, 832
    pairs = [plain.random_matrix(rng, r, c) for r, c in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
    gate, up, down = (_resident(fa, *p) for p in pairs)
    host = fa.Weights.from_host_fp8(pairs[0][0], pairs[0][1], ffn, hidden)
    for batch in (1, 5, 80):
        x = to_dev(_activations(rng, batch, hidden))
        y = gate.gemm(x)
        assert torch.equal(host.gemm(x), y)
        a, b = fa.gemm_pair(gate, up, x)
        assert torch.equal(a, y) and torch.equal(b, up.gemm(x))
        assert torch.equal(gate.gemm_noalloc(x, torch.empty_like(y)), y)
        assert torch.equal(gate.gemv(x[0]), gate.gemm(x[:1])[0]) and torch.equal(gate.gemv(x[0], act_mode=fa.ACT_INT8), gate.gemm(x[:1])[0])
        g, u = fa.gemv_multi([gate, up], x[0])
        assert torch.equal(g, gate.gemv(x[0])) and torch.equal(u, up.gemv(x[0]))
        got = fa.ffn_swiglu(gate, up, down, x[0])
        act = (g * u / (1 + torch.exp(-g.double())).float())
        # (silu by another exponential: the last bits of the intermediate, whose quantization may move a value to the next
        # code, a step of 1/8 of it at most)
        want = down.gemv(act.contiguous())
        assert float((got - want).norm() / want.norm()) < 0.02


def _groups(rng, counts):
    off = np.zeros(len(counts) + 1, np.int32)
    off[1:] = np.cumsum(counts)
    return off


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,counts,x_rows", [
    (1, 1, [1], 1), (17, 129, [0, 3, 0, 1], 4), (130, 300, [16, 17, 1, 64, 65, 0, 130], 50), (64, 256, [1] * 40, 8),
    (768, 2048, [1, 0] * 8, 1), (200, 512, [300, 5], 77), (48, 96, [0] * 1000 + [2] + [0] * 23, 2), (2880, 160, [3, 90, 33], 126),
    (144, 640, [0, 0, 700], 700), (36, 260, [2, 1, 5, 0, 8] * 30, 19),
    (24, 7168, [4, 1, 0, 5], 6), (5, 66000, [2, 0, 1], 3), (24, 7296, [4, 1, 0, 17], 6), (270, 160, [24, 23, 25], 72), (270, 160, [24, 23, 24], 71),
])
def test_grouped_against_64_bits(fa, rows, cols, counts, x_rows):
    print("fp8 grouped", rows, cols, len(counts), x_rows, flush=True)
    rng = np.random.default_rng(rows + cols + x_rows)
    codes, scales = plain.random_matrix(rng, rows, cols, matrices=len(counts))
    off = _groups(rng, counts)
    x = _activations(rng, x_rows, cols)
    gather = rng.integers(0, x_rows, off[-1]).astype(np.int32)  # (the same row several times)
    got = fa.gemm_grouped(_resident(fa, codes, scales), len(counts), to_dev(off), to_dev(x), gather=to_dev(gather)).cpu().numpy()
    for g in range(len(counts)):
        s = slice(off[g], off[g + 1])
        if counts[g]:
            want, room = plain.product(codes[g], scales[g], x[gather[s]])
            assert (np.abs(got[s] - want) <= room).all(), g


@pytest.mark.gpu
def test_grouped_without_a_list_reads_the_rows_in_order(fa):
    rng = np.random.default_rng(6)
    codes, scales = plain.random_matrix(rng, 40, 200, matrices=3)
    off = _groups(rng, [5, 0, 90])
    x = _activations(rng, 95, 200)
    w = _resident(fa, codes, scales)
    got = fa.gemm_grouped(w, 3, to_dev(off), to_dev(x))
    again = fa.gemm_grouped(w, 3, to_dev(off), to_dev(x), gather=to_dev(np.arange(95, dtype=np.int32)))
    assert np.array_equal(got.cpu().numpy(), again.cpu().numpy())
    want, room = plain.product(codes[2], scales[2], x[5:])
    assert (np.abs(got[5:].cpu().numpy() - want) <= room).all()


@pytest.mark.gpu
def test_lists_that_point_outside_are_clamped(fa):
    """Offsets outside 0 .. pairs or out of order and gather entries outside x: rows of no group stay as they were, a
    group's range is from the largest offset so far."""
    import torch
    rng = np.random.default_rng(2)
    codes, scales = plain.random_matrix(rng, 33, 140, matrices=4)
    x = _activations(rng, 6, 140)
    w = _resident(fa, codes, scales)
    gather = np.array([-5, 0, 99, 5, 2, 2147483647, -2147483648, 3, 1, 4], np.int32)
    for off in ([2, 5, 3, 4, 8], [-7, 4, 1000, 2, 6], [3, 3, 3, 3, 3], [0, 10, 0, 10, 0]):
        y = torch.full((10, 33), 7.5, device="cuda")
        fa.gemm_grouped(w, 4, to_dev(np.array(off, np.int32)), to_dev(x), gather=to_dev(gather), out=y)
        got = y.cpu().numpy()
        top = np.maximum.accumulate(np.clip(off, 0, 10))
        seen = np.zeros(10, bool)
        for g in range(4):
            s = slice(top[g], top[g + 1])
            seen[s] = True
            if top[g + 1] > top[g]:
                want, room = plain.product(codes[g], scales[g], x[np.clip(gather[s], 0, 5)])
                assert (np.abs(got[s] - want) <= room).all(), (off, g)
        assert (got[~seen] == 7.5).all(), off


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 40, 300])
def test_unaligned_operands(fa, batch):
    """Activations and outputs that start 4 bytes past a 16-byte boundary: the aligned call's bits."""
    import torch
    rng = np.random.default_rng(batch)
    codes, scales = plain.random_matrix(rng, 132, 256)
    w = _resident(fa, codes, scales)
    x = to_dev(_activations(rng, batch, 256))
    room = torch.zeros(x.numel() + 1, device="cuda")
    shifted = room[1:].view(batch, 256)
    shifted.copy_(x)
    y = torch.full((batch * 132 + 2,), 3.0, device="cuda")
    w.gemm(shifted, out=y[1:-1])
    assert torch.equal(y[1:-1].view(batch, 132), w.gemm(x)) and float(y[0]) == 3.0 and float(y[-1]) == 3.0
    bytes_ = torch.zeros(codes.size + 1, dtype=torch.uint8, device="cuda")
    bytes_[1:] = to_dev(codes).flatten()
    odd = fa.Weights.from_device_fp8(bytes_[1:], to_dev(scales), 132, 256)
    assert torch.equal(odd.gemm(x), w.gemm(x))


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 24, 200])
def test_captured_and_replayed_on_another_stream(fa, batch):
    import torch
    rng = np.random.default_rng(4)
    codes, scales = plain.random_matrix(rng, 260, 512)
    w = _resident(fa, codes, scales)
    stacked = _resident(fa, *plain.random_matrix(rng, 64, 512, matrices=4))
    off = to_dev(np.array([0, batch // 3, batch // 2, batch, batch], np.int32))
    x = to_dev(_activations(rng, batch, 512))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    y, z = torch.empty((batch, 260), device="cuda"), torch.empty((batch, 64), device="cuda")
    with torch.cuda.stream(other):
        w.gemm(x, out=y)  # (the shape once before the capture)
        fa.gemm_grouped(stacked, 4, off, x, out=z)
    other.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=other):
        w.gemm(x, out=y)
        fa.gemm_grouped(stacked, 4, off, x, out=z)
    for i in range(3):
        x.copy_(to_dev(_activations(rng, batch, 512)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w.gemm(x)) and torch.equal(z, fa.gemm_grouped(stacked, 4, off, x)), i


# ---- refusals, without a device ----

def _null():
    import frink_amd
    return frink_amd.lib(), frink_amd


def test_the_kind_is_outside_the_seam():
    L, fa = _null()
    assert fa.matvec_kernel(fa.FP8_BLOCK) is None and not L.frk_hip_has_launch(fa.FP8_BLOCK) and not L.frk_hip_gemm_supported(fa.FP8_BLOCK)
    assert L.frk_hip_block_bytes(fa.FP8_BLOCK) == 0
    h = C.c_void_p()
    buf = np.zeros(256, np.uint8)
    assert L.frk_hip_weights_register(fa.FP8_BLOCK, C.c_void_p(buf.ctypes.data), 256, 2, 128, C.byref(h)) == fa.ERR_UNSUPPORTED
    assert L.frk_hip_weights_from_device(fa.FP8_BLOCK, C.c_void_p(buf.ctypes.data), 256, 2, 128, None, C.byref(h)) == fa.ERR_UNSUPPORTED


@pytest.mark.parametrize("rows,cols,matrices,needle", [
    (0, 128, 1, "empty"), (4, 0, 1, "empty"), (4, 128, 0, "empty"), (7, 128, 2, "divide"), (2 ** 31, 1, 1, "too large"), (1, 2 ** 31, 1, "too large"), (1, 2 ** 23 + 1, 1, "too large"),
    (70000, 8, 70000, "65535"),
])
def test_shapes_refused_before_any_device_call(rows, cols, matrices, needle):
    L, fa = _null()
    p = C.c_void_p(4096)
    h = C.c_void_p(1)
    assert L.frk_hip_weights_from_device_fp8(p, p, rows, cols, matrices, None, C.byref(h)) == fa.ERR_SHAPE
    assert needle in fa.last_error() and not h.value
    assert L.frk_hip_weights_register_fp8(p, p, rows, cols, matrices, C.byref(h)) == fa.ERR_SHAPE


@pytest.mark.parametrize("name", ["frk_f8.hip", "frk_f8_tile.hip"])
def test_no_register_is_read_before_its_wait(tmp_path, name):
    """The compiler does not count the wait states behind a matrix instruction across a branch that splits and joins: one such
    branch in the loop over the blocks once left a sum's readers two instructions behind it."""
    import os
    import subprocess

    import isa_mfma_lint
    import isa_wait_lint
    from frink_amd import build as fb
    out = tmp_path / "kernels.s"
    cmd = [fb.hipcc()] + fb.HIPCC_FLAGS + ["-x", "hip", "--cuda-device-only", "-S", os.path.join(fb.CSRC, name), "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    asm = out.read_text()
    assert "v_mfma" in asm and isa_mfma_lint.violations(asm) == []
    for k in isa_wait_lint.kernels(asm):
        assert isa_wait_lint.violations(asm, k) == [], k


def test_null_arguments():
    L, fa = _null()
    p, h = C.c_void_p(4096), C.c_void_p()
    for args in ((None, p, C.byref(h)), (p, None, C.byref(h)), (p, p, None)):
        assert L.frk_hip_weights_from_device_fp8(args[0], args[1], 1, 1, 1, None, args[2]) == fa.ERR_ARG
        assert L.frk_hip_weights_register_fp8(args[0], args[1], 1, 1, 1, args[2]) == fa.ERR_ARG


def test_python_checks_lengths():
    _, fa = _null()
    for codes, scales, rows, cols, matrices in ((10, 1, 2, 6, 1), (12, 2, 2, 6, 1), (12, 1, 2, 6, 3), (12, 1, 2, 6, 2)):
        with pytest.raises(ValueError):
            fa.Weights.from_host_fp8(np.zeros(codes, np.uint8), np.zeros(scales, np.float32), rows, cols, matrices)


@pytest.mark.gpu
def test_calls_refused_on_a_handle(fa):
    import torch
    rng = np.random.default_rng(0)
    w = _resident(fa, *plain.random_matrix(rng, 16, 256, matrices=2))
    x = torch.zeros((2, 256), device="cuda")
    off = to_dev(np.array([0, 1, 2, 2], np.int32))
    with pytest.raises(fa.BackendError, match="names 3 groups") as e:
        fa.gemm_grouped(_resident(fa, *plain.random_matrix(rng, 6, 256, matrices=2)), 3, off, x)
    assert e.value.code == fa.ERR_SHAPE
    for call in (lambda: w.gemv(x[0], act_mode=fa.ACT_F32_DOT), lambda: w.gemm_q8k(fa.quantize_q8_k(x), 2), lambda: w.gemv_q8k(fa.quantize_q8_k(x[0])),
                 lambda: w.gemm_acts(fa.BatchActs(4, 256).quantize(x)), lambda: w.keep_decoded()):
        with pytest.raises(fa.BackendError) as e:
            call()
        assert e.value.code == fa.ERR_UNSUPPORTED


# ---- the layer of experts behind the router ----

def _layer(fa, rng, experts, hidden, ffn):
    parts = [plain.random_matrix(rng, r, c, matrices=experts) for r, c in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
    return parts, [_resident(fa, *p) for p in parts]


def _plain_layer(parts, x, ids, weights):
    """f64, and how far f32 may be from it: an intermediate is off by what product() says of gate and up, and where a border
    between two codes lies within that, its code may be the next one."""
    out, room = np.zeros((x.shape[0], parts[2][0].shape[1])), np.zeros((x.shape[0], parts[2][0].shape[1]))
    for t in range(x.shape[0]):
        for e, w in zip(ids[t], weights[t]):
            if e < 0 or e >= parts[0][0].shape[0]:
                continue
            (g, rg), (u, ru) = (plain.product(codes[e], scales[e], x[t:t + 1]) for codes, scales in parts[:2])
            dw = plain.dequant(parts[2][0][e], parts[2][1][e])
            sig = 1 / (1 + np.exp(np.minimum(-g, 700)))
            act = g * sig * u
            off = rg * np.abs(u) * 1.1 + ru * np.abs(g) + 4 * 2.0 ** -24 * np.abs(act)  # |d silu| <= 1.1
            q = plain.quantize(act)
            moved = np.abs(plain.quantize(act + off) - q) + np.abs(plain.quantize(act - off) - q)
            y = (q @ dw.T)[0]
            out[t] += w * y
            room[t] += np.abs(w) * ((moved @ np.abs(dw).T)[0] + (128 + dw.shape[1] / 128 + 12) * 2.0 ** -24 * (np.abs(q) @ np.abs(dw).T)[0])
    return out, room


@pytest.mark.gpu
@pytest.mark.parametrize("batch,experts,k,hidden,ffn", [
    (1, 4, 2, 260, 130), (3, 8, 8, 128, 384), (16, 6, 3, 384, 100), (33, 5, 2, 640, 256), (70, 3, 1, 132, 513), (200, 4, 2, 256, 128),
    (1, 64, 8, 512, 192), (40, 128, 4, 256, 96), (4, 16, 3, 1028, 700), (8, 32, 8, 260, 1300), (1, 3, 1, 24576, 40), (1, 3, 1, 24704, 40),
    (1, 2, 1, 16, 1)])
def test_expert_layer_against_64_bits(fa, batch, experts, k, hidden, ffn):
    print("fp8 experts", batch, experts, k, hidden, ffn, flush=True)
    rng = np.random.default_rng(batch + experts * hidden)
    parts, (gate, up, down) = _layer(fa, rng, experts, hidden, ffn)
    x = _activations(rng, batch, hidden)
    logits = rng.standard_normal((batch, experts)).astype(np.float32)
    if batch > 2:
        logits[1, 1:] = -np.inf  # (one expert left: slots of id -1)
    ids, w = fa.route(to_dev(logits), k, score="sigmoid", scale=2.5)
    got = fa.moe_ffn(gate, up, down, experts, to_dev(x), ids, w).cpu().numpy()
    want, room = _plain_layer(parts, x, ids.cpu().numpy(), w.cpu().numpy())
    assert (np.abs(got - want) <= room * 1.01 + 1e-30).all()


@pytest.mark.gpu
def test_router_and_experts_captured_together(fa):
    import torch
    rng = np.random.default_rng(9)
    _, (gate, up, down) = _layer(fa, rng, 16, 256, 128)
    bias = to_dev((rng.standard_normal(16) * 0.1).astype(np.float32))
    for batch in (1, 5, 60):
        x, logits = to_dev(_activations(rng, batch, 256)), to_dev(rng.standard_normal((batch, 16)).astype(np.float32))
        rule = dict(score="sigmoid", bias=bias, groups=4, top_groups=2, group_best=2)

        def step(out=None):
            ids, w = fa.route(logits, 4, **rule)
            return fa.moe_ffn(gate, up, down, 16, x, ids, w, out=out)
        y = torch.empty((batch, 256), device="cuda")
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(y)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(y)
        for _ in range(3):
            x.copy_(to_dev(_activations(rng, batch, 256)))
            logits.copy_(to_dev(rng.standard_normal((batch, 16)).astype(np.float32)))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, step())


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,ffn", [(640, 832), (256, 130), (24576, 48)])
def test_a_layer_of_one_expert_is_the_ffn(fa, hidden, ffn):
    import torch
    rng = np.random.default_rng(hidden)
    _, (gate, up, down) = _layer(fa, rng, 1, hidden, ffn)
    x = to_dev(_activations(rng, 1, hidden))
    y = fa.moe_ffn(gate, up, down, 1, x, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.ones((1, 1), device="cuda"))
    want = fa.ffn_swiglu(gate, up, down, x[0])
    assert torch.equal(y[0], want)  # the same sums in the same order


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [((512, 300), 1024), ((4096, 64), 640), ((40, 9000), 300), ((2880, 2880), 2880)])
def test_a_pair_is_its_matrices(fa, rows, cols):
    """Pairs of one quantization and of two, whichever kernels their plans name; captured and replayed."""
    import torch
    rng = np.random.default_rng(cols)
    w0, w1 = (_resident(fa, *plain.random_matrix(rng, r, cols)) for r in rows)
    for batch in (1, 4, 6, 8, 16, 17, 40, 64, 65, 130, 300):
        x = to_dev(_activations(rng, batch, cols))
        want = w0.gemm(x), w1.gemm(x)
        got = fa.gemm_pair(w0, w1, x)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), batch
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        fa.gemm_pair(w0, w1, x, outs=got)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        fa.gemm_pair(w0, w1, x, outs=got)
    for _ in range(3):
        x.copy_(to_dev(_activations(rng, batch, cols)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], w0.gemm(x)) and torch.equal(got[1], w1.gemm(x))


@pytest.mark.gpu
def test_tensors_of_another_device_are_refused(fa):
    import torch

    class Elsewhere:  # (a tensor of a second device, which this one need not have)
        def __init__(self, t):
            self.t = t

        def __getattr__(self, name):
            return getattr(self.t, name)

        def get_device(self):
            return self.t.get_device() + 1
    rng = np.random.default_rng(2)
    codes, scales = plain.random_matrix(rng, 16, 128)
    w = _resident(fa, codes, scales)
    x = Elsewhere(torch.zeros((1, 128), device="cuda"))
    ids, weights = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.ones((1, 1), device="cuda")
    for call in (lambda: w.gemm(x), lambda: w.gemv(x), lambda: w.gemm_noalloc(x, torch.zeros((1, 16), device="cuda")), lambda: fa.gemm_pair(w, w, x),
                 lambda: fa.gemv_multi([w, w], x), lambda: fa.gemm_grouped(w, 1, to_dev(np.array([0, 1], np.int32)), x),
                 lambda: fa.moe_ffn(w, w, w, 1, x, ids, weights), lambda: fa.Weights.from_device_fp8(Elsewhere(to_dev(codes)), to_dev(scales), 16, 128)):
        with pytest.raises(ValueError, match="current device"):
            call()


@pytest.mark.gpu
def test_two_threads_on_two_streams(fa):
    """Calls of one handle from two threads at once, each on its own stream: the results of calls one after the other."""
    import threading

    import torch
    rng = np.random.default_rng(21)
    w = _resident(fa, *plain.random_matrix(rng, 500, 1300))
    stack = _resident(fa, *plain.random_matrix(rng, 96, 300, matrices=4))
    jobs, want = [], []
    for batch in (2, 9, 33, 150):
        x, g = to_dev(_activations(rng, batch, 1300)), to_dev(_activations(rng, batch, 300))
        off = to_dev(_groups(rng, [batch // 2, 0, batch - batch // 2, 0]))
        jobs.append((x, g, off))
        want.append((w.gemm(x), fa.gemm_grouped(stack, 4, off, g)))
    torch.cuda.synchronize()
    wrong = []

    def work(order):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for i in order * 10:
                got = w.gemm(jobs[i][0]), fa.gemm_grouped(stack, 4, jobs[i][2], jobs[i][1])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
                stream.synchronize()
    threads = [threading.Thread(target=work, args=(o,)) for o in ([0, 1, 2, 3], [3, 2, 1, 0])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


@pytest.mark.gpu
def test_expert_layers_refused(fa):
    import torch
    rng = np.random.default_rng(1)
    _, (gate, up, down) = _layer(fa, rng, 4, 130, 64)
    x = torch.zeros((2, 130), device="cuda")
    ids, w = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros((2, 2), device="cuda")
    with pytest.raises(fa.BackendError, match="multiple of four") as e:
        fa.moe_ffn(gate, up, down, 4, x, ids, w)
    assert e.value.code == fa.ERR_SHAPE
    _, (gate, up, down) = _layer(fa, rng, 4, 128, 64)
    x = torch.zeros((2, 128), device="cuda")
    with pytest.raises(fa.BackendError, match="shapes disagree|names 2 experts"):
        fa.moe_ffn(gate, up, down, 2, x, ids, w)
    q8 = fa.Weights.from_device(fa.Q8_0, torch.zeros(4 * 128 * 2 * 34, dtype=torch.uint8, device="cuda"), 4 * 128, 64)
    with pytest.raises(fa.BackendError) as e:
        fa.moe_ffn(gate, up, q8, 4, x, ids, w)
    assert e.value.code == fa.ERR_UNSUPPORTED
