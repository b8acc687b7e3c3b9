"""MXFP4 (4-bit floating point, a power of two for every 32 values): quantization to blocks and to activation rows, the values back, and
products with both operands in it, against the definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import mxfp4_plain as plain
from test_gpu_parity import fa, to_dev  # noqa: F401 (fa: the module's fixture)

TYPES = ("float32", "bfloat16", "float16")


def _resident(fa, codes, scales):
    return fa.Weights.from_device(fa.MXFP4, to_dev(plain.blocks(codes, scales).reshape(-1)), *codes.shape)


def _activations(rng, rows, cols):
    """Rows of different sizes, a few large channels, some zeros."""
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-6, 7, (rows, 1))
    x[:, rng.integers(0, cols, max(1, cols // 64))] *= 30
    x[rng.random((rows, cols)) < 0.05] = 0
    return x.astype(np.float32)


def _borders(rng, rows, cols):
    """Values on every border between two codes, at and beside powers of two and the largest code, at the ends of f32's range."""
    x = (rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-20, 20, (rows, 1))).astype(np.float32)
    half = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], np.float32)
    for r in range(0, rows, 2):
        s = np.float32(2.0 ** int(rng.integers(-140, 120)))
        with np.errstate(over="ignore"):
            x[r, :16], x[r, 16:32] = half * s, -half * s
        for k in range(32, cols - 31, 32):
            x[r, k:k + 16] = np.nextafter(half, np.float32(rng.choice([-9, 9]))) * rng.choice([1, -1], 16)
    x[1 % rows, :3] = np.array([1, -2, 3]) * np.float32(2.0 ** -149)
    x[1 % rows, 3:32] = 0
    x[rows - 1, -32:] = np.finfo(np.float32).max
    if rows > 2:
        x[2, :32] = 0
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (5, 2880), (33, 512), (300, 416), (61, 4096), (1025, 256)])
@pytest.mark.parametrize("kind", TYPES)
def test_blocks_and_back(fa, rows, cols, kind):
    """Codes and scale bytes, bit for bit; what they stand for; a resident matrix of them."""
    import torch
    print("mxfp4 blocks", rows, cols, kind, flush=True)
    rng = np.random.default_rng(rows + cols)
    x = to_dev(_borders(rng, rows, cols)).to(getattr(torch, kind))
    x[~torch.isfinite(x)] = 1.0  # (f16: what it does not hold)
    codes, scales = plain.quantize(x.double().cpu().numpy())
    got = fa.quantize_mxfp4(x)
    assert got.shape == (rows, cols // 32 * 17) and got.dtype == torch.uint8
    assert np.array_equal(got.cpu().numpy().reshape(rows, -1, 17), plain.blocks(codes, scales))
    want = plain.values(codes, scales).astype(np.float32)
    assert np.array_equal(fa.dequantize_mxfp4(got, cols).cpu().numpy(), want)
    assert np.array_equal(fa.Weights.from_device(fa.MXFP4, got.flatten(), rows, cols).dequant().cpu().numpy(), want)
    # an odd place in memory, for the input and the output
    n = x.numel()
    room = torch.zeros(n + 1, dtype=x.dtype, device="cuda")
    room[1:] = x.flatten()
    out = torch.full((n // 32 * 17 + 2,), 7, dtype=torch.uint8, device="cuda")
    fa.quantize_mxfp4(room[1:].view(rows, cols), out=out[1:-1])
    assert torch.equal(out[1:-1], got.flatten()) and out[0] == 7 and out[-1] == 7
    assert torch.equal(fa.dequantize_mxfp4(out[1:-1], cols), fa.dequantize_mxfp4(got, cols))


@pytest.mark.gpu
def test_every_code_under_every_scale(fa):
    codes = np.tile(np.arange(32, dtype=np.uint8) % 16, (256, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    got = fa.dequantize_mxfp4(to_dev(plain.blocks(codes, scales).reshape(-1)), 32).cpu().numpy()
    with np.errstate(over="ignore"):
        want = plain.values(codes, scales).astype(np.float32)
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,cols", [(1, 32), (5, 2880), (70, 96), (300, 4128)])
def test_activation_rows(fa, batch, cols):
    """What a BatchActs holds; blocks that are no numbers."""
    rng = np.random.default_rng(batch)
    x = _borders(rng, batch, cols)
    acts = fa.BatchActs(batch + 3, cols, "mxfp4")
    assert np.array_equal(acts.quantize(to_dev(x)).values().cpu().numpy(), plain.values(*plain.quantize(x)).astype(np.float32))
    bad = rng.choice(batch, max(1, batch // 4), replace=False)
    x[bad, rng.integers(0, cols, bad.size)] = rng.choice([np.inf, -np.inf, np.nan], bad.size)
    got = acts.quantize(to_dev(x)).values().cpu().numpy()
    assert np.array_equal(got, plain.values(*plain.quantize(x)).astype(np.float32), equal_nan=True)
    back = fa.dequantize_mxfp4(fa.quantize_mxfp4(to_dev(x)), cols).cpu().numpy()
    assert np.array_equal(got, back, equal_nan=True)


# both sides of every number of tokens, strips, wavefronts, tiles and shares of the columns that the plan tells apart
SHAPES = [(1, 32, 1), (15, 64, 2), (16, 480, 1), (17, 512, 4), (129, 544, 5), (300, 992, 17), (64, 96, 33), (257, 2880, 61), (1000, 544, 65),
          (144, 14336, 5), (576, 2304, 9), (33, 1152, 200), (272, 384, 257), (512, 1152, 300), (31, 4096, 1), (7200, 160, 1), (7200, 160, 7), (7201, 96, 40),
          (12801, 96, 1), (12801, 128, 3), (13000, 64, 20), (12900, 96, 32), (12900, 96, 64), (40, 28672, 1), (33, 65536, 1), (33, 65536, 2), (20, 7168, 4), (20, 8192, 3),
          (100, 1024, 700), (4096, 128, 7), (2880, 160, 97), (300, 8192, 64), (200, 16384, 100), (70, 14336, 48), (513, 4128, 30), (1030, 512, 1100),
          (65, 32, 65), (3001, 288, 513),
          # each tile and share of the columns, with rows, tokens and stages that end inside
          (8200, 544, 1500), (2049, 1056, 2050), (14337, 1312, 257), (14337, 1568, 130), (8200, 1568, 257), (8200, 32, 200), (3001, 544, 700), (3001, 8224, 65),
          (1537, 16416, 65), (8200, 8224, 6), (257, 2336, 33), (257, 3360, 97), (513, 800, 33), (300, 1056, 70)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,batch", SHAPES)
def test_product_against_64_bits(fa, rows, cols, batch):
    import torch
    print("mxfp4 product", rows, cols, batch, flush=True)
    rng = np.random.default_rng(rows * 7 + cols * 3 + batch)
    codes, scales = plain.random_matrix(rng, rows, cols)
    w = _resident(fa, codes, scales)
    x = _activations(rng, batch, cols)
    want, room = plain.product(codes, scales, x)
    xd = to_dev(x)
    got = w.gemm_mxfp4(xd)
    assert (np.abs(got.cpu().numpy() - want) <= room).all()
    assert torch.equal(got, w.gemm_mxfp4(xd))  # the same bits again
    acts = fa.BatchActs(batch, cols, "mxfp4").quantize(xd)
    kept = w.gemm_acts(acts)
    assert (np.abs(kept.cpu().numpy() - want) <= room).all()
    if batch > 4:
        assert torch.equal(kept, got)
    # into and out of an odd place in memory; what lies beside stays
    y = torch.full((batch * rows + 2,), 3.0, device="cuda")
    xo = torch.zeros(xd.numel() + 1, device="cuda")
    xo[1:] = xd.flatten()
    w.gemm_mxfp4(xo[1:].view(batch, cols), out=y[1:-1])
    assert torch.equal(y[1:-1].view(batch, rows), got) and float(y[0]) == 3.0 and float(y[-1]) == 3.0


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 7, 24, 40, 100, 300])
def test_scales_far_apart(fa, batch):
    """Blocks whose scales differ by up to 2^80 within a row: small ones are lost beside large ones, and no more than that."""
    rng = np.random.default_rng(batch)
    codes, scales = plain.random_matrix(rng, 140, 1312, spread=20)
    x = (rng.standard_normal((batch, 1312)) * np.repeat(2.0 ** rng.integers(-20, 20, (batch, 41)), 32, 1)).astype(np.float32)
    want, room = plain.product(codes, scales, x)
    got = _resident(fa, codes, scales).gemm_mxfp4(to_dev(x)).cpu().numpy()
    assert (np.abs(got - want) <= room).all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 16, 40, 100])
@pytest.mark.parametrize("ends", [(0, 254), (254, 0), (1, 200), (20, 234)])
def test_scales_at_the_ends(fa, batch, ends):
    """One operand's scales at the end of E8M0's range, the other's at the other end: the products are ordinary numbers."""
    rng = np.random.default_rng(batch)
    w_byte, x_byte = ends
    codes, scales = plain.random_matrix(rng, 70, 160)
    scales[:] = w_byte
    xc = rng.integers(0, 16, (batch, 160), dtype=np.uint8)
    xc[:, ::32] = 7  # (a block's largest: between 4 and 8 under its scale)
    x_byte = min(x_byte, 252)
    x = plain.values(xc, np.full((batch, 5), x_byte, np.uint8)).astype(np.float32)
    want, room = plain.product(codes, scales, x)
    assert np.isfinite(want).all() and np.abs(want).max() < 2.0 ** 127
    got = _resident(fa, codes, scales).gemm_mxfp4(to_dev(x)).cpu().numpy()
    assert (np.abs(got - want) <= room + 160 * 2.0 ** -126).all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 3, 16, 40, 70, 300])
@pytest.mark.parametrize("cols", [288, 1312])
def test_values_that_are_no_numbers_stay_in_their_rows(fa, batch, cols):
    """Infinities and NaN in activations, the scale byte 255 in weights; in the padding behind a row's last block nothing of the kind counts."""
    rng = np.random.default_rng(batch)
    rows = 140
    codes, scales = plain.random_matrix(rng, rows, cols)
    codes[:, -16:] |= 0xf  # (what follows a row's codes are its scales, what follows those the next row's codes)
    scales[7, 3], scales[139, -1] = 255, 255
    w = _resident(fa, codes, scales)
    x = _activations(rng, batch, cols)
    bad = rng.choice(batch, max(1, batch // 4), replace=False)
    x[bad, rng.integers(0, cols, bad.size)] = rng.choice([np.inf, -np.inf, np.nan], bad.size)
    got = w.gemm_mxfp4(to_dev(x)).cpu().numpy()
    ok = np.ones(rows, bool)
    ok[[7, 139]] = False
    keep = np.setdiff1d(np.arange(batch), bad)
    want = np.full((batch, rows), np.nan)
    good, room = plain.product(codes[ok], scales[ok], x[keep])
    want[np.ix_(keep, ok)] = good
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert (np.abs(got[np.ix_(keep, ok)] - good) <= room).all()


@pytest.mark.gpu
def test_zero_activations_give_zero(fa):
    rng = np.random.default_rng(1)
    w = _resident(fa, *plain.random_matrix(rng, 200, 480))
    for batch in (1, 16, 40, 100):
        assert not w.gemm_mxfp4(to_dev(np.zeros((batch, 480), np.float32))).any()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [3, 40, 300])
def test_on_several_streams_and_in_graphs(fa, batch):
    """Calls on two streams at once; two graphs of one stream, replayed between each other and the stream's own calls."""
    import torch
    rng = np.random.default_rng(batch)
    parts = [plain.random_matrix(rng, 700, 2304) for _ in range(2)]
    ws = [_resident(fa, *p) for p in parts]
    xs = [to_dev(_activations(rng, batch, 2304)) for _ in range(2)]
    want = [w.gemm_mxfp4(x) for w, x in zip(ws, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ws[i].gemm_mxfp4(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    ys = [torch.zeros_like(v) for v in want]
    graphs = []
    with torch.cuda.stream(streams[0]):
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[0]):
                ws[i].gemm_mxfp4(xs[i], out=ys[i])
            graphs.append(g)
        for rep in range(3):
            for i in (0, 1):
                ys[i].zero_()
                graphs[i].replay()
                assert torch.equal(ws[1 - i].gemm_mxfp4(xs[1 - i]), want[1 - i])
                streams[0].synchronize()
                assert torch.equal(ys[i], want[i]), rep


@pytest.mark.gpu
def test_matrices_past_32_bits(fa):
    """4.4 GB of blocks: the first and the last rows, by every kernel."""
    import torch
    print("mxfp4, weights past 2^32 bytes", flush=True)
    rows, cols = 3600000, 2304
    blocks = torch.randint(0, 256, (rows, cols // 32, 17), dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    blocks[..., 0] = 118 + (blocks[..., 0] & 3)
    w = fa.Weights.from_device(fa.MXFP4, blocks.flatten(), rows, cols)
    picked = [slice(0, 100), slice(rows // 2, rows // 2 + 100), slice(rows - 100, rows)]
    parts = []
    for s in picked:
        b = blocks[s].cpu().numpy()
        parts.append((np.concatenate([b[:, :, 1:] & 15, b[:, :, 1:] >> 4], 2).reshape(100, cols), b[:, :, 0]))
    del blocks
    x = _activations(np.random.default_rng(1), 70, cols)
    for batch in (1, 12, 30, 70):
        y = w.gemm_mxfp4(to_dev(x[:batch]))
        for s, p in zip(picked, parts):
            want, room = plain.product(*p, x[:batch])
            assert (np.abs(y[:, s].cpu().numpy() - want) <= room).all(), (batch, s)


@pytest.mark.gpu
def test_batches_past_32_bits(fa):
    """8.9 GB of activations, 2^31 results and more, in blocks of GGUF's 2^32 bytes; the first and the last tokens."""
    import torch
    print("mxfp4, activations past 2^32 bytes", flush=True)
    rows, cols, batch = 4160, 4224, 2 ** 19 + 5
    rng = np.random.default_rng(2)
    codes, scales = plain.random_matrix(rng, rows, cols)
    w = _resident(fa, codes, scales)
    x = torch.randn((batch, cols), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    acts = fa.BatchActs(batch, cols, "mxfp4").quantize(x)
    y = w.gemm_acts(acts)
    assert y.numel() > 2 ** 31
    picked = [slice(0, 3), slice(batch // 2, batch // 2 + 3), slice(batch - 7, batch)]
    for s in picked:
        want, room = plain.product(codes, scales, x[s].cpu().numpy())
        assert (np.abs(y[s].cpu().numpy() - want) <= room).all(), s
    del y
    values = acts.values()
    back = fa.dequantize_mxfp4(fa.quantize_mxfp4(x), cols)
    for s in picked:
        want = plain.values(*plain.quantize(x[s].cpu().numpy())).astype(np.float32)
        assert np.array_equal(values[s].cpu().numpy(), want) and np.array_equal(back[s].cpu().numpy(), want)


@pytest.mark.gpu
def test_a_feed_forward_block_in_four_bits(fa):
    """As a decoder uses them: weights quantized, the norm's rows quantized once for gate and up, the down projection over its own quantization."""
    import torch
    rng = np.random.default_rng(5)
    hidden, ffn, batch = 1280, 2080, 37
    mats = [rng.standard_normal(s).astype(np.float32) * 0.05 for s in ((ffn, hidden), (ffn, hidden), (hidden, ffn))]
    gate, up, down = (fa.Weights.from_device(fa.MXFP4, fa.quantize_mxfp4(to_dev(m)).flatten(), *m.shape) for m in mats)
    x, res = _activations(rng, batch, hidden), _activations(rng, batch, hidden)
    weight = rng.uniform(0.5, 1.5, hidden).astype(np.float32)
    acts = fa.BatchActs(64, hidden, "mxfp4")
    a, h = fa.rms_norm(to_dev(x), to_dev(weight), 1e-5, residual=to_dev(res), acts=acts)
    g, u = gate.gemm_acts(a), up.gemm_acts(a)
    act = torch.nn.functional.silu(g) * u
    y = down.gemm_mxfp4(act) + h
    ph, pn = plain.norm(x, res, weight, 1e-5, lambda v: v.astype(np.float64))
    q = [plain.quantize(m) for m in mats]
    assert np.array_equal(h.cpu().numpy(), ph.astype(np.float32))
    for got, m in ((g, q[0]), (u, q[1])):
        want, room = plain.product(*m, pn)
        assert (np.abs(got.cpu().numpy() - want) <= room).all()
    want, room = plain.product(*q[2], act.cpu().numpy())
    assert (np.abs(y.cpu().numpy() - (want + ph)) <= room + 2.0 ** -23 * (np.abs(want) + np.abs(ph))).all()


# ---- refusals ----
def test_python_refuses_before_anything_runs():
    import torch

    import frink_amd as fa
    x = torch.zeros((2, 64))
    for call in (lambda: fa.quantize_mxfp4(x), lambda: fa.dequantize_mxfp4(torch.zeros(34, dtype=torch.uint8), 32), lambda: fa.rms_norm(x)):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
    with pytest.raises(ValueError, match="form"):
        fa.BatchActs(4, 64, "q4")


def test_the_library_refuses_before_anything_runs():
    import frink_amd as fa
    L = fa.lib()
    room = np.zeros(256, np.uint8)
    p = C.c_void_p(room.ctypes.data)
    h = C.c_void_p()
    for rc, status in [(L.frk_hip_quantize_mxfp4_dev(0, None, 32, p, None), fa.ERR_ARG), (L.frk_hip_quantize_mxfp4_dev(0, p, 32, None, None), fa.ERR_ARG),
                       (L.frk_hip_quantize_mxfp4_dev(3, p, 32, p, None), fa.ERR_UNSUPPORTED), (L.frk_hip_quantize_mxfp4_dev(0, p, 33, p, None), fa.ERR_SHAPE),
                       (L.frk_hip_quantize_mxfp4_dev(0, p, 0, p, None), fa.ERR_SHAPE), (L.frk_hip_dequantize_mxfp4_dev(p, 31, p, None), fa.ERR_SHAPE),
                       (L.frk_hip_dequantize_mxfp4_dev(None, 32, p, None), fa.ERR_ARG), (L.frk_hip_gemm_mxfp4_dev(None, p, 1, p, None), fa.ERR_ARG),
                       (L.frk_hip_batch_acts_create_form(4, 64, 3, C.byref(h)), fa.ERR_UNSUPPORTED), (L.frk_hip_batch_acts_create_form(4, 48, 2, C.byref(h)), fa.ERR_SHAPE),
                       (L.frk_hip_batch_acts_create_form(0, 64, 2, C.byref(h)), fa.ERR_SHAPE), (L.frk_hip_batch_acts_create_form(4, 0, 1, C.byref(h)), fa.ERR_SHAPE),
                       (L.frk_hip_batch_acts_create_form(4, (1 << 23) + 32, 2, C.byref(h)), fa.ERR_SHAPE), (L.frk_hip_batch_acts_create_form(4, 64, 2, None), fa.ERR_ARG),
                       (L.frk_hip_batch_acts_create_form((1 << 30) + 1, 64, 1, C.byref(h)), fa.ERR_SHAPE), (L.frk_hip_batch_acts_values_dev(None, p, None), fa.ERR_ARG)]:
        assert rc == status and fa.last_error()


@pytest.mark.gpu
def test_operands_that_do_not_fit_are_refused(fa):
    import torch
    rng = np.random.default_rng(3)
    w = _resident(fa, *plain.random_matrix(rng, 64, 128))
    x, y = torch.zeros((3, 128), device="cuda"), torch.zeros((3, 64), device="cuda")
    w.gemm_mxfp4(x, out=y)
    for bad in (x.half(), x[:, :64], x[:, :96].contiguous(), x.cpu(), torch.zeros((128, 3), device="cuda").t()):
        with pytest.raises(ValueError):
            w.gemm_mxfp4(bad)
    for bad in (y.flatten()[:191], y.half(), torch.zeros((64, 3), device="cuda").t()):
        with pytest.raises(ValueError, match="contiguous floats"):
            w.gemm_mxfp4(x, out=bad)
    other = fa.Weights.from_device_fp8(torch.zeros((64, 128), dtype=torch.uint8, device="cuda"), torch.ones((1, 1), device="cuda"), 64, 128)
    acts = {f: fa.BatchActs(4, 128, f) for f in ("fp8", "mxfp4")}
    for call in (lambda: other.gemm_mxfp4(x), lambda: w.gemm_acts(acts["fp8"].quantize(x)), lambda: other.gemm_acts(acts["mxfp4"].quantize(x))):
        with pytest.raises(fa.BackendError) as e:
            call()
        assert e.value.code == fa.ERR_UNSUPPORTED
    for a in acts.values():
        with pytest.raises(fa.BackendError) as e:
            a.quantize(torch.zeros((5, 128), device="cuda"))
        assert e.value.code == fa.ERR_SHAPE
    fresh = fa.BatchActs(4, 128, "mxfp4")
    for call in (lambda: w.gemm_acts(fresh, out=y), lambda: fresh.values(out=y)):
        with pytest.raises(fa.BackendError) as e:  # nothing is in it yet
            call()
        assert e.value.code == fa.ERR_ARG
    narrow = fa.BatchActs(4, 96, "mxfp4").quantize(torch.zeros((2, 96), device="cuda"))
    with pytest.raises(fa.BackendError) as e:
        w.gemm_acts(narrow)
    assert e.value.code == fa.ERR_SHAPE
    for bad in (torch.zeros((2, 33), device="cuda"), torch.zeros((0, 32), device="cuda"), torch.zeros((2, 32), dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            fa.quantize_mxfp4(bad)
    for blocks, cols in ((torch.zeros(33, dtype=torch.uint8, device="cuda"), 32), (torch.zeros(34, dtype=torch.uint8, device="cuda"), 33), (torch.zeros(34, device="cuda"), 32)):
        with pytest.raises(ValueError):
            fa.dequantize_mxfp4(blocks, cols)
