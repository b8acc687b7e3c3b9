"""Root-mean-square norms with the residual's addition, their result as it is or quantized for the products behind: against the
definition in 64 bits, bit for bit."""
import ctypes as C

import numpy as np
import pytest

import fp8_plain
import mxfp4_plain as plain
import oracle as fo
from test_gpu_parity import fa, make_weights, to_dev  # noqa: F401 (fa: the module's fixture)

EPS = 1e-5


def _rounded(kind):
    """f32 -> the type's numbers, in 64 bits."""
    import torch

    def to(v):
        return torch.from_numpy(np.ascontiguousarray(v, np.float32)).to(getattr(torch, kind)).double().numpy()
    return to


def _rows(rng, batch, cols, kind):
    """Rows of different sizes with a few large channels, of the type's numbers (f64)."""
    x = rng.standard_normal((batch, cols)) * 2.0 ** rng.integers(-5, 5, (batch, 1))
    x[:, rng.integers(0, cols, max(1, cols // 100))] *= 20
    return _rounded(kind)(x)


def _dev(v, kind):
    import torch
    return torch.from_numpy(np.ascontiguousarray(v)).to(getattr(torch, kind)).cuda()


# chunks of 256 a wavefront: one, two (the last not whole), four, more than sixteen wavefronts hold; rows that are not whole pieces of four
SHAPES = [(1, 1), (3, 5), (2, 130), (7, 256), (5, 260), (61, 301), (33, 515), (4, 1028), (61, 2880), (1, 4096), (300, 4100), (700, 640), (2, 8200), (600, 8192),
          (3, 16384), (2, 16388), (3, 20001), (1, 40000), (1500, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("batch,cols", SHAPES)
@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16"])
def test_norm_against_64_bits(fa, batch, cols, kind):
    import torch
    print("norm", batch, cols, kind, flush=True)
    rng = np.random.default_rng(batch * 3 + cols)
    x, res = (_rows(rng, batch, cols, kind) for _ in range(2))
    weight = rng.uniform(0.5, 1.5, cols).astype(np.float32)
    rounded = _rounded(kind)
    for weight_kind, r in ((None, res), ("float32", res), (kind, None), ("float32", None)):
        w = None if weight_kind is None else _dev(weight, weight_kind)
        y, h = fa.rms_norm(_dev(x, kind), w, EPS, residual=None if r is None else _dev(r, kind))
        ph, py = plain.norm(x, r, None if w is None else w.float().cpu().numpy(), EPS, rounded)
        assert np.array_equal(h.double().cpu().numpy(), ph)
        assert y.dtype == getattr(torch, kind) and np.array_equal(y.double().cpu().numpy(), rounded(py)), (weight_kind, r is None)
    # an odd place in memory; h in x's or the residual's place, y in x's
    w = _dev(weight, "float32")
    ph, py = plain.norm(x, res, weight, EPS, rounded)
    for in_place in ("none", "sum in x", "sum in residual", "y in x", "y in residual", "both"):
        rooms = [torch.full((batch * cols + 2,), 3.0, dtype=getattr(torch, kind), device="cuda") for _ in range(4)]
        views = [r[1:-1].view(batch, cols) for r in rooms]
        views[0].copy_(_dev(x, kind)), views[1].copy_(_dev(res, kind))
        to_sum = {"sum in x": views[0], "sum in residual": views[1], "both": views[1]}.get(in_place, views[2])
        to_y = {"y in x": views[0], "y in residual": views[1], "both": views[0]}.get(in_place, views[3])
        y, h = fa.rms_norm(views[0], w, EPS, residual=views[1], sum_out=to_sum, out=to_y)
        assert y.data_ptr() == to_y.data_ptr() and h.data_ptr() == to_sum.data_ptr()
        assert np.array_equal(h.double().cpu().numpy(), ph) and np.array_equal(y.double().cpu().numpy(), rounded(py)), in_place
        assert all(float(r[0]) == 3.0 and float(r[-1]) == 3.0 for r in rooms)


FORMS = {"q8_k": [256, 1024, 2816, 4096, 16640], "fp8": [3, 128, 300, 1300, 2880, 4096, 17000], "mxfp4": [32, 480, 512, 1312, 4096, 16416]}


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 2, 8, 9, 16, 17, 33, 64, 65, 200, 700])
@pytest.mark.parametrize("form", list(FORMS))
def test_quantized_output_is_the_quantization_of_the_output(fa, batch, form):
    """Values and products, bit for bit, as of the plain output quantized by itself; the plain output beside it; a larger batch before."""
    import torch
    for cols in FORMS[form]:
        print("norm", form, batch, cols, flush=True)
        rng = np.random.default_rng(batch + cols)
        x, res, weight = to_dev(_rows(rng, batch, cols, "float32").astype(np.float32)), to_dev(_rows(rng, batch, cols, "float32").astype(np.float32)), to_dev(rng.uniform(0.5, 1.5, cols).astype(np.float32))
        y, h = fa.rms_norm(x, weight, EPS, residual=res)
        room = batch + 40
        want = fa.BatchActs(room, cols, form).quantize(y)
        acts = fa.BatchActs(room, cols, form).quantize(torch.ones((room, cols), device="cuda"))
        beside = torch.zeros_like(y)
        got, h2 = fa.rms_norm(x, weight, EPS, residual=res, out=beside, acts=acts)
        assert got is acts and acts.batch == batch and torch.equal(h, h2) and torch.equal(beside, y)
        values = acts.values()
        assert values.shape == (batch, cols) and torch.equal(values, want.values())
        if form == "q8_k":
            q, d, _ = fo.quantize_q8_k(y[batch - 1].cpu().numpy())
            assert np.array_equal(values[batch - 1].cpu().numpy(), (q.reshape(-1, 256) * d[:, None]).astype(np.float32).reshape(-1))
            ws = [fa.Weights.from_host(k, make_weights(k, 96, cols, seed=k), 96, cols) for k in (fo.Q4_K, fo.Q5_K, fo.Q6_K)]
        elif form == "fp8":
            assert np.array_equal(values.cpu().numpy(), fp8_plain.quantize(y.cpu().numpy()).astype(np.float32))
            codes, scales = fp8_plain.random_matrix(rng, 140, cols)
            ws = [fa.Weights.from_device_fp8(to_dev(codes), to_dev(scales), 140, cols)]
            p, room_ = fp8_plain.product(codes[0], scales[0], y.cpu().numpy())
        else:
            assert np.array_equal(values.cpu().numpy(), plain.values(*plain.quantize(y.cpu().numpy())).astype(np.float32))
            codes, scales = plain.random_matrix(rng, 140, cols)
            ws = [fa.Weights.from_device(fa.MXFP4, to_dev(plain.blocks(codes, scales).reshape(-1)), 140, cols)]
            p, room_ = plain.product(codes, scales, y.cpu().numpy())
        for w in ws:
            a, b = w.gemm_acts(acts), w.gemm_acts(want)
            assert torch.equal(a, b)
        if form != "q8_k":
            assert (np.abs(a.cpu().numpy() - p) <= room_).all()
        if form == "fp8" and batch >= 9:
            assert torch.equal(a, ws[0].gemm(y))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("form", list(FORMS))
def test_quantized_output_of_two_byte_rows(fa, kind, form):
    """What is quantized is y in f32, not rounded to the rows' type."""
    rng = np.random.default_rng(4)
    for batch, cols in ((3, 768), (70, 1280), (1, 17152)):
        x, res = (_rows(rng, batch, cols, kind) for _ in range(2))
        weight = rng.uniform(0.5, 1.5, cols).astype(np.float32)
        acts = fa.BatchActs(batch, cols, form)
        fa.rms_norm(_dev(x, kind), to_dev(weight), EPS, residual=_dev(res, kind), acts=acts)
        _, y = plain.norm(x, res, weight, EPS, _rounded(kind))
        assert np.array_equal(acts.values().cpu().numpy(), fa.BatchActs(batch, cols, form).quantize(to_dev(y)).values().cpu().numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [200, 4096, 20000])
def test_rows_that_are_no_numbers_or_zero(fa, cols):
    rng = np.random.default_rng(cols)
    x = _rows(rng, 9, cols, "float32")
    x[1, 7], x[3, -1], x[5, 0], x[6] = np.nan, np.inf, -np.inf, 0
    x[7] = np.float32(3e38)
    x[8] *= 2.0 ** -140
    x = x.astype(np.float32).astype(np.float64)
    for eps in (EPS, 0.0, 1e-300):
        y, h = fa.rms_norm(to_dev(x.astype(np.float32)), None, eps)
        _, want = plain.norm(x, None, None, eps, None)
        assert np.array_equal(y.cpu().numpy(), want, equal_nan=True), eps
    for form in ("fp8", "mxfp4"):
        n = cols // 32 * 32
        acts = fa.BatchActs(9, n, form)
        fa.rms_norm(to_dev(x[:, :n].astype(np.float32)), None, EPS, acts=acts)
        _, want = plain.norm(x[:, :n], None, None, EPS, None)
        want = fp8_plain.quantize(want) if form == "fp8" else plain.values(*plain.quantize(want))
        assert np.array_equal(acts.values().cpu().numpy(), want.astype(np.float32), equal_nan=True)


@pytest.mark.gpu
def test_sums_past_the_range_of_the_type(fa):
    """f16 rows whose sum with the residual is an infinity there; bf16 sums halfway between two numbers."""
    x = _rounded("float16")(np.full((1, 64), 60000.0))
    y, h = fa.rms_norm(_dev(x, "float16"), None, EPS, residual=_dev(x, "float16"))
    assert np.isinf(h.float().cpu().numpy()).all() and np.isnan(y.float().cpu().numpy()).all()
    a = np.tile(np.array([1.0, 1.0 + 2.0 ** -7, 2.0, -1.0]), 16)[None]
    b = np.full((1, 64), 2.0 ** -8)
    _, h = fa.rms_norm(_dev(a, "bfloat16"), None, EPS, residual=_dev(b, "bfloat16"))
    assert np.array_equal(h.double().cpu().numpy(), _rounded("bfloat16")(a + b))


@pytest.mark.gpu
def test_on_several_streams_and_in_a_graph(fa):
    """A decoding step: the norm, three projections over its quantized rows; captured, replayed between eager calls of other batches."""
    import torch
    rng = np.random.default_rng(6)
    cols = 1024
    for form in ("q8_k", "fp8", "mxfp4"):
        print("norm in a graph", form, flush=True)
        if form == "q8_k":
            ws = [fa.Weights.from_host(k, make_weights(k, 300, cols, seed=k), 300, cols) for k in (fo.Q4_K, fo.Q5_K, fo.Q6_K)]
        elif form == "fp8":
            ws = [fa.Weights.from_device_fp8(*(to_dev(v) for v in fp8_plain.random_matrix(rng, 300, cols)), 300, cols) for _ in range(3)]
        else:
            ws = [fa.Weights.from_device(fa.MXFP4, to_dev(plain.blocks(*plain.random_matrix(rng, 300, cols)).reshape(-1)), 300, cols) for _ in range(3)]
        weight = to_dev(rng.uniform(0.5, 1.5, cols).astype(np.float32))
        for batch in (1, 20, 200):
            xs = [to_dev(_rows(rng, b, cols, "float32").astype(np.float32)) for b in (batch, 7)]
            res = [to_dev(_rows(rng, b, cols, "float32").astype(np.float32)) for b in (batch, 7)]
            acts = [fa.BatchActs(max(batch, 7), cols, form) for _ in range(2)]
            stream = torch.cuda.Stream()
            h, ys = torch.zeros_like(xs[0]), [torch.zeros((batch, 300), device="cuda") for _ in ws]

            def step(i, out=None, sum_out=None):
                a, s = fa.rms_norm(xs[i], weight, EPS, residual=res[i], sum_out=sum_out, acts=acts[i])
                return [s] + [w.gemm_acts(a, out=None if out is None else o) for w, o in zip(ws, out or ws)]
            want, other = step(0), step(1)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                step(0, ys, h)
                stream.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    step(0, ys, h)
                for rep in range(3):
                    for t in [h] + ys:
                        t.zero_()
                    g.replay()
                    for a, b in zip(step(1), other):
                        assert torch.equal(a, b)
                    stream.synchronize()
                    assert all(torch.equal(a, b) for a, b in zip([h] + ys, want)), rep


@pytest.mark.gpu
def test_rows_past_32_bits(fa):
    import torch
    print("norm past 2^32 bytes", flush=True)
    batch, cols = 2 ** 19 + 5, 4224
    x = torch.randn((batch, cols), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    weight = torch.rand(cols, device="cuda")
    acts = fa.BatchActs(batch, cols, "fp8")
    y, h = fa.rms_norm(x, weight, EPS, residual=x, out=torch.empty_like(x), acts=acts)[0], None
    values, plain_y = acts.values(), fa.rms_norm(x, weight, EPS, residual=x)[0]
    for s in (slice(0, 3), slice(batch // 2, batch // 2 + 3), slice(batch - 7, batch)):
        ph, py = plain.norm(x[s].cpu().numpy(), x[s].cpu().numpy(), weight.cpu().numpy(), EPS, lambda v: v.astype(np.float64))
        assert np.array_equal(plain_y[s].cpu().numpy(), py)
        assert np.array_equal(values[s].cpu().numpy(), fp8_plain.quantize(py).astype(np.float32))


# ---- refusals ----
def test_the_library_refuses_before_anything_runs():
    import frink_amd as fa
    L = fa.lib()
    room = np.zeros(4096, np.float32)
    p, q = C.c_void_p(room.ctypes.data), C.c_void_p(room.ctypes.data + 8192)

    def norm(kind=0, x=p, residual=None, weight_kind=0, weight=None, eps=EPS, batch=1, cols=64, total=None, y=q, acts=None):
        return L.frk_hip_rms_norm_dev(kind, x, residual, weight_kind, weight, eps, batch, cols, total, y, acts, None)
    for rc, status in [(norm(x=None), fa.ERR_ARG), (norm(y=None), fa.ERR_ARG), (norm(total=q), fa.ERR_ARG), (norm(kind=3), fa.ERR_UNSUPPORTED),
                       (norm(kind=-1), fa.ERR_UNSUPPORTED), (norm(weight=p, weight_kind=9), fa.ERR_UNSUPPORTED), (norm(eps=-1e-9), fa.ERR_ARG),
                       (norm(eps=float("nan")), fa.ERR_ARG), (norm(eps=float("inf")), fa.ERR_ARG), (norm(batch=0), fa.ERR_SHAPE), (norm(cols=0), fa.ERR_SHAPE),
                       (norm(batch=(1 << 30) + 1), fa.ERR_SHAPE), (norm(cols=(1 << 23) + 1), fa.ERR_SHAPE)]:
        assert rc == status and fa.last_error()


@pytest.mark.gpu
def test_operands_that_do_not_fit_are_refused(fa):
    import torch
    x = torch.ones((3, 64), device="cuda")
    w = torch.ones(64, device="cuda")
    fa.rms_norm(x, w)
    for call in (lambda: fa.rms_norm(x.double()), lambda: fa.rms_norm(x.t()), lambda: fa.rms_norm(x[:0]), lambda: fa.rms_norm(x, w[:63]), lambda: fa.rms_norm(x, w.cpu()),
                 lambda: fa.rms_norm(x, w, residual=x.half()), lambda: fa.rms_norm(x, w, residual=x[:2]), lambda: fa.rms_norm(x, w, residual=x.cpu()),
                 lambda: fa.rms_norm(x, w, out=x[:2]), lambda: fa.rms_norm(x, w, out=x.bfloat16()), lambda: fa.rms_norm(x, w, sum_out=x[:, :32]),
                 lambda: fa.rms_norm(torch.ones((), device="cuda"))):
        with pytest.raises(ValueError):
            call()
    y = torch.empty_like(x)
    with pytest.raises(fa.BackendError) as e:
        fa.rms_norm(x, w, residual=x, out=y, sum_out=y)
    assert e.value.code == fa.ERR_ARG
    acts = fa.BatchActs(2, 64, "fp8")
    for bad in (x, x[:2, :32].contiguous()):
        with pytest.raises(fa.BackendError) as e:
            fa.rms_norm(bad, None, acts=acts)
        assert e.value.code == fa.ERR_SHAPE and acts.batch == 0


@pytest.mark.gpu
@pytest.mark.parametrize("form", list(FORMS))
def test_a_refused_norm_leaves_the_batch_as_it_was(fa, form):
    """The outputs of values() and gemm_acts are sized by what the object holds, also behind a refusal."""
    import torch
    x = torch.randn((3, 256), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    acts = fa.BatchActs(3, 256, form).quantize(x)
    want = acts.values()
    for bad in (torch.ones((4, 256), device="cuda"), x[:, :128].contiguous()):
        with pytest.raises(fa.BackendError):
            fa.rms_norm(bad, acts=acts)
        assert acts.batch == 3 and torch.equal(acts.values(), want)
    with pytest.raises(ValueError):
        fa.rms_norm(x, acts=acts, out=torch.empty((2, 256), device="cuda"))
    assert acts.batch == 3 and torch.equal(acts.values(torch.empty((3, 256), device="cuda")), want)
    with pytest.raises(ValueError):
        acts.values(torch.empty((2, 256), device="cuda"))
    acts.release()
    with pytest.raises(ValueError):
        fa.rms_norm(x, acts=acts, sum_out=torch.empty_like(x))
