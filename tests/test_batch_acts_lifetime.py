"""How long a BatchActs lives: released or dropped while something is captured, and beside the graphs that it is part of."""
import ctypes as C
import gc

import numpy as np
import pytest

import mxfp4_plain as plain
import oracle as fo
from test_gpu_parity import fa, make_weights, to_dev  # noqa: F401 (fa: the module's fixture)

FORMS = ("q8_k", "fp8", "mxfp4")


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("how", ["released", "dropped"])
def test_an_object_that_ends_during_a_capture_leaves_the_capture_alone(fa, form, how):
    """A norm is captured; between its calls an object that it has nothing to do with ends."""
    import torch
    print("an object", how, "during a capture", form, flush=True)
    rng = np.random.default_rng(1)
    x, weight = to_dev(rng.standard_normal((3, 256)).astype(np.float32)), to_dev(rng.uniform(0.5, 1.5, 256).astype(np.float32))
    want = fa.rms_norm(x, weight)[0]
    acts = fa.BatchActs(3, 256, form).quantize(x)
    assert np.isfinite(acts.values().cpu().numpy()).all()
    y, z, stream, graph = torch.empty_like(x), torch.empty_like(x), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        fa.rms_norm(x, weight, out=y)
        if how == "released":
            acts.release()
            assert not acts.handle
        del acts
        gc.collect()
        fa.rms_norm(x, weight, out=z)
    for _ in range(3):
        y.zero_(), z.zero_()
        graph.replay()
        assert torch.equal(fa.rms_norm(x, weight)[0], want)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(z, want)


@pytest.mark.gpu
@pytest.mark.parametrize("decoded", [False, True])
def test_a_matrix_dropped_during_a_capture_leaves_the_capture_alone(fa, decoded):
    import torch
    print("a matrix dropped during a capture", decoded, flush=True)
    rng = np.random.default_rng(3)
    x, weight = to_dev(rng.standard_normal((3, 256)).astype(np.float32)), to_dev(rng.uniform(0.5, 1.5, 256).astype(np.float32))
    want = fa.rms_norm(x, weight)[0]
    w = fa.Weights.from_device(fa.MXFP4, to_dev(plain.blocks(*plain.random_matrix(rng, 64, 256)).reshape(-1)), 64, 256)
    if decoded:
        w.keep_decoded()
    y, stream, graph = torch.empty_like(x), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        del w
        gc.collect()
        fa.rms_norm(x, weight, out=y)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


class _Library:
    """The library's entry points, of which the calls are kept and nothing else."""

    def __init__(self):
        self.released = []

    def frk_hip_batch_acts_create_form(self, max_batch, cols, form, out):
        out._obj.value = 4096 + form
        return 0

    def frk_hip_batch_acts_release(self, handle):
        self.released.append(handle.value)
        return 0

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("use", ["quantize", "values", "rms_norm", "gemm_acts", "nothing"])
@pytest.mark.parametrize("stream,capturing", [(0, False), (7, False), (7, True)])
def test_what_a_graph_holds_is_kept_until_its_release(monkeypatch, form, use, stream, capturing):
    """Dropped, an object frees its memory, in every form; not one that a captured call has used.  (On the CPU: a graph over freed memory is not run.)"""
    import torch

    import frink_amd as fa
    library = _Library()
    monkeypatch.setattr(fa, "_lib", library)
    monkeypatch.setattr(fa, "lib", lambda: library)
    monkeypatch.setattr(fa, "_stream_raw", lambda torch: stream)
    monkeypatch.setattr(fa, "_stream", lambda: C.c_void_p(stream))
    monkeypatch.setattr(fa, "_fp8_stream", lambda torch, x, others=(): stream)
    monkeypatch.setattr(fa, "_float_type", lambda torch, x, which=None: 0)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    x, y = torch.zeros((2, 256)), torch.zeros((2, 256))
    for again in (False, True):  # (a later call that no graph holds changes nothing)
        acts = fa.BatchActs(2, 256, form)
        acts.batch = 2
        for n in range(1 + again):
            if n:
                monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
            if use == "quantize":
                acts.quantize(x)
            elif use == "values":
                acts.values(out=y)
            elif use == "rms_norm":
                fa.rms_norm(x, out=y, acts=acts)
            elif use == "gemm_acts":
                fa.Weights(None, fa.MXFP4, 256, 256).gemm_acts(acts, out=y)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
        handle = acts.handle.value
        del acts
        gc.collect()
        kept = capturing and use != "nothing"
        assert library.released == ([] if kept else [handle]), (form, use)
        library.released.clear()
    if capturing:
        acts = fa.BatchActs(2, 256, form).quantize(x)
        acts.release()  # (the caller's word that no graph is replayed any more)
        assert library.released == [4096 + FORMS.index(form)] and acts.handle is None
        del acts
        gc.collect()
        assert len(library.released) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_an_object_dropped_behind_its_calls(fa, form):
    """Calls are under way when the object ends, and its memory is asked for again at once; a graph's object that its program dropped."""
    import torch
    print("dropped behind its calls", form, flush=True)
    rng = np.random.default_rng(2)
    cols, rows, batch = 1024, 640, 40
    x = to_dev(rng.standard_normal((batch, cols)).astype(np.float32))
    if form == "q8_k":
        w = fa.Weights.from_host(fo.Q4_K, make_weights(fo.Q4_K, rows, cols, seed=3), rows, cols)
    elif form == "fp8":
        w = fa.Weights.from_device_fp8(torch.randint(0, 100, (rows, cols), dtype=torch.uint8, device="cuda"), torch.ones((5, 8), device="cuda"), rows, cols)
    else:
        w = fa.Weights.from_device(fa.MXFP4, to_dev(plain.blocks(*plain.random_matrix(rng, rows, cols)).reshape(-1)), rows, cols)
    acts = fa.BatchActs(batch, cols, form)
    want = w.gemm_acts(fa.rms_norm(x, acts=acts)[0])
    torch.cuda.synchronize()
    ys = [torch.empty_like(want) for _ in range(4)]
    for y in ys:
        mine = fa.BatchActs(batch, cols, form)
        w.gemm_acts(fa.rms_norm(x, acts=mine)[0], out=y)
        del mine
        fa.BatchActs(batch, cols, form).quantize(torch.full_like(x, 9.0))
    assert all(torch.equal(y, want) for y in ys)
    stream, graph, y = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.empty_like(want)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        w.gemm_acts(fa.rms_norm(x, acts=acts)[0], out=y)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        w.gemm_acts(fa.rms_norm(x, acts=acts)[0], out=y)
    del acts
    gc.collect()
    for _ in range(3):
        y.zero_()
        others = [fa.BatchActs(batch, cols, form).quantize(torch.full_like(x, 9.0)) for _ in range(4)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and len(others) == 4
