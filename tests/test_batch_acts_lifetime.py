"""How long a BatchActs lives: released or dropped while something is captured, and beside the graphs that it is part of."""
import gc

import numpy as np
import pytest

import mxfp4_plain as plain
from test_gpu_parity import fa, to_dev  # noqa: F401 (fa: the module's fixture)

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
