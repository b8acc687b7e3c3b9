"""The shapes that a norm's operands may have."""
import numpy as np
import pytest

from test_gpu_parity import fa, to_dev  # noqa: F401 (fa: the module's fixture)

OTHERS = [(64, 3), (192,), (1, 192), (3, 64, 1), (1, 3, 64), (6, 32)]  # as many values as (3, 64)


class _Library:
    def __init__(self):
        self.norms = 0

    def frk_hip_rms_norm_dev(self, *args):
        self.norms += 1
        return 0


@pytest.mark.parametrize("which", ["residual", "sum_out", "out"])
@pytest.mark.parametrize("shape", OTHERS)
def test_operands_of_another_shape_are_refused(monkeypatch, which, shape):
    """Also where they have as many values: read in x's order they would be other rows."""
    import torch

    import frink_amd as fa
    library = _Library()
    monkeypatch.setattr(fa, "lib", lambda: library)
    monkeypatch.setattr(fa, "_fp8_stream", lambda torch, x, others=(): 0)
    monkeypatch.setattr(fa, "_float_type", lambda torch, x, which=None: 0)
    x = torch.ones((3, 64))
    with pytest.raises(ValueError, match="beside activations"):
        fa.rms_norm(x, **{which: torch.ones(shape)})
    assert library.norms == 0
    fa.rms_norm(x, **{which: torch.ones((3, 64))})
    fa.rms_norm(torch.ones(shape), **{which: torch.ones(shape)})
    assert library.norms == 2


@pytest.mark.gpu
@pytest.mark.parametrize("shape", OTHERS + [(64,), (2, 3, 5, 32)])
def test_rows_of_any_number_of_dimensions(fa, shape):
    """All but the last dimension are rows; outputs have the operands' shape."""
    import torch
    rng = np.random.default_rng(len(shape))
    x, res = (to_dev(rng.standard_normal(shape).astype(np.float32)) for _ in range(2))
    flat = x.view(-1, shape[-1])
    want, h = fa.rms_norm(flat, residual=res.view(flat.shape))
    y, s = torch.empty_like(x), torch.empty_like(x)
    for got in (fa.rms_norm(x, residual=res), fa.rms_norm(x, residual=res, out=y, sum_out=s)):
        assert got[0].shape == got[1].shape == x.shape
        assert torch.equal(got[0].view(flat.shape), want) and torch.equal(got[1].view(flat.shape), h)
