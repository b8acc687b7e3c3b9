"""Calls over weights in 8-bit floating point together with other kinds, at the ends of the range, and what they refuse."""
import numpy as np
import pytest

import fp8_plain as plain
import oracle as fo
from test_fp8_blocks import _activations, _resident
from test_gpu_parity import fa, make_weights, to_dev  # noqa: F401 (fa: the module's fixture)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [28672, 32768])
def test_several_kinds_over_one_activation(fa, cols):
    """Both sides of the longest row that its product's launch quantizes; a second call finds the scratch memory as large as it needs."""
    import torch
    print("fp8 beside K-quants", cols, flush=True)
    rng = np.random.default_rng(cols)
    rows = 64
    f8 = [_resident(fa, *plain.random_matrix(rng, rows, cols)) for _ in range(2)]
    k = [fa.Weights.from_host(kind, make_weights(kind, rows, cols, seed=kind), rows, cols) for kind in (fo.Q4_K, fo.Q5_K, fo.Q6_K)]
    x = to_dev(_activations(rng, 1, cols)[0])
    alone = {w: w.gemv(x) for w in f8}
    acts = fa.quantize_q8_k(x)
    alone.update((w, w.gemv_q8k(acts)) for w in k)
    for ws in ([f8[0], k[0]], [k[0], f8[0], k[1], f8[1], k[2]], [k[2], f8[1]], [f8[0], f8[1], k[1]]):
        for _ in range(2):
            for got, w in zip(fa.gemv_multi(ws, x), ws):
                assert torch.equal(got, alone[w])
    hidden = 96
    down = fa.Weights.from_host(fo.Q8_0, make_weights(fo.Q8_0, hidden, rows, seed=1), hidden, rows)
    d = down.dequant().cpu().numpy().astype(np.float64).reshape(hidden, rows)
    for gate, up in ((f8[0], k[0]), (k[2], f8[1])):
        g, u = (alone[w].cpu().numpy().astype(np.float64) for w in (gate, up))
        with np.errstate(over="ignore"):
            act = g / (1 + np.exp(-g)) * u
        # an exponential of a few units in its last place, a sum, a quotient, a product; then `rows` products and sums in f32
        room = (16 + 2 * rows) * 2.0 ** -24 * (np.abs(d) @ np.abs(act))
        for _ in range(2):
            got = fa.ffn_swiglu(gate, up, down, x).cpu().numpy()
            assert (np.abs(got - d @ act) <= room).all()
