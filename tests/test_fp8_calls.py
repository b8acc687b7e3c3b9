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


def _ends(rng, end, matrices, rows, cols, batch):
    """Codes, scales and activations whose products are f32's largest (the results far below) or smallest (far above)."""
    sign = rng.integers(0, 2, (matrices, rows, cols), dtype=np.uint8) << 7
    blocks = (matrices, -(-rows // 128), -(-cols // 128))
    if end == "largest":
        codes, scales = sign | np.uint8(0x7e), np.full(blocks, 2.0 ** -30, np.float32)
        x = rng.uniform(0.5, 1.0, (batch, cols)) * np.finfo(np.float32).max
    else:
        codes, scales = sign | rng.integers(0, 4, sign.shape, dtype=np.uint8), np.full(blocks, 2.0 ** 100, np.float32)
        x = rng.integers(0, 20, (batch, cols)) * 2.0 ** -109
    x *= rng.choice([-1, 1], x.shape)
    x[batch // 2] = np.abs(x[batch // 2])
    if end == "largest" and batch != 4:
        x[batch // 2, :128] = np.finfo(np.float32).max  # with rows of one sign the largest sum there is
    return codes, scales, x.astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("end", ["largest", "smallest"])
@pytest.mark.parametrize("batch", [1, 4, 16, 30, 64, 100, 300])
def test_products_at_the_ends_of_the_range(fa, end, batch):
    """Sums of codes times activations that f32 does not hold, or holds as subnormal numbers only, under scales that bring them back."""
    print("fp8 range", end, batch, flush=True)
    rng = np.random.default_rng(batch)
    codes, scales, x = _ends(rng, end, 2, 140, 1300, batch)
    for m in range(2):  # one sign: the sums reach the end
        codes[m, ::5] &= 0x7f
    want, room = np.empty((batch, 280)), np.empty((batch, 280))
    for m in range(2):
        want[:, 140 * m:140 * (m + 1)], room[:, 140 * m:140 * (m + 1)] = plain.product(codes[m], scales[m], x)
    w = _resident(fa, codes, scales)
    got = w.gemm(to_dev(x)).cpu().numpy()
    assert (np.abs(got - want) <= room).all()
    off = np.array([0, batch // 3, batch], np.int32)
    got = fa.gemm_grouped(w, 2, to_dev(off), to_dev(x)).cpu().numpy()
    for m in range(2):
        s, r = slice(off[m], off[m + 1]), slice(140 * m, 140 * (m + 1))
        assert (np.abs(got[s] - want[s, r]) <= room[s, r]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 60])
def test_expert_layer_over_the_largest_activations(fa, batch):
    from test_fp8_blocks import _plain_layer
    rng = np.random.default_rng(batch)
    experts, hidden, ffn = 4, 260, 200
    codes, _, x = _ends(rng, "largest", 2 * experts, ffn, hidden, batch)
    scales = np.full((2 * experts, 2, 3), 2.0 ** -132, np.float32)
    parts = [(codes[:experts], scales[:experts]), (codes[experts:], scales[experts:]), plain.random_matrix(rng, hidden, ffn, matrices=experts)]
    gate, up, down = (_resident(fa, *p) for p in parts)
    ids = rng.integers(0, experts, (batch, 2)).astype(np.int32)
    weights = rng.uniform(0.2, 1, (batch, 2)).astype(np.float32)
    got = fa.moe_ffn(gate, up, down, experts, to_dev(x), to_dev(ids), to_dev(weights)).cpu().numpy()
    want, room = _plain_layer(parts, x, ids, weights)
    assert (np.abs(got - want) <= room * 1.01).all()
    y = fa.ffn_swiglu(_resident(fa, codes[:1], scales[:1]), _resident(fa, codes[4:5], scales[:1]), _resident(fa, *(p[:1] for p in parts[2])), to_dev(x[0]))
    want, room = _plain_layer([(codes[:1], scales[:1]), (codes[4:5], scales[:1]), tuple(p[:1] for p in parts[2])], x[:1], [[0]], [[1.0]])
    assert (np.abs(y.cpu().numpy() - want[0]) <= room[0] * 1.01).all()


class _On:
    """A tensor that says it is on a device `step` further on, which this machine need not have."""

    def __init__(self, t, step=1):
        self.t, self.step = t, step

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.t.get_device() + self.step


@pytest.mark.gpu
def test_every_tensor_of_a_call_is_on_the_current_device(fa):
    import torch
    rng = np.random.default_rng(2)
    w = _resident(fa, *plain.random_matrix(rng, 128, 128))
    x, y = torch.zeros((1, 128), device="cuda"), torch.zeros((1, 128), device="cuda")
    ids, weights = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.ones((1, 1), device="cuda")
    off = to_dev(np.array([0, 1], np.int32))
    calls = [lambda t: w.gemm(x, out=t(y)), lambda t: w.gemv(x, out=t(y)), lambda t: w.gemm_noalloc(x, t(y)), lambda t: fa.gemm_pair(w, w, x, outs=(y, t(y))),
             lambda t: fa.gemv_multi([w, w], x, outs=[t(y), y]), lambda t: fa.ffn_swiglu(w, w, w, t(x)), lambda t: fa.ffn_swiglu(w, w, w, x, out=t(y)),
             lambda t: fa.moe_ffn(w, w, w, 1, x, t(ids), weights), lambda t: fa.moe_ffn(w, w, w, 1, x, ids, t(weights)),
             lambda t: fa.moe_ffn(w, w, w, 1, x, ids, weights, out=t(y)), lambda t: fa.gemm_grouped(w, 1, t(off), x),
             lambda t: fa.gemm_grouped(w, 1, off, x, gather=t(ids)), lambda t: fa.gemm_grouped(w, 1, off, x, out=t(y)), lambda t: w.get_rows(t(ids))]
    for call in calls:
        call(lambda t: t)
        with pytest.raises(ValueError, match="current device"):
            call(_On)
    for call in calls[7:10]:  # (host memory)
        with pytest.raises(ValueError, match="device -1"):
            call(lambda t: t.cpu())


@pytest.mark.gpu
def test_the_other_kinds_take_a_peers_memory(fa):
    """As they did before there were FP8_BLOCK matrices; host memory has to be page-locked."""
    import torch
    n = 256
    q = fa.Weights.from_host(fo.Q8_0, make_weights(fo.Q8_0, n, n, seed=1), n, n)
    gate, down = (fa.Weights.from_host(fo.Q4_K, make_weights(fo.Q4_K, 2 * n, n, seed=s), 2 * n, n) for s in (2, 3))
    rng = np.random.default_rng(3)
    x = to_dev(rng.standard_normal((2, n)).astype(np.float32))
    ids, weights = to_dev(np.array([[0], [1]], np.int32)), torch.ones((2, 1), device="cuda")
    off = to_dev(np.array([0, 1, 2], np.int32))
    for call in (lambda t: q.gemm(t(x)), lambda t: q.gemv(t(x[0])), lambda t: q.gemm_noalloc(t(x), torch.zeros_like(x)), lambda t: fa.gemm_pair(gate, down, t(x))[1],
                 lambda t: fa.gemv_multi([q, q], t(x[0]))[1], lambda t: fa.ffn_swiglu(q, q, q, t(x[0])), lambda t: fa.gemm_grouped(gate, 2, t(off), t(x)),
                 lambda t: fa.moe_ffn(gate, gate, down, 2, t(x), t(ids), t(weights)), lambda t: q.get_rows(t(ids[:, 0].contiguous()))):
        assert torch.equal(call(lambda t: t), call(_On))
    want = fa.moe_ffn(gate, gate, down, 2, x, ids, weights)
    assert torch.equal(fa.moe_ffn(gate, gate, down, 2, x, ids.cpu().pin_memory(), weights.cpu().pin_memory()), want)
    for call in (lambda: fa.moe_ffn(gate, gate, down, 2, x, ids.cpu(), weights), lambda: fa.moe_ffn(gate, gate, down, 2, x, ids, weights.cpu()),
                 lambda: fa.gemv_multi([q], x[0].cpu()), lambda: fa.ffn_swiglu(q, q, q, x[0].cpu())):
        with pytest.raises(AssertionError):
            call()


@pytest.mark.gpu
def test_operands_without_room_are_refused(fa):
    """Nothing is launched: the calls would read or write past a tensor's end, or into other values than floats."""
    import torch
    rng = np.random.default_rng(2)
    n = 256
    w = _resident(fa, *plain.random_matrix(rng, n, n))
    x, y = torch.zeros((3, n), device="cuda"), torch.zeros((3, n), device="cuda")
    ids, weights, off = torch.zeros((3, 1), dtype=torch.int32, device="cuda"), torch.ones((3, 1), device="cuda"), to_dev(np.array([0, 3], np.int32))
    for call in (lambda out: w.gemv(x[0], out=out), lambda out: w.gemm(x, out=out), lambda out: fa.gemm_pair(w, w, x, outs=(y, out)),
                 lambda out: fa.gemv_multi([w, w], x[0], outs=[y[0], out]), lambda out: fa.ffn_swiglu(w, w, w, x[0], out=out),
                 lambda out: fa.moe_ffn(w, w, w, 1, x, ids, weights, out=out), lambda out: fa.gemm_grouped(w, 1, off, x, out=out)):
        call(y)
        for bad in (y.flatten()[:n - 1], y.half(), y.int(), torch.zeros((n, 3), device="cuda").t()):
            with pytest.raises(ValueError, match="contiguous floats"):
                call(bad)
    for call in (lambda: fa.moe_ffn(w, w, w, 1, x[:2], ids, weights), lambda: fa.moe_ffn(w, w, w, 1, x, ids, weights[:2])):
        with pytest.raises(ValueError, match="3 x 1 ids"):
            call()
    for bad in (x[0, :n - 1], x[0].double(), x[:, 0].repeat(n, 1)[:, 0]):
        for call in (lambda: fa.gemv_multi([w], bad), lambda: fa.ffn_swiglu(w, w, w, bad)):
            with pytest.raises(ValueError, match="contiguous floats"):
                call()
    with pytest.raises(ValueError, match="outputs"):
        fa.gemv_multi([w, w], x[0], outs=[y[0]])


def test_host_codes_are_bytes():
    import frink_amd
    for codes in (np.full((2, 6), 1.5, np.float32), np.full((2, 6), 300), np.full((2, 6), -1)):
        with pytest.raises(ValueError, match="bytes"):
            frink_amd.Weights.from_host_fp8(codes, np.ones(1, np.float32), 2, 6)


@pytest.mark.gpu
def test_host_codes_of_any_byte_type(fa):
    """One byte a code, taken as it lies; whole numbers that are bytes."""
    codes = np.random.default_rng(1).permutation(256).astype(np.uint8).reshape(4, 64)
    codes[(codes & 0x7f) == 0x7f] = 0
    for c in (codes, codes.view(np.int8), codes.astype(np.int64), codes.view(np.dtype("V1"))):
        got = fa.Weights.from_host_fp8(c, np.full(1, 2.0), 4, 64).dequant().cpu().numpy()
        assert np.array_equal(got, plain.VALUES[codes].astype(np.float32) * 2)


@pytest.mark.gpu
def test_matrices_past_32_bits(fa):
    """4.8 GB of codes, as one matrix and as a stack: the first and the last rows."""
    import torch
    print("fp8, weights past 2^32 bytes", flush=True)
    rows, cols, stack = 8 * (2 ** 18 + 128), 2304, 8
    gen = torch.Generator("cuda").manual_seed(1)
    codes = torch.randint(0, 127, (rows, cols), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.rand((rows // 128, cols // 128), device="cuda", generator=gen) * 2.0 ** -8
    w = fa.Weights.from_device_fp8(codes, scales, rows, cols)
    rng = np.random.default_rng(1)
    x = _activations(rng, 100, cols)
    picked = [slice(0, 128), slice(rows - 128, rows), slice(rows // 2, rows // 2 + 128)]
    parts = [(codes[s].cpu().numpy(), scales[s.start // 128:s.start // 128 + 1].cpu().numpy()) for s in picked]
    for batch in (1, 12, 40, 100):
        y = w.gemm(to_dev(x[:batch]))
        for s, p in zip(picked, parts):
            want, room = plain.product(*p, x[:batch])
            assert (np.abs(y[:, s].cpu().numpy() - want) <= room).all(), (batch, s)
    assert np.array_equal(w.get_rows(to_dev(np.array([rows - 1], np.int32))).cpu().numpy()[0], plain.dequant(*parts[1])[-1].astype(np.float32))
    w = fa.Weights.from_device_fp8(codes, scales, rows, cols, matrices=stack)
    del codes
    for pairs in (10, 100):
        off = np.minimum(np.arange(stack + 1) * (pairs // stack), pairs).astype(np.int32)
        off[-1] = pairs
        y = fa.gemm_grouped(w, stack, to_dev(off), to_dev(x[:pairs]))
        want, room = plain.product(*parts[1], x[off[-2]:pairs])
        assert (np.abs(y[off[-2]:, -128:].cpu().numpy() - want) <= room).all(), pairs


@pytest.mark.gpu
def test_batches_past_32_bits(fa):
    """8.9 GB of activations, 4.4 GB quantized, 2^31 results and more: the first and the last tokens."""
    import torch
    print("fp8, activations past 2^32 bytes", flush=True)
    rows, cols, batch = 4160, 4224, 2 ** 19 + 5
    rng = np.random.default_rng(2)
    codes, scales = plain.random_matrix(rng, rows, cols)
    w = _resident(fa, codes, scales)
    x = torch.randn((batch, cols), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    y = w.gemm(x)
    assert y.numel() > 2 ** 31
    for s in (slice(0, 3), slice(batch // 2, batch // 2 + 3), slice(batch - 7, batch)):
        want, room = plain.product(codes[0], scales[0], x[s].cpu().numpy())
        assert (np.abs(y[s].cpu().numpy() - want) <= room).all(), s


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [34, 300])
def test_lists_that_point_outside_over_tiles(fa, pairs):
    """As for a few pairs: offsets are clamped and made non-decreasing, gather entries clamped, rows of no group left as they were."""
    import torch
    rng = np.random.default_rng(pairs)
    codes, scales = plain.random_matrix(rng, 150, 140, matrices=4)
    x = _activations(rng, 6, 140)
    w = _resident(fa, codes, scales)
    gather = rng.integers(-3, 9, pairs).astype(np.int32)
    gather[[0, 7]] = 2 ** 31 - 1, -2 ** 31
    for off in ([2, 5, 3, 4, 8], [-7, 4, 100000, 2, 6], [3] * 5, [0, pairs, 0, pairs, 0], [9, 40, 31, 33, pairs - 1], [-2 ** 31, 20, 2 ** 31 - 1, 0, 0]):
        y = torch.full((pairs, 150), 7.5, device="cuda")
        fa.gemm_grouped(w, 4, to_dev(np.array(off, np.int32)), to_dev(x), gather=to_dev(gather), out=y)
        got = y.cpu().numpy()
        top = np.maximum.accumulate(np.clip(off, 0, pairs))
        seen = np.zeros(pairs, bool)
        for g in range(4):
            s = slice(top[g], top[g + 1])
            seen[s] = True
            if top[g + 1] > top[g]:
                want, room = plain.product(codes[g], scales[g], x[np.clip(gather[s], 0, 5)])
                assert (np.abs(got[s] - want) <= room).all(), (off, g)
        assert (got[~seen] == 7.5).all(), off


@pytest.mark.gpu
@pytest.mark.parametrize("batch,k", [(1, 6), (4, 6), (20, 6), (300, 3)])
def test_expert_layer_over_any_ids(fa, batch, k):
    """The same expert twice, ids that are no expert's, tokens without any: what is no expert adds nothing."""
    from test_fp8_blocks import _layer, _plain_layer
    rng = np.random.default_rng(batch)
    experts, hidden, ffn = 8, 260, 132
    parts, (gate, up, down) = _layer(fa, rng, experts, hidden, ffn)
    x = _activations(rng, batch, hidden)
    ids = rng.integers(-2, experts + 2, (batch, k)).astype(np.int32)
    ids[0, 0], ids[0, 1] = 2 ** 31 - 1, -2 ** 31
    ids[0, 2:4] = 5 if k > 3 else 1
    ids[batch // 2] = ids[batch // 2] if batch < 3 else -1
    weights = rng.standard_normal((batch, k)).astype(np.float32)
    got = fa.moe_ffn(gate, up, down, experts, to_dev(x), to_dev(ids), to_dev(weights)).cpu().numpy()
    want, room = _plain_layer(parts, x, ids, weights)
    assert (np.abs(got - want) <= room * 1.01).all()
    if batch > 2:
        assert (got[batch // 2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,batch", [(517, 4100, 70), (1000, 8192, 130), (999, 7000, 300)])
def test_shares_of_the_columns_into_unaligned_outputs(fa, rows, cols, batch):
    import torch
    rng = np.random.default_rng(rows)
    w = _resident(fa, *plain.random_matrix(rng, rows, cols))
    x = to_dev(_activations(rng, batch, cols))
    want = w.gemm(x)
    y = torch.full((batch * rows + 2,), 3.0, device="cuda")
    w.gemm(x, out=y[1:-1])
    assert torch.equal(y[1:-1].view(batch, rows), want) and float(y[0]) == 3.0 and float(y[-1]) == 3.0
