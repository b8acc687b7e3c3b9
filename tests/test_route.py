"""Routing by a rule against its definition in 64 bits: scores, bias, groups, ties, masks; refusals."""
import ctypes as C

import numpy as np
import pytest

import fp8_plain as plain
from test_gpu_parity import fa, to_dev  # noqa: F401 (fa: the module's fixture)


def _check(fa, logits, k, bias=None, **rule):
    ids, w = fa.route(to_dev(logits), k, bias=None if bias is None else to_dev(bias), **rule)
    want_ids, want = plain.route(logits, k, bias=bias, **rule)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    # rounded to f32 once, behind a handful of roundings in 64 bits and two exponentials of a few units in its last places
    got = w.cpu().numpy()
    assert (np.abs(got - want) <= np.abs(want) * (2.0 ** -24 + 2.0 ** -45) + 2.0 ** -150).all()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("n_experts", [1, 2, 5, 63, 64, 65, 100, 128, 129, 256, 257, 384, 512, 513, 1000, 1024])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_number_of_experts(fa, n_experts, score):
    rng = np.random.default_rng(n_experts)
    logits = (rng.standard_normal((9, n_experts)) * 2).astype(np.float32)
    logits[1] = 0.25
    logits[2] = np.round(logits[2])  # many equal ones
    logits[3] *= 20
    logits[4, rng.random(n_experts) < 0.7] = -np.inf
    logits[5] = -np.inf
    logits[6, rng.random(n_experts) < 0.3] = np.nan
    logits[7, rng.integers(0, n_experts, 2)] = np.inf
    bias = (rng.standard_normal(n_experts) * 0.1).astype(np.float32)
    for k in sorted({1, min(8, n_experts), min(64, n_experts)}):
        for norm in (False, True):
            for b in (None, bias):
                _check(fa, logits, k, bias=b, score=score, norm=norm, scale=1.0 if norm else 2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("groups,size", [(2, 1), (2, 7), (8, 32), (4, 64), (8, 20), (3, 100), (16, 16), (64, 16), (64, 1), (12, 5), (33, 31),
                                         (32, 8), (4, 32), (8, 64), (2, 128), (3, 64), (6, 8), (5, 4)])
@pytest.mark.parametrize("group_best", [1, 2])
def test_groups(fa, groups, size, group_best):
    rng = np.random.default_rng(groups * size)
    n = groups * size
    logits = (rng.standard_normal((7, n)) * 1.5).astype(np.float32)
    logits[1] = 1.0                                 # all groups equal
    logits[2] = np.round(logits[2])
    logits[3, : (groups - 1) * size] = -np.inf      # one group left
    logits[4, ::2] = -np.inf
    logits[5] = -np.inf
    logits[6, size // 2:: size] = np.nan
    bias = (rng.standard_normal(n) * 0.2).astype(np.float32)
    for top_groups in sorted({1, (groups + 1) // 2, groups}):
        k = min(8, top_groups * size)
        for score in ("softmax", "sigmoid"):
            for b in (None, bias):
                _check(fa, logits, k, bias=b, score=score, groups=groups, top_groups=top_groups, group_best=group_best)


@pytest.mark.gpu
def test_scores_closer_than_an_f32_step_are_told_apart(fa):
    """Sigmoids above 15 are one in f32, and a bias of 1 swallows the last bits of small scores: the logits still decide."""
    logits = np.full((2, 130), -30, np.float32)
    logits[0, [3, 70, 129, 5]] = 20.0, 20.5, 21.0, 19.5
    logits[1, [9, 8, 100]] = -18.0, -18.5, -17.5
    bias = np.ones(130, np.float32)
    ids, _ = fa.route(to_dev(logits), 3, score="sigmoid", bias=to_dev(bias))
    assert ids.cpu().numpy().tolist() == [[129, 70, 3], [100, 9, 8]]
    _check(fa, logits, 3, bias=bias, score="sigmoid")


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 2, 3, 5, 64, 1000, 4099])
def test_batches(fa, batch):
    rng = np.random.default_rng(batch)
    logits = rng.standard_normal((batch, 48)).astype(np.float32)
    _check(fa, logits, 6, bias=(rng.standard_normal(48) * 0.1).astype(np.float32), score="sigmoid", groups=4, top_groups=2, group_best=2, scale=2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 128, 256, 512, 1024])
def test_logits_and_biases_of_any_alignment(fa, n):
    rng = np.random.default_rng(n)
    logits, bias = rng.standard_normal((5, n)).astype(np.float32), (rng.standard_normal(n) * 0.1).astype(np.float32)
    rule = dict(score="sigmoid", groups=4, top_groups=2, group_best=2)
    want_ids, want = plain.route(logits, 8, bias=bias, **rule)
    for logits_at, bias_at in ((1, 0), (0, 1), (2, 3)):
        x, b = (to_dev(np.concatenate([np.zeros(at, np.float32), v.ravel()]))[at:] for v, at in ((logits, logits_at), (bias, bias_at)))
        ids, w = fa.route(x.view(5, n), 8, bias=b, **rule)
        assert np.array_equal(ids.cpu().numpy(), want_ids) and np.allclose(w.cpu().numpy(), want, rtol=2.0 ** -23, atol=0)


@pytest.mark.gpu
def test_biases_that_are_no_numbers(fa):
    """A bias of -inf or NaN takes an expert out of the choice; one of +inf puts it first."""
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((4, 40)).astype(np.float32)
    bias = np.zeros(40, np.float32)
    bias[[4, 30]], bias[17], bias[25] = -np.inf, np.inf, np.nan
    for score in ("softmax", "sigmoid"):
        _check(fa, logits, 39, bias=bias, score=score)
        _check(fa, logits, 5, bias=bias, score=score, groups=4, top_groups=2, group_best=2)


@pytest.mark.gpu
def test_captured_and_replayed(fa):
    import torch
    rng = np.random.default_rng(4)
    logits = to_dev(rng.standard_normal((33, 256)).astype(np.float32))
    bias = to_dev((rng.standard_normal(256) * 0.1).astype(np.float32))
    rule = dict(score="sigmoid", bias=bias, groups=8, top_groups=4, group_best=2, scale=2.5)
    fa.route(logits, 8, **rule)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, w = fa.route(logits, 8, **rule)
    for _ in range(3):
        logits.copy_(to_dev(rng.standard_normal((33, 256)).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        again = fa.route(logits, 8, **rule)
        assert torch.equal(ids, again[0]) and torch.equal(w, again[1])


@pytest.mark.parametrize("batch,n,k,rule,code,needle", [
    (0, 8, 1, {}, "ERR_SHAPE", "empty"), (1, 0, 1, {}, "ERR_SHAPE", "empty"), (1, 8, 0, {}, "ERR_SHAPE", "top-k"),
    (1, 8, 9, {}, "ERR_SHAPE", "top-k"), (1, 1025, 8, {}, "ERR_SHAPE", "1024"), (1, 128, 65, {}, "ERR_SHAPE", "max 64"),
    (1, 8, 1, {"score": 2}, "ERR_UNSUPPORTED", "score"), (1, 8, 1, {"groups": 3}, "ERR_SHAPE", "groups"),
    (1, 8, 1, {"groups": 0}, "ERR_SHAPE", "groups"), (1, 130, 1, {"groups": 65}, "ERR_SHAPE", "groups"),
    (1, 8, 1, {"groups": 4, "top_groups": 5}, "ERR_SHAPE", "of 4 groups"), (1, 8, 1, {"groups": 4, "top_groups": 0}, "ERR_SHAPE", "of 4 groups"),
    (1, 8, 1, {"group_best": 3}, "ERR_SHAPE", "best"), (1, 8, 5, {"groups": 4, "top_groups": 2}, "ERR_SHAPE", "fewer"),
    (2 ** 31, 8, 1, {}, "ERR_SHAPE", "batch"),
])
def test_refusals(batch, n, k, rule, code, needle):
    import frink_amd as fa
    r = fa.RouteRule(0, 1, 1, 1, 1, 1.0, None)
    for name, v in rule.items():
        setattr(r, name, v)
    p = C.c_void_p(4096)
    assert fa.lib().frk_hip_route_dev(p, batch, n, k, C.byref(r), p, p, None) == getattr(fa, code)
    assert needle in fa.last_error()


def test_null_arguments():
    import frink_amd as fa
    r = fa.RouteRule(0, 1, 1, 1, 1, 1.0, None)
    p = C.c_void_p(4096)
    for args in ((None, C.byref(r), p, p), (p, None, p, p), (p, C.byref(r), None, p), (p, C.byref(r), p, None)):
        assert fa.lib().frk_hip_route_dev(args[0], 1, 8, 1, args[1], args[2], args[3], None) == fa.ERR_ARG


def test_python_refuses_an_unknown_score():
    import frink_amd as fa
    import types
    import torch
    fake = types.SimpleNamespace(dtype=torch.float32, is_cuda=True, dim=lambda: 2, contiguous=lambda: types.SimpleNamespace(shape=(1, 8)))
    with pytest.raises(ValueError, match="score"):
        fa.route(fake, 1, score="cosine")
