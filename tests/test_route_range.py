"""Routing by a rule at the ends of its range: more tokens than one launch holds, scores that 64 bits do not tell apart."""
import numpy as np
import pytest

import fp8_plain as plain
from test_gpu_parity import fa, to_dev  # noqa: F401 (fa: the module's fixture)


@pytest.mark.gpu
def test_more_tokens_than_a_launch_holds(fa):
    import torch
    print("route, 2^25 + 7 tokens", flush=True)
    logits = torch.randn((2 ** 25 + 7, 2), generator=torch.Generator("cuda").manual_seed(3), device="cuda")
    ids, w = fa.route(logits, 1, norm=False)
    assert torch.equal(ids[:, 0], (logits[:, 1] > logits[:, 0]).int())
    want = 1 / (1 + torch.exp(-(logits[:, 0].double() - logits[:, 1].double()).abs()))
    # (rounded to f32 once, behind a handful of roundings in 64 bits)
    assert bool(((w[:, 0].double() - want).abs() <= want * (2.0 ** -24 + 2.0 ** -45)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rule,logits,bias,chosen", [
    (dict(score="sigmoid"), {3: 40.0, 9: 60.0, 20: 50.0, 30: 20.0}, None, [3, 9, 20, 30]),          # all one but the last
    (dict(score="sigmoid"), {i: -900.0 + i for i in range(40)}, None, [0, 1, 2, 3]),                # all zero
    (dict(score="sigmoid"), {i: (i + 1) * 1e-25 for i in range(40)}, None, [0, 1, 2, 3]),           # all a half
    (dict(score="softmax"), {i: -800.0 + i for i in range(39)} | {39: 0.0, 38: -1.0}, None, [39, 38, 0, 1]),
    (dict(score="sigmoid"), {i: i / 8 for i in range(40)}, 2.0 ** 60, [0, 1, 2, 3]),                # the bias alone
    (dict(score="sigmoid", groups=4, top_groups=2, group_best=2), {5: 40.0, 6: 41.0, 12: 90.0, 13: 90.0, 33: 50.0, 34: 50.0}, None, [5, 6, 12, 13])])
def test_scores_that_are_equal_in_64_bits_go_by_index(fa, rule, logits, bias, chosen):
    l = np.full((3, 40), -5.0, np.float32)
    l[:, list(logits)] = list(logits.values())
    b = None if bias is None else np.full(40, bias, np.float32)
    ids, w = fa.route(to_dev(l), 4, bias=None if b is None else to_dev(b), **rule)
    assert ids.cpu().numpy().tolist() == [chosen] * 3
    with np.errstate(over="ignore"):
        want_ids, want = plain.route(l, 4, bias=b, **rule)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    assert (np.abs(w.cpu().numpy() - want) <= want * (2.0 ** -24 + 2.0 ** -45) + 2.0 ** -150).all()


@pytest.mark.parametrize("rule", [dict(groups=2 ** 32 + 1), dict(groups=2, top_groups=2 ** 32 + 2), dict(group_best=2 ** 35 + 1), dict(groups=1 - 2 ** 32)])
def test_numbers_of_groups_past_32_bits(rule):
    import types

    import frink_amd
    import torch

    class Logits(types.SimpleNamespace):
        def contiguous(self):
            return self
    logits = Logits(dtype=torch.float32, is_cuda=True, dim=lambda: 2, shape=(1, 8))
    with pytest.raises(ValueError, match="groups"):
        frink_amd.route(logits, 1, **rule)
