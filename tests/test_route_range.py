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
