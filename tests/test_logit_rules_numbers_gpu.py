"""Penalties given as numbers are fp32 numbers: what is no positive one there is refused as a repetition penalty."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_repetition_penalties_at_the_end_of_the_range(cuda):
    import torch_ggml_ops_b200 as tgo

    x = torch.tensor([[1.0, -1.0, 0.0, 2.0 ** -100]], device="cuda")
    h = torch.arange(4, device="cuda")
    for bad in (1e-60, 2.0 ** -151, 0.0, -1e-60, math.nan):
        with pytest.raises(RuntimeError, match="positive"):
            tgo.logit_rules(x, history=h, repetition_penalty=bad)
    least = 2.0 ** -149
    assert tgo.logit_rules(x, history=h, repetition_penalty=least).tolist() == [[math.inf, -least, 0.0, 2.0 ** 49]]
    assert tgo.logit_rules(x, history=h, repetition_penalty=2.0 ** 120).tolist() == [[2.0 ** -120, -(2.0 ** 120), 0.0, 0.0]]
