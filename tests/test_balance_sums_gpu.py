"""The balance loss over very many tokens that are all alike, whose additions all round the same way."""
import pytest
import torch

from routing_ref import U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,experts,scoring", [(1 << 28, 3, "softmax"), ((1 << 26) + 7, 8, "sigmoid"), ((1 << 21) + 1, 200, "softmax")])
def test_many_equal_tokens(cuda, tokens, experts, scoring):
    import torch_ggml_ops_b200 as tgo

    row = torch.randn(1, experts, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    loss, counts = tgo.moe_balance_loss(row.expand(tokens, experts).contiguous(), torch.zeros(tokens, 1, dtype=torch.int32, device="cuda"), scoring=scoring)
    x = row[0].double()
    score = torch.softmax(x, 0) if scoring == "softmax" else torch.sigmoid(x) / torch.sigmoid(x).sum()
    want = float(experts * score[0])
    # 256 tokens of a warp and 8 warps are added in fp32, each step off by U of the sum at most; a share by some 60 U (exponents, their sum, the division)
    assert abs(float(loss) - want) <= (256 + 8 + 60) * U * want
    assert counts.tolist() == [tokens] + [0] * (experts - 1)
