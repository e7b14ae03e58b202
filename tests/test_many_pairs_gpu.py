"""Nearly 2^31 pairs, where the last blocks' pair numbers pass 2^31, and the sizes at which the sort of moe_dispatch changes its kernels."""
import pytest
import torch

pytestmark = pytest.mark.gpu

K, TOKENS = 128, 2 ** 24 - 1
PAIRS = K * TOKENS                    # 2^31 - 128: less than a block below 2^31


def ids_of(experts):
    """All pairs to expert 0 but the last token's: to the last expert, and its last two to none."""
    ids = torch.zeros(TOKENS, K, dtype=torch.int32, device="cuda")
    ids[-1] = experts - 1
    ids[-1, -2], ids[-1, -1] = -1, experts
    return ids


def is_arange(t, n, step=1 << 28):
    return all(torch.equal(t[i:min(i + step, n)], torch.arange(i, min(i + step, n), dtype=t.dtype, device="cuda")) for i in range(0, n, step))


@pytest.mark.parametrize("experts", [2, 1025])
def test_dispatch_and_combine(cuda, experts):
    import torch_ggml_ops_b200 as tgo

    torch.cuda.empty_cache()
    ids = ids_of(experts)
    x = torch.arange(TOKENS, device="cuda").remainder(7).bfloat16()[:, None].expand(TOKENS, 8).contiguous()
    rows, at, indices, ends = tgo.moe_dispatch(x, ids, experts)
    del ids
    flat = at.reshape(-1)
    assert is_arange(flat, PAIRS - 2) and flat[-2:].tolist() == [-1, -1]
    assert ends.tolist() == [PAIRS - K] * (experts - 1) + [PAIRS - 2] and is_arange(indices, experts)
    assert torch.equal(rows[-K:-2], x[-1:].expand(K - 2, 8)) and not rows[-2:].any() and torch.equal(rows[::K], x)
    y = tgo.moe_combine(rows, at)
    assert torch.equal(y[:-1], (x[:-1].float() * K).bfloat16()) and torch.equal(y[-1], (x[-1].float() * (K - 2)).bfloat16())


def test_the_sort_and_the_plan_of_one_rank(cuda):
    from torch_ggml_ops_b200 import native

    torch.cuda.empty_cache()
    ids = ids_of(2).reshape(-1)
    to_pair, to_sorted, _, ends = native.route_sort(ids, 2)
    del ids
    assert ends.tolist() == [PAIRS - K, PAIRS - 2]
    assert is_arange(to_pair, PAIRS - 2) and is_arange(to_sorted, PAIRS - 2) and to_sorted[-2:].tolist() == [-1, -1]
    del to_pair
    row, plan_ends, overflow = torch.empty(PAIRS, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    native.local_plan(to_sorted, ends, PAIRS - 70, row, plan_ends, overflow)
    assert is_arange(row, PAIRS - 70) and bool((row[-70:] == -1).all()) and plan_ends.tolist() == [PAIRS - K, PAIRS - 70] and overflow.tolist() == [1]


@pytest.mark.parametrize("tokens,k,experts", [(4096, 1, 7), (4097, 1, 7), (512, 8, 1024), (512, 8, 1025), (1025, 4, 1024), (1025, 4, 1025), (2000, 8, 4096), (5, 1024, 300),
                                              (4, 1024, 300)])
def test_where_the_sort_changes(cuda, tokens, k, experts):
    """Up to 4096 pairs in one launch, more by counts per block, and with more than 1024 experts by the sort of the expert-parallel layer."""
    import torch_ggml_ops_b200 as tgo
    from torch_ggml_ops_b200 import native

    g = torch.Generator(device="cuda").manual_seed(tokens)
    for low, high in ((-1, experts + 1), (experts - 1, experts), (-3, 0)):      # any, all to the last, none
        ids = torch.randint(low, high, (tokens, k), device="cuda", generator=g, dtype=torch.int32)
        x = torch.randn(tokens, 16, device="cuda", generator=g).bfloat16()
        rows, at, indices, ends = tgo.moe_dispatch(x, ids, experts)
        named = ((ids >= 0) & (ids < experts)).reshape(-1)
        order = torch.sort(torch.where(named, ids.reshape(-1).long(), experts), stable=True).indices
        n = int(named.sum())
        want_at = torch.full((tokens * k,), -1, dtype=torch.int32, device="cuda")
        want_at[order[:n]] = torch.arange(n, dtype=torch.int32, device="cuda")
        counts = torch.bincount(ids.reshape(-1)[named], minlength=experts)
        assert torch.equal(at.reshape(-1), want_at) and torch.equal(ends.long(), counts.cumsum(0)) and torch.equal(indices, torch.arange(experts, device="cuda"))
        assert torch.equal(rows[:n], x[order[:n] // k]) and not rows[n:].any()
        _, to_sorted, ei, eo = native.route_sort(ids.reshape(-1), experts)
        assert torch.equal(to_sorted, at.reshape(-1)) and torch.equal(ei, indices) and torch.equal(eo, ends)
