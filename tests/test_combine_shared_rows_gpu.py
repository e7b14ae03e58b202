"""The gradient of ``moe_combine`` for maps that name rows many times: the sum over the pairs, in their order, in a time that is linear in the
pairs.  Small whole numbers make every sum exact, so that the rows' gradients are equal to torch's."""
import pytest
import torch

import routing_ref as ref
from routing_ref import U, near

pytestmark = pytest.mark.gpu


def maps():
    """name -> (row_of_pair, rows)"""
    g = torch.Generator(device="cuda").manual_seed(8)
    rand = lambda lo, hi, *s: torch.randint(lo, hi, s, device="cuda", generator=g).int()   # noqa: E731
    twice = torch.randperm(6000, device="cuda", generator=g).remainder(3000).int().reshape(-1, 4)
    return {
        "every row by two": (twice, 3000),
        "one row": (torch.zeros(1500, 3, dtype=torch.int32, device="cuda"), 5),
        "the last row": (torch.full((700, 2), 255, dtype=torch.int32, device="cuda"), 256),
        "few rows": (rand(-2, 9, 2100, 2), 7),
        "256 and 257 rows": (rand(0, 257, 1025, 3), 257),
        "some rows twice": (torch.where(rand(0, 20, 4000, 1) == 0, rand(0, 4100, 4000, 1), torch.arange(4000, device="cuda").int()[:, None]), 4100),
        "a step and one pair": (rand(0, 400, 1025, 1), 400),
        "many rows": (rand(-1, 70001, 30000, 3), 70000),
        "very many rows": (torch.cat([rand(0, 1 << 24, 3000, 2), rand((1 << 24) - 9, (1 << 24) + 70, 3000, 2)]), (1 << 24) + 60),
        "one pair": (torch.zeros(1, 1, dtype=torch.int32, device="cuda"), 3),
        "one token": (torch.tensor([[2, 2, 0, 2]], dtype=torch.int32, device="cuda"), 3),
    }


@pytest.mark.parametrize("name", ["every row by two", "one row", "the last row", "few rows", "256 and 257 rows", "some rows twice", "a step and one pair", "many rows",
                                  "very many rows", "one pair", "one token"])
def test_sums_of_whole_numbers(cuda, name):
    import torch_ggml_ops_b200 as tgo

    at, n = maps()[name]
    g = torch.Generator(device="cuda").manual_seed(1)
    for width in (8, 264, 1288) if n < 1 << 20 else (8,):
        rows = torch.ones(n, width, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        for weights in (None, torch.randint(-2, 3, at.shape, device="cuda", generator=g).float().requires_grad_()):
            dy = torch.randint(-2, 3, (at.shape[0], width), device="cuda", generator=g).bfloat16()
            named = ((at >= 0) & (at < n)).reshape(-1)
            each = dy.float().repeat_interleave(at.shape[1], 0) * (1.0 if weights is None else weights.detach().reshape(-1, 1))
            want = torch.zeros(n, width, device="cuda").index_add_(0, at.reshape(-1)[named].long(), each[named]).bfloat16()
            leaves = [rows] if weights is None else [rows, weights]
            y = tgo.moe_combine(rows, at, weights)
            got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
            assert torch.equal(got[0], want)
            if weights is not None:
                assert torch.equal(got[1].reshape(-1), torch.where(named, dy.float().sum(1).repeat_interleave(at.shape[1]), 0.0))
            for _ in range(2):
                assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy, retain_graph=True), got))


def test_sums_of_any_numbers(cuda):
    """Against 64 bits; the same bits every time, as the order of a sum is that of the pairs."""
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator().manual_seed(2)
    at = torch.randint(-1, 41, (300, 5), generator=g).int()
    rows, w, dy = torch.randn(40, 72, generator=g).bfloat16(), torch.randn(300, 5, generator=g), torch.randn(300, 72, generator=g).bfloat16()
    d_rows, size, d_w, w_size = ref.combine_grad(dy, rows, at, w)
    rd, wd = rows.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = tgo.moe_combine(rd, at.cuda(), wd)
    got = torch.autograd.grad(y, [rd, wd], dy.cuda(), retain_graph=True)
    most = int(torch.bincount(at[(at >= 0) & (at < 40)]).max())
    # a sum of c products in fp32: each of its c steps is off by U of no more than the sum of the sizes; then the rounding to bf16
    room = most * U * size
    near(got[0], d_rows, room + 2.0 ** -8 * (d_rows.abs() + room))
    near(got[1], d_w, (72 / 32 + 8) * U * w_size)
    for _ in range(5):
        again = torch.autograd.grad(y, [rd, wd], dy.cuda(), retain_graph=True)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


def test_captured_with_maps_that_change(cuda):
    """A graph's map may name rows once in one replay and many times in the next."""
    import torch_ggml_ops_b200 as tgo

    once = torch.arange(600, device="cuda").int().reshape(200, 3)
    often = once.remainder(17).contiguous()
    at, rows = once.clone(), torch.randn(600, 24, device="cuda").bfloat16()
    dy = torch.randn(200, 24, device="cuda").bfloat16()

    def step():
        leaf = rows.detach().requires_grad_()
        return torch.autograd.grad(tgo.moe_combine(leaf, at), leaf, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for m in (often, once, often, once):
        at.copy_(m)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())


def test_half_a_million_pairs(cuda):
    """Every row named by two pairs, and every pair naming one row: milliseconds, where a search of the map for every pair took seconds."""
    ops = torch.ops.torch_ggml_ops_b200
    pairs, k, width = 1 << 19, 8, 64
    dy = torch.ones(pairs // k, width, dtype=torch.bfloat16, device="cuda")
    for at, n, want in ((torch.randperm(pairs, device="cuda").remainder(pairs // 2).int(), pairs // 2, 2.0), (torch.zeros(pairs, dtype=torch.int32, device="cuda"), 1, float(pairs))):
        at = at.reshape(-1, k)
        ops.moe_combine_rows_grad(dy, at, None, n)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        d = ops.moe_combine_rows_grad(dy, at, None, n)
        end.record()
        torch.cuda.synchronize()
        assert bool((d == want).all())
        assert start.elapsed_time(end) < 200.0
