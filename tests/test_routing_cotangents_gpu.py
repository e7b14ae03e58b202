"""Cotangents of the routing operators as autograd makes them: parts of a larger tensor that start at any element, transposed ones, numbers
that were expanded.  Each gives the bits that the same values in a plain tensor give."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def data():
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(-1, 9, (21, 3), device="cuda", generator=g).int()
    x = torch.randn(21, 24, device="cuda", generator=g).bfloat16().requires_grad_()
    w = torch.rand(21, 3, device="cuda", generator=g).requires_grad_()
    logits = torch.randn(21, 16, device="cuda", generator=g).requires_grad_()
    return ids, x, w, logits


def programs():
    import torch_ggml_ops_b200 as tgo

    ids, x, w, logits = data()
    rows, at, _, _ = tgo.moe_dispatch(x, ids, 8)
    r = rows.detach().requires_grad_()
    return [(lambda: tgo.moe_dispatch(x, ids, 8)[0], [x]), (lambda: tgo.moe_combine(r, at, w), [r, w]), (lambda: tgo.moe_combine(r, at), [r]),
            (lambda: tgo.moe_router(logits, 3)[0], [logits]), (lambda: tgo.moe_balance_loss(logits, ids.clamp(max=15))[0].reshape(1, 1), [logits])]


def test_parts_of_a_larger_tensor(cuda):
    for make, leaves in programs():
        y = make()
        dy = torch.randn_like(y)
        want = torch.autograd.grad(y, leaves, dy)
        for off in (0, 1, 3, 4, 8, 11):
            flat = torch.zeros(y.numel() + 16, dtype=y.dtype, device="cuda")
            part = flat[off:off + y.numel()].view(y.shape)
            part.copy_(dy)
            assert part.is_contiguous() and part.data_ptr() % 16 == off * y.element_size() % 16
            for a, b in zip(torch.autograd.grad(make(), leaves, part), want):
                assert torch.equal(a, b)
            # the same from a program: elements joined in front
            joined = torch.cat([torch.zeros(off, dtype=y.dtype, device="cuda"), make().reshape(-1)])
            for a, b in zip(torch.autograd.grad(joined, leaves, torch.cat([flat[:off], dy.reshape(-1)])), want):
                assert torch.equal(a, b)
        for a, b in zip(torch.autograd.grad(make(), leaves, dy.t().contiguous().t()), want):
            assert torch.equal(a, b)
        one = torch.ones((), dtype=y.dtype, device="cuda").expand(y.shape)
        for a, b in zip(torch.autograd.grad(make(), leaves, one), torch.autograd.grad(make(), leaves, torch.ones_like(y))):
            assert torch.equal(a, b)


def test_in_a_compiled_program(cuda):
    for make, leaves in programs():
        y = make()
        total = lambda: (torch.cat([y.new_ones(3), make().reshape(-1)]) * torch.arange(3 + y.numel(), device="cuda").to(y.dtype)).float().sum()   # noqa: E731
        torch._dynamo.reset()
        compiled = torch.compile(total, backend="aot_eager")
        for a, b in zip(torch.autograd.grad(compiled(), leaves), torch.autograd.grad(total(), leaves)):
            assert torch.equal(a, b)


def test_the_gradient_of_dispatch_by_itself(cuda):
    """The operator, its refusals and its own gradient: the sum over a token's pairs, so that of a row is its token's."""
    import torch_ggml_ops_b200 as tgo

    op = torch.ops.torch_ggml_ops_b200.moe_dispatch_grad
    ids, x, _, _ = data()
    rows, at, _, _ = tgo.moe_dispatch(x.detach(), ids, 8)
    g = torch.randn_like(rows).requires_grad_()
    d = op(g, at)
    assert torch.equal(d, tgo.moe_combine(g.detach(), at))
    dd = torch.randn_like(d)
    (back,) = torch.autograd.grad(d, g, dd)
    assert torch.equal(back, tgo.moe_dispatch(dd, ids, 8)[0])
    assert op(g[:0], at).eq(0).all() and op(g.detach(), at[:0]).shape == (0, 24)
    for bad, needle in (((g.float(), at), "like the rows"), ((g[None], at), "like the rows"), ((g[:, :12], at), "like the rows"), ((g, at.long()), "row_of_pair"),
                        ((g, at.cpu()), "row_of_pair"), ((g, at[:, :0]), "top_k")):
        with pytest.raises(RuntimeError, match=needle):
            op(*bad)
    torch.library.opcheck(op.default, (g, at), test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
