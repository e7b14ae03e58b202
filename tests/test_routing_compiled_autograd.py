"""Backward passes of the routing operators under compiled autograd: on meta tensors, without a GPU, and on one, where they give the eager
pass's bits, whatever was compiled before them."""
import pytest
import torch

DEVICES = ["meta", pytest.param("cuda", marks=pytest.mark.gpu)]


def compiled(program):
    from torch._dynamo import compiled_autograd

    with compiled_autograd._enable(lambda g: torch.compile(g, backend="aot_eager")):
        return program()


def same(got, want, device):
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.shape == b.shape and a.dtype == b.dtype and (device == "meta" or torch.equal(a, b))


def data(device, n, experts=16, k=3, width=24):
    if device == "cuda":
        torch.manual_seed(n)
    logits = torch.randn(n, experts, device=device, requires_grad=True)
    x = torch.randn(n, width, device=device).bfloat16().requires_grad_()
    rows = torch.randn(n * k, width, device=device).bfloat16().requires_grad_()
    w = torch.rand(n, k, device=device).requires_grad_()
    ids = (torch.arange(n * k, device=device).reshape(n, k) * 7 % (experts + 2) - 1).int()
    at = (n * k - 1 - torch.arange(n * k, device=device)).reshape(n, k).int()
    return logits, x, rows, w, ids, at


@pytest.mark.parametrize("device", DEVICES)
def test_each_operator_in_every_form(device):
    import torch_ggml_ops_b200 as tgo

    torch._dynamo.reset()
    for n in (9, 9, 14, 5):                               # a graph again, and of other sizes
        logits, x, rows, w, ids, at = data(device, n)
        programs = [(lambda s=s, v=v: tgo.moe_router(logits, 3, scoring=s, normalize=v)[0], [logits]) for s in ("softmax", "sigmoid") for v in (True, False)]
        programs += [(lambda s=s: tgo.moe_balance_loss(logits, ids, scoring=s)[0], [logits]) for s in ("softmax", "sigmoid")]
        programs += [(lambda: tgo.moe_dispatch(x, ids, 16)[0], [x])]
        for leaves in ([rows, w], [rows], [w]):
            programs += [(lambda: tgo.moe_combine(rows, at, w), leaves)]
        programs += [(lambda: tgo.moe_combine(rows, at), [rows]), (lambda: tgo.moe_combine(rows.detach(), at, w), [w]), (lambda: tgo.moe_combine(rows, at, w.detach()), [rows])]
        for make, leaves in programs:
            y = make()
            dy = torch.ones_like(y) if device == "meta" else torch.randn_like(y)
            want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
            same(compiled(lambda: torch.autograd.grad(y, leaves, dy, retain_graph=True)), want, device)
            same(torch.autograd.grad(y, leaves, dy), want, device)          # what the graph keeps is as it was
            with pytest.raises(RuntimeError, match="second time"):
                compiled(lambda: torch.autograd.grad(y, leaves, dy))
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone() if device == "cuda" else t, lambda t: t):
                z = make()
            same(compiled(lambda: torch.autograd.grad(z, leaves, dy)), want, device)


@pytest.mark.parametrize("device", DEVICES)
def test_a_layer(device):
    import torch_ggml_ops_b200 as tgo

    torch._dynamo.reset()

    def step(logits, x):
        weights, ids = tgo.moe_router(logits, 3)
        rows, at, _, _ = tgo.moe_dispatch(x, ids, 16)
        (tgo.moe_combine(tgo.swiglu(rows, rows * 2), at, weights).float().sum() + tgo.moe_balance_loss(logits, ids)[0]).backward()
        got = [t.grad for t in (logits, x)]
        logits.grad = x.grad = None
        return got

    for n in (9, 30, 17):
        logits, x = data(device, n)[:2]
        want = step(logits, x)
        same(compiled(lambda: step(logits, x)), want, device)
