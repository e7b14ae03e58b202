"""What ``moe_combine`` holds until its backward pass: the rows only for a gradient of the weights, the weights only for one of the rows.  On
meta tensors, without a GPU, and on one."""
import pytest
import torch


@pytest.mark.parametrize("device", ["meta", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_what_is_not_needed_is_not_kept(device):
    import torch_ggml_ops_b200 as tgo

    def inputs():
        leaf_r = torch.ones(12, 16, device=device, dtype=torch.bfloat16, requires_grad=True)
        leaf_w = torch.full((4, 3), 0.5, device=device, requires_grad=True)
        return leaf_r, leaf_w, torch.arange(12, device=device).reshape(4, 3).int()

    for weights in ("none", "plain", "wanted"):
        leaf_r, leaf_w, at = inputs()
        rows = leaf_r * 1
        w = {"none": None, "plain": leaf_w.detach().clone(), "wanted": leaf_w * 1}[weights]
        y = tgo.moe_combine(rows, at, w)
        with torch.no_grad():
            rows.zero_()                                   # written over after the forward pass
        if weights == "wanted":
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                torch.autograd.grad(y.float().sum(), leaf_r)
            continue
        (d,) = torch.autograd.grad(y.float().sum(), leaf_r)
        assert d.shape == leaf_r.shape
        if device == "cuda":
            assert bool((d == (1.0 if w is None else 0.5)).all())
    # weights alone: the rows are needed, the weights themselves are not
    leaf_r, leaf_w, at = inputs()
    w = leaf_w * 1
    y = tgo.moe_combine(leaf_r.detach(), at, w)
    with torch.no_grad():
        w.zero_()
    (d,) = torch.autograd.grad(y.float().sum(), leaf_w)
    assert d.shape == leaf_w.shape and (device == "meta" or bool((d == 16.0).all()))
    # rows alone: the weights are needed
    leaf_r, leaf_w, at = inputs()
    w = leaf_w.detach().clone()
    y = tgo.moe_combine(leaf_r, at, w)
    w.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y.float().sum(), leaf_r)


@pytest.mark.gpu
def test_the_rows_memory_is_free_until_the_backward_pass(cuda):
    import torch_ggml_ops_b200 as tgo

    n, width = 1 << 14, 2048                               # 64 MB of rows
    at = torch.arange(n, device="cuda").reshape(-1, 8).int()
    leaf = torch.ones(1, width, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = tgo.moe_combine(leaf.expand(n, width).contiguous(), at)
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert held < 1 << 20, held
    (d,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert d.shape == leaf.shape


@pytest.mark.gpu
def test_the_gradient_of_rows_alone_has_the_same_bits(cuda):
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator(device="cuda").manual_seed(3)
    ops = torch.ops.torch_ggml_ops_b200
    rows = torch.randn(70, 264, device="cuda", generator=g).bfloat16()
    at = torch.randint(-2, 75, (30, 4), device="cuda", generator=g).int()
    w = torch.randn(30, 4, device="cuda", generator=g)
    dy = torch.randn(30, 264, device="cuda", generator=g).bfloat16()
    for weights in (w, None):
        want = ops.moe_combine_grad(dy, rows, at, weights, True, True)[0]
        assert torch.equal(ops.moe_combine_rows_grad(dy, at, weights, 70), want)
        leaf = rows.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(tgo.moe_combine(leaf, at, weights), leaf, dy)[0], want)
    assert ops.moe_combine_rows_grad(dy, at, w, 0).shape == (0, 264)
    assert ops.moe_combine_rows_grad(dy[:0], at[:0], w[:0], 5).eq(0).all()
    for bad, needle in (((dy, at, w, -1), "number of rows"), ((dy, at, w, 1 << 31), "number of rows"), ((dy[:3], at, w, 70), "grad must be"), ((dy, at.long(), w, 70), "row_of_pair"),
                        ((dy, at, w[:3], 70), "one entry per pair"), ((dy[:, :12], at, w, 70), "multiple of 8"), ((dy.float(), at, w, 70), "bfloat16"),
                        ((dy, at[:, :0], None, 70), "top_k")):
        with pytest.raises(RuntimeError, match=needle):
            ops.moe_combine_rows_grad(*bad)
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(ops.moe_combine_rows_grad.default, (dy, at, w, 70), test_utils=tests)
