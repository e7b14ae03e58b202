"""GPU tests of the routing operators (``routing.py``) against their definitions in 64 bits (``routing_ref.py``), at the
sizes and masks where they can go wrong, and of a whole layer built from them."""
import math

import pytest
import torch

import routing_ref as ref
from routing_ref import HALF_STEP, TINY, U, near

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def scores(tokens, experts, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + 1000 * tokens + experts)
    return (torch.randn(tokens, experts, generator=g) * spread).to(dtype)


def check_router(logits, k, scoring, normalize, mask=None, grad=True):
    import torch_ggml_ops_b200 as tgo

    x = logits.cuda().requires_grad_(grad)
    m = None if mask is None else mask.cuda()
    w, ids = tgo.moe_router(x, k, scoring=scoring, normalize=normalize, token_mask=m)
    want_w, want_ids = ref.router(logits, k, scoring, normalize, mask)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and not ids.requires_grad
    assert torch.equal(ids.cpu(), want_ids)
    # exponents are off by U of themselves, expf, log1pf and the division by a few U, the sum by one U per step of 5 + 32
    c = (2 * ref.spread(logits, scoring) + 50) * U
    near(w, want_w, c * want_w + 2.0 ** -126)
    if not grad:
        return w, ids
    g = torch.randn(w.shape, generator=torch.Generator().manual_seed(5))
    (dx,) = torch.autograd.grad(w, x, g.cuda())
    assert dx.dtype == logits.dtype and dx.shape == x.shape
    want, size = ref.router_grad(logits, want_ids, g, scoring, normalize)
    near(dx, want, 2 * c * size + HALF_STEP[logits.dtype] * (want.abs() + 2 * c * size) + TINY[logits.dtype] + 2.0 ** -120)
    return w, ids


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 256, 8), (3, 5, 5), (17, 32, 32), (9, 33, 2), (20, 64, 6), (7, 100, 7), (33, 128, 8), (70, 256, 8),
                                              (13, 255, 9), (5, 257, 10), (11, 512, 4), (6, 1000, 4), (4, 1024, 32), (3, 1023, 31)])
def test_router(cuda, dtype, scoring, normalize, tokens, experts, k):
    check_router(scores(tokens, experts, dtype), k, scoring, normalize)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_router_of_equal_scores_takes_the_lower_expert(cuda, dtype, scoring, normalize):
    x = scores(40, 96, dtype).round().clamp(-1, 1)       # three values only
    x[0] = 0.0
    x[1, ::2], x[1, 1::2] = 0.0, -0.0                     # zeros of both signs are equal
    x[2, 17:] = x[2, :79].clone()
    check_router(x, 9, scoring, normalize)
    y = torch.full((3, 300), 1.5, dtype=dtype)            # all equal, wider than a chunk of a lane
    check_router(y, 12, scoring, normalize)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("experts,k", [(8, 8), (40, 12), (64, 20), (128, 32), (100, 9), (256, 32), (512, 32), (1024, 32), (777, 17)])
def test_router_of_sorted_scores(cuda, dtype, experts, k):
    """The best all lie together, so that one lane of a warp holds many of them, or all that it has."""
    x = torch.empty(5, experts)
    ramp = torch.arange(experts) / 8.0
    x[0], x[1], x[2], x[3] = ramp, -ramp, ramp - 7, (ramp - experts / 16).abs()
    x[4] = torch.where(torch.arange(experts) % 32 < 4, 50 + ramp / 64, ramp / 64)
    check_router(x.to(dtype), k, "softmax", True)
    x[:, ::2] = -math.inf
    check_router(x.to(dtype), k, "softmax", False)


def test_router_of_nearly_equal_scores(cuda):
    """fp32 scores that differ in their last bits only, in every order."""
    base = torch.tensor([1.0, -1.0, 3.1, 1e-30, -1e-30, 77.0, 2.0 ** -130])
    x = torch.empty(7 * 6, 200)
    g = torch.Generator().manual_seed(2)
    for i in range(x.shape[0]):
        b = base[i % 7].view(torch.int32) + torch.randint(0, 4 if i < 21 else 4000, (200,), generator=g, dtype=torch.int32)
        x[i] = b.view(torch.float32)
    for k in (1, 8, 20, 32):
        check_router(x, k, "softmax", True, grad=False)
    # equal numbers among the best, and one behind them that is larger by the last bit only
    y = torch.zeros(64, 70)
    for i in range(64):
        y[i, : i + 3] = 2.0
        y[i, i + 5] = torch.nextafter(torch.tensor(2.0), torch.tensor(3.0))
        y[i, 69] = torch.nextafter(torch.tensor(2.0), torch.tensor(1.0))
    for k in (1, 4, 7, 31, 32):
        check_router(y, k, "sigmoid", True, grad=False)
        check_router(scores(30, 70, torch.float32, k).bfloat16().float(), k, "softmax", False, grad=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_router_with_experts_switched_off_and_padded_tokens(cuda, dtype, scoring, normalize):
    x = scores(24, 40, dtype)
    x[0] = -math.inf                                      # nothing left
    x[1, 3:] = -math.inf                                  # fewer left than asked for
    x[2, ::3] = -math.inf
    x[3] = torch.finfo(dtype).min                         # the type's lowest value is a score like any other
    x[4, 7] = torch.finfo(dtype).max
    x[5, :39] = torch.finfo(dtype).min
    x[6] = -100.0                                         # sigmoids that fp32 holds as (nearly) nothing
    x[7] = 100.0
    check_router(x, 6, scoring, normalize)
    mask = torch.arange(24) % 3 != 0
    dead = x.clone()
    dead[~mask] = math.nan                                # what padded tokens hold is not looked at
    w, ids = check_router(torch.where(mask[:, None], x, torch.zeros_like(x)), 6, scoring, normalize, mask)
    import torch_ggml_ops_b200 as tgo

    d = dead.cuda().requires_grad_()
    w2, ids2 = tgo.moe_router(d, 6, scoring=scoring, normalize=normalize, token_mask=mask.cuda())
    assert torch.equal(w, w2) and torch.equal(ids, ids2)
    (dx,) = torch.autograd.grad(w2.sum(), d)
    assert not dx[~mask.cuda()].any() and not torch.isnan(dx).any()
    none = torch.zeros(24, dtype=torch.bool)
    w3, ids3 = tgo.moe_router(d, 6, scoring=scoring, normalize=normalize, token_mask=none.cuda())
    assert not w3.any() and bool((ids3 == -1).all())


@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_router_shows_nan(cuda, scoring, normalize):
    import torch_ggml_ops_b200 as tgo

    x = scores(6, 50, torch.float32)
    clean, clean_ids = tgo.moe_router(x.cuda(), 4, scoring=scoring, normalize=normalize)
    x[1, 9] = math.nan
    x[2] = math.nan
    x[3, 5] = math.inf
    w, ids = tgo.moe_router(x.cuda(), 4, scoring=scoring, normalize=normalize)
    assert torch.isnan(w[1]).all() and torch.isnan(w[2]).all() and bool((ids[2] == -1).all()) and 9 not in ids[1]
    y = scores(6, 50, torch.float32)
    y.view(torch.int32)[4, 49] = -1                       # a NaN with its sign set
    for dtype in DTYPES:
        z = y.to(dtype)
        if dtype != torch.float32:
            z.view(torch.int16)[4, 49] = -1
        wy, idy = tgo.moe_router(z.cuda(), 4, scoring=scoring, normalize=normalize)
        assert torch.isnan(wy[4]).all() and 49 not in idy[4] and bool(torch.isfinite(wy[:4]).all())
    assert int(ids[3, 0]) == 5 and (torch.isnan(w[3, 0]) if scoring == "softmax" else bool(torch.isfinite(w[3]).all()))
    for t in (0, 4, 5):
        assert torch.equal(w[t], clean[t]) and torch.equal(ids[t], clean_ids[t])


def test_router_layouts(cuda):
    """Leading dimensions, rows that lie apart, rows that start at odd places, no tokens."""
    import torch_ggml_ops_b200 as tgo

    base = scores(15, 77, torch.bfloat16).cuda()
    w, ids = tgo.moe_router(base, 3)
    w2, ids2 = tgo.moe_router(base.reshape(3, 5, 77), 3)
    assert w2.shape == (3, 5, 3) and torch.equal(w2.reshape(15, 3), w) and torch.equal(ids2.reshape(15, 3), ids)
    w1, ids1 = tgo.moe_router(base[4], 3)
    assert w1.shape == (3,) and torch.equal(w1, w[4]) and torch.equal(ids1, ids[4])
    for at in (0, 1, 8):
        wide = torch.full((15, 96), 50.0, dtype=torch.bfloat16, device="cuda")
        wide[:, at:at + 77] = base
        view = wide[:, at:at + 77].detach().requires_grad_()
        w3, ids3 = tgo.moe_router(view, 3, normalize=False)
        plain = base.clone().requires_grad_()
        w4, ids4 = tgo.moe_router(plain, 3, normalize=False)
        assert torch.equal(w3, w4) and torch.equal(ids3, ids4)
        g = torch.randn_like(w3)
        assert torch.equal(torch.autograd.grad(w3, view, g)[0], torch.autograd.grad(w4, plain, g)[0])
    # a cotangent that is no plain tensor
    x = base.clone().requires_grad_()
    w5, _ = tgo.moe_router(x, 3)
    (dx,) = torch.autograd.grad(w5.sum(), x, retain_graph=True)
    assert torch.equal(dx, torch.autograd.grad(w5, x, torch.ones_like(w5))[0])
    e = torch.empty(0, 77, device="cuda", requires_grad=True)
    w6, ids6 = tgo.moe_router(e, 3)
    assert w6.shape == (0, 3) and ids6.shape == (0, 3) and torch.autograd.grad(w6.sum(), e)[0].shape == (0, 77)


@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_router_gradient_against_differences(cuda, scoring, normalize):
    import torch_ggml_ops_b200 as tgo

    x = scores(8, 12, torch.float32, 6)
    g = torch.randn(8, 3, generator=torch.Generator().manual_seed(1))
    xd = x.cuda().requires_grad_()
    w, ids = tgo.moe_router(xd, 3, scoring=scoring, normalize=normalize)
    (dx,) = torch.autograd.grad(w, xd, g.cuda())
    h = 2.0 ** -11                                        # no two scores are as near, so the choice stays
    for t in range(8):
        for e in range(12):
            ends = []
            for step in (h, -h):
                y = x[t:t + 1].double().clone()
                y[0, e] += step
                wy, iy = ref.router(y, 3, scoring, normalize)
                assert torch.equal(iy[0], ids[t].cpu())
                ends.append(float((wy[0] * g[t].double()).sum()))
            # third derivatives of the weights are below 1: h^2 / 6 of the cotangent's size, and fp32
            assert abs((ends[0] - ends[1]) / (2 * h) - float(dx[t, e])) < 1e-6 * (1 + float(g[t].abs().sum()))


def test_combine_gradients_against_differences(cuda):
    """The sums are linear in the rows and in the weights: the change of <out, dy> is the gradient, up to the sums' roundings."""
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator().manual_seed(12)
    at = ref.sort_rows(expert_ids(6, 3, 8, 5, 0.2), 8)[0]
    rows, w = torch.randn(18, 16, generator=g).bfloat16(), torch.randn(6, 3, generator=g)
    dy = torch.randn(6, 16, generator=g).bfloat16()
    rd, wd = rows.cuda().requires_grad_(), w.cuda().requires_grad_()
    d_rows, d_w = torch.autograd.grad(tgo.moe_combine(rd, at.cuda(), wd), [rd, wd], dy.cuda())
    value = lambda r, v: float((ref.combine(r, at, v)[0] * dy.double()).sum())   # noqa: E731
    base = value(rows, w)
    for t, s in ((0, 0), (2, 1), (5, 2)):
        moved = w.double().clone()
        moved[t, s] += 1.0
        assert abs(value(rows, moved) - base - float(d_w[t, s])) < 1e-4
    for r, c in ((0, 0), (7, 3), (17, 15)):
        moved = rows.double().clone()
        moved[r, c] += 1.0
        assert abs(value(moved, w) - base - float(d_rows[r, c])) <= 2.0 ** -8 * abs(float(d_rows[r, c])) + 1e-9


def test_refusals(cuda):
    import torch_ggml_ops_b200 as tgo

    x, ids = torch.randn(4, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    rows, w = torch.randn(8, 16, device="cuda").bfloat16(), torch.rand(4, 2, device="cuda")
    for call, needle in ((lambda: tgo.moe_router(x.double(), 2), "dtype"), (lambda: tgo.moe_router(x, 0), "top_k"), (lambda: tgo.moe_router(x, 9), "top_k"),
                         (lambda: tgo.moe_router(torch.zeros(2, 1025, device="cuda"), 2), "1024 experts"), (lambda: tgo.moe_router(x.t(), 2), "contiguous"),
                         (lambda: tgo.moe_router(x.reshape(2, 2, 8).transpose(0, 1), 2), "contiguous"),
                         (lambda: tgo.moe_router(x[:1].expand(4, 8), 2), "contiguous"), (lambda: tgo.moe_router(x[:, :0], 1), "empty"),
                         (lambda: tgo.moe_router(x, 2, token_mask=torch.ones(3, dtype=torch.bool, device="cuda")), "one entry per token"),
                         (lambda: tgo.moe_router(x, 2, token_mask=torch.ones(4, device="cuda")), "token_mask"),
                         (lambda: tgo.moe_router(x, 2, token_mask=torch.ones(4, dtype=torch.bool)), "token_mask"),
                         (lambda: tgo.moe_balance_loss(x, ids.long()), "expert_ids"), (lambda: tgo.moe_balance_loss(x, ids[:3]), "one row per row"),
                         (lambda: tgo.moe_balance_loss(x, ids.t().contiguous().t()), "contiguous"), (lambda: tgo.moe_balance_loss(x, ids[:, :0]), "top_k"),
                         (lambda: tgo.moe_dispatch(rows[:4].float(), ids, 8), "bfloat16"), (lambda: tgo.moe_dispatch(rows[:3], ids, 8), "one row per row"),
                         (lambda: tgo.moe_dispatch(rows[:4, :12].contiguous(), ids, 8), "multiple of 8"), (lambda: tgo.moe_dispatch(rows[:4], ids, 0), "num_experts"),
                         (lambda: tgo.moe_dispatch(rows[:4], ids, 4097), "num_experts"), (lambda: tgo.moe_dispatch(rows[:4], ids.long(), 8), "expert_ids"),
                         (lambda: tgo.moe_dispatch(rows.reshape(-1)[1:65].reshape(4, 16), ids, 8), "16 bytes"),
                         (lambda: tgo.moe_dispatch(rows[::2], ids, 8), "contiguous"), (lambda: tgo.moe_combine(rows, ids.long(), w), "row_of_pair"),
                         (lambda: tgo.moe_combine(rows, ids, w[:3]), "one entry per pair"), (lambda: tgo.moe_combine(rows, ids, w.half()), "weights"),
                         (lambda: tgo.moe_combine(rows, ids, w.cpu()), "weights"), (lambda: tgo.moe_combine(rows.reshape(2, 4, 16), ids, w), "rows, width"),
                         (lambda: tgo.moe_combine(rows.half(), ids, w), "bfloat16"), (lambda: tgo.moe_combine(rows, ids[:, :0], w[:, :0]), "top_k")):
        with pytest.raises(RuntimeError, match=needle):
            call()
    with pytest.raises(RuntimeError, match="device"):
        tgo.moe_balance_loss(x, ids.cpu())


def test_router_of_many_tokens(cuda):
    """More tokens than blocks run at once, compared among themselves and with torch's own top-k of distinct scores."""
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.rand(200003, 24, device="cuda", generator=g).argsort(1).float() / 7 - 1
    w, ids = tgo.moe_router(x, 5)
    top = torch.topk(x.double(), 5)
    assert torch.equal(ids.long(), top.indices)
    near(w, torch.softmax(top.values, 1), 60 * U)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 256, 8), (7, 5, 2), (300, 33, 4), (90, 64, 6), (2500, 8, 2), (41, 256, 8), (19, 1000, 4), (10, 1024, 32)])
def test_balance_loss(cuda, dtype, scoring, tokens, experts, k):
    import torch_ggml_ops_b200 as tgo

    logits = scores(tokens, experts, dtype, 1)
    ids = ref.router(logits, k, "softmax", True)[1]
    ids[::5, 0] = -1
    ids[::7] = -1
    ids[::11, -1] = experts + 3
    x = logits.cuda().requires_grad_()
    loss, counts = tgo.moe_balance_loss(x, ids.cuda(), scoring=scoring)
    want, want_counts, want_dx, size = ref.balance(logits, ids, scoring)
    assert loss.dtype == torch.float32 and loss.shape == () and counts.dtype == torch.int32 and not counts.requires_grad
    assert torch.equal(counts.cpu().long(), want_counts)
    # sums of positive numbers: one U per step (tokens of a warp, the warps, the blocks), and the exponents' error
    c = (2 * ref.spread(logits, scoring) + 60) * U
    near(loss, want, (c + 400 * U) * want)
    (dx,) = torch.autograd.grad(loss, x, torch.tensor(0.7, device="cuda"))
    near(dx, 0.7 * want_dx, 2 * c * size + HALF_STEP[dtype] * (want_dx.abs() + 2 * c * size) + TINY[dtype])
    again = tgo.moe_balance_loss(x, ids.cuda(), scoring=scoring)
    assert torch.equal(again[0], loss) and torch.equal(again[1], counts)


def test_balance_loss_against_differences(cuda):
    import torch_ggml_ops_b200 as tgo

    logits = scores(12, 20, torch.float32, 4)
    for scoring in ("softmax", "sigmoid"):
        ids = ref.router(logits, 3, scoring, True)[1]
        x = logits.cuda().requires_grad_()
        (dx,) = torch.autograd.grad(tgo.moe_balance_loss(x, ids.cuda(), scoring=scoring)[0], x)
        h = 2.0 ** -10
        for t, e in ((0, 0), (3, 7), (11, 19)):
            up, down = logits.double().clone(), logits.double().clone()
            up[t, e] += h
            down[t, e] -= h
            slope = (ref.balance(up, ids, scoring)[0] - ref.balance(down, ids, scoring)[0]) / (2 * h)
            assert abs(float(slope) - float(dx[t, e])) < 1e-6     # h^2 / 6 of a third derivative below 1, and fp32


def test_balance_loss_without_tokens(cuda):
    import torch_ggml_ops_b200 as tgo

    x = scores(9, 12, torch.float32).cuda()
    x[2] = math.nan
    x.requires_grad_()
    loss, counts = tgo.moe_balance_loss(x, torch.full((9, 2), -1, dtype=torch.int32, device="cuda"))
    assert float(loss.detach()) == 0.0 and not counts.any()
    assert not torch.autograd.grad(loss, x)[0].any()
    e = torch.empty(0, 12, device="cuda", requires_grad=True)
    loss, counts = tgo.moe_balance_loss(e, torch.empty(0, 2, dtype=torch.int32, device="cuda"))
    assert float(loss.detach()) == 0.0 and counts.shape == (12,) and torch.autograd.grad(loss, e)[0].shape == (0, 12)
    # one padded token among others may hold anything
    ids = torch.zeros(9, 2, dtype=torch.int32, device="cuda")
    ids[2] = -1
    loss, _ = tgo.moe_balance_loss(x, ids)
    assert math.isfinite(float(loss.detach())) and bool(torch.isfinite(torch.autograd.grad(loss, x)[0]).all())
    # a row with every expert switched off that names one all the same
    y = scores(3, 12, torch.float32).cuda()
    y[1] = -math.inf
    y.requires_grad_()
    loss, _ = tgo.moe_balance_loss(y, ids[:3] * 0)
    (dy,) = torch.autograd.grad(loss, y)
    assert math.isfinite(float(loss.detach())) and not dy[1].any() and bool(torch.isfinite(dy).all())


def test_an_even_use_costs_one(cuda):
    import torch_ggml_ops_b200 as tgo

    ids = torch.arange(64, dtype=torch.int32, device="cuda").reshape(32, 2) % 8
    loss, counts = tgo.moe_balance_loss(torch.zeros(32, 8, device="cuda"), ids)
    assert float(loss) == 1.0 and bool((counts == 8).all())


def expert_ids(tokens, k, experts, seed, dropped=0.1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(experts, generator=g)[:k] for _ in range(tokens)]).int()
    ids[torch.rand(tokens, k, generator=g) < dropped] = -1
    ids[torch.rand(tokens, k, generator=g) < dropped / 4] = experts
    return ids


@pytest.mark.parametrize("tokens,k,experts,width", [(1, 1, 1, 8), (1, 8, 256, 2048), (3, 2, 5, 16), (16, 8, 256, 512), (33, 4, 1000, 264), (128, 8, 64, 72),
                                                    (130, 8, 64, 8), (600, 6, 40, 40), (50, 1, 4096, 24), (1, 32, 32, 4104)])
@pytest.mark.parametrize("dropped", [0.0, 0.2, 1.0])
def test_dispatch(cuda, tokens, k, experts, width, dropped):
    import torch_ggml_ops_b200 as tgo

    ids = expert_ids(tokens, k, experts, tokens + k, dropped)
    x = torch.randn(tokens, width, generator=torch.Generator().manual_seed(1)).bfloat16()
    xd = x.cuda().requires_grad_()
    rows, at, indices, offsets = tgo.moe_dispatch(xd, ids.cuda(), experts)
    want_at, want_ends = ref.sort_rows(ids, experts)
    assert torch.equal(at.cpu(), want_at) and torch.equal(offsets.cpu(), want_ends) and torch.equal(indices.cpu(), torch.arange(experts))
    want = torch.zeros(tokens * k, width, dtype=torch.bfloat16)
    for t in range(tokens):
        for s in range(k):
            if want_at[t, s] >= 0:
                want[want_at[t, s]] = x[t]
    assert torch.equal(rows.detach().cpu(), want)
    g = torch.randn(tokens * k, width, generator=torch.Generator().manual_seed(2)).bfloat16()
    (dx,) = torch.autograd.grad(rows, xd, g.cuda())
    y, size = ref.combine(g, want_at, None)
    near(dx, y, k * U * size + 2.0 ** -8 * y.abs() * (1 + 2.0 ** -7))


@pytest.mark.parametrize("tokens,k,experts,width", [(1, 1, 1, 8), (1, 8, 256, 2048), (3, 2, 5, 16), (16, 8, 64, 512), (33, 4, 100, 264), (70, 10, 40, 1000),
                                                    (5, 3, 7, 4104), (2, 32, 32, 520)])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("dropped", [0.0, 0.3, 1.0])
def test_combine_and_its_gradients(cuda, tokens, k, experts, width, weighted, dropped):
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator().manual_seed(7)
    at = ref.sort_rows(expert_ids(tokens, k, experts, 3 * tokens + k, dropped), experts)[0]
    rows = torch.randn(tokens * k, width, generator=g).bfloat16()
    w = torch.randn(tokens, k, generator=g) if weighted else None
    dy = torch.randn(tokens, width, generator=g).bfloat16()
    rd, wd = rows.cuda().requires_grad_(), None if w is None else w.cuda().requires_grad_()
    y = tgo.moe_combine(rd, at.cuda(), wd)
    want, size = ref.combine(rows, at, w)
    near(y, want, 2 * k * U * size + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7))
    got = torch.autograd.grad(y, [rd, wd] if weighted else [rd], dy.cuda())
    d_rows, rows_size, d_w, w_size = ref.combine_grad(dy, rows, at, w)
    near(got[0], d_rows, 2 * U * rows_size + 2.0 ** -8 * d_rows.abs() * (1 + 2.0 ** -7))
    if weighted:
        near(got[1], d_w, (width / 32 + 8) * U * w_size)


def test_combine_gradient_of_one_input_alone(cuda):
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator().manual_seed(9)
    at = ref.sort_rows(expert_ids(20, 4, 16, 4), 16)[0].cuda()
    rows, w = torch.randn(80, 64, generator=g).bfloat16().cuda(), torch.rand(20, 4, generator=g).cuda()
    dy = torch.randn(20, 64, generator=g).bfloat16().cuda()
    both_r, both_w = rows.clone().requires_grad_(), w.clone().requires_grad_()
    want_r, want_w = torch.autograd.grad(tgo.moe_combine(both_r, at, both_w), [both_r, both_w], dy)
    one = rows.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(tgo.moe_combine(one, at, w), one, dy)[0], want_r)
    one = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(tgo.moe_combine(rows, at, one), one, dy)[0], want_w)


def test_combine_of_any_map(cuda):
    """A map that is no result of a dispatch: rows named twice and more, rows that do not exist, more rows than pairs."""
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator().manual_seed(11)
    at = torch.tensor([[0, 0, 3], [5, 3, -1], [2 ** 31 - 1, 9, -(2 ** 31)], [3, 10, 19], [20, 19, 1]], dtype=torch.int32)
    for n in (20, 4, 12):
        rows, w = torch.randn(n, 296, generator=g).bfloat16(), torch.randn(5, 3, generator=g)
        dy = torch.randn(5, 296, generator=g).bfloat16()
        rd, wd = rows.cuda().requires_grad_(), w.cuda().requires_grad_()
        y = tgo.moe_combine(rd, at.cuda(), wd)
        want, size = ref.combine(rows, at, w)
        near(y, want, 6 * U * size + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7))
        got = torch.autograd.grad(y, [rd, wd], dy.cuda())
        d_rows, rows_size, d_w, w_size = ref.combine_grad(dy, rows, at, w)
        near(got[0], d_rows, 8 * U * rows_size + 2.0 ** -8 * d_rows.abs() * (1 + 2.0 ** -7))
        near(got[1], d_w, 20 * U * w_size)


def test_dispatch_and_combine_layouts(cuda):
    import torch_ggml_ops_b200 as tgo

    x = torch.randn(6, 16, device="cuda").bfloat16()
    ids = expert_ids(6, 2, 4, 1).cuda()
    rows, at, _, _ = tgo.moe_dispatch(x, ids, 4)
    rows2, at2, _, _ = tgo.moe_dispatch(x.reshape(2, 3, 16), ids.reshape(2, 3, 2), 4)
    assert torch.equal(rows, rows2) and torch.equal(at.reshape(2, 3, 2), at2)
    w = torch.rand(2, 3, 2, device="cuda")
    y = tgo.moe_combine(rows, at2, w)
    assert y.shape == (2, 3, 16) and torch.equal(y.reshape(6, 16), tgo.moe_combine(rows, at, w.reshape(6, 2)))
    one = tgo.moe_combine(rows, at[3], w.reshape(6, 2)[3])
    assert one.shape == (16,) and torch.equal(one, y.reshape(6, 16)[3])
    # no tokens, no rows
    none = torch.empty(0, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    r, a, i, o = tgo.moe_dispatch(none, torch.empty(0, 2, dtype=torch.int32, device="cuda"), 4)
    assert r.shape == (0, 16) and a.shape == (0, 2) and i.tolist() == [0, 1, 2, 3] and o.tolist() == [0] * 4
    assert torch.autograd.grad(r.sum(), none)[0].shape == (0, 16)
    assert tgo.moe_combine(r, a, torch.empty(0, 2, device="cuda")).shape == (0, 16)
    empty = none.detach().requires_grad_()
    y = tgo.moe_combine(empty, at, w.reshape(6, 2))
    assert not y.detach().any() and torch.autograd.grad(y.sum(), empty)[0].shape == (0, 16)
    # a cotangent that is an expanded number
    xg = x.clone().requires_grad_()
    rows, at, _, _ = tgo.moe_dispatch(xg, ids, 4)
    (dx,) = torch.autograd.grad(rows.sum(), xg)
    assert torch.equal(dx[:, 0].float(), (at >= 0).sum(1).float())


def test_dispatch_of_many_pairs(cuda):
    """Every size of the sort, against native.route_sort's result for the same ids and rows moved by indexing."""
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator(device="cuda").manual_seed(3)
    for tokens, k, experts in ((1023, 1, 7), (1025, 1, 7), (4096, 8, 256), (9001, 8, 300)):
        ids = torch.randint(-1, experts + 1, (tokens, k), device="cuda", generator=g, dtype=torch.int32)
        x = torch.randn(tokens, 64, device="cuda", generator=g).bfloat16()
        rows, at, _, offsets = tgo.moe_dispatch(x, ids, experts)
        named = ((ids >= 0) & (ids < experts)).reshape(-1)
        order = torch.sort(torch.where(named, ids.reshape(-1).long(), experts), stable=True).indices
        n = int(named.sum())
        want_at = torch.full_like(ids.reshape(-1), -1)
        want_at[order[:n]] = torch.arange(n, dtype=torch.int32, device="cuda")
        assert torch.equal(at.reshape(-1), want_at) and int(offsets[-1]) == n
        assert torch.equal(rows[:n], x[order[:n] // k]) and not rows[n:].any()


# ------------------------------------------------------------------ a layer, as it is used
def layer(tokens, dtype=torch.float32):
    import numpy as np  # noqa: F401
    from oracle import ref as oref
    from helpers import expert_case, to_dev

    E, H, F, k = 12, 512, 256, 3
    qt_gu, qt_d = oref.Q4_K, oref.Q6_K
    (wg, Wg), (wu, Wu), (wd, Wd) = (expert_case(qt, E, n, kk, s) for qt, n, kk, s in ((qt_gu, F, H, 1), (qt_gu, F, H, 2), (qt_d, H, F, 3)))
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, H, generator=g).bfloat16()
    gate = (torch.randn(E, H, generator=g) * 0.05).to(dtype)
    return E, H, F, k, qt_gu, qt_d, [to_dev(w) for w in (wg, wu, wd)], [torch.from_numpy(W).double() for W in (Wg, Wu, Wd)], x, gate


def run_layer(tgo, x, gate, ws, E, F, k, qt_gu, qt_d, mask=None):
    logits = x.float() @ gate.t()
    weights, ids = tgo.moe_router(logits, k, token_mask=mask)
    balance, counts = tgo.moe_balance_loss(logits, ids)
    rows, at, experts, ends = tgo.moe_dispatch(x, ids, E)
    return tgo.moe_combine(tgo.moe_mlp(rows, *ws, experts, ends, qt_gu, qt_d, F), at, weights), balance, counts, weights, ids


@pytest.mark.parametrize("tokens", [1, 5, 64, 301])
def test_a_layer_and_its_gradients(cuda, tokens):
    """router -> dispatch -> experts -> combine with the balance loss, forward and backward, against the same in 64 bits (the
    experts' products round to bf16 between: their own tolerances)."""
    import torch_ggml_ops_b200 as tgo

    E, H, F, k, qt_gu, qt_d, ws, (Wg, Wu, Wd), x, gate = layer(tokens)
    mask = torch.ones(tokens, dtype=torch.bool)
    mask[tokens // 2 + 1::4] = False
    xd, gd = x.cuda().requires_grad_(), gate.cuda().requires_grad_()
    y, balance, counts, weights, ids = run_layer(tgo, xd, gd, ws, E, F, k, qt_gu, qt_d, mask.cuda())
    dy = torch.randn(tokens, H, generator=torch.Generator().manual_seed(1)).bfloat16()
    dx, dgate = torch.autograd.grad([y, balance], [xd, gd], [dy.cuda(), torch.tensor(3.0, device="cuda")])
    assert bool((ids[~mask.cuda()] == -1).all()) and int(counts.sum()) == int(mask.sum()) * k

    xf, gf = x.double().requires_grad_(), gate.double().requires_grad_()
    logits = xf @ gf.t()
    at = ids.cpu().long()
    want, probs = torch.zeros(tokens, H, dtype=torch.float64), []
    for t in torch.nonzero(mask)[:, 0].tolist():
        w = torch.softmax(logits[t, at[t]], 0)
        probs.append(torch.softmax(logits[t], 0))
        for s in range(k):
            e = at[t, s]
            h = torch.nn.functional.silu(Wg[e] @ xf[t]) * (Wu[e] @ xf[t])
            want = want.index_add(0, torch.tensor([t]), (w[s] * (Wd[e] @ h))[None])
    f = torch.bincount(at[at >= 0], minlength=E).double()
    want_balance = E * (f / f.sum() * torch.stack(probs).mean(0)).sum()
    want_dx, want_dgate = torch.autograd.grad([want, want_balance], [xf, gf], [dy.double(), torch.tensor(3.0, dtype=torch.float64)])
    far = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())   # noqa: E731
    assert far(y.detach(), want.detach()) < 1e-2
    assert abs(float(balance.detach()) / float(want_balance.detach()) - 1) < 1e-5
    assert far(dx, want_dx) < 1.5e-2
    assert far(dgate, want_dgate) < 2e-2


def test_a_layer_equals_the_expert_parallel_one(cuda):
    """PeerMoEMLP.plan takes what moe_router gives, padded tokens too; it weights inside its activation kernels."""
    import torch_ggml_ops_b200 as tgo
    from torch_ggml_ops_b200.moe_parallel import PeerMoEMLP

    tokens = 200
    E, H, F, k, qt_gu, qt_d, ws, _, x, gate = layer(tokens)
    mask = (torch.arange(tokens) % 5 != 0).cuda()
    with torch.no_grad():
        y, _, _, weights, ids = run_layer(tgo, x.cuda(), gate.cuda(), ws, E, F, k, qt_gu, qt_d, mask)
        peer = PeerMoEMLP(*ws, qt_gu, qt_d, E, H, F, capacity_rows=tokens * k, tokens_per_rank=tokens, top_k=k)
        peer.plan(ids, weights)
        z = peer.forward(x.cuda())
    assert float((y.float() - z.float()).norm() / y.float().norm()) < 1e-2
    assert not y[~mask].any() and not z[~mask].any()


def test_a_layer_captured_and_replayed(cuda):
    import torch_ggml_ops_b200 as tgo

    tokens = 48
    E, H, F, k, qt_gu, qt_d, ws, _, x, gate = layer(tokens)
    gate = gate.cuda()
    inputs = [x.cuda(), torch.randn(tokens, H, device="cuda").bfloat16()]
    still = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        run_layer(tgo, still, gate, ws, E, F, k, qt_gu, qt_d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = run_layer(tgo, still, gate, ws, E, F, k, qt_gu, qt_d)
    for v in (inputs[1], inputs[0], inputs[1]):
        still.copy_(v)
        graph.replay()
        with torch.no_grad():
            want = run_layer(tgo, v, gate, ws, E, F, k, qt_gu, qt_d)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_gradients_captured_and_replayed(cuda):
    import torch_ggml_ops_b200 as tgo

    at = ref.sort_rows(expert_ids(30, 4, 16, 4), 16)[0].cuda()
    ids = expert_ids(30, 4, 16, 4).cuda()
    leaves = [torch.randn(30, 16, device="cuda"), torch.randn(120, 64, device="cuda").bfloat16(), torch.rand(30, 4, device="cuda"),
              torch.randn(30, 64, device="cuda").bfloat16()]

    def step(logits, rows, w, x):
        v = [t.detach().requires_grad_() for t in (logits, rows, w, x)]
        rw, _ = tgo.moe_router(v[0], 4, normalize=False)
        loss, _ = tgo.moe_balance_loss(v[0], ids)
        r, _, _, _ = tgo.moe_dispatch(v[3], ids, 16)
        total = (rw * w).sum() + loss + tgo.moe_combine(v[1], at, v[2]).float().square().sum() + r.float().pow(3).sum()
        return torch.autograd.grad(total, v)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*leaves)
    for scale in (1.0, -0.5):
        for t in leaves:
            t.mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        for a, b in zip(got, step(*leaves)):
            assert torch.equal(a, b)


def test_other_streams(cuda):
    import torch_ggml_ops_b200 as tgo

    x = torch.randn(500, 64, device="cuda")
    want = tgo.moe_router(x, 6)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            w, ids = tgo.moe_router(x, 6)
            got.append((w, ids, *tgo.moe_balance_loss(x, ids), *tgo.moe_dispatch(torch.ones(500, 8, device="cuda").bfloat16(), ids, 64)))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], want[0]) and torch.equal(g[1], want[1])
        for a, b in zip(g, got[0]):
            assert torch.equal(a, b)


def test_second_derivatives_are_refused(cuda):
    import torch_ggml_ops_b200 as tgo

    x = torch.randn(5, 8, device="cuda", requires_grad=True)
    w, ids = tgo.moe_router(x, 2)
    (dx,) = torch.autograd.grad(w.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="higher-order"):
        dx.sum().backward()
    (dx,) = torch.autograd.grad(tgo.moe_balance_loss(x, ids)[0], x, create_graph=True)
    with pytest.raises(RuntimeError, match="higher-order"):
        dx.square().sum().backward()
    rows = torch.randn(10, 8, device="cuda").bfloat16().requires_grad_()
    at = torch.arange(10, dtype=torch.int32, device="cuda").reshape(5, 2)
    (dr,) = torch.autograd.grad(tgo.moe_combine(rows, at).float().square().sum(), rows, create_graph=True)
    with pytest.raises(RuntimeError, match="higher-order"):
        dr.float().sum().backward()


def test_what_autograd_keeps(cuda):
    """Two passes over one graph, a second one after it was freed, inputs that were written over, forward mode, hooks on what is kept."""
    import torch_ggml_ops_b200 as tgo

    x = torch.randn(5, 8, device="cuda", requires_grad=True)
    ids = torch.arange(10, dtype=torch.int32, device="cuda").reshape(5, 2) % 8
    t = torch.randn(5, 16, device="cuda").bfloat16().requires_grad_()
    rows, at, _, _ = tgo.moe_dispatch(t, ids, 8)
    r, w = rows.detach().requires_grad_(), torch.rand(5, 2, device="cuda", requires_grad=True)
    for make, leaf in ((lambda: tgo.moe_router(x * 1, 2)[0], x), (lambda: tgo.moe_balance_loss(x * 1, ids)[0], x), (lambda: tgo.moe_dispatch(t * 1, ids, 8)[0], t),
                       (lambda: tgo.moe_combine(r * 1, at, w), r), (lambda: tgo.moe_combine(r.detach(), at, w * 1), w)):
        y = make()
        g = torch.ones_like(y)
        (a,) = torch.autograd.grad(y, leaf, g, retain_graph=True)
        (b,) = torch.autograd.grad(y, leaf, g)
        assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, leaf, g)
        with torch.autograd.graph.save_on_cpu():
            z = make()
        assert torch.equal(torch.autograd.grad(z, leaf, g)[0], a)
    for change in ("x", "w"):
        v = x * 1
        weights, _ = tgo.moe_router(v, 2, normalize=False)
        total = weights.sum()
        with torch.no_grad():
            (v if change == "x" else weights).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            total.backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach().requires_grad_(), torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            tgo.moe_router(dual, 2)
    # leaves that share a node with others, and one that wants nothing
    loss = tgo.moe_combine(tgo.moe_dispatch(t, ids, 8)[0], at, tgo.moe_router(x, 2)[0]).float().sum() + tgo.moe_balance_loss(x, ids)[0]
    loss.backward()
    assert x.grad.shape == x.shape and t.grad.shape == t.shape and tgo.moe_router(x.detach(), 2)[0].grad_fn is None


def test_compiled_and_checked_by_torch(cuda):
    import torch_ggml_ops_b200 as tgo

    E, H, F, k, qt_gu, qt_d, ws, _, x, gate = layer(20)
    step = lambda a, g: run_layer(tgo, a, g, ws, E, F, k, qt_gu, qt_d)   # noqa: E731
    a, g = x.cuda().requires_grad_(), gate.cuda().requires_grad_()
    eager, compiled = step(a, g), torch.compile(step, fullgraph=True, backend="aot_eager")(a, g)
    for p, q in zip(eager, compiled):
        assert torch.equal(p, q)
    dy = torch.ones_like(eager[0])
    for p, q in zip(torch.autograd.grad(eager[0], [a, g], dy), torch.autograd.grad(compiled[0], [a, g], dy)):
        assert torch.equal(p, q)
    ops = torch.ops.torch_ggml_ops_b200
    logits = torch.randn(6, 16, device="cuda", requires_grad=True)
    ids = expert_ids(6, 2, 16, 1).cuda()
    rows = torch.randn(12, 8, device="cuda").bfloat16().requires_grad_()
    at = torch.arange(12, dtype=torch.int32, device="cuda").reshape(6, 2)
    w = torch.rand(6, 2, device="cuda", requires_grad=True)
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    for op, args in ((ops.moe_router, (logits, 3, 0, True, None)), (ops.moe_balance_loss, (logits, ids, 1)),
                     (ops.moe_dispatch, (rows[:6].detach().requires_grad_(), ids, 16)), (ops.moe_combine, (rows, at, w)), (ops.moe_combine, (rows, at, None)),
                     (ops.moe_router_grad, (torch.rand(6, 2, device="cuda"), logits.detach(), ids, w.detach(), 0, True)),
                     (ops.moe_combine_grad, (rows[:6].detach(), rows.detach(), at, w.detach(), True, False))):
        torch.library.opcheck(op.default, args, test_utils=tests)


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 scores, and rows of more than 2^31 elements: what is behind them is found."""
    import torch_ggml_ops_b200 as tgo

    tokens = 2 ** 31 // 512 + 5
    x = torch.zeros(tokens, 512, dtype=torch.bfloat16, device="cuda")
    x[-3:, 100] = 4.0
    x[-3:, 511] = 3.0
    x.requires_grad_()
    w, ids = tgo.moe_router(x, 2, normalize=False)
    assert ids[-3:].tolist() == [[100, 511]] * 3 and ids[:3].tolist() == [[0, 1]] * 3
    (dx,) = torch.autograd.grad(w[-1, 0], x)
    assert not dx[:-1].any() and float(dx[-1, 100]) > 0 > float(dx[-1, 511])
    loss, counts = tgo.moe_balance_loss(x, ids)
    assert counts[[0, 1, 100, 511]].tolist() == [tokens - 3, tokens - 3, 3, 3]
    (dx,) = torch.autograd.grad(loss, x)
    assert float(dx[-1, 0]) > 0 and torch.equal(dx[0], dx[-4])
    del x, dx
    tokens = 2 ** 31 // (2 * 2048) + 3
    t = torch.zeros(tokens, 2048, dtype=torch.bfloat16, device="cuda")
    t[-1] = 1.0
    t.requires_grad_()
    ids = torch.zeros(tokens, 2, dtype=torch.int32, device="cuda")
    ids[:, 1] = 1
    rows, at, _, ends = tgo.moe_dispatch(t, ids, 2)
    assert at[-1].tolist() == [tokens - 1, 2 * tokens - 1] and ends.tolist() == [tokens, 2 * tokens]
    assert bool((rows[-1] == 1).all()) and bool((rows[tokens - 1] == 1).all()) and not rows[tokens:-1].any()
    y = tgo.moe_combine(rows, at, torch.full((tokens, 2), 0.75, device="cuda"))
    assert bool((y[-1] == 1.5).all()) and not y[:-1].any()
    (dt,) = torch.autograd.grad(y[-1].sum(), t)
    assert bool((dt[-1] == 1.5).all()) and not dt[:-1].any()


def small_step(tgo, logits, tokens):
    weights, ids = tgo.moe_router(logits, 4, normalize=False)
    balance, _ = tgo.moe_balance_loss(logits, ids)
    rows, at, _, _ = tgo.moe_dispatch(tokens, ids, 32)
    return tgo.moe_combine(rows * 2, at, weights), balance


def test_batches_of_any_size_in_one_graph(cuda):
    import torch_ggml_ops_b200 as tgo

    torch._dynamo.reset()
    compiled = torch.compile(lambda a, b: small_step(tgo, a, b), dynamic=True, fullgraph=True, backend="aot_eager")
    for n in (40, 17, 90):
        a, b = torch.randn(n, 32, device="cuda", requires_grad=True), torch.randn(n, 64, device="cuda").bfloat16().requires_grad_()
        want, got = small_step(tgo, a, b), compiled(a, b)
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        for p, q in zip(*(torch.autograd.grad(y.float().sum() + loss, [a, b]) for y, loss in (want, got))):
            assert torch.equal(p, q)


def test_a_backward_pass_into_leaves_captured(cuda):
    import torch_ggml_ops_b200 as tgo

    a, b = torch.randn(40, 32, device="cuda", requires_grad=True), torch.randn(40, 64, device="cuda").bfloat16().requires_grad_()

    def step():
        a.grad = b.grad = None
        y, loss = small_step(tgo, a, b)
        (y.float().sum() + loss).backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    want = a.grad.clone(), b.grad.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a.grad, want[0]) and torch.equal(b.grad, want[1])


def test_without_autograd_twice_and_from_several_threads(cuda):
    import threading

    import torch_ggml_ops_b200 as tgo

    x, t = torch.randn(40, 32, device="cuda"), torch.randn(40, 64, device="cuda").bfloat16()
    with torch.inference_mode():
        want = small_step(tgo, x, t)
    # dispatch is linear: the second derivative of the rows' cubes is 6 x for each of the 4 pairs
    leaf = t.clone().requires_grad_()
    ids = tgo.moe_router(x, 4)[1]
    (g,) = torch.autograd.grad((tgo.moe_dispatch(leaf, ids, 32)[0].float() ** 3).sum(), leaf, create_graph=True)
    (h,) = torch.autograd.grad(g.float().sum(), leaf)
    near(h, 24 * t.double(), 2.0 ** -6 * t.double().abs().cpu() * 24)   # two passes, each with two roundings to bf16
    found = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                y, loss = small_step(tgo, x, t)
            torch.cuda.current_stream().synchronize()
            found.append(torch.equal(y, want[0]) and torch.equal(loss, want[1]))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(5)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert found == [True] * 5
