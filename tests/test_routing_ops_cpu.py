"""Refusals and traced shapes of the routing operators and logit_rules, without a GPU: the C boundary refuses before any
device work, the Python side before it reaches a kernel."""
import ctypes

import pytest
import torch


def test_the_c_boundary_refuses_before_any_device_work():
    from torch_ggml_ops_b200 import native

    lib = native.lib()
    buf = (ctypes.c_char * 64)()
    p = ctypes.addressof(buf) & ~15
    router = lambda logits=p, dtype=0, tokens=2, experts=8, stride=8, k=2, scoring=0, ids=p: lib.tgo_moe_router(   # noqa: E731
        logits, dtype, tokens, experts, stride, k, scoring, 1, None, p, ids, None)
    balance = lambda tokens=2, experts=8, k=2, ws=1 << 20: lib.tgo_moe_balance_loss(p, 2, tokens, experts, experts, p, k, 0, p, p, p, p, ws, None)   # noqa: E731
    dispatch = lambda x=p, tokens=2, k=2, experts=8, width=8, ws=1 << 20: lib.tgo_moe_dispatch(   # noqa: E731
        x, p, tokens, k, experts, width, p, p, p, p, p, ws, None)
    grad = lambda dy=p, rows=p, n=4, d_rows=p, d_w=p, ws=16: lib.tgo_moe_combine_grad(dy, rows, n, p, None, d_rows, d_w, 2, 2, 8, p, ws, None)   # noqa: E731

    def rules(logits=p, dtype=0, rows=2, vocab=8, stride=8, history=None, n=0, id_bytes=8, bias=None, values=None, nb=0):
        return lib.tgo_logit_rules(logits, p, dtype, rows, vocab, stride, stride, history, None, n, n, id_bytes, 8, None, 1.0, None, 0.0, None, 0.0,
                                   bias, values, nb, nb, nb, 8, None, 0, None)

    cases = [
        (lambda: router(logits=None), "null"), (lambda: router(ids=None), "null"), (lambda: router(dtype=7), "type"),
        (lambda: router(tokens=0), "zero-row"), (lambda: router(experts=1025, stride=1025), "1..1024"), (lambda: router(experts=0), "1..1024"),
        (lambda: router(k=0), "top_k"), (lambda: router(k=9), "top_k"), (lambda: router(experts=64, stride=64, k=33), "top_k"),
        (lambda: router(tokens=1 << 31), "2^31"), (lambda: router(stride=7), "overlap"), (lambda: router(logits=p + 1), "aligned"),
        (lambda: router(scoring=2), "scoring"),
        (lambda: balance(ws=8), "workspace"), (lambda: balance(k=0), "top_k"), (lambda: balance(tokens=0), "zero-row"),
        (lambda: dispatch(x=None), "null"), (lambda: dispatch(x=p + 2), "16-byte"), (lambda: dispatch(width=12), "multiple of 8"),
        (lambda: dispatch(experts=4097), "4096"), (lambda: dispatch(k=1025), "1024"), (lambda: dispatch(tokens=1 << 30), "2^31"),
        (lambda: dispatch(tokens=5000, ws=4), "workspace"), (lambda: dispatch(tokens=0), "zero-row"),
        (lambda: lib.tgo_moe_combine(p, -1, p, None, p, 2, 2, 8, None), "negative"), (lambda: lib.tgo_moe_combine(p, 4, p, None, p + 8, 2, 2, 8, None), "16-byte"),
        (lambda: lib.tgo_moe_combine(None, 4, p, None, p, 2, 2, 8, None), "null"),
        (lambda: grad(dy=None), "null"), (lambda: grad(rows=None), "null"), (lambda: grad(d_rows=None, d_w=None), "no gradient"),
        (lambda: grad(ws=15), "workspace"),
        (lambda: rules(logits=None), "null"), (lambda: rules(dtype=3), "type"), (lambda: rules(rows=0), "zero-row"), (lambda: rules(vocab=0), "vocabulary"),
        (lambda: rules(vocab=1 << 31, stride=1 << 31), "vocabulary"), (lambda: rules(stride=7), "overlap"), (lambda: rules(logits=p + 1), "aligned"),
        (lambda: rules(history=p, n=4, id_bytes=2), "4 or 8"), (lambda: rules(bias=p, nb=4), "values"), (lambda: rules(n=-1), "negative"),
    ]
    for call, needle in cases:
        assert call() < 0
        assert needle in native.last_error(), (needle, native.last_error())
    assert lib.tgo_moe_balance_workspace_bytes(0, 8) == -1 and lib.tgo_moe_balance_workspace_bytes(4, 2000) == -1
    assert lib.tgo_moe_dispatch_workspace_bytes(4096, 8) == 0 < lib.tgo_moe_dispatch_workspace_bytes(4097, 8)
    assert lib.tgo_moe_dispatch_workspace_bytes(-1, 8) == -1 and lib.tgo_moe_dispatch_workspace_bytes(4, 0) == -1


def test_traced_shapes():
    import torch_ggml_ops_b200 as tgo

    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")   # noqa: E731
    logits, ids = meta(3, 5, 40), meta(3, 5, 6, dtype=torch.int32)
    w, e = tgo.moe_router(logits, 6, scoring="sigmoid")
    assert w.shape == e.shape == (3, 5, 6) and w.dtype == torch.float32 and e.dtype == torch.int32
    loss, counts = tgo.moe_balance_loss(logits, ids)
    assert loss.shape == () and loss.dtype == torch.float32 and counts.shape == (40,) and counts.dtype == torch.int32
    rows, at, indices, offsets = tgo.moe_dispatch(meta(3, 5, 64), ids, 40)
    assert rows.shape == (90, 64) and at.shape == (3, 5, 6) and indices.shape == offsets.shape == (40,)
    assert (rows.dtype, at.dtype, indices.dtype, offsets.dtype) == (torch.bfloat16, torch.int32, torch.int64, torch.int32)
    y = tgo.moe_combine(rows, at, meta(3, 5, 6, dtype=torch.float32))
    assert y.shape == (3, 5, 64) and y.dtype == torch.bfloat16
    out = tgo.logit_rules(meta(4, 100), history=meta(4, 9, dtype=torch.int64), repetition_penalty=1.2)
    assert out.shape == (4, 100) and out.dtype == torch.bfloat16
    # with gradients: shapes of the formulas' operators
    x = meta(7, 40).requires_grad_()
    w, _ = tgo.moe_router(x, 6)
    assert torch.autograd.grad(w.sum() + tgo.moe_balance_loss(x, meta(7, 6, dtype=torch.int32))[0], x)[0].shape == (7, 40)
    r, g = meta(20, 64).requires_grad_(), meta(5, 2, dtype=torch.float32).requires_grad_()
    dr, dg = torch.autograd.grad(tgo.moe_combine(r, meta(5, 2, dtype=torch.int32), g).sum(), [r, g])
    assert dr.shape == (20, 64) and dg.shape == (5, 2) and dg.dtype == torch.float32
    t = meta(5, 64).requires_grad_()
    assert torch.autograd.grad(tgo.moe_dispatch(t, meta(5, 2, dtype=torch.int32), 8)[0].sum(), t)[0].shape == (5, 64)


def test_there_is_no_cpu_implementation():
    import torch_ggml_ops_b200 as tgo

    with pytest.raises((NotImplementedError, RuntimeError)):
        tgo.moe_router(torch.zeros(2, 8), 2)
    with pytest.raises((NotImplementedError, RuntimeError)):
        tgo.moe_combine(torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises((NotImplementedError, RuntimeError)):
        tgo.logit_rules(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="scoring"):
        tgo.moe_router(torch.zeros(2, 8), 2, scoring="tanh")
    with pytest.raises(RuntimeError, match="no gradient"):
        tgo.logit_rules(torch.zeros(2, 8, requires_grad=True))
