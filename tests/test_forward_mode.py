"""No operator has a forward-mode derivative: a tangent on any differentiable input is refused, whether or not the input (or another) wants
a gradient too.  On meta tensors, without a GPU, and on one."""
import pytest
import torch
from torch.autograd import forward_ad as fwd

ops, own = torch.ops.torch_ggml_ops, torch.ops.torch_ggml_ops_b200


def programs(device):
    """(call, its differentiable inputs) for every operator."""
    import torch_ggml_ops_b200 as tgo

    half = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=device)   # noqa: E731
    f32 = lambda *s: torch.zeros(s, device=device)                           # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)       # noqa: E731
    i64 = lambda *s: torch.zeros(*s, dtype=torch.int64, device=device)       # noqa: E731
    byte = lambda n: torch.zeros(n, dtype=torch.uint8, device=device)        # noqa: E731
    qt, block, n = 12, 144, 256                                              # Q4_K: 144 bytes hold 256 weights
    w, we, ei, eo = byte(n * block), torch.zeros(2, n * block, dtype=torch.uint8, device=device), torch.arange(2, device=device), i32(2)
    ids = i32(3, 2)
    return {
        "mmq": (lambda x: tgo.mmq(x, w, qt, n), [half(3, 256)]),
        "mmq_grad_input": (lambda d: ops.mmq_grad_input(d, w, qt, 256), [half(3, n)]),
        "grouped_mmq": (lambda x: tgo.grouped_mmq(x, we, ei, eo, qt, n), [half(3, 256)]),
        "grouped_mmq_grad_input": (lambda d: ops.grouped_mmq_grad_input(d, we, ei, eo, qt, 256), [half(3, n)]),
        "grouped_mmq_pair": (lambda x: tgo.grouped_mmq_pair(x, we, we, ei, eo, qt, n), [half(3, 256)]),
        "grouped_mmq_pair_grad_input": (lambda a, b: ops.grouped_mmq_pair_grad_input(a, b, we, we, ei, eo, qt, 256), [half(3, n), half(3, n)]),
        "mmq_multi": (lambda x: tgo.mmq_multi(x, [w, w], qt, n), [half(3, 256)]),
        "swiglu": (tgo.swiglu, [half(3, 8), half(3, 8)]),
        "swiglu_grad": (own.swiglu_grad, [half(3, 8), half(3, 8), half(3, 8)]),
        "lm_head_loss": (lambda x: own.lm_head_loss(x, w, qt, n, i64(3), 2, 1.0), [half(3, 256)]),
        "moe_router": (lambda x: tgo.moe_router(x, 2), [f32(3, 8)]),
        "moe_router_grad": (lambda g, x, v: own.moe_router_grad(g, x, ids, v, 0, True), [f32(3, 2), f32(3, 8), f32(3, 2)]),
        "moe_balance_loss": (lambda x: tgo.moe_balance_loss(x, ids), [f32(3, 8)]),
        "moe_balance_grad": (lambda g, x, c: own.moe_balance_grad(g, x, ids, c, 0), [f32(), f32(3, 8), f32(8)]),
        "moe_dispatch": (lambda x: tgo.moe_dispatch(x, ids, 8), [half(3, 16)]),
        "moe_combine": (lambda r, v: tgo.moe_combine(r, ids, v), [half(6, 16), f32(3, 2)]),
        "moe_combine_grad": (lambda d, r, v: own.moe_combine_grad(d, r, ids, v, True, True), [half(3, 16), half(6, 16), f32(3, 2)]),
        "moe_combine_rows_grad": (lambda d, v: own.moe_combine_rows_grad(d, ids, v, 6), [half(3, 16), f32(3, 2)]),
        "moe_dispatch_grad": (lambda d: own.moe_dispatch_grad(d, ids), [half(6, 16)]),
        "logit_rules": (lambda x, v, a, b, c: tgo.logit_rules(x, bias_ids=ids, bias_values=v, repetition_penalty=a, presence_penalty=b, frequency_penalty=c),
                        [f32(3, 8), f32(3, 2), f32(3), f32(3), f32(3)]),
        "logit_rules_out": (lambda x, v, a, b, c, o: tgo.logit_rules(x, bias_ids=ids, bias_values=v, repetition_penalty=a, presence_penalty=b, frequency_penalty=c,
                                                                     out=o), [f32(3, 8), f32(3, 2), f32(3), f32(3), f32(3), f32(3, 8)]),
    }


@pytest.mark.parametrize("device", ["meta", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("name", sorted(programs("meta")))
def test_a_tangent_is_refused(device, name):
    call, inputs = programs(device)[name]
    for i, at in enumerate(inputs):
        for wants in ("nothing", "this one", "all", "all but this one"):
            with fwd.dual_level():
                v = [t.clone().requires_grad_(wants == "all" or wants == "this one" and j == i or wants == "all but this one" and j != i) for j, t in enumerate(inputs)]
                v[i] = fwd.make_dual(v[i], torch.ones_like(at))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*v)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*v)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, tuple(inputs), tuple(torch.ones_like(t) for t in inputs))
