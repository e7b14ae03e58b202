"""What the C entries of the routing operators and of logit_rules refuse before any device work: pointers that are not multiples of their type's
size, at which a kernel would fault."""
import ctypes

import pytest


def entries():
    from torch_ggml_ops_b200 import native

    lib = native.lib()
    buf = (ctypes.c_char * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15
    ws = 1 << 30
    # name -> (call with pointers by name, {name: bytes that it has to be a multiple of})
    def rules(t=0, id_bytes=8, length_bytes=8, **q):
        return lib.tgo_logit_rules(q["logits"], q["out"], t, 2, 8, 8, 8, q["history"], q["lengths"], 4, 4, id_bytes, length_bytes, q["rep"], 1.0, q["pres"], 0.0,
                                   q["freq"], 0.0, q["bias_ids"], q["values"], 4, 4, 4, id_bytes, q["allowed"], 1, None)

    return p, {
        "router": (lambda **q: lib.tgo_moe_router(q["logits"], 2, 2, 8, 8, 2, 0, 1, None, q["weights"], q["ids"], None), {"logits": 4, "weights": 4, "ids": 4}),
        "router_grad": (lambda **q: lib.tgo_moe_router_grad(q["logits"], 0, 2, 8, 8, q["ids"], q["weights"], q["dw"], 2, 0, 1, q["dx"], None),
                        {"logits": 2, "ids": 4, "weights": 4, "dw": 4, "dx": 2}),
        "router_grad fp32": (lambda **q: lib.tgo_moe_router_grad(p, 2, 2, 8, 8, p, p, p, 2, 0, 1, q["dx"], None), {"dx": 4}),
        "balance": (lambda **q: lib.tgo_moe_balance_loss(q["logits"], 1, 2, 8, 8, q["ids"], 2, 0, q["loss"], q["counts"], q["coef"], q["ws"], ws, None),
                    {"logits": 2, "ids": 4, "loss": 4, "counts": 4, "coef": 4, "ws": 8}),
        "balance_grad": (lambda **q: lib.tgo_moe_balance_grad(q["logits"], 2, 2, 8, 8, q["ids"], 2, 0, q["coef"], q["dloss"], q["dx"], None),
                         {"logits": 4, "ids": 4, "coef": 4, "dloss": 4, "dx": 4}),
        "dispatch": (lambda **q: lib.tgo_moe_dispatch(q["x"], q["ids"], 5000, 1, 8, 8, q["rows"], q["at"], q["indices"], q["ends"], q["ws"], ws, None),
                     {"x": 16, "ids": 4, "rows": 16, "at": 4, "indices": 8, "ends": 4, "ws": 4}),
        "combine": (lambda **q: lib.tgo_moe_combine(q["rows"], 4, q["at"], q["weights"], q["out"], 2, 2, 8, None), {"rows": 16, "at": 4, "weights": 4, "out": 16}),
        "combine_grad": (lambda **q: lib.tgo_moe_combine_grad(q["dy"], q["rows"], 4, q["at"], q["weights"], q["d_rows"], q["dw"], 2, 2, 8, q["ws"], ws, None),
                         {"dy": 16, "rows": 16, "at": 4, "weights": 4, "d_rows": 16, "dw": 4, "ws": 4}),
        "rules": (rules, {"logits": 2, "out": 2, "history": 8, "lengths": 8, "rep": 4, "pres": 4, "freq": 4, "bias_ids": 8, "values": 4, "allowed": 4}),
        "rules of 4-byte ids": (lambda **q: rules(2, 4, 4, **q), {"logits": 4, "out": 4, "history": 4, "lengths": 4, "rep": 4, "pres": 4, "freq": 4, "bias_ids": 4,
                                                                "values": 4, "allowed": 4}),
    }


@pytest.mark.parametrize("name", ["router", "router_grad", "router_grad fp32", "balance", "balance_grad", "dispatch", "combine", "combine_grad", "rules", "rules of 4-byte ids"])
def test_misaligned_pointers_are_refused(name):
    from torch_ggml_ops_b200 import native

    p, every = entries()
    call, pointers = every[name]
    for which, size in pointers.items():
        assert call(**{k: p + (size // 2 if k == which else 0) for k in pointers}) < 0
        assert "align" in native.last_error(), (which, native.last_error())


def test_a_result_that_meets_the_logits_is_refused():
    """out is the logits themselves or shares nothing with them; nothing is left to do for logits that no rule names, so that a legal call needs no
    device."""
    from torch_ggml_ops_b200 import native

    lib = native.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) & ~63

    def call(out, rows=3, vocab=8, in_stride=20, out_stride=20, allowed=p):
        return lib.tgo_logit_rules(p, out, 2, rows, vocab, in_stride, out_stride, None, None, 0, 0, 8, 8, None, 1.0, None, 0.0, None, 0.0, None, None, 0, 0, 0, 8, allowed, 1, None)

    for kw in (dict(out=p, out_stride=24), dict(out=p, in_stride=8), dict(out=p + 4), dict(out=p + 28), dict(out=p + 80), dict(out=p + 52), dict(out=p + 4, rows=1),
               dict(out=p + 28, rows=1), dict(out=p + 100), dict(out=p + 160, out_stride=16)):
        assert call(**kw) < 0 and "no memory" in native.last_error(), (kw, native.last_error())
    assert call(out=p, allowed=None) == 0 and call(out=p, rows=1, in_stride=0, out_stride=0, allowed=None) == 0
