"""GPU tests of ``logit_rules`` against its definition in 64 bits (``routing_ref.py``), of its refusals, and of a decode
step that uses it behind the head's product."""
import math

import pytest
import torch

import routing_ref as ref
from routing_ref import HALF_STEP, TINY, U, near

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def case(rows, vocab, n_history, n_bias, mask, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * rows + vocab)
    c = {"logits": (torch.randn(rows, vocab, generator=g) * 3).to(dtype)}
    if n_history is not None:
        c["history"] = (torch.rand(rows, n_history, generator=g).pow(3) * (vocab + 2)).long() - 1     # some outside the vocabulary
        c["lengths"] = torch.randint(-1, n_history + 3, (rows,), generator=g)
        c["repetition"] = 0.7 + torch.rand(rows, generator=g)
        c["presence"] = torch.rand(rows, generator=g) - 0.3
        c["frequency"] = torch.rand(rows, generator=g) * 0.3 - 0.1
    if n_bias:
        c["bias_ids"] = torch.randint(-2, vocab + 2, (rows, n_bias), generator=g)
        c["bias_values"] = torch.randn(rows, n_bias, generator=g) * 2
    if mask:
        words = torch.randint(-(1 << 31), 1 << 31, (rows, (vocab + 31) // 32), generator=g)
        words[0] = 0                    # nothing allowed
        if rows > 1:
            words[1] = -1               # everything
        if rows > 2:
            words[2, 1:] = 0
        c["allowed"] = words.to(torch.int32)
    return c


def call(c, **more):
    import torch_ggml_ops_b200 as tgo

    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    names = {"lengths": "history_lengths", "repetition": "repetition_penalty", "presence": "presence_penalty", "frequency": "frequency_penalty"}
    logits = d.pop("logits")
    return tgo.logit_rules(logits, **{names.get(k, k): v for k, v in d.items()}, **more)


def check(c, got=None):
    got = call(c) if got is None else got
    want, size = ref.rules(**c)
    dtype = c["logits"].dtype
    limit = torch.finfo(dtype).max * (1 + HALF_STEP[dtype])
    want = torch.where(want.abs() >= limit, torch.copysign(torch.full_like(want, math.inf), want), want)
    # a handful of fp32 operations on numbers of this size, a U each (biases: one each), then the rounding to the type
    n = 8 + (c["bias_ids"].shape[-1] if "bias_ids" in c else 0)
    room = torch.where(torch.isfinite(want), n * U * size + HALF_STEP[dtype] * (want.abs() + n * U * size) + TINY[dtype], 0.0)
    near(got, want, room)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (2, 33), (3, 1000), (5, 1023), (4, 1025), (2, 9000), (1, 20011)])
@pytest.mark.parametrize("n_history,n_bias,mask", [(None, 0, True), (50, 0, False), (0, 3, True), (300, 0, True), (None, 40, False), (700, 70, True)])
def test_rules(cuda, dtype, rows, vocab, n_history, n_bias, mask):
    c = case(rows, vocab, n_history, n_bias, mask, dtype)
    got = check(c)
    assert got.dtype == dtype and torch.equal(got, call(c))
    # in place: the same bits
    inplace = c["logits"].cuda()
    import torch_ggml_ops_b200 as tgo  # noqa: F401

    d = dict(c, logits=inplace)
    assert call(d, out=inplace) is inplace
    assert torch.equal(inplace, got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(cuda, dtype):
    """Infinities, NaN and the lowest value among the logits, allowed and not, penalised and not."""
    lowest = torch.finfo(dtype).min
    x = torch.tensor([[math.nan, math.inf, -math.inf, lowest, -0.0, 0.0, 1.0, -1.0] * 8] * 3, dtype=dtype)
    c = {"logits": x, "history": torch.arange(16).repeat(3, 1), "repetition": torch.tensor([1.5, 1.0, 2.0]), "presence": torch.tensor([0.0, 0.5, -0.5]),
         "frequency": torch.tensor([0.0, 0.0, 0.25]), "allowed": torch.tensor([[0x0F0F0F0F, -1]] * 3, dtype=torch.int32)}
    got = check(c).cpu()
    off = torch.tensor([(0x0F0F0F0F >> i) & 1 == 0 for i in range(32)] + [False] * 32)
    assert bool((got[:, off] == -math.inf).all())
    assert torch.isnan(got[:, ~off][:, 0]).all()
    # what no rule names keeps its bits (the sign of a zero, too)
    plain = call({"logits": x, "history": torch.full((3, 2), -1), "repetition": torch.full((3,), 2.0)}).cpu()
    width = {2: torch.int16, 4: torch.int32}[x.element_size()]
    assert torch.equal(plain.view(width), x.view(width))


def test_numbers_for_all_rows_and_rows_for_all(cuda):
    c = case(4, 500, 60, 9, True, torch.float32)
    one = dict(c, history=c["history"][0], bias_ids=c["bias_ids"][0], bias_values=c["bias_values"][0], allowed=c["allowed"][2], repetition=1.3, presence=0.25,
               frequency=0.125)
    del one["lengths"]
    got = check(one)
    full = {k: (v if k == "logits" else v.expand(4, *v.shape).contiguous() if isinstance(v, torch.Tensor) else torch.full((4,), v)) for k, v in one.items()}
    assert torch.equal(got, call(full))


@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_layouts(cuda, ids):
    """Rows that lie apart, logits and result that start at odd places, ids of either size, one row without its dimension."""
    import torch_ggml_ops_b200 as tgo

    for dtype in DTYPES:
        c = case(3, 777, 40, 5, True, dtype)
        c["history"], c["lengths"], c["bias_ids"] = c["history"].to(ids), c["lengths"].to(ids), c["bias_ids"].to(ids)
        want = check(c)
        for at in (0, 1, 3, 8):
            apart = lambda t, w: torch.zeros(3, w, dtype=t.dtype).index_copy_(1, torch.arange(at, at + t.shape[1]), t).cuda()[:, at:at + t.shape[1]]   # noqa: E731
            d = dict(c, logits=apart(c["logits"], 1000), history=apart(c["history"], 99), bias_ids=apart(c["bias_ids"], 20), bias_values=apart(c["bias_values"], 21),
                     allowed=apart(c["allowed"], 40))
            assert torch.equal(call(d), want)
            out = torch.zeros(3, 900, dtype=dtype, device="cuda")
            call(d, out=out[:, 5:782])
            assert torch.equal(out[:, 5:782], want) and not out[:, :5].any() and not out[:, 782:].any()
            call(dict(d), out=d["logits"])
            assert torch.equal(d["logits"], want)
        row = tgo.logit_rules(c["logits"][2].cuda(), history=c["history"][2].cuda(), history_lengths=c["lengths"][2:].cuda(),
                              repetition_penalty=c["repetition"][2:].cuda(), presence_penalty=c["presence"][2:].cuda(),
                              frequency_penalty=c["frequency"][2:].cuda(), bias_ids=c["bias_ids"][2].cuda(), bias_values=c["bias_values"][2].cuda(),
                              allowed=c["allowed"][2].cuda())
        assert row.shape == (777,) and torch.equal(row, want[2])
    assert tgo.logit_rules(torch.empty(0, 50, device="cuda"), presence_penalty=1.0).shape == (0, 50)
    x = torch.randn(2, 50, device="cuda")
    assert torch.equal(tgo.logit_rules(x), x)


def test_the_same_token_again_and_again(cuda):
    """Counts beyond 16 bits, biases that name one token many times."""
    x = torch.zeros(2, 4000)
    x[:, 7] = 1.0
    h = torch.full((2, 70001), 7)
    h[1, 70000:] = 9
    check({"logits": x, "history": h, "frequency": 0.5, "presence": 1.0})
    n = 333
    c = {"logits": x, "bias_ids": torch.full((2, n), 11), "bias_values": torch.randn(2, n, generator=torch.Generator().manual_seed(1))}
    c["bias_ids"][:, ::3] = 3999
    got = check(c)
    assert torch.equal(got, call(c))
    # sums that are zero in between, tokens that history names too, more entries than tokens
    c = {"logits": torch.randn(2, 40, generator=torch.Generator().manual_seed(2)), "history": torch.arange(0, 40, 3).repeat(2, 9), "repetition": 1.5,
         "frequency": 0.25, "bias_ids": torch.arange(40).repeat(2, 64), "bias_values": torch.tensor([1.0, -1.0, 2.0, -2.0]).repeat_interleave(40).repeat(2, 16)}
    c["bias_values"][1, 7::120] = 3.0
    check(c)
    for n in (1, 33, 65, 97):
        d = dict(c, bias_ids=torch.full((2, n), 9), bias_values=torch.tensor([1.0 if j // 32 % 2 == 0 else -1.0 for j in range(n)]).repeat(2, 1))
        check(d)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,n_history,n_bias,mask", [(3, 30011, 8150, 42, True), (3, 30011, 8150, 43, False), (2, 100003, 9000, 300, True),
                                                              (1, 70000, 70000, 0, True), (1, 3000, 66000, 3000, False), (2, 5000, 3, 9000, True), (33, 700, 16400, 5, True),
                                                              (32, 90000, 16384, 0, False), (40, 3, 70000, 1, False)])
def test_long_histories_and_lists(cuda, dtype, rows, vocab, n_history, n_bias, mask):
    """Every size of a block, counts of 16 and 32 bits, one slice and several."""
    import torch_ggml_ops_b200 as tgo

    c = case(rows, vocab, n_history, n_bias, mask, dtype)
    got = check(c)
    d = {k: v.cuda() for k, v in c.items()}
    args = dict(history=d["history"], history_lengths=d["lengths"], repetition_penalty=d["repetition"], presence_penalty=d["presence"],
                frequency_penalty=d["frequency"], bias_ids=d.get("bias_ids"), bias_values=d.get("bias_values"), allowed=d.get("allowed"))
    for _ in range(2):
        x = d["logits"].clone()
        tgo.logit_rules(x, out=x, **args)
        assert torch.equal(x, got) and torch.equal(tgo.logit_rules(d["logits"], **args), got)


def test_a_large_vocabulary_and_many_rows(cuda):
    """Every slice of a row, and more rows than run at once; the definition in elementary operations."""
    import torch_ggml_ops_b200 as tgo

    g = torch.Generator(device="cuda").manual_seed(5)
    for rows, vocab, n in ((2, 248320, 5000), (1, 1000003, 3000), (700, 5003, 64)):
        x = torch.randn(rows, vocab, device="cuda", generator=g)
        h = torch.randint(0, vocab, (rows, n), device="cuda", generator=g)
        h[:, n // 2:] = h[:, : n - n // 2]
        words = torch.randint(-(1 << 31), 1 << 31, (rows, (vocab + 31) // 32), device="cuda", generator=g).to(torch.int32)
        counts = torch.zeros_like(x).scatter_add_(1, h, torch.ones_like(h, dtype=torch.float32))
        by = torch.full_like(x, 1.25)   # by a number torch multiplies with its rounded reciprocal
        want = torch.where(counts > 0, torch.where(x > 0, x / by, x * by) - (counts * 0.5 + 0.25), x)
        token = torch.arange(vocab, device="cuda")
        want = torch.where((words[:, token // 32] >> (token % 32)) & 1 != 0, want, -math.inf)
        got = tgo.logit_rules(x, history=h, repetition_penalty=1.25, presence_penalty=0.25, frequency_penalty=0.5, allowed=words)
        assert torch.equal(got, want)


def test_refusals(cuda):
    import torch_ggml_ops_b200 as tgo

    x = torch.randn(3, 64, device="cuda")
    h = torch.zeros(3, 4, dtype=torch.long, device="cuda")
    ok = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for kw, needle in (({"history": h[:2]}, "one row per row"), ({"history": h.float()}, "int32 or torch.int64"), ({"history": h.t().contiguous().t()}, "last dimension"),
                       ({"history_lengths": h[:, 0].contiguous()}, "need a history"), ({"history": h, "history_lengths": h[:2, 0].contiguous()}, "history_lengths"),
                       ({"repetition_penalty": 0.0}, "positive"), ({"repetition_penalty": -1.0}, "positive"), ({"presence_penalty": torch.zeros(2, device="cuda")}, "one entry"),
                       ({"presence_penalty": torch.zeros(3, device="cuda").double()}, "contiguous"), ({"bias_ids": h}, "together"),
                       ({"bias_ids": h, "bias_values": torch.zeros(3, 3, device="cuda")}, "same length"),
                       ({"bias_ids": h, "bias_values": torch.zeros(3, 4, device="cuda").half()}, "float32"), ({"allowed": ok[:, :1].contiguous()}, "one bit per token"),
                       ({"allowed": ok.long()}, "int32"), ({"history": h.cpu()}, "device"), ({"out": torch.empty(3, 64, device="cuda").half()}, "out must be"),
                       ({"out": torch.empty(2, 64, device="cuda")}, "out must be"), ({"out": torch.empty(1, 64, device="cuda").expand(3, 64)}, "memory|overlap|single")):
        with pytest.raises(RuntimeError, match=needle):
            tgo.logit_rules(x, **kw)
    base = torch.randn(4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="overlap|memory"):
        tgo.logit_rules(base[:3], out=base[1:])
    wide = torch.randn(3, 300, device="cuda")
    for bad in (wide[:, 8:72], wide[:, 63:127], wide.reshape(-1)[:192].reshape(3, 64)):
        with pytest.raises(RuntimeError, match="no memory"):
            tgo.logit_rules(wide[:, :64], out=bad)
    beside = wide[:, 64:128]
    assert torch.equal(tgo.logit_rules(wide[:, :64], bias_ids=h[0], bias_values=torch.ones(4, device="cuda"), out=beside),
                       tgo.logit_rules(wide[:, :64], bias_ids=h[0], bias_values=torch.ones(4, device="cuda")))
    with pytest.raises(RuntimeError, match="overlap|memory"):
        tgo.logit_rules(base, bias_ids=h[0], bias_values=base[0, :4], out=base)
    with pytest.raises(RuntimeError, match="contiguous"):
        tgo.logit_rules(torch.randn(64, 3, device="cuda").t())
    with pytest.raises(RuntimeError, match="rows, vocab"):
        tgo.logit_rules(x[None])
    with pytest.raises(RuntimeError, match="dtype"):
        tgo.logit_rules(x.double())


def test_captured_and_on_other_streams(cuda):
    import torch_ggml_ops_b200 as tgo

    c = {k: v.cuda() for k, v in case(3, 5000, 200, 9, True, torch.bfloat16).items()}
    want = call(c).clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = call(c)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    with torch.cuda.graph(graph):
        out = call(c)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    c["lengths"].zero_()
    c["bias_values"].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call(c)) and not torch.equal(out, want)
    compiled = torch.compile(lambda x, h: tgo.logit_rules(x, history=h, presence_penalty=0.5), fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(c["logits"], c["history"]), tgo.logit_rules(c["logits"], history=c["history"], presence_penalty=0.5))
    ops = torch.ops.torch_ggml_ops_b200
    args = (c["logits"], c["history"], None, None, 1.1, None, 0.0, None, 0.5, None, None, None)
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(ops.logit_rules.default, args, test_utils=tests)
    torch.library.opcheck(ops.logit_rules_out.default, (*args, torch.empty_like(c["logits"])), test_utils=tests)
    inplace = torch.compile(lambda x, h: tgo.logit_rules(x, history=h, presence_penalty=0.5, out=x), fullgraph=True, backend="aot_eager")
    x = c["logits"].clone()
    inplace(x, c["history"])
    assert torch.equal(x, tgo.logit_rules(c["logits"], history=c["history"], presence_penalty=0.5))


def test_a_decode_step(cuda):
    """Hidden states through the router, the experts, the head and the rules, token by token: a token that a rule forbids is
    never taken, one that came before is penalised by what its count says."""
    import torch_ggml_ops_b200 as tgo
    from helpers import dense_case, to_dev
    from oracle import ref as oref
    from test_routing_ops_gpu import layer, run_layer

    tokens, vocab = 6, 2000
    E, H, F, k, qt_gu, qt_d, ws, _, x, gate = layer(tokens)
    head = to_dev(dense_case(oref.Q6_K, vocab, H, 8)[0])
    hidden, history = x.cuda(), torch.full((tokens, 5), -1, dtype=torch.long, device="cuda")
    words = torch.full((tokens, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
    words[0] = 0
    words[0, 3] = 1 << 7                # one token left: 103
    with torch.no_grad():
        for step in range(5):
            y = run_layer(tgo, hidden, gate.cuda(), ws, E, F, k, qt_gu, qt_d)[0]
            logits = tgo.mmq((y.float() * 0.01).bfloat16(), head, oref.Q6_K, vocab)
            rules = dict(history=history, repetition_penalty=1.1, frequency_penalty=0.1, allowed=words)
            want, size = ref.rules(logits, history=history, repetition=1.1, frequency=0.1, allowed=words)
            new = tgo.logit_rules(logits, **rules)
            near(new, want, torch.where(torch.isfinite(want), 8 * U * size + 2.0 ** -8 * (want.abs() + 8 * U * size), 0.0))
            token = new.float().argmax(1)
            assert int(token[0]) == 103
            history[:, step] = token
            hidden = (hidden.float() * 0.9 + y.float() * 0.01).bfloat16()


def test_offsets_beyond_32_bits(cuda):
    import torch_ggml_ops_b200 as tgo

    rows, vocab = 2 ** 31 // 248320 + 3, 248320
    x = torch.ones(rows, vocab, dtype=torch.bfloat16, device="cuda")
    h = torch.tensor([5, vocab - 1], device="cuda").expand(rows, 2)
    words = torch.full((rows, vocab // 32), -1, dtype=torch.int32, device="cuda")
    words[-1, 0] = ~4
    y = tgo.logit_rules(x, history=h, repetition_penalty=2.0, allowed=words)
    assert float(y[-1, 5]) == float(y[-1, -1]) == float(y[0, 5]) == 0.5 and float(y[-1, 2]) == -math.inf
    assert int((y[-1] == 1).sum()) == vocab - 3 and int((y[-2] == 1).sum()) == vocab - 2
    tgo.logit_rules(x, history=h, repetition_penalty=2.0, allowed=words, out=x)
    assert torch.equal(x[-2:], y[-2:]) and torch.equal(x[:2], y[:2])
