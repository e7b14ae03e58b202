"""The routing of a mixture-of-experts layer and the rules on a head's logits: what is timed and compared.

``kind`` says which operator a case calls:

* ``router``: ``moe_router``, scores of a gate -> the experts of every token and their weights;
* ``balance``: ``moe_balance_loss``, how evenly the experts are used, and the pairs of every expert;
* ``dispatch``: ``moe_dispatch``, tokens to rows sorted by expert, as the grouped products take them;
* ``combine``: ``moe_combine``, the experts' rows back to tokens, weighted;
* ``rules``: ``logit_rules``, biases, penalties for repeated tokens and a grammar's mask on logits.

``train`` adds the gradients, as a training program takes them.  ``padded`` is the share of tokens that
only fill a batch up.  With ``own`` false, ``run`` computes the same in elementary torch operations.
"""
import math

import torch

own = False

EXPERTS, HIDDEN, TOP_K, VOCAB = 256, 2048, 8, 248320
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the gate of a decode batch: all latency
        {"name": "router_decode_16", "kind": "router", "tokens": 16, "experts": EXPERTS, "top_k": TOP_K, "dtype": "bf16",
         "scoring": "softmax", "normalize": True, "padded": 0.0, "train": False},
        # a prompt through a gate that scores every expert for itself, an expert count that is no power of two
        {"name": "router_prompt_1291", "kind": "router", "tokens": 1291, "experts": 1000, "top_k": 4, "dtype": "fp32",
         "scoring": "sigmoid", "normalize": True, "padded": 0.0, "train": False},
        # fine-tuning, plain probabilities as weights, padded sequences
        {"name": "router_train_8200", "kind": "router", "tokens": 8200, "experts": EXPERTS, "top_k": TOP_K, "dtype": "fp32",
         "scoring": "softmax", "normalize": False, "padded": 0.1, "train": True},
        # fine-tuning, a large batch
        {"name": "router_train_65536", "kind": "router", "tokens": 65536, "experts": EXPERTS, "top_k": TOP_K, "dtype": "bf16",
         "scoring": "softmax", "normalize": True, "padded": 0.0, "train": True},
        # the balance of one padded sequence, few experts
        {"name": "balance_train_600", "kind": "balance", "tokens": 600, "experts": 64, "top_k": 6, "dtype": "fp32",
         "scoring": "sigmoid", "padded": 0.2, "train": True},
        # the balance of a large batch
        {"name": "balance_train_65536", "kind": "balance", "tokens": 65536, "experts": EXPERTS, "top_k": TOP_K, "dtype": "bf16",
         "scoring": "softmax", "padded": 0.0, "train": True},
        # a decode batch to its experts: all latency
        {"name": "dispatch_decode_16", "kind": "dispatch", "tokens": 16, "experts": EXPERTS, "top_k": TOP_K, "width": HIDDEN,
         "padded": 0.0, "train": False},
        # fine-tuning, there and the gradient back
        {"name": "dispatch_train_16384", "kind": "dispatch", "tokens": 16384, "experts": EXPERTS, "top_k": TOP_K, "width": HIDDEN,
         "padded": 0.05, "train": True},
        # a prompt's rows back to its tokens
        {"name": "combine_prompt_600", "kind": "combine", "tokens": 600, "experts": EXPERTS, "top_k": TOP_K, "width": HIDDEN,
         "padded": 0.0, "train": False},
        # fine-tuning: gradients of the rows and of the routing weights
        {"name": "combine_train_8192", "kind": "combine", "tokens": 8192, "experts": EXPERTS, "top_k": TOP_K, "width": HIDDEN,
         "padded": 0.05, "train": True},
        # a decode batch with everything: ragged histories, biases, a grammar
        {"name": "rules_decode_16", "kind": "rules", "rows": 16, "vocab": VOCAB, "history": 8192, "bias": 16, "mask": True, "dtype": "bf16"},
        # a wide decode batch, an odd vocabulary, penalties and masks
        {"name": "rules_decode_200", "kind": "rules", "rows": 200, "vocab": VOCAB - 7, "history": 1500, "bias": 0, "mask": True, "dtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("router", "router", "balance", "dispatch", "combine", "rules"))
    if kind == "rules":
        vocab = _log_int(rng, 1000, VOCAB)
        history = 0 if rng.random() < 0.15 else _log_int(rng, 1, 16384)
        return {"kind": kind, "rows": _log_int(rng, 1, 200), "vocab": vocab, "history": history, "bias": rng.choice((0, 1, 16, 300)),
                "mask": rng.random() < 0.6 or history == 0, "dtype": rng.choice(("bf16", "fp16", "fp32"))}
    experts = rng.choice((EXPERTS, EXPERTS, 128, 64, 8, _log_int(rng, 4, 1024)))
    top_k = rng.randint(1, min(experts, 10))
    tokens = _log_int(rng, 1, 65536 if kind in ("router", "balance") else 16384 * TOP_K // max(TOP_K, top_k))
    case = {"kind": kind, "tokens": tokens, "experts": experts, "top_k": top_k, "padded": rng.choice((0.0, 0.0, 0.05, 0.3)),
            "train": rng.random() < (0.6 if tokens >= 64 else 0.2)}
    if kind in ("router", "balance"):
        case["dtype"] = rng.choice(("bf16", "fp16", "fp32"))
        case["scoring"] = rng.choice(("softmax", "softmax", "sigmoid"))
        if kind == "router":
            case["normalize"] = rng.random() < 0.7
    else:
        case["width"] = HIDDEN if rng.random() < 0.5 else 8 * _log_int(rng, 8, 256)
    return case


# ------------------------------------------------------------------------------ inputs
def _scores(gen, case):
    """Scores of a gate with favourites [tokens, experts], in the type that the program keeps them in."""
    bias = torch.randn(case["experts"], device="cuda", generator=gen) * 0.5
    x = torch.randn(case["tokens"], case["experts"], device="cuda", generator=gen) * 2.0 + bias
    return x.to(DTYPES[case.get("dtype", "fp32")])


def _live(gen, case):
    return torch.rand(case["tokens"], device="cuda", generator=gen) >= case["padded"] if case["padded"] else None


def _experts_of(gen, case, scores):
    """Experts of every token, best first; none (-1) for the tokens that only fill the batch up."""
    ids = torch.topk(scores.float(), case["top_k"]).indices.to(torch.int32)
    live = _live(gen, case)
    return ids if live is None else torch.where(live[:, None], ids, -1)


def _rows(gen, rows, width):
    return torch.empty(rows, width, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "rules":
        b, v, n = case["rows"], case["vocab"], case["history"]
        s["logits"] = (torch.randn(b, v, device="cuda", generator=gen) * 3.0).to(DTYPES[case["dtype"]])
        if n:
            # some tokens come again and again; rows of every length up to the longest
            s["history"] = (torch.rand(b, n, device="cuda", generator=gen).pow_(4) * v).long()
            s["lengths"] = (torch.rand(b, device="cuda", generator=gen) * (n + 1)).int()
            s["lengths"][0] = n
            s["repetition"] = 1.0 + 0.3 * torch.rand(b, device="cuda", generator=gen)
            s["presence"] = 0.5 * torch.rand(b, device="cuda", generator=gen)
            s["frequency"] = 0.2 * torch.rand(b, device="cuda", generator=gen)
        if case["bias"]:
            s["bias_ids"] = torch.randint(-1, v, (b, case["bias"]), device="cuda", generator=gen)
            s["bias_ids"][:, -1] = s["bias_ids"][:, 0]   # named twice
            s["bias_values"] = torch.randn(b, case["bias"], device="cuda", generator=gen) * 2.0
        if case["mask"]:
            words = (v + 31) // 32
            draw = [torch.randint(-(1 << 31), 1 << 31, (b, words), device="cuda", generator=gen) for _ in range(3)]
            # grammars that allow one token in eight and ones that forbid one in eight
            tight = torch.rand(b, 1, device="cuda", generator=gen) < 0.5
            s["allowed"] = torch.where(tight, draw[0] & draw[1] & draw[2], draw[0] | draw[1] | draw[2]).to(torch.int32)
        return s
    scores = _scores(gen, case)
    if case["kind"] in ("router", "balance"):
        s["logits"] = scores.requires_grad_(case["train"])
        if case["kind"] == "router":
            s["mask"] = _live(gen, case)
            s["dw"] = torch.randn(case["tokens"], case["top_k"], device="cuda", generator=gen)
        else:
            s["ids"] = _experts_of(gen, case, scores.detach())
            s["dloss"] = torch.rand((), device="cuda", generator=gen) + 0.5
        return s
    t, k, h = case["tokens"], case["top_k"], case["width"]
    s["ids"] = _experts_of(gen, case, scores)
    if case["kind"] == "dispatch":
        s["x"] = _rows(gen, t, h).requires_grad_(case["train"])
        s["drows"] = _rows(gen, t * k, h) if case["train"] else None
        return s
    s["rows"] = _rows(gen, t * k, h).requires_grad_(case["train"])
    s["row_of_pair"] = _sorted_rows(s["ids"], case["experts"])[0]
    gate = torch.rand(t, k, device="cuda", generator=gen) + 0.25
    s["weights"] = (gate / gate.sum(1, keepdim=True)).requires_grad_(case["train"])
    s["dy"] = _rows(gen, t, h) if case["train"] else None
    return s


def _sorted_rows(ids, experts):
    """Row of every pair when the pairs are sorted by expert (-1: it names none), the pairs in that order, and how many there are."""
    flat = ids.reshape(-1).long()
    named = (flat >= 0) & (flat < experts)
    order = torch.sort(torch.where(named, flat, experts), stable=True).indices
    row = torch.empty_like(flat)
    row[order] = torch.arange(flat.numel(), device=flat.device)
    return torch.where(named, row, -1).to(torch.int32).reshape(ids.shape), order, named


# ------------------------------------------------------------------------------ one pass
def run(state):
    return _OWN[state["kind"]](state) if own else _PLAIN[state["kind"]](state)


def _router_own(s):
    import torch_ggml_ops_b200 as tgo

    w, ids = tgo.moe_router(s["logits"], s["top_k"], scoring=s["scoring"], normalize=s["normalize"], token_mask=s["mask"])
    return (w.detach(), ids, *torch.autograd.grad(w, s["logits"], s["dw"])) if s["train"] else (w, ids)


def _balance_own(s):
    import torch_ggml_ops_b200 as tgo

    loss, counts = tgo.moe_balance_loss(s["logits"], s["ids"], scoring=s["scoring"])
    return (loss.detach(), counts, *torch.autograd.grad(loss, s["logits"], s["dloss"])) if s["train"] else (loss, counts)


def _dispatch_own(s):
    import torch_ggml_ops_b200 as tgo

    rows, row_of_pair, indices, offsets = tgo.moe_dispatch(s["x"], s["ids"], s["experts"])
    return (rows.detach(), row_of_pair, indices, offsets, *(torch.autograd.grad(rows, s["x"], s["drows"]) if s["train"] else ()))


def _combine_own(s):
    import torch_ggml_ops_b200 as tgo

    y = tgo.moe_combine(s["rows"], s["row_of_pair"], s["weights"])
    return (y.detach(), *torch.autograd.grad(y, (s["rows"], s["weights"]), s["dy"])) if s["train"] else (y,)


def _rules_own(s):
    import torch_ggml_ops_b200 as tgo

    if "lengths" not in s:   # nothing has been generated yet
        return tgo.logit_rules(s["logits"], bias_ids=s.get("bias_ids"), bias_values=s.get("bias_values"), allowed=s.get("allowed"))
    return tgo.logit_rules(s["logits"], history=s["history"], history_lengths=s["lengths"], repetition_penalty=s["repetition"],
                           presence_penalty=s["presence"], frequency_penalty=s["frequency"], bias_ids=s.get("bias_ids"),
                           bias_values=s.get("bias_values"), allowed=s.get("allowed"))


def _log_scores(x, scoring):
    """Scores on a logarithmic scale, and their slope."""
    if scoring == "softmax":
        return x, torch.ones_like(x)
    far = torch.exp(-x.abs())
    return torch.clamp(x, max=0.0) - torch.log1p(far), torch.where(x > 0, far, 1.0) / (1.0 + far)


def _shares(u):
    """exp(u) over its sum, row by row; zeros for a row of -inf."""
    top = u.amax(1, keepdim=True)
    e = torch.exp(u - torch.where(top == -math.inf, 0.0, top))
    return e / torch.clamp(e.sum(1, keepdim=True), min=1e-30)


def _router_plain(s):
    x = s["logits"].detach().float()
    k, mask = s["top_k"], s["mask"]
    if mask is not None:
        x = torch.where(mask[:, None], x, -math.inf)
    value, order = torch.sort(x, dim=1, descending=True, stable=True)   # of equal scores the lower expert
    value, order = value[:, :k], order[:, :k]
    taken = value > -math.inf
    ids = torch.where(taken, order, -1).to(torch.int32)
    u, slope = _log_scores(x, s["scoring"])
    picked = u.gather(1, order)
    if s["normalize"]:
        w = _shares(picked)
    elif s["scoring"] == "softmax":
        w = _shares(u).gather(1, order)
    else:
        w = torch.exp(picked)
    w = torch.where(taken, w, 0.0)
    if not s["train"]:
        return w, ids
    g = torch.where(taken, s["dw"], 0.0)
    inner = (g * w).sum(1, keepdim=True)
    own_part = w * (g - inner) if s["normalize"] else w * g
    dx = torch.zeros_like(x)
    dx.scatter_(1, order, torch.where(taken, own_part, 0.0) * slope.gather(1, order))
    if s["scoring"] == "softmax" and not s["normalize"]:
        dx -= _shares(u) * inner
    return w, ids, dx.to(s["logits"].dtype)


def _balance_plain(s):
    x, experts, ids = s["logits"].detach().float(), s["experts"], s["ids"].long()
    named = (ids >= 0) & (ids < experts)
    live = named.any(1)
    counts = torch.zeros(experts, dtype=torch.int32, device=x.device)
    counts.scatter_add_(0, torch.where(named, ids, 0).reshape(-1), named.to(torch.int32).reshape(-1))
    u, slope = _log_scores(x, s["scoring"])
    p = torch.where(live[:, None], _shares(u), 0.0)
    n, pairs = torch.clamp(live.sum(), min=1), torch.clamp(named.sum(), min=1)
    share = counts.float() / pairs
    loss = experts * (share * (p.double().sum(0) / n).float()).sum()
    if not s["train"]:
        return loss, counts
    c = experts * share / n * s["dloss"]
    dx = p * (c - (p * c).sum(1, keepdim=True)) * slope
    return loss, counts, dx.to(s["logits"].dtype)


def _dispatch_plain(s):
    x, k, experts = s["x"].detach(), s["top_k"], s["experts"]
    row_of_pair, order, named = _sorted_rows(s["ids"], experts)
    rows = torch.where(named[order][:, None], x[order // k], 0)
    counts = torch.bincount(torch.where(named, s["ids"].reshape(-1).long(), experts), minlength=experts + 1)[:experts]
    out = (rows, row_of_pair, torch.arange(experts, device=x.device), torch.cumsum(counts, 0).to(torch.int32))
    if not s["train"]:
        return out
    index = torch.clamp(row_of_pair, min=0).reshape(-1).long()
    dx = torch.where(named[:, None], s["drows"][index].float(), 0.0).reshape(-1, k, x.shape[1]).sum(1)
    return *out, dx.to(x.dtype)


def _combine_plain(s):
    rows, w, k = s["rows"].detach(), s["weights"].detach(), s["top_k"]
    index, named = s["row_of_pair"].reshape(-1).long(), s["row_of_pair"] >= 0
    picked = torch.where(named[:, :, None], rows[torch.clamp(index, min=0)].float().reshape(-1, k, rows.shape[1]), 0.0)
    y = (picked * w[:, :, None]).sum(1).to(rows.dtype)
    if not s["train"]:
        return (y,)
    dy = s["dy"].float()
    dw = (picked * dy[:, None, :]).sum(2)
    drows = torch.zeros_like(rows)
    drows[index[named.reshape(-1)]] = (dy[:, None, :] * w[:, :, None]).to(rows.dtype)[named]
    return y, drows, dw


def _rules_plain(s):
    x = s["logits"].float()
    b, v = x.shape
    if "bias_ids" in s:
        ids = s["bias_ids"]
        x = x + torch.zeros_like(x).scatter_add_(1, torch.clamp(ids, min=0), torch.where(ids >= 0, s["bias_values"], 0.0))
    if "lengths" in s:
        ids, at = s["history"], torch.arange(s["history"].shape[1], device=x.device)
        counts = torch.zeros_like(x).scatter_add_(1, ids, (at < s["lengths"][:, None]).float())
        again = torch.where(x > 0, x / s["repetition"][:, None], x * s["repetition"][:, None])
        again = again - (counts * s["frequency"][:, None] + s["presence"][:, None])
        x = torch.where(counts > 0, again, x)
    if "allowed" in s:
        token = torch.arange(v, device=x.device)
        x = torch.where((s["allowed"][:, token // 32] >> (token % 32)) & 1 != 0, x, -math.inf)
    return x.to(s["logits"].dtype)


_OWN = {"router": _router_own, "balance": _balance_own, "dispatch": _dispatch_own, "combine": _combine_own, "rules": _rules_own}
_PLAIN = {"router": _router_plain, "balance": _balance_plain, "dispatch": _dispatch_plain, "combine": _combine_plain, "rules": _rules_plain}


# ------------------------------------------------------------------------------ what a pass needs
def work(case):
    """Every input once, every output once; an operation for each score, product and sum."""
    if case["kind"] == "rules":
        b, v, n = case["rows"], case["vocab"], case["history"]
        words = (v + 31) // 32 if case["mask"] else 0
        return {"bytes": b * (2 * v * SIZE[case["dtype"]] + n * 4 + words * 4 + case["bias"] * 12), "flops": 4 * b * v}
    t, k, e, train = case["tokens"], case["top_k"], case["experts"], case["train"]
    if case["kind"] in ("router", "balance"):
        scores = t * e * SIZE[case["dtype"]]
        if case["kind"] == "router":
            return {"bytes": scores + t * k * 8 + (t * k * 4 + scores if train else 0), "flops": (6 if train else 4) * t * e}
        return {"bytes": scores + t * k * 4 + e * 4 + (scores if train else 0), "flops": (8 if train else 4) * t * e}
    token, pairs = t * case["width"] * 2, t * k * case["width"] * 2
    if case["kind"] == "dispatch":
        return {"bytes": (token + pairs) * (2 if train else 1) + t * k * 8 + e * 12, "flops": t * k * case["width"] if train else 0}
    return {"bytes": token + pairs + t * k * 8 + (token + pairs + t * k * 4 if train else 0),
            "flops": (5 if train else 2) * t * k * case["width"]}


# ------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s)


def _router_exact(s):
    k, train = s["top_k"], s["train"]
    x = s["logits"].detach().double()
    live = torch.isfinite(x) if s["mask"] is None else torch.isfinite(x) & s["mask"][:, None]
    # rank of every expert in its row: those above it, and those before it that are its equal
    step = max(1, (1 << 27) // (x.shape[1] ** 2))
    rank = torch.cat([((p[:, None, :] > p[:, :, None]) | ((p[:, None, :] == p[:, :, None]) & (_before(x.shape[1]))[None])).sum(2)
                      for p in x.split(step)])
    slots = torch.argsort(rank, dim=1)[:, :k]
    taken = live.gather(1, slots)
    if s["scoring"] == "softmax":
        score = torch.softmax(x, 1)
    else:
        score = torch.sigmoid(x)
    chosen = torch.zeros_like(live).scatter_(1, slots, True) & live
    total = (score * chosen).sum(1, keepdim=True)
    weight = torch.where(chosen, score / total, 0.0) if s["normalize"] else score * chosen
    out = (weight.gather(1, slots), torch.where(taken, slots, -1).to(torch.int32))
    if not train:
        return out
    g = torch.zeros_like(x).scatter_(1, slots, s["dw"].double() * taken)
    dscore = g * chosen
    if s["normalize"]:
        dscore = torch.where(chosen, (dscore - (dscore * weight).sum(1, keepdim=True)) / total, 0.0)
    if s["scoring"] == "softmax":
        dx = score * (dscore - (dscore * score).sum(1, keepdim=True))
    else:
        dx = dscore * score * torch.sigmoid(-x)
    return *out, dx


def _before(n):
    i = torch.arange(n, device="cuda")
    return i[None, :] < i[:, None]


def _balance_exact(s):
    x, ids, experts = s["logits"].detach().double().requires_grad_(s["train"]), s["ids"], s["experts"]
    live = ids[:, 0] >= 0
    score = torch.softmax(x, 1) if s["scoring"] == "softmax" else torch.sigmoid(x) / torch.sigmoid(x).sum(1, keepdim=True)
    counts = torch.bincount(ids[ids >= 0].long(), minlength=experts)
    if not bool(live.any()):
        zero = torch.zeros((), dtype=torch.float64, device="cuda")
        return (zero, counts.to(torch.int32), torch.zeros_like(x)) if s["train"] else (zero, counts.to(torch.int32))
    loss = experts * torch.dot(counts.double() / counts.sum(), score[live].mean(0))
    if not s["train"]:
        return loss, counts.to(torch.int32)
    return loss.detach(), counts.to(torch.int32), *torch.autograd.grad(loss, x, s["dloss"].double())


def _dispatch_exact(s):
    t, k, experts = s["tokens"], s["top_k"], s["experts"]
    ids = s["ids"].reshape(-1).long().cpu()
    row_of_pair = torch.full((t * k,), -1, dtype=torch.int32)
    ends, at, pairs = [], 0, []
    for e in range(experts):
        mine = torch.nonzero(ids == e)[:, 0]
        row_of_pair[mine] = torch.arange(at, at + mine.numel(), dtype=torch.int32)
        pairs.append(mine)
        at += mine.numel()
        ends.append(at)
    pairs = torch.cat(pairs).cuda()
    rows = torch.zeros(t * k, s["width"], dtype=torch.float64, device="cuda")
    rows[:at] = s["x"].detach().double()[pairs // k]
    out = (rows, row_of_pair.reshape(t, k), torch.arange(experts), torch.tensor(ends, dtype=torch.int32))
    if not s["train"]:
        return out
    return *out, torch.zeros(t, s["width"], dtype=torch.float64, device="cuda").index_add_(0, pairs // k, s["drows"][:at].double())


def _combine_exact(s):
    rows, w = s["rows"].detach(), s["weights"].detach().double()
    t, k, h = s["tokens"], s["top_k"], s["width"]
    y, dw = torch.zeros(t, h, dtype=torch.float64, device="cuda"), torch.zeros(t, k, dtype=torch.float64, device="cuda")
    drows = torch.zeros(t * k, h, dtype=torch.float64, device="cuda")
    for j in range(k):
        tokens = torch.nonzero(s["row_of_pair"][:, j] >= 0)[:, 0]
        at = s["row_of_pair"][tokens, j].long()
        y[tokens] += w[tokens, j, None] * rows[at].double()
        if s["train"]:
            dw[tokens, j] = torch.linalg.vecdot(rows[at].double(), s["dy"][tokens].double())
            drows[at] = w[tokens, j, None] * s["dy"][tokens].double()
    return (y, drows, dw) if s["train"] else (y,)


def _rules_exact(s):
    x = s["logits"].double()
    b, v = x.shape
    row = torch.arange(b, device="cuda")[:, None]
    if "bias_ids" in s:
        named = s["bias_ids"] >= 0
        x = x.index_put((row.expand_as(named)[named], s["bias_ids"][named]), s["bias_values"].double()[named], accumulate=True)
    if "lengths" in s:
        inside = torch.arange(s["history"].shape[1], device="cuda")[None, :] < s["lengths"][:, None]
        counts = torch.bincount((row * v + s["history"])[inside], minlength=b * v).reshape(b, v)
        for i in range(b):
            seen = torch.nonzero(counts[i])[:, 0]
            old, n = x[i, seen], counts[i, seen]
            rep, freq, pres = (s[name][i].double() for name in ("repetition", "frequency", "presence"))
            x[i, seen] = torch.where(old > 0, old / rep, old * rep) - n * freq - pres
    if "allowed" in s:
        for bit in range(32):
            words = (s["allowed"] >> bit) & 1
            x[:, bit::32] = torch.where(words[:, : x[:, bit::32].shape[1]] != 0, x[:, bit::32], -math.inf)
    return x


_EXACT = {"router": _router_exact, "balance": _balance_exact, "dispatch": _dispatch_exact, "combine": _combine_exact, "rules": _rules_exact}
