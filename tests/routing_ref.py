"""The routing operators and the rules on logits in 64 bits, token by token, and how far fp32 arithmetic
may take a result from them.  U = 2^-24: what one fp32 operation is off by, relative to its result."""
import math

import torch

U = 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}   # half the least subnormal


def log_scores(x, scoring):
    """u and du/dx for scores x (double)."""
    if scoring == "softmax":
        return x, torch.ones_like(x)
    return torch.nn.functional.logsigmoid(x), torch.sigmoid(-x)


def softmax(u):
    top = u.max()
    if top == -math.inf:
        return torch.zeros_like(u)
    e = torch.exp(u - top)
    return e / e.sum()


def router(logits, k, scoring, normalize, mask=None):
    x = logits.detach().double().cpu().reshape(-1, logits.shape[-1])
    mask = None if mask is None else mask.cpu().reshape(-1)
    ids = torch.full((x.shape[0], k), -1, dtype=torch.int32)
    w = torch.zeros(x.shape[0], k, dtype=torch.float64)
    for t in range(x.shape[0]):
        if mask is not None and not mask[t]:
            continue
        row = x[t].tolist()
        order = sorted((e for e in range(len(row)) if row[e] > -math.inf), key=lambda e: (-row[e], e))[:k]
        if not order:
            continue
        ids[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
        u = log_scores(x[t], scoring)[0]
        if normalize:
            w[t, :len(order)] = softmax(u[order])
        elif scoring == "softmax":
            w[t, :len(order)] = softmax(u)[order]
        else:
            w[t, :len(order)] = torch.exp(u[order])
    return w.reshape(*logits.shape[:-1], k), ids.reshape(*logits.shape[:-1], k)


def router_grad(logits, ids, g, scoring, normalize):
    """Gradient of sum(g * weights) and, for each entry, the sum of the sizes of what it is the difference of."""
    x, ids, g = logits.detach().double().cpu().reshape(-1, logits.shape[-1]), ids.cpu().reshape(-1, ids.shape[-1]), g.double().cpu().reshape(-1, ids.shape[-1])
    dx, size = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[0]):
        named = ids[t] >= 0
        if not named.any():
            continue
        at, gt = ids[t][named].long(), g[t][named]
        u, slope = log_scores(x[t], scoring)
        p = torch.zeros_like(u)
        if normalize:
            p[at] = softmax(u[at])
        else:
            p = softmax(u) if scoring == "softmax" else torch.exp(u)
        full = torch.zeros_like(u)
        full[at] = gt
        if normalize or scoring == "softmax":
            dx[t] = p * (full - (full * p).sum()) * slope
            size[t] = p * (full.abs() + (full * p).abs().sum()) * slope
        else:
            dx[t] = p * full * slope
            size[t] = dx[t].abs()
    return dx.reshape(logits.shape), size.reshape(logits.shape)


def spread(logits, scoring):
    """Largest distance of a finite u from its row's largest: an exponent's error grows with it."""
    u = log_scores(logits.detach().double().cpu().reshape(-1, logits.shape[-1]), scoring)[0]
    u = torch.where(torch.isfinite(u), u, torch.nan)
    top = torch.nan_to_num(u, nan=-math.inf).amax(1, keepdim=True)
    return float(torch.nan_to_num(torch.minimum(top - u, torch.full_like(u, 110.0)) + u.abs().clamp(max=110.0), nan=0.0).max())


def balance(logits, ids, scoring):
    """loss, counts, gradient and the sizes of its parts."""
    e = logits.shape[-1]
    x, ids = logits.detach().double().cpu().reshape(-1, e), ids.cpu().reshape(-1, ids.shape[-1]).long()
    named = (ids >= 0) & (ids < e)
    counts = torch.bincount(ids[named], minlength=e)
    live = named.any(1)
    n = int(live.sum())
    dx, size = torch.zeros_like(x), torch.zeros_like(x)
    if n == 0:
        return torch.zeros((), dtype=torch.float64), counts, dx.reshape(logits.shape), size.reshape(logits.shape)
    f = counts.double() / counts.sum()
    total = torch.zeros(e, dtype=torch.float64)
    c = e * f / n
    for t in torch.nonzero(live)[:, 0].tolist():
        u, slope = log_scores(x[t], scoring)
        p = softmax(u)
        total += p
        inner = (c * p).sum()
        dx[t], size[t] = p * (c - inner) * slope, p * (c + inner) * slope
    return e * (f * total / n).sum(), counts, dx.reshape(logits.shape), size.reshape(logits.shape)


def sort_rows(ids, experts):
    """row_of_pair and end rows of a stable sort by expert."""
    flat = ids.cpu().reshape(-1).tolist()
    row, ends, at = [-1] * len(flat), [], 0
    for e in range(experts):
        for i, v in enumerate(flat):
            if v == e:
                row[i] = at
                at += 1
        ends.append(at)
    return torch.tensor(row, dtype=torch.int32).reshape(ids.shape), torch.tensor(ends, dtype=torch.int32)


def combine(rows, row_of_pair, w):
    """Result and, entry by entry, the sum of the products' sizes."""
    r, at = rows.detach().double().cpu(), row_of_pair.cpu().reshape(-1, row_of_pair.shape[-1])
    w = torch.ones(at.shape, dtype=torch.float64) if w is None else w.detach().double().cpu().reshape(at.shape)
    y, size = torch.zeros(at.shape[0], r.shape[1], dtype=torch.float64), torch.zeros(at.shape[0], r.shape[1], dtype=torch.float64)
    for t in range(at.shape[0]):
        for s in range(at.shape[1]):
            if 0 <= at[t, s] < r.shape[0]:
                y[t] += w[t, s] * r[at[t, s]]
                size[t] += (w[t, s] * r[at[t, s]]).abs()
    shape = (*row_of_pair.shape[:-1], r.shape[1])
    return y.reshape(shape), size.reshape(shape)


def combine_grad(dy, rows, row_of_pair, w):
    """d_rows and its size, d_weights and its size."""
    r, at = rows.detach().double().cpu(), row_of_pair.cpu().reshape(-1, row_of_pair.shape[-1])
    dy = dy.double().cpu().reshape(at.shape[0], -1)
    w = torch.ones(at.shape, dtype=torch.float64) if w is None else w.detach().double().cpu().reshape(at.shape)
    d_rows, rows_size = torch.zeros_like(r), torch.zeros_like(r)
    d_w, w_size = torch.zeros(at.shape, dtype=torch.float64), torch.zeros(at.shape, dtype=torch.float64)
    for t in range(at.shape[0]):
        for s in range(at.shape[1]):
            if 0 <= at[t, s] < r.shape[0]:
                d_rows[at[t, s]] += w[t, s] * dy[t]
                rows_size[at[t, s]] += (w[t, s] * dy[t]).abs()
                d_w[t, s] = (dy[t] * r[at[t, s]]).sum()
                w_size[t, s] = (dy[t] * r[at[t, s]]).abs().sum()
    return d_rows, rows_size, d_w.reshape(row_of_pair.shape), w_size.reshape(row_of_pair.shape)


def rules(logits, history=None, lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias_ids=None, bias_values=None, allowed=None):
    """Result (double) and the sizes of its parts, token by token."""
    x = logits.detach().double().cpu()
    b, v = x.shape
    size = x.abs().clone()

    def row_of(t, i):
        return None if t is None else (t[i] if t.dim() == 2 else t).cpu().tolist()

    def number(p, i):
        return float(p[i].double()) if isinstance(p, torch.Tensor) else float(torch.tensor(p, dtype=torch.float32))

    for i in range(b):
        ids, values = row_of(bias_ids, i), row_of(bias_values, i)
        for j, t in enumerate(ids or []):
            if 0 <= t < v:
                x[i, t] += values[j]
                size[i, t] += abs(values[j])
        counts = {}
        h = row_of(history, i) or []
        n = len(h) if lengths is None else max(0, min(len(h), int(lengths[i])))
        for t in h[:n]:
            if 0 <= t < v:
                counts[t] = counts.get(t, 0) + 1
        for t, c in counts.items():
            rep, pres, freq = number(repetition, i), number(presence, i), number(frequency, i)
            a = float(x[i, t])
            a = a / rep if a > 0 else a * rep
            x[i, t] = a - (c * freq + pres)
            size[i, t] = size[i, t] * max(rep, 1 / rep) + abs(c * freq) + abs(pres)
        words = row_of(allowed, i)
        if words is not None:
            on = torch.tensor([(words[t // 32] >> (t % 32)) & 1 for t in range(v)], dtype=torch.bool)
            x[i][~on] = -math.inf
    return x, size


def near(got, want, room):
    """got within room (entry by entry) of want; infinities and NaN where want has them."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    ok = same | ((got - want).abs() <= room)
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} entries off; worst {float(torch.nan_to_num((got - want).abs() / torch.as_tensor(room)).max()):.3g} times the room"
