"""The routing of a mixture-of-experts layer on one GPU, around the grouped products: from a gate's scores to
every token's experts (``moe_router``), how evenly they are used (``moe_balance_loss``), tokens to rows sorted by
expert and back (``moe_dispatch``, ``moe_combine``).  With ``moe_mlp`` or the grouped products between the last two
a layer is

    weights, ids = moe_router(x @ gate.t(), top_k)
    rows, row_of_pair, experts, ends = moe_dispatch(x, ids, num_experts)
    y = moe_combine(moe_mlp(rows, w_gate, w_up, w_down, experts, ends, qt, qt_down, ffn), row_of_pair, weights)
    balance, pairs = moe_balance_loss(x @ gate.t(), ids)

and differentiable with respect to ``x`` and the gate.  The reference leaves all of it to its caller (its grouped
operators take rows sorted by expert: csrc/mmq_hip.cu:325-406).  ``PeerMoEMLP.plan`` takes what ``moe_router`` gives.

Kernels: ``csrc/router.cu`` and ``csrc/dispatch.cu``; registered in ``csrc/torch_ext_routing.cpp``.  No CPU or eager
fallback.
"""
from __future__ import annotations

import torch

_NS = "torch_ggml_ops_b200"
_ops = torch.ops.torch_ggml_ops_b200
SCORINGS = {"softmax": 0, "sigmoid": 1}


@torch.library.register_fake(f"{_NS}::moe_router")
def _(logits, top_k, scoring, normalize, token_mask):
    shape = (*logits.shape[:-1], top_k)
    return logits.new_empty(shape, dtype=torch.float32), logits.new_empty(shape, dtype=torch.int32)


@torch.library.register_fake(f"{_NS}::moe_router_grad")
def _(grad, logits, expert_ids, weights, scoring, normalize):
    return logits.new_empty(logits.shape)


@torch.library.register_fake(f"{_NS}::moe_balance_loss")
def _(logits, expert_ids, scoring):
    e = logits.shape[-1]
    return (logits.new_empty((), dtype=torch.float32), logits.new_empty((e,), dtype=torch.int32), logits.new_empty((e,), dtype=torch.float32))


@torch.library.register_fake(f"{_NS}::moe_balance_grad")
def _(grad, logits, expert_ids, coef, scoring):
    return logits.new_empty(logits.shape)


@torch.library.register_fake(f"{_NS}::moe_dispatch")
def _(input, expert_ids, num_experts):
    return (input.new_empty((expert_ids.numel(), input.shape[-1])), torch.empty_like(expert_ids),
            expert_ids.new_empty((num_experts,), dtype=torch.int64), expert_ids.new_empty((num_experts,)))


@torch.library.register_fake(f"{_NS}::moe_dispatch_grad")
def _(grad, row_of_pair):
    return grad.new_empty((*row_of_pair.shape[:-1], grad.shape[1]))


@torch.library.register_fake(f"{_NS}::moe_combine")
def _(rows, row_of_pair, weights):
    return rows.new_empty((*row_of_pair.shape[:-1], rows.shape[1]))


@torch.library.register_fake(f"{_NS}::moe_combine_grad")
def _(grad, rows, row_of_pair, weights, need_rows, need_weights):
    return (torch.empty_like(rows) if need_rows else rows.new_empty((0, rows.shape[1])),
            rows.new_empty(row_of_pair.shape if need_weights else (0,), dtype=torch.float32))


@torch.library.register_fake(f"{_NS}::moe_combine_rows_grad")
def _(grad, row_of_pair, weights, n_rows):
    return grad.new_empty((n_rows, grad.shape[-1]))


def _scoring(name: str) -> int:
    try:
        return SCORINGS[name]
    except KeyError:
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid'; got {name!r}") from None


def moe_router(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", normalize: bool = True,
               token_mask: torch.Tensor | None = None):
    """Experts of every token and their weights from a gate's scores ``logits`` [..., experts] (bf16, fp16 or fp32;
    up to 1024 experts; a matrix may have rows that lie apart).  Returns ``(weights, expert_ids)``, fp32 and int32
    [..., top_k] (top_k up to 32).

    ``expert_ids``: the largest scores, largest first; of equal ones the lower expert first.  ``weights``: with
    ``normalize`` they add up to one, as softmax of the chosen scores (``scoring="softmax"``) or as
    sigmoid(score) over the sum of the chosen (``"sigmoid"``); without it softmax over all experts, or sigmoid(score).

    ``token_mask`` (bool [...]): tokens that only fill a batch up are False; they get expert -1 and weight 0, as do
    choices for which only scores of -inf (experts switched off) or NaN are left.  Pairs with expert -1 are what
    ``moe_dispatch`` and ``PeerMoEMLP.plan`` drop.  A NaN among a token's scores makes its weights NaN.

    The weights are differentiable with respect to ``logits``, once."""
    return _ops.moe_router.default(logits, top_k, _scoring(scoring), normalize, token_mask)


def moe_balance_loss(logits: torch.Tensor, expert_ids: torch.Tensor, *, scoring: str = "softmax"):
    """``(loss, counts)``: loss = experts * sum over experts of f * P, with f an expert's share of all pairs (token,
    expert id) and P the mean over the tokens of its probability (softmax of ``logits``, or sigmoid over the sum of
    the sigmoids); 1 where the experts are used evenly.  ``counts`` (int32 [experts]): pairs of every expert.

    ``expert_ids`` [..., top_k] int32 as ``moe_router`` gives them.  A token all of whose ids are outside the experts
    (padding) takes no part; without any token the loss is 0.  The loss is differentiable with respect to
    ``logits`` (the counts are constants), once; the same call gives the same bits.  That gradient is of the order of one over
    the tokens and has the logits' type: of fp16 logits of thousands of tokens it falls among fp16's subnormals, so scale the
    loss, as one does in fp16, or give the scores in bf16 or fp32."""
    return _ops.moe_balance_loss.default(logits, expert_ids, _scoring(scoring))[:2]


def moe_dispatch(input: torch.Tensor, expert_ids: torch.Tensor, num_experts: int):
    """Token rows ``input`` [..., width] (bf16, width a multiple of 8) to rows sorted by expert: returns ``(rows,
    row_of_pair, expert_indices, expert_offsets)``.  ``rows`` [pairs, width] with the last two are what
    ``grouped_mmq``, ``grouped_mmq_pair`` and ``moe_mlp`` take (every expert a group, empty ones too; up to 4096
    experts).  ``row_of_pair`` (int32, like ``expert_ids`` [..., top_k]): each pair's row, for ``moe_combine``; -1 for
    pairs whose id names no expert.  Rows behind the last expert's are zeros; the grouped products leave theirs as they are.

    ``rows`` is differentiable with respect to ``input`` (the pairs' gradients are added in fp32)."""
    return _ops.moe_dispatch.default(input, expert_ids, num_experts)


def moe_combine(rows: torch.Tensor, row_of_pair: torch.Tensor, weights: torch.Tensor | None = None):
    """``out[..., :] = sum over a token's pairs of weights * rows[row_of_pair]`` (fp32 sums, one rounding): rows
    [rows, width] bf16 sorted by expert back to tokens.  ``row_of_pair`` int32 [..., top_k] as ``moe_dispatch`` gives
    it, ``weights`` fp32 of the same shape (None: 1).  Pairs whose row is not in ``rows`` add nothing.

    Differentiable with respect to ``rows`` and ``weights``, once (a row that no pair names gets a gradient of
    zeros, one that several name their sum).  Only a gradient of the weights needs ``rows`` again: without one they are
    not kept for the backward pass and may be written over."""
    return _ops.moe_combine.default(rows, row_of_pair, weights)


__all__ = ["moe_balance_loss", "moe_combine", "moe_dispatch", "moe_router"]
