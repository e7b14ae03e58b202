"""What a generation step does to a head's logits (``mmq`` on the head's weight) before a token is taken from them:
biases, penalties for tokens that came before and a grammar's mask, in one launch (``csrc/logit_rules.cu``;
registered in ``csrc/torch_ext_routing.cpp``).  The reference stops at the head's product."""
from __future__ import annotations

import torch

_NS = "torch_ggml_ops_b200"
_ops = torch.ops.torch_ggml_ops_b200


@torch.library.register_fake(f"{_NS}::logit_rules")
def _(logits, history, history_lengths, repetition, repetition_all, presence, presence_all, frequency, frequency_all, bias_ids, bias_values, allowed):
    return logits.new_empty(logits.shape)


@torch.library.register_fake(f"{_NS}::logit_rules_out")
def _(logits, history, history_lengths, repetition, repetition_all, presence, presence_all, frequency, frequency_all, bias_ids, bias_values, allowed, out):
    return None


def logit_rules(logits: torch.Tensor, *, history: torch.Tensor | None = None, history_lengths: torch.Tensor | None = None,
                repetition_penalty: float | torch.Tensor = 1.0, presence_penalty: float | torch.Tensor = 0.0,
                frequency_penalty: float | torch.Tensor = 0.0, bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None,
                allowed: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Applies, row by row of ``logits`` ([rows, vocab] or [vocab]; bf16, fp16 or fp32), in this order and in fp32:

    * biases: ``x += bias_values[j]`` for every j with ``bias_ids[j]`` = token (one token's biases are added up first);
    * penalties, with c = occurrences of the token in the row's history, where c > 0: ``x = x / repetition_penalty`` if
      x > 0, else ``x * repetition_penalty``; then ``x -= c * frequency_penalty + presence_penalty``;
    * the mask: ``x = -inf`` where bit ``token % 32`` of ``allowed[token // 32]`` is 0.

    ``history`` (int32 or int64 [rows, n]): ids of prompt and answer so far, of which the first ``history_lengths``
    (int32 or int64 [rows]; None: all) count.  The penalties are numbers or fp32 tensors [rows]; a repetition
    penalty has to be positive.  ``bias_ids`` (int32 or int64) and ``bias_values`` (fp32) [rows, n], ``allowed`` (int32
    [rows, at least vocab / 32]).  Of history, biases and mask one row ([n]) may serve all rows; their rows may lie
    apart.  Ids outside the vocabulary name nothing (pad with -1).  A row whose mask leaves no token is -inf throughout.

    Returns a new tensor like ``logits``, or writes ``out``, which may be ``logits`` itself: then only what changes is
    written.  For generation: no gradient, and tensors that want one are refused."""
    rep, rep_all = (repetition_penalty, 1.0) if isinstance(repetition_penalty, torch.Tensor) else (None, repetition_penalty)
    pres, pres_all = (presence_penalty, 0.0) if isinstance(presence_penalty, torch.Tensor) else (None, presence_penalty)
    freq, freq_all = (frequency_penalty, 0.0) if isinstance(frequency_penalty, torch.Tensor) else (None, frequency_penalty)
    args = (logits, history, history_lengths, rep, rep_all, pres, pres_all, freq, freq_all, bias_ids, bias_values, allowed)
    if out is None:
        return _ops.logit_rules.default(*args)
    _ops.logit_rules_out.default(*args, out)
    return out


__all__ = ["logit_rules"]
