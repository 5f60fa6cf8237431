"""Log probabilities of sequences under a causal LM, with their gradient: the
policy-update side of the log probabilities that `generate(return_logprobs)`
reports (the reference trainer's log-softmax + gather over rollout tokens).

Log probability, entropy and their gradient are fg_token_logprobs /
fg_token_logprobs_backward on the logits of a chunk of positions.  No more than
one chunk's logits are kept: where there are several, each is made again in its
backward pass (and its gradient, of the same size, lives with it).
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable
from torch.utils.checkpoint import checkpoint

from .. import ops
from .verify import unwrap_causal_lm


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        r = ops.token_logprobs(logits, tokens, temperature=temperature)
        # (the entropy is an output, which the caller may change in place)
        ctx.save_for_backward(logits, tokens, r.lse, r.entropy.clone())
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return r.logp, r.entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logp, grad_entropy):
        if grad_logp is None and grad_entropy is None:
            return None, None, None
        logits, tokens, lse, entropy = ctx.saved_tensors
        g = torch.zeros_like(lse) if grad_logp is None else grad_logp.float().contiguous()
        h = None if grad_entropy is None else grad_entropy.float().contiguous()
        return ops.token_logprobs_backward(logits, tokens, lse, entropy, g, h, temperature=ctx.temperature), None, None


def _check_ids(ids: torch.Tensor, least: int | None, end: int, name: str):
    """Refuses ids outside [least, end): one host sync where they are on the
    GPU, so not during a capture."""
    if ids.is_cuda and torch.cuda.is_current_stream_capturing():
        return
    bad = ids >= end if least is None else (ids >= end) | (ids < least)
    if bool(bad.any()):
        raise ValueError(f"{name} must be below the vocabulary's {end} entries"
                         + ("" if least is None else f" and at least {least}"))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0):
    """(log probability, entropy) f32 [n] of tokens (int32 [n], negative:
    padded, zeros) under softmax(logits / temperature), logits [n, vocab] with
    contiguous rows; differentiable with respect to the logits.  A token
    behind the vocabulary is refused (outside stream captures, in which it
    gets zeros and sets the device error word)."""
    if logits.shape[0] != tokens.shape[0]:  # the gradient has one row per token
        raise ValueError("logits and tokens must have one row each per entry")
    # the kernel would give such an entry zeros and record it in the device
    # error word, which nobody reads here
    _check_ids(tokens, None, logits.shape[-1], "tokens")
    return _TokenLogprobs.apply(logits, tokens, float(temperature))


def sequence_logprobs(causal_lm, input_ids: torch.Tensor, attention_mask: torch.Tensor, *, prompt_len: int,
                      temperature: float = 1.0, chunk: int = 4096):
    """(log probability, entropy) f32 [B, S - prompt_len] of the tokens from
    position prompt_len on (at least 1), each given the tokens before it;
    zeros at positions with attention_mask 0.  Differentiable; `chunk`
    positions' logits are made and kept at a time (in training the lm_head of
    more than one chunk runs twice).  Ids outside the embedding or the lm_head
    are refused before anything runs."""
    B, S = input_ids.shape
    if not 1 <= prompt_len < S:
        raise ValueError("prompt_len must leave at least one token on each side")
    if attention_mask.shape != input_ids.shape:
        raise ValueError("attention_mask must have the shape of input_ids")
    base = unwrap_causal_lm(causal_lm)
    _check_ids(input_ids, 0, base.model.get_input_embeddings().weight.shape[0], "input_ids")
    scored = torch.where(attention_mask.to(input_ids.device) > 0, input_ids, 0)[:, prompt_len:]
    _check_ids(scored, 0, base.lm_head.weight.shape[0], "scored input_ids")
    dev = base.lm_head.weight.device
    ids, mask = input_ids.to(dev), attention_mask.to(dev).long()
    pos = (mask.cumsum(-1) - 1).clamp(min=0)
    hidden = base.model(input_ids=ids, attention_mask=mask, position_ids=pos, use_cache=False,
                        return_dict=True).last_hidden_state
    hidden = hidden[:, prompt_len - 1:S - 1].reshape(-1, hidden.shape[-1])
    tokens = torch.where(mask > 0, ids, -1)[:, prompt_len:].reshape(-1).to(torch.int32)

    def score(h, t):
        return _TokenLogprobs.apply(base.lm_head(h), t, float(temperature))

    n, chunk = hidden.shape[0], int(chunk)
    if torch.is_grad_enabled() and n > chunk:
        score = functools.partial(checkpoint, score, use_reentrant=False)
    out = [score(hidden[a:a + chunk], tokens[a:a + chunk].contiguous()) for a in range(0, n, chunk)]
    logp, entropy = (torch.cat(x).view(B, S - prompt_len) for x in zip(*out))
    return logp, entropy
