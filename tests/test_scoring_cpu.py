"""The differentiable log probabilities on the CPU: the launches are replaced by
the formulas, what is tested is what lies around them (autograd, refusals)."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture
def scoring(monkeypatch):
    """engine.scoring with fg_token_logprobs and its gradient computed by torch on the CPU, into the tensors that the
    wrappers pass."""
    from flashgrpo_b200 import ops
    from flashgrpo_b200.engine import scoring as s

    known = {}  # address -> tensor: the stand-in of a launch sees pointers alone

    def ptr(t):
        if t is None:
            return None
        known[t.data_ptr()] = t
        return t.data_ptr()

    def call(t, name, *a, **kw):
        get = lambda p: None if p is None else known[p]  # noqa: E731
        if name == "fg_token_logprobs":
            logits, tok, T = get(a[0]), get(a[6]), a[8]
            logp, ent, lse = map(get, a[9:12])
            n = tok.numel()
            x = logits[:n].detach().float() / T
            z = torch.log_softmax(x, 1)
            live = tok >= 0
            zero = torch.zeros(())
            logp.copy_(torch.where(live, z.gather(1, tok.clamp(min=0).long()[:, None])[:, 0], zero))
            ent.copy_(torch.where(live, -(z.exp() * z).sum(1), zero))
            lse.copy_(torch.where(live, torch.logsumexp(x, 1), zero))
        else:
            assert name == "fg_token_logprobs_backward"
            logits, tok, n, T = get(a[0]), get(a[4]), a[5], a[6]
            lse, ent, g, h, out = map(get, a[7:12])
            z = logits[:n].detach().float() / T - lse[:, None]
            one = torch.zeros_like(z).scatter_(1, tok.clamp(min=0).long()[:, None], 1.0)
            d = g[:, None] * (one - z.exp())
            if h is not None:
                d = d - h[:, None] * z.exp() * (z + ent[:, None])
            out[:n].copy_((d / T).masked_fill((tok < 0)[:, None], 0.0))

    monkeypatch.setattr(ops, "_ptr", ptr)
    monkeypatch.setattr(ops, "_call", call)
    monkeypatch.setattr(ops, "_stream", lambda t: None)
    monkeypatch.setattr(ops, "_need", lambda t, name, dtype=None, contiguous=True: None)
    return s


def plain(logits, tok, T=1.0):
    z = torch.log_softmax(logits / T, -1)
    live = tok >= 0
    lp = z.gather(1, tok.clamp(min=0).long()[:, None])[:, 0]
    return torch.where(live, lp, torch.zeros(())), torch.where(live, -(z.exp() * z).sum(1), torch.zeros(()))


def case(n=7, V=31):
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, V, (n,), generator=g, dtype=torch.int32)
    tok[2] = -1
    return torch.randn(n, V, generator=g).requires_grad_(), tok, torch.randn(n, generator=g)


@pytest.mark.parametrize("change", [lambda lp, w: lp.mul_(w), lambda lp, w: lp.__setitem__(w > 0, 0.0),
                                    lambda lp, w: lp.detach().zero_()], ids=["mul_", "setitem", "detached"])
def test_log_probabilities_can_be_changed_in_place(scoring, change):
    """What a trainer does to them behind the call (a mask, a weight); the entropy stays usable.  fp32 sums of 31 terms
    on both sides."""
    logits, tok, w = case()
    lp, ent = scoring.token_logprobs(logits, tok)
    change(lp, w)
    (lp.sum() + (w * ent).sum()).backward()
    x = logits.detach().clone().requires_grad_()
    lp2, ent2 = plain(x, tok)
    lp2 = lp2.clone()
    change(lp2, w)
    (lp2.sum() + (w * ent2).sum()).backward()
    assert (logits.grad - x.grad).abs().max() < 64 * 2.0 ** -24 * 8


def test_outputs_are_tensors_of_their_own(scoring):
    from flashgrpo_b200 import ops

    logits, tok, _ = case()
    r = ops.token_logprobs(logits.detach(), tok)
    assert all(t._base is None for t in (r.logp, r.entropy, r.lse))
    assert len({t.untyped_storage().data_ptr() for t in (r.logp, r.entropy, r.lse)}) == 3


@pytest.mark.parametrize("change", [lambda e, w: e.mul_(w), lambda e, w: e.__setitem__(w > 0, 0.0),
                                    lambda e, w: e.detach().zero_()], ids=["mul_", "setitem", "detached"])
def test_entropies_can_be_changed_in_place(scoring, change):
    """The gradient reads the entropy of the forward, not what the caller made of it."""
    logits, tok, w = case()
    lp, ent = scoring.token_logprobs(logits, tok)
    change(ent, w)
    ((w * lp).sum() + ent.sum()).backward()
    x = logits.detach().clone().requires_grad_()
    lp2, ent2 = plain(x, tok)
    ent2 = ent2.clone()
    change(ent2, w)
    ((w * lp2).sum() + ent2.sum()).backward()
    assert (logits.grad - x.grad).abs().max() < 64 * 2.0 ** -24 * 8


def test_logits_rows_behind_the_tokens_are_refused(scoring):
    """Their gradient would lack those rows, which autograd notices in the backward pass alone."""
    logits, tok, _ = case()
    for bad in (tok[:5], tok[:0]):
        with pytest.raises(ValueError):
            scoring.token_logprobs(logits, bad)


@pytest.fixture(scope="module")
def causal_lm():
    from flashgrpo_b200.utils import synthetic

    return synthetic.build_model(1)


def sequences(B=3, S=20):
    ids = torch.randint(0, 4096, (B, S), generator=torch.Generator().manual_seed(2))
    mask = torch.ones_like(ids)
    mask[1, :4] = 0
    return ids, mask


@pytest.mark.parametrize("chunk", [7, 1000])
def test_sequence_logprobs_keep_one_chunk_of_logits(scoring, causal_lm, chunk):
    """Between the forward and the backward pass no [positions, vocab] tensor of several chunks is saved, and the
    gradient is that of the whole (fp32 sums over the vocabulary of 4096 and the positions in another order)."""
    ids, mask = sequences()
    w = causal_lm.lm_head.weight.requires_grad_(True)
    saved = []
    try:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(tuple(t.shape)) or t, lambda t: t):
            lp, ent = scoring.sequence_logprobs(causal_lm, ids, mask, prompt_len=5, chunk=chunk)
        kept = [s for s in saved if len(s) == 2 and s[1] == 4096 and s[0] != 256]  # (256: the lm_head, transposed)
        assert len(kept) == (1 if chunk >= 45 else 0), kept
        got = torch.autograd.grad(lp.sum() + 0.3 * ent.sum(), w)[0]
        pos = (mask.cumsum(-1) - 1).clamp(min=0)
        logits = causal_lm(input_ids=ids, attention_mask=mask, position_ids=pos).logits[:, 4:-1].reshape(-1, 4096)
        lp2, ent2 = plain(logits, torch.where(mask > 0, ids, -1)[:, 5:].reshape(-1).int())
        want = torch.autograd.grad(lp2.sum() + 0.3 * ent2.sum(), w)[0]
        assert (lp.reshape(-1) - lp2).abs().max() < 1e-4 and (got - want).norm() <= 2.5e-4 * want.norm()
    finally:
        causal_lm.lm_head.weight.requires_grad_(False)


def test_sequence_logprobs_without_gradients(scoring, causal_lm):
    ids, mask = sequences()
    with torch.no_grad():
        a = scoring.sequence_logprobs(causal_lm, ids, mask, prompt_len=5, chunk=7)
        b = scoring.sequence_logprobs(causal_lm, ids, mask, prompt_len=5)
    assert all((x - y).abs().max() < 1e-4 and not x.requires_grad for x, y in zip(a, b))


@pytest.mark.parametrize("bad", [31, 32, 1 << 30])
def test_tokens_behind_the_vocabulary_are_refused(scoring, bad):
    """The kernel would give such an entry log probability 0 and no gradient."""
    logits, tok, _ = case()
    tok[3] = bad
    with pytest.raises(ValueError):
        scoring.token_logprobs(logits, tok)
    tok[3] = 30
    scoring.token_logprobs(logits, tok)


@pytest.mark.parametrize("at,bad", [((0, 9), 4096), ((0, 1), 5000), ((1, 2), 4096), ((2, 19), -1)],
                         ids=["scored", "prompt", "masked", "negative"])
def test_sequences_with_bad_ids_are_refused_before_the_model_runs(scoring, causal_lm, monkeypatch, at, bad):
    ids, mask = sequences()
    ids[at] = bad
    monkeypatch.setattr(causal_lm.model, "forward", lambda *a, **k: pytest.fail("the model ran"))
    with pytest.raises(ValueError):
        scoring.sequence_logprobs(causal_lm, ids, mask, prompt_len=5)


def test_scored_ids_that_the_lm_head_lacks_are_refused(scoring, causal_lm, monkeypatch):
    """An embedding with more rows than the lm_head (added pad tokens): such ids may stand in the prompt and in masked
    places, not among the scored tokens."""
    ids, mask = sequences()
    monkeypatch.setattr(causal_lm, "lm_head", torch.nn.Linear(256, 4000, bias=False))
    ids.clamp_(max=3999)
    ids[0, 2], ids[1, 1] = 4095, 4000
    mask[2, 17:] = 0
    ids[2, 18] = 4095
    scoring.sequence_logprobs(causal_lm, ids, mask, prompt_len=5)
    ids[0, 7] = 4000
    with pytest.raises(ValueError):
        scoring.sequence_logprobs(causal_lm, ids, mask, prompt_len=5)


def test_alternatives_without_log_probabilities_are_refused():
    from flashgrpo_b200.decoding.flash_medusa_decoder import FlashMedusaConfig, FlashMedusaDecoder

    with pytest.raises(ValueError):
        FlashMedusaDecoder(None, None, None, FlashMedusaConfig(logprob_alternatives=3))
    FlashMedusaDecoder(None, None, None, FlashMedusaConfig(logprob_alternatives=3, return_logprobs=True))
