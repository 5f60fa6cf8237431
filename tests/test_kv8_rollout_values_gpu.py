"""Rollouts over an 8-bit cache with blocks in use, against an HF forward (fp32
on the CPU) whose attention reads the K/V of finished blocks as the plain form
stores them: wrong layers, rows, blocks or lengths in the engine's load, commit
or attention show in the log probabilities."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

BLK = 32


class _Tok:
    pad_token_id = 0
    eos_token_id = 1


# ------------------------------------------------------------ plain form (CPU)
def stored(x):
    """[H, n * 32, D] -> the values that e4m3 blocks with power-of-two scales hold."""
    b = x.double().unflatten(1, (-1, BLK))
    e = torch.ceil(torch.log2(b.abs().amax((2, 3), keepdim=True) / 448.0)).clamp(min=-126)
    m, ex = torch.frexp(b * torch.exp2(-e))
    step = torch.exp2((ex - 1).clamp(min=-6).double() - 3)
    return (torch.round(b * torch.exp2(-e) / step) * step * torch.exp2(e)).flatten(1, 2).to(x.dtype)


class Oracle:
    """The model's logits for one sequence; position p's query was fed in a round that began with starts[p] tokens
    in the cache (0: the prefill) and reads whole blocks of those as stored."""

    def __init__(self, model, cache_dtype):
        from transformers import AttentionInterface

        AttentionInterface.register("kv8_plain", self.attention)
        model.config._attn_implementation = "kv8_plain"
        self.model, self.cache_dtype = model, cache_dtype

    def attention(self, module, query, key, value, attention_mask, scaling=None, **kw):
        S, layer = query.shape[2], module.layer_idx
        n = S // BLK * BLK
        k, v = (x[0].to(self.cache_dtype).to(x.dtype) for x in (key, value))
        k8, v8 = k.clone(), v.clone()
        k8[:, :n], v8[:, :n] = stored(k[:, :n]), stored(v[:, :n])
        self.kept[layer] = k8, v8
        at = torch.arange(S)
        in8 = at[None, :] < (self.starts // BLK * BLK)[:, None]
        hidden = at[None, :] > at[:, None]
        # planted mistakes
        if self.plant == "not quantised":
            k8, v8 = k, v
        elif self.plant == "length a block short":
            hidden = hidden | in8 & (at[None, :] >= (self.starts // BLK * BLK - BLK)[:, None])
        elif self.plant == "another row":
            m = min(n, self.other[layer][0].shape[1])
            k8[:, :m], v8[:, :m] = (x[:, :m] for x in self.other[layer])
        elif self.plant == "another layer" and layer == 1:
            v8[:, :n] = self.kept[0][1][:, :n]
        elif self.plant == "blocks exchanged":
            v8 = torch.cat([v8[:, BLK:2 * BLK], v8[:, :BLK], v8[:, 2 * BLK:]], 1)
        G = query.shape[1] // k.shape[0]
        k, v, k8, v8 = (x.repeat_interleave(G, 0) for x in (k, v, k8, v8))
        s = torch.where(in8, query[0] @ k8.transpose(1, 2), query[0] @ k.transpose(1, 2)) * scaling
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        return ((p * in8) @ v8 + (p * ~in8) @ v).transpose(0, 1)[None], None

    def __call__(self, ids, starts, prompt, plant=None, other=None):
        self.starts, self.plant, self.other, self.kept = starts, plant, other, {}
        with torch.no_grad():
            logits = self.model(input_ids=ids[None]).logits[0, prompt - 1:-1]
        return torch.log_softmax(logits, -1).gather(1, ids[prompt:, None])[:, 0], logits


PLANTS = ("length a block short", "another row", "another layer", "blocks exchanged")


def rollout(dec, monkeypatch, ids, mask, **kw):
    """generate() in eager rounds, and every round's row lengths at its start: [(state rows, lengths)]."""
    from flashgrpo_b200.engine.verify import VerifyEngine

    rounds, inner = [], VerifyEngine.run_round

    def run_round(self, st, rb, *a, **k):
        rows = st.rows.tolist() if hasattr(st, "rows") else list(range(st.B))
        lens = (st.base if hasattr(st, "rows") else st).row_len.tolist()
        rounds.append({r: lens[r] for r in rows})
        return inner(self, st, rb, *a, **k)

    with monkeypatch.context() as m:
        m.setattr(VerifyEngine, "run_round", run_round)
        return dec.generate(ids, mask, **kw), rounds


def check(dec, captured, oracle, monkeypatch, lengths, most, repeats, tolerance):
    """tolerance(logits, effect of the quantisation) -> bounds of the largest and of the rms difference."""
    from flashgrpo_b200 import _native
    from flashgrpo_b200.utils import synthetic

    ids, mask = synthetic.random_prompts(len(lengths), max(lengths), 4096, seed=5)
    mask = mask.clone()
    for r, n in enumerate(lengths):
        mask[r, :max(lengths) - n] = 0
    kw = dict(repeated_generate_nums=repeats, max_length=most)
    res, rounds = rollout(dec, monkeypatch, ids, mask, **kw)
    again = captured.generate(ids, mask, **kw)
    assert again["generated_token_ids"] == res["generated_token_ids"]
    assert again["generated_logprobs"] == res["generated_logprobs"]
    found, kept = {p: 0 for p in PLANTS}, []
    for row, toks in enumerate(res["generated_token_ids"]):
        n = lengths[row // repeats]
        seq = torch.cat([ids[row // repeats, max(lengths) - n:], torch.tensor(toks)])
        begins = sorted({r[row] for r in rounds if row in r})
        assert begins[0] == n
        starts = torch.zeros(seq.numel(), dtype=torch.long)
        for b in begins:
            starts[b:] = b
        got = torch.tensor(res["generated_logprobs"][row])
        want, logits = oracle(seq, starts, n)
        mine = dict(oracle.kept)
        plain = oracle(seq, starts, n, "not quantised")[0]
        biggest, rms = tolerance(logits, plain - want)
        size = lambda d: (float(d.abs().max()), float(d.pow(2).mean().sqrt()))  # noqa: E731
        far = size(got - want)
        assert far[0] <= biggest and far[1] <= rms, (row, far, biggest, rms)
        # the oracle's own planted mistakes are outside those bounds (where the row is long enough to have them)
        for plant in PLANTS:
            if plant == "another row" and not kept:
                continue
            off = size(oracle(seq, starts, n, plant, kept[0] if kept else None)[0] - got)
            found[plant] += off[0] > biggest or off[1] > rms
        if row % repeats == 0 and not kept:
            kept.append(mine)
    rows = len(res["generated_token_ids"])
    assert all(v >= rows - repeats for v in found.values()), found
    assert _native.read_device_error(clear=True) == 0


def test_fp32_rollout_over_blocks(monkeypatch):
    """head_dim 64 in fp32.  Both sides compute the same logits in other orders: 688 * 2^-24 * 8 * 10 = 3e-3 (sums of up
    to 688 terms, an lm_head scaled by 8, logits of size 10).  A K or V value that a last-bit difference puts on the
    other side of a code's border moves by a step; all of them together (2 layers, 2 heads, 130 tokens, 64 dims, K and
    V: 2^16.0 values) move a log probability by less than 0.1, one by 0.1 / 2^8 = 4e-4: five of those are allowed."""
    from flashgrpo_b200.decoding.flash_medusa_decoder import FlashMedusaConfig, FlashMedusaDecoder
    from flashgrpo_b200.utils import synthetic

    heads = {k: v.cuda() for k, v in synthetic.medusa_head_tensors(1).items()}
    cfg = dict(tree_mode="fixed", max_tree_nodes_per_seq=16, max_tree_depth=4, fixed_tree_topk_by_depth=(4, 2, 2),
               top_p=1.0, sampling_seed=11, kv_cache_dtype="fp8", return_logprobs=True)
    gpu = synthetic.build_model(1).cuda()
    make = lambda graphs: FlashMedusaDecoder(gpu, heads, _Tok(), FlashMedusaConfig(  # noqa: E731
        use_cuda_graphs=graphs, **cfg))

    def tolerance(logits, effect):
        assert effect.abs().max() > 5e-3 * 2  # reading the cache unquantised would show, too
        return 5e-3, 5e-3

    check(make(False), make(True), Oracle(synthetic.build_model(1), torch.float32), monkeypatch, (70, 40, 96), 140, 2,
          tolerance)


@pytest.mark.parametrize("tree", [True, False])
def test_bf16_rollout_over_blocks(monkeypatch, tree):
    """Two layers of the 1.5B shape (head_dim 128, the tensor-core kernel), with trees and with one token a round.
    Roundings to bf16 between a token and its logits: per layer norm, QKV, RoPE, attention, O + residual, norm, gate,
    product, down + residual, then norm and logits, 20 of at most 2^-8 each.  The largest difference is bounded by their
    sum on the largest logit, the rms by independent ones on the logits' rms.  Codes that the roundings put on the other
    side of a border are further errors of e4m3's own kind: at most the quantisation's effect once more."""
    from flashgrpo_b200.decoding.flash_medusa_decoder import FlashMedusaConfig, FlashMedusaDecoder
    from flashgrpo_b200.utils import synthetic

    heads = {}
    g = torch.Generator().manual_seed(0)
    for i in range(3):
        heads[f"heads.{i}.norm.weight"] = torch.ones(1536).bfloat16().cuda()
        heads[f"heads.{i}.norm.bias"] = torch.zeros(1536).bfloat16().cuda()
        heads[f"heads.{i}.fc.weight"] = (torch.randn(1536, 1536, generator=g) * 0.02).bfloat16().cuda()
        heads[f"heads.{i}.fc.bias"] = torch.zeros(1536).bfloat16().cuda()
    cfg = dict(tree_mode="fixed", max_tree_nodes_per_seq=13, max_tree_depth=4, fixed_tree_topk_by_depth=(4, 2),
               top_p=1.0, sampling_seed=5, kv_cache_dtype="fp8", return_logprobs=True, autotune_dense=False,
               enable_medusa_spec_after=0 if tree else 1 << 30)
    gpu = synthetic.build_model(2, layers=2, vocab=4096).cuda()
    make = lambda graphs: FlashMedusaDecoder(gpu, heads, _Tok(), FlashMedusaConfig(  # noqa: E731
        use_cuda_graphs=graphs, **cfg))

    def tolerance(logits, effect):
        return (20 * 2.0 ** -8 * float(logits.abs().max()) + float(effect.abs().max()),
                20 ** 0.5 * 2.0 ** -8 * float(logits.pow(2).mean().sqrt()) + float(effect.pow(2).mean().sqrt()))

    oracle = Oracle(synthetic.build_model(2, layers=2, vocab=4096).float(), torch.bfloat16)
    check(make(False), make(True), oracle, monkeypatch, (90, 64, 131), 175, 1, tolerance)
