"""generate() in the calls that follow one another on a decoder: several
lengths, with both caches."""
from __future__ import annotations

import pytest
import torch

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


class _Tok:
    pad_token_id = 0
    eos_token_id = 1


@pytest.fixture(scope="module")
def bf16_model():
    """Two layers of the 1.5B shape: head_dim 128, the tensor-core kernels."""
    from flashgrpo_b200.utils import synthetic

    return synthetic.build_model(2, layers=2, vocab=4096).cuda()


def bf16_heads(n=3):
    g = torch.Generator().manual_seed(0)
    heads = {}
    for i in range(n):
        heads[f"heads.{i}.norm.weight"] = torch.ones(1536).bfloat16().cuda()
        heads[f"heads.{i}.norm.bias"] = torch.zeros(1536).bfloat16().cuda()
        heads[f"heads.{i}.fc.weight"] = (torch.randn(1536, 1536, generator=g) * 0.02).bfloat16().cuda()
        heads[f"heads.{i}.fc.bias"] = torch.zeros(1536).bfloat16().cuda()
    return heads


def bf16_decoder(model, **kw):
    from flashgrpo_b200.decoding.flash_medusa_decoder import FlashMedusaConfig, FlashMedusaDecoder

    cfg = dict(tree_mode="fixed", max_tree_nodes_per_seq=13, max_tree_depth=4, fixed_tree_topk_by_depth=(4, 2),
               top_p=1.0, sampling_seed=7, autotune_dense=False)
    return FlashMedusaDecoder(model, bf16_heads(), _Tok(), FlashMedusaConfig(**{**cfg, **kw}))


@pytest.mark.parametrize("cache", ["model", "fp8"])
def test_one_decoder_with_two_capacities(bf16_model, cache):
    """Short, long, short: the long call's split plan needs a larger workspace of another layout on the same round
    buffers, and the captured rounds of the short one are replayed behind it.  Every call gives the tokens of its first
    run and of eager rounds (the same kernels with the same plans: the same bits)."""
    from flashgrpo_b200 import _native, ops
    from flashgrpo_b200.utils import synthetic

    kw = dict(kv_cache_dtype=cache, return_logprobs=True)
    size = ops.kv8_attention_workspace_bytes if cache == "fp8" else ops.attention_workspace_bytes
    most = "max_q_len" if cache == "fp8" else "max_kv_len"
    calls = [(500, 524), (2500, 2524)]
    need = [size(2, 13, 12, 2, 128, num_splits=0, **{most: m + 15}) for _, m in calls]
    assert 0 < need[0] < need[1]
    dec = bf16_decoder(bf16_model, **kw)
    got = []
    for which in (0, 0, 1, 1, 0, 1, 0):
        n, most_len = calls[which]
        ids, mask = synthetic.random_prompts(1, n, 4096, seed=3)
        r = dec.generate(ids, mask, repeated_generate_nums=2, max_length=most_len)
        got.append((which, r["generated_token_ids"], r["generated_logprobs"]))
    for which in (0, 1):
        n, most_len = calls[which]
        ids, mask = synthetic.random_prompts(1, n, 4096, seed=3)
        r = bf16_decoder(bf16_model, use_cuda_graphs=False, **kw).generate(ids, mask, repeated_generate_nums=2,
                                                                           max_length=most_len)
        for w, toks, lps in got:
            if w == which:
                assert toks == r["generated_token_ids"] and lps == r["generated_logprobs"]
    assert _native.read_device_error(clear=True) == 0


def test_sequence_logprobs_memory_goes_by_the_chunk():
    """What a forward leaves on the device, and the peak of the backward behind it: of 4096 positions and a vocabulary
    of 4096 in fp32 (64 MB of logits) the chunks of 256 (4 MB, twice with the gradient) keep no more than one."""
    from flashgrpo_b200.engine.scoring import sequence_logprobs
    from flashgrpo_b200.utils import synthetic

    m = synthetic.build_model(1).cuda()
    m.lm_head.weight.requires_grad_(True)
    ids = torch.randint(0, 4096, (16, 264), generator=torch.Generator().manual_seed(5)).cuda()
    mask = torch.ones_like(ids)
    held, peak, grads = {}, {}, {}
    for chunk in (256, 4096, 256):
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        lp, ent = sequence_logprobs(m, ids, mask, prompt_len=8, chunk=chunk)
        held[chunk] = torch.cuda.memory_allocated() - start
        torch.cuda.reset_peak_memory_stats()
        grads[chunk], = torch.autograd.grad(lp.sum() + 0.1 * ent.sum(), m.lm_head.weight)
        peak[chunk] = torch.cuda.max_memory_allocated() - start
        del lp, ent
    mb = 1 << 20
    assert held[256] + 56 * mb < held[4096], held
    assert peak[256] < held[256] + 32 * mb < peak[4096], (held, peak)
    assert (grads[256] - grads[4096]).norm() <= 2.5e-4 * grads[4096].norm()


@pytest.mark.parametrize("k,sample", [(0, True), (3, True), (2, False)])
def test_a_correction_keeps_the_log_probabilities_of_its_draw(bf16_model, monkeypatch, k, sample):
    """A round's correction is the next round's root.  What is reported for it is what its parent's tree logits say in
    the round that drew it, bit for bit, whatever the next proposal's own GEMM and rounding make of the same hidden
    state; rows that finish earlier leave the batch in between."""
    from flashgrpo_b200 import _native, ops
    from flashgrpo_b200.engine.verify import VerifyEngine
    from flashgrpo_b200.utils import synthetic

    dec = bf16_decoder(bf16_model, return_logprobs=True, logprob_alternatives=k, use_cuda_graphs=False,
                       do_sample=sample, temperature=0.8 if sample else 1.0)
    T = 0.8 if sample else 1.0
    want, seen, sizes = {}, [0], set()
    inner = VerifyEngine.accept

    def accept(self, st, rb, cfg, phase_event=None):
        inner(self, st, rb, cfg, phase_event=phase_event)
        names = ["logp", "entropy"] + (["top_idx", "top_logp"] if k else [])
        here = st.rows.tolist() if hasattr(st, "rows") else list(range(st.B))
        sizes.add(st.B)
        for i, row in enumerate(here):
            if row in want:
                seen[0] += 1
                tok, vals = want.pop(row)
                assert int(rb.out["acc_tokens"][i, 0]) == tok
                for name in names:
                    assert torch.equal(rb.logprobs[k][name][i, 0], vals[name]), (row, name)
            if int(st.pending[i]) >= 0:
                at = rb.tree["slot"][i, int(rb.out["last_node"][i])].view(1)
                r = ops.token_logprobs(rb.tree_logits, st.pending[i:i + 1].contiguous(), rows=at.contiguous(),
                                       temperature=T, k=k)
                want[row] = int(st.pending[i]), {n: getattr(r, n)[0].clone() for n in names}

    monkeypatch.setattr(VerifyEngine, "accept", accept)
    ids, mask = synthetic.random_prompts(3, 40, 4096, seed=8)
    mask[0, :9], mask[2, :30] = 0, 0
    res = dec.generate(ids, mask, repeated_generate_nums=2, max_length=60)
    monkeypatch.undo()
    assert seen[0] > 40 and len(sizes) > 1
    # captured rounds, twice on one decoder: the same values
    dec = bf16_decoder(bf16_model, return_logprobs=True, logprob_alternatives=k, do_sample=sample,
                       temperature=0.8 if sample else 1.0)
    for _ in range(2):
        again = dec.generate(ids, mask, repeated_generate_nums=2, max_length=60)
        for key in ("generated_token_ids", "generated_logprobs", "generated_entropies"):
            assert again[key] == res[key]
        assert again.get("generated_alternatives") == res.get("generated_alternatives")
    assert _native.read_device_error(clear=True) == 0


def test_one_decoder_with_two_batches(bf16_model):
    """One row, many rows, one row: the proposal's workspace grows in between, and the captured rounds of the small
    batch are replayed behind it."""
    from flashgrpo_b200 import _native
    from flashgrpo_b200.utils import synthetic

    dec = bf16_decoder(bf16_model, return_logprobs=True)
    ids, mask = synthetic.random_prompts(1, 20, 4096, seed=3)
    got = {1: [], 48: []}
    for n in (1, 1, 48, 48, 1, 48, 1):
        r = dec.generate(ids, mask, repeated_generate_nums=n, max_length=44)
        got[n].append((r["generated_token_ids"], r["generated_logprobs"]))
    assert all(x == got[1][0] for x in got[1]) and all(x == got[48][0] for x in got[48])
    assert _native.read_device_error(clear=True) == 0
