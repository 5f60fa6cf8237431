"""Workspaces of the engine's rounds: captured rounds hold their addresses, so
a round of another size or capacity must not replace them (no GPU, no kernels)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch


def engine(kv8: bool):
    from flashgrpo_b200.engine.verify import ModelSpec, VerifyEngine

    e = object.__new__(VerifyEngine)
    e.spec = ModelSpec(n_layers=2, hidden=1536, n_q_heads=12, n_kv_heads=2, head_dim=128, inter=8960, vocab=4096,
                       eps=1e-6, dtype=torch.bfloat16)
    e.device, e.kv8, e._graphs = torch.device("cpu"), kv8, {}
    return e


@pytest.mark.parametrize("kv8", [False, True])
def test_attention_workspaces_of_two_capacities(kv8):
    """Small, large, small capacity on one set of round buffers: the first workspace stays, and each is zero-filled
    and large enough for its own plan."""
    from flashgrpo_b200 import ops

    e = engine(kv8)
    rb = SimpleNamespace(N=13, attn_ws={})
    size = ops.kv8_attention_workspace_bytes if kv8 else ops.attention_workspace_bytes
    small, large = (SimpleNamespace(B=4, capacity=c) for c in (1056, 4128))
    need = [size(4, 13, 12, 2, 128, num_splits=0, **{"max_q_len" if kv8 else "max_kv_len": st.capacity})
            for st in (small, large)]
    assert 0 < need[0] < need[1]
    a = e._attn_workspace(rb, small, 0)
    at = a.data_ptr()
    assert a.numel() * 4 >= need[0] and not a.any()
    a.fill_(7)  # what a plan leaves in its partials must not be another plan's counters
    b = e._attn_workspace(rb, large, 0)
    assert b.numel() * 4 >= need[1] and not b.any() and b.data_ptr() != at
    again = e._attn_workspace(rb, small, 0)
    assert again.data_ptr() == at and (again == 7).all()
    c = e._attn_workspace(rb, small, 3)
    assert c.data_ptr() not in (at, b.data_ptr()) and not c.any()
    assert e._attn_workspace(rb, large, 1) is None


@pytest.mark.parametrize("call", [lambda e, big: e._lm_head_ws(200 if big else 8, 0, 4),
                                  lambda e, big: e._propose_ws(64 if big else 2, 3, 4),
                                  lambda e, big: e._chain_ws(200 if big else 8, 4)],
                         ids=["lm_head", "propose", "chain"])
def test_a_replaced_workspace_stays(call):
    """A larger batch takes a new workspace; the one that captured rounds of the smaller batch hold is not freed (a
    weak reference to it lives) and serves no other tensor."""
    import weakref

    e = engine(False)
    e.heads = SimpleNamespace(chain={"state_proj.weight": torch.empty(256, 1536)})
    small = call(e, False)
    at, ref = small.data_ptr(), weakref.ref(small)
    del small
    large = call(e, True)
    assert large.data_ptr() != at and large.numel() > ref().numel()
    assert ref() is not None and ref().data_ptr() == at
    assert call(e, True) is large
