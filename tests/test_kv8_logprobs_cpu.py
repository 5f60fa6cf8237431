"""Refusals of the 8-bit cache's and the log probabilities' entry points: all
come before any CUDA call, so they are checked without a GPU."""
from __future__ import annotations

import ctypes

import pytest

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 8)


@pytest.fixture(scope="module")
def N():
    from flashgrpo_b200 import _native

    _native.load()
    return _native


def cache(N, **kw):
    f = dict(k8=1 << 20, v8=1 << 20, k_scale=1 << 20, v_scale=1 << 20, k_tail=1 << 20, v_tail=1 << 20,
             dtype=N.FG_DTYPE_BF16, n_layers=2, batch=4, n_kv_heads=2, head_dim=128, capacity=64, tail_capacity=48,
             rows=None)
    f.update(kw)
    return ctypes.byref(N.Kv8Cache(*f.values()))


BAD_CACHES = [
    (dict(k8=None), "FG_EINVAL"), (dict(v_scale=None), "FG_EINVAL"), (dict(k_tail=None), "FG_EINVAL"),
    (dict(n_layers=0), "FG_EINVAL"), (dict(batch=0), "FG_EINVAL"), (dict(n_kv_heads=0), "FG_EINVAL"),
    (dict(capacity=0), "FG_EINVAL"), (dict(capacity=48), "FG_EUNSUPPORTED"), (dict(tail_capacity=31), "FG_EINVAL"),
    (dict(head_dim=0), "FG_EUNSUPPORTED"), (dict(head_dim=144), "FG_EUNSUPPORTED"),
    (dict(head_dim=72), "FG_EUNSUPPORTED"), (dict(dtype=2), "FG_EUNSUPPORTED"), (dict(dtype=7), "FG_EUNSUPPORTED"),
    (dict(k8=(1 << 20) + 8), "FG_EINVAL"), (dict(v_tail=(1 << 20) + 4), "FG_EINVAL"), (dict(batch=3), "FG_EINVAL"),
]


@pytest.mark.parametrize("bad,status", BAD_CACHES)
def test_bad_caches(N, bad, status):
    lib, c, want = N.load(), cache(N, **bad), getattr(N, status)
    assert lib.fg_kv8_load(c, 0, P, P, 1, 1, 1, 33, P, 4, 1, P, ODD, None) == want
    assert lib.fg_kv8_commit(c, P, 4, P, 4, P, ODD, None, None, None) == want
    assert lib.fg_tree_attention_kv8(P, c, 0, P, P, P, 4, 8, 4, 1.0, P, None, 0, 1, 64, None) == want


def test_load_refusals(N):
    lib = N.load()
    call = lambda c=cache(N), layer=0, k=P, src=33, lens=P, n=4, rep=1, q=P, t=ODD: lib.fg_kv8_load(  # noqa: E731
        c, layer, k, P, 128, 128, 128, src, lens, n, rep, q, t, None)
    assert call(n=0) == N.FG_OK
    for kw in (dict(layer=-1), dict(layer=2), dict(k=None), dict(src=-1), dict(lens=None), dict(n=-1), dict(rep=0),
               dict(q=None), dict(t=None), dict(t=P), dict(n=5), dict(n=2, rep=3), dict(c=None)):
        assert call(**kw) == N.FG_EINVAL, kw
    assert call(src=96) == N.FG_ECAPACITY


def test_commit_refusals(N):
    lib = N.load()
    call = lambda c=cache(N), nodes=P, dcap=4, acc=P, B=4, q=P, t=ODD, qo=None, to=None: lib.fg_kv8_commit(  # noqa: E731
        c, nodes, dcap, acc, B, q, t, qo, to, None)
    other = ctypes.c_void_p(1 << 21)
    assert call(B=0) == N.FG_OK
    for kw in (dict(nodes=None), dict(acc=None), dict(q=None), dict(t=None), dict(dcap=0), dict(B=-1), dict(B=5),
               dict(qo=other), dict(to=other), dict(qo=other, to=other), dict(qo=P, to=other), dict(qo=other, to=ODD),
               dict(qo=ODD, to=P), dict(t=P)):
        assert call(**kw) == N.FG_EINVAL, kw
    assert call(dcap=17) == N.FG_ECAPACITY


def test_attention_refusals(N):
    lib = N.load()

    def call(c=cache(N), q=P, layer=0, ql=P, tl=P, anc=P, B=4, nodes=8, hq=4, scale=1.0, out=P, ws=None, nbytes=0,
             splits=1, most=64):
        return lib.fg_tree_attention_kv8(q, c, layer, ql, tl, anc, B, nodes, hq, scale, out, ws, nbytes, splits, most,
                                         None)

    assert call(B=0) == N.FG_OK
    for kw in (dict(q=None), dict(ql=None), dict(tl=None), dict(anc=None), dict(out=None), dict(layer=2),
               dict(layer=-1), dict(nodes=0), dict(hq=3), dict(hq=0), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(most=-1), dict(splits=65), dict(q=ODD),
               dict(out=ODD), dict(B=-1), dict(B=5)):
        assert call(**kw) == N.FG_EINVAL, kw
    for kw in (dict(nodes=129), dict(nodes=49), dict(splits=2), dict(splits=2, ws=P, nbytes=64),
               dict(splits=2, ws=ODD, nbytes=1 << 30)):
        assert call(**kw) == N.FG_ECAPACITY, kw
    size = lambda *a: lib.fg_tree_attention_kv8_workspace_size(*a)  # noqa: E731
    assert size(64, 13, 12, 2, 128, 1, 1024) == 0 and size(64, 13, 12, 2, 128, 2, 1024) > 0
    for bad in ((0, 13, 12, 2, 128, 2, 9), (1, 0, 12, 2, 128, 2, 9), (1, 1, 12, 5, 128, 2, 9), (1, 1, 12, 0, 128, 2, 9),
                (1, 1, 12, 2, 128, 65, 9), (1, 1, 12, 2, 128, 2, -1)):
        assert size(*bad) == 0


def test_logprobs_refusals(N):
    lib = N.load()
    call = lambda x=P, dt=1, ld=100, V=100, rows_n=8, rows=None, tok=P, n=8, T=1.0, logp=P, k=0, ti=P, tl=P: (  # noqa: E731
        lib.fg_token_logprobs(x, dt, ld, V, rows_n, rows, tok, n, T, logp, P, P, k, ti, tl, None))
    assert call(n=0) == N.FG_OK
    for kw in (dict(x=None), dict(dt=3), dict(dt=-1), dict(ld=99), dict(V=0), dict(rows_n=7), dict(rows_n=0),
               dict(rows_n=0, rows=P), dict(tok=None), dict(n=-1), dict(T=0.0), dict(T=-1.0), dict(T=float("nan")),
               dict(T=float("inf")), dict(logp=None), dict(k=-1), dict(k=2, ti=None), dict(k=2, tl=None)):
        assert call(**kw) == N.FG_EINVAL, kw
    for kw in (dict(k=17), dict(k=5, V=4)):
        assert call(**kw) == N.FG_ECAPACITY, kw
    far = ctypes.c_void_p(1 << 30)

    def back(x=P, dt=1, ld=100, V=100, tok=P, n=8, T=1.0, lse=P, ent=P, g=P, h=P, out=far, ldo=100):
        return lib.fg_token_logprobs_backward(x, dt, ld, V, tok, n, T, lse, ent, g, h, out, ldo, None)

    assert back(n=0) == N.FG_OK
    near = ctypes.c_void_p((1 << 20) + 256)
    for kw in (dict(x=None), dict(dt=3), dict(ld=99), dict(ldo=99), dict(V=0), dict(tok=None), dict(n=-1),
               dict(T=0.0), dict(T=float("nan")), dict(lse=None), dict(g=None), dict(ent=None), dict(out=None),
               dict(out=near), dict(out=P, ldo=101)):
        assert back(**kw) == N.FG_EINVAL, kw


def test_decoder_options():
    from flashgrpo_b200.decoding.flash_medusa_decoder import FlashMedusaConfig, FlashMedusaDecoder

    FlashMedusaDecoder(None, None, None, FlashMedusaConfig(kv_cache_dtype="fp8", return_logprobs=True,
                                                           logprob_alternatives=16))
    for bad in (dict(kv_cache_dtype="int8"), dict(logprob_alternatives=17), dict(logprob_alternatives=-1)):
        with pytest.raises(ValueError):
            FlashMedusaDecoder(None, None, None, FlashMedusaConfig(**bad))


# ------------------------------------------------------ tensors of two devices
@pytest.fixture
def fake(monkeypatch):
    """The wrappers over tensors without memory (so of any device); the calls that pass their checks are listed."""
    from flashgrpo_b200 import ops
    from torch._subclasses.fake_tensor import FakeTensorMode

    called = []
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else 1 << 20)
    monkeypatch.setattr(ops, "_stream", lambda t: None)
    monkeypatch.setattr(ops, "_call", lambda t, name, *a, **k: called.append(name))
    with FakeTensorMode():
        yield ops, called


def two_devices(call, args, called, name):
    """call(**args) on one device runs; with any one tensor on another it is refused before the launch."""
    import torch

    call(**args)
    assert called == [name]
    for key, t in args.items():
        if isinstance(t, torch.Tensor):
            with pytest.raises(ValueError):
                call(**{**args, key: torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda:1")})
    assert called == [name]


def test_cache_calls_with_tensors_of_two_devices(fake):
    import torch

    ops, called = fake
    on = dict(device="cuda:0")
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, **on)  # noqa: E731
    cache = ops.Kv8Cache.empty(1, 2, 2, 64, 128, max_nodes=8, dtype=torch.bfloat16, **on)
    kv = dict(dtype=torch.bfloat16, **on)
    two_devices(lambda **a: ops.kv8_load(cache, 0, **a),
                dict(k=torch.empty(2, 2, 40, 128, **kv), v=torch.empty(2, 2, 40, 128, **kv), lengths=i32(2),
                     q_len=i32(2), tail_len=i32(2)), called, "fg_kv8_load")
    called.clear()
    two_devices(lambda **a: ops.kv8_commit(cache, **a),
                dict(acc_nodes=i32(2, 4), acc_len=i32(2), q_len=i32(2), tail_len=i32(2), q_len_out=i32(2),
                     tail_len_out=i32(2)), called, "fg_kv8_commit")
    called.clear()
    q = torch.empty(2, 8, 4, 128, **kv)
    two_devices(lambda **a: ops.tree_attention_kv8(cache=cache, layer=0, scale=1.0, **a),
                dict(q=q, q_len=i32(2), tail_len=i32(2), anc=i32(8, 4), out=torch.empty_like(q), workspace=i32(64)),
                called, "fg_tree_attention_kv8")


def test_logprob_calls_with_tensors_of_two_devices(fake):
    import torch

    ops, called = fake
    on = dict(device="cuda:0")
    f = lambda *s: torch.empty(s, **on)  # noqa: E731
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, **on)  # noqa: E731
    names = ops.TokenLogprobs._fields
    two_devices(lambda logits, tokens, rows, **o: ops.token_logprobs(logits, tokens, rows=rows, k=2,
                                                                     out=ops.TokenLogprobs(**o)),
                dict(logits=f(4, 50), tokens=i32(4), rows=i32(4),
                     **dict(zip(names, (f(4), f(4), f(4), i32(4, 2), f(4, 2))))), called, "fg_token_logprobs")
    called.clear()
    two_devices(ops.token_logprobs_backward,
                dict(logits=f(4, 50), tokens=i32(4), lse=f(4), entropy=f(4), grad_logp=f(4), grad_entropy=f(4),
                     out=f(4, 50)), called, "fg_token_logprobs_backward")


# ------------------------------------------------ lengths that share memory
@pytest.mark.parametrize("lens,q,t,rows", [(0, 0, 64, None), (0, 64, 0, None), (0, 64, 12, None), (0, -12, 64, None),
                                           (0, 64, 72, None), (0, 64, 128, 64), (0, 64, 128, 140)])
def test_load_lengths_that_share_memory(N, lens, q, t, rows):
    """A CTA writes a row's lengths while others still read the source's."""
    lib, at = N.load(), lambda off: None if off is None else ctypes.c_void_p((1 << 22) + off)  # noqa: E731
    c = cache(N, rows=None if rows is None else (1 << 22) + rows)
    assert lib.fg_kv8_load(c, 0, P, P, 128, 128, 128, 33, at(lens), 4, 1, at(q), at(t), None) == N.FG_EINVAL


@pytest.mark.parametrize("nodes,acc,q,t,qo,to,rows", [
    (0, 64, 64, 128, None, None, None), (0, 64, 128, 64, None, None, None), (0, 128, 60, 192, None, None, None),
    (0, 128, 192, 200, None, None, None), (0, 128, 192, 256, None, None, 192), (0, 128, 192, 256, None, None, 250),
    (0, 128, 192, 256, 128, 320, None), (0, 128, 192, 256, 320, 48, None), (0, 128, 192, 256, 320, 332, None),
    (0, 128, 192, 256, 196, 320, None), (0, 128, 192, 256, 320, 384, 384)])
def test_commit_lengths_that_share_memory(N, nodes, acc, q, t, qo, to, rows):
    lib, at = N.load(), lambda off: None if off is None else ctypes.c_void_p((1 << 22) + off)  # noqa: E731
    c = cache(N, rows=None if rows is None else (1 << 22) + rows)
    assert lib.fg_kv8_commit(c, at(nodes), 4, at(acc), 4, at(q), at(t), at(qo), at(to), None) == N.FG_EINVAL


@pytest.mark.parametrize("T", [1e-45, 1e-40, 4.2e-39])
def test_temperatures_without_a_finite_reciprocal(N, T):
    """log2 e / T is infinite in fp32: every row's maximum would become NaN."""
    lib, far = N.load(), ctypes.c_void_p(1 << 30)
    assert lib.fg_token_logprobs(P, 1, 100, 100, 8, None, P, 8, T, P, P, P, 0, P, P, None) == N.FG_EINVAL
    assert lib.fg_token_logprobs_backward(P, 1, 100, 100, P, 8, T, P, P, P, P, far, 100, None) == N.FG_EINVAL
