"""The 8-bit KV cache (load, commit) and the tree attention over it, against
plain 64-bit implementations.

Load and commit are exact: scales are powers of two and the codes the nearest
e4m3 values, so codes, scales, tails and lengths have to be equal.  The
attention's tolerance counts its roundings: weights and the result to the
model's type (finfo.eps / 2 each), fp32 scores (one rounding per product and
partial sum, 2^-24 each, counted twice for accumulators that truncate) and
fp32 sums over the slots.
"""
from __future__ import annotations

import math

import pytest
import torch

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

DEV = "cuda"
BLK = 32


@pytest.fixture(scope="module")
def ops():
    from flashgrpo_b200 import _native, ops as o

    _native.load()
    _native.read_device_error(clear=True)
    yield o
    assert _native.read_device_error(clear=True) == 0


# ------------------------------------------------------- plain forms (CPU)
def e4m3(x):
    """Nearest e4m3 value of x (float64, |x| <= 448), ties to even."""
    m, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def quantise(block):
    """[32, D] -> (code values, scale), float64."""
    b = block.double()
    if not bool(b.isfinite().all()):
        return torch.full_like(b, math.nan), math.nan
    amax = float(b.abs().max())
    e = -126
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e4m3(b * 2.0 ** -e), 2.0 ** e


class Plain:
    """The cache as float64 tensors on the CPU."""

    def __init__(self, cache):
        self.codes = [cache.k8.double().cpu(), cache.v8.double().cpu()]
        self.scale = [cache.k_scale.double().cpu(), cache.v_scale.double().cpu()]
        self.tail = [cache.k_tail.double().cpu(), cache.v_tail.double().cpu()]

    def put(self, kv, layer, row, q0, tokens):
        """tokens [H, n, D] appended from 8-bit slot q0 on: whole blocks, then the tail; returns the lengths."""
        H, n, D = tokens.shape
        whole, rest = n // BLK, n % BLK
        for h in range(H):
            for i in range(whole):
                c, s = quantise(tokens[h, i * BLK:(i + 1) * BLK])
                self.codes[kv][layer, row, h, q0 + i * BLK:q0 + (i + 1) * BLK] = c
                self.scale[kv][layer, row, h, q0 // BLK + i] = s
            self.tail[kv][layer, row, h, :rest] = tokens[h, whole * BLK:].double()
        return q0 + whole * BLK, rest

    def same(self, cache):
        for kv, (c, s, t) in enumerate(((cache.k8, cache.k_scale, cache.k_tail),
                                        (cache.v8, cache.v_scale, cache.v_tail))):
            for got, want in ((c, self.codes), (s, self.scale), (t, self.tail)):
                got = got.double().cpu()
                assert ((got == want[kv]) | (got.isnan() & want[kv].isnan())).all()


def fill(cache, g, dtype):
    """Any values in every slot, as an earlier use of the buffers leaves them."""
    for t in (cache.k8, cache.v8):
        t.view(torch.uint8).copy_(torch.randint(0, 127, t.shape, generator=g, dtype=torch.uint8))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.exp2(torch.randint(-9, 3, t.shape, generator=g).float()))
    for t in (cache.k_tail, cache.v_tail):
        t.copy_(torch.randn(t.shape, generator=g).to(dtype))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# -------------------------------------------------------------------- load
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,repeats,H,D,cap", [([0], 1, 1, 16, 32), ([1], 2, 2, 128, 64), ([31, 32, 33], 1, 2, 64, 64),
                                                     ([95, 64, 7, 0, 96], 3, 1, 128, 96), ([130, 257], 1, 3, 112, 256)])
def test_load(ops, dtype, lengths, repeats, H, D, cap):
    g = torch.Generator().manual_seed(sum(lengths) + D)
    P, S = len(lengths), max(lengths)
    cache = ops.Kv8Cache.empty(2, P * repeats, H, cap, D, max_nodes=5, dtype=dtype, device=DEV)
    fill(cache, g, dtype)
    plain = Plain(cache)
    k = (torch.randn(P, H, S, D, generator=g) * torch.exp(torch.randn(P, H, S, 1, generator=g) * 3)).to(dtype)
    v = torch.randn(P, H, S, D, generator=g).to(dtype)
    q = torch.full((P * repeats,), 99, dtype=torch.int32, device=DEV)
    t = q.clone()
    ops.kv8_load(cache, 1, k.to(DEV), v.to(DEV), i32(lengths), q, t, repeats=repeats)
    for b in range(P * repeats):
        p = b // repeats
        for kv, x in enumerate((k, v)):
            got = plain.put(kv, 1, b, 0, x[p, :, :lengths[p]])
        assert (int(q[b]), int(t[b])) == got == (lengths[p] // BLK * BLK, lengths[p] % BLK)
    plain.same(cache)


def test_load_values_at_the_borders(ops):
    """Blocks around the scale's borders, ties, the smallest and largest values, zeros, infinities and NaN."""
    D = 16
    cache = ops.Kv8Cache.empty(1, 1, 1, 12 * BLK, D, max_nodes=1, dtype=torch.float32, device=DEV)
    plain = Plain(cache)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(12, BLK, D, generator=g)
    x[0] = 0.0
    x[1] = x[1].clamp(-1, 1)
    x[1, 0, 0] = 448.0                       # scale 1
    x[2, 0, 0] = 448.0 * (1 + 2.0 ** -23)    # just above: scale 2
    x[3] = torch.arange(BLK * D).view(BLK, D).float() * 2.0 ** -10  # ties and subnormal codes
    x[3, 0, 0] = 448.0
    x[4] *= 1e38
    x[5] *= 1e-38
    x[6] = 2.0 ** -149
    x[7, 3, 5] = math.inf
    x[8, 31, 15] = math.nan
    x[9, 0, 1] = -math.inf
    x[10] = 2.0 ** 127
    x[11] = -torch.finfo(torch.float32).max
    k = x.view(1, 1, 12 * BLK, D)
    q, t = i32([0]), i32([0])
    ops.kv8_load(cache, 0, k.to(DEV), k.flip(2).contiguous().to(DEV), i32([12 * BLK]), q, t)
    plain.put(0, 0, 0, 0, k[0])
    plain.put(1, 0, 0, 0, k.flip(2)[0])
    plain.same(cache)


@pytest.mark.parametrize("layout", ["transposed", "offset", "expanded"])
def test_load_strides(ops, layout):
    """[B, S, H, D] storage, rows that start off a 16-byte boundary, one source row for all."""
    g = torch.Generator().manual_seed(5)
    P, H, S, D = 3, 2, 70, 64
    lens = [70, 33, 64]

    def make():
        if layout == "transposed":
            return torch.randn(P, S, H, D, generator=g).bfloat16().to(DEV).transpose(1, 2)
        if layout == "offset":
            return torch.randn(P, H, S, D + 3, generator=g).bfloat16().to(DEV)[..., 1:D + 1]
        return torch.randn(1, H, S, D, generator=g).bfloat16().to(DEV).expand(P, H, S, D)

    k, v = make(), make()
    cache = ops.Kv8Cache.empty(1, 6, H, 96, D, max_nodes=4, dtype=torch.bfloat16, device=DEV)
    rows = i32([4, 0, 5])
    plain, q, t = Plain(cache), i32([0] * 3), i32([0] * 3)
    ops.kv8_load(cache.view(rows), 0, k, v, i32(lens), q, t)
    for p in range(P):
        for kv, x in enumerate((k, v)):
            plain.put(kv, 0, int(rows[p]), 0, x.cpu()[p, :, :lens[p]])
    plain.same(cache)


def test_load_bad_lengths_and_rows(ops):
    from flashgrpo_b200 import _native as N

    cache = ops.Kv8Cache.empty(1, 3, 1, 64, 16, max_nodes=2, dtype=torch.float32, device=DEV)
    plain = Plain(cache)
    k = torch.ones(3, 1, 64, 16, device=DEV)
    q, t = i32([9] * 3), i32([9] * 3)
    ops.kv8_load(cache, 0, k, k, i32([-1, 65, 40]), q, t)
    assert N.read_device_error(clear=True) == N.FG_EINVAL
    assert q.tolist() == [0, 0, 32] and t.tolist() == [0, 0, 8]
    for kv in range(2):
        plain.put(kv, 0, 2, 0, k[2, :, :40].cpu())
    plain.same(cache)
    ops.kv8_load(cache.view(i32([3, -1, 2])), 0, k, k, i32([40, 40, 40]), q, t)
    assert N.read_device_error(clear=True) == N.FG_EINVAL
    assert q.tolist() == [0, 0, 32] and t.tolist() == [0, 0, 8]
    plain.same(cache)


# ------------------------------------------------------------------ commit
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,L,H,D,N,dcap", [(torch.bfloat16, 2, 2, 128, 13, 4), (torch.float32, 1, 3, 64, 16, 16),
                                                (torch.bfloat16, 3, 1, 48, 1, 1), (torch.bfloat16, 1, 2, 128, 128, 8)])
def test_commit(ops, dtype, L, H, D, N, dcap, in_place):
    g = torch.Generator().manual_seed(N * 10 + dcap)
    cap = 96
    rowlens = [0, 1, 31, 30, 32, 63, 64, 95, 17, 5]
    B = len(rowlens)
    cache = ops.Kv8Cache.empty(L, B + 2, H, cap, D, max_nodes=N, dtype=dtype, device=DEV)
    fill(cache, g, dtype)
    plain = Plain(cache)
    rows = torch.randperm(B + 2, generator=g)[:B].to(torch.int32)
    acc = [int(torch.randint(0, min(dcap, N) + 1, (1,), generator=g)) for _ in range(B)]
    acc[2], acc[7] = min(dcap, N), 0
    path = torch.full((B, dcap), -1, dtype=torch.int32)
    for b in range(B):
        path[b, :acc[b]] = torch.randperm(N, generator=g)[:acc[b]].sort().values.to(torch.int32)
    ql, tl = [x // BLK * BLK for x in rowlens], [x % BLK for x in rowlens]
    want = []
    for b in range(B):
        at = list(range(tl[b])) + [tl[b] + int(path[b, j]) for j in range(acc[b])]
        r = int(rows[b])
        for layer in range(L):
            for kv in range(2):
                new = plain.put(kv, layer, r, ql[b], plain.tail[kv][layer, r][:, at].clone())
        want.append(new)
    q, t = i32(ql), i32(tl)
    qo, to = (q, t) if in_place else (i32([7] * B), i32([7] * B))
    ops.kv8_commit(cache.view(rows.to(DEV)), path.to(DEV), i32(acc), q, t, q_len_out=None if in_place else qo,
                   tail_len_out=None if in_place else to)
    assert list(zip(qo.tolist(), to.tolist())) == want
    if not in_place:
        assert q.tolist() == ql and t.tolist() == tl
    plain.same(cache)


def test_commit_of_a_long_tail(ops):
    """A tail of several blocks (a cache whose tail also holds unquantised prompts)."""
    g = torch.Generator().manual_seed(8)
    cache = ops.Kv8Cache.empty(1, 2, 2, 160, 32, max_nodes=120, dtype=torch.bfloat16, device=DEV)
    fill(cache, g, torch.bfloat16)
    plain = Plain(cache)
    tl, acc = [100, 127], [[0, 3, 5], [2]]
    for b in range(2):
        at = list(range(tl[b])) + [tl[b] + n for n in acc[b]]
        for kv in range(2):
            plain.put(kv, 0, b, 32 * b, plain.tail[kv][0, b][:, at].clone())
    q, t = i32([0, 32]), i32(tl)
    ops.kv8_commit(cache, i32([[0, 3, 5], [2, -1, -1]]), i32([3, 1]), q, t)
    assert q.tolist() == [96, 160] and t.tolist() == [7, 0]
    plain.same(cache)


def test_commit_refuses_rows_that_do_not_fit(ops):
    """Each such row stays as it is, its lengths too, and the others are committed."""
    from flashgrpo_b200 import _native as N

    g = torch.Generator().manual_seed(3)
    bad = [dict(q=33), dict(q=-32), dict(q=160), dict(t=-1), dict(t=36), dict(a=-1), dict(a=4), dict(path=[0, 0, 1]),
           dict(path=[-1, 0, 1]), dict(path=[0, 1, 30]), dict(row=9), dict(row=-1)]
    for k, case in enumerate([*bad, dict(q=128, t=31, err=N.FG_ECAPACITY)]):
        cache = ops.Kv8Cache.empty(1, 2, 1, 128, 16, max_nodes=4, dtype=torch.bfloat16, device=DEV)
        fill(cache, g, torch.bfloat16)
        plain = Plain(cache)
        q, t = i32([case.get("q", 32), 0]), i32([case.get("t", 7), 2])
        before = q.tolist(), t.tolist()
        path = i32([case.get("path", [0, 1, 2]), [1, 3, -1]])
        at = [0, 1, 2 + 1, 2 + 3]
        for kv in range(2):
            plain.put(kv, 0, 1, 0, plain.tail[kv][0, 1][:, at].clone())
        ops.kv8_commit(cache.view(i32([case.get("row", 0), 1])), path, i32([case.get("a", 3), 2]), q, t)
        assert N.read_device_error(clear=True) == case.get("err", N.FG_EINVAL), case
        assert (int(q[0]), int(t[0])) == (before[0][0], before[1][0]) and (int(q[1]), int(t[1])) == (0, 4)
        plain.same(cache)


# --------------------------------------------------------------- attention
def tree_bits(n, g, empty=()):
    words, depth = [], []
    for j in range(n):
        above = [i for i in range(j) if depth[i] < 6]
        p = above[int(torch.randint(len(above), (1,), generator=g))] if above else -1
        w = list(words[p]) if p >= 0 else [0, 0, 0, 0]
        w[j >> 5] |= 1 << (j & 31)
        words.append(w)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    for j in empty:
        words[j] = [0, 0, 0, 0]
    return torch.tensor([[x - (1 << 32) if x >> 31 else x for x in w] for w in words], dtype=torch.int32)


def attention_reference(q, cache, layer, rows, q_len, tail_len, anc, scale):
    """(out, tolerance) in float64: every visible slot of every row, and what the roundings can add up to."""
    B, N, hq, D = q.shape
    H = cache.n_kv_heads
    G = hq // H
    half = torch.finfo(q.dtype).eps / 2
    bits = torch.tensor([[(int(w) >> j) & 1 for w in r for j in range(32)][:N] for r in anc.tolist()], device=DEV).bool()
    out = torch.zeros(B, N, hq, D, dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    for b in range(B):
        r, n, t = int(rows[b]), int(q_len[b]), int(tail_len[b])
        part = lambda c, s, x: torch.cat([  # noqa: E731
            c[layer, r, :, :n].double() * s[layer, r, :, :n // BLK].double().repeat_interleave(BLK, -1)[..., None],
            x[layer, r, :, :t + N].double()], 1)
        k, v = part(cache.k8, cache.k_scale, cache.k_tail), part(cache.v8, cache.v_scale, cache.v_tail)
        see = torch.cat([torch.ones(N, n + t, dtype=torch.bool, device=DEV), bits], 1)
        for h in range(H):
            qq = q[b, :, h * G:(h + 1) * G].double()
            s = (torch.einsum("ngd,td->ngt", qq, k[h]) * scale).masked_fill(~see[:, None], -math.inf)
            s_abs = (torch.einsum("ngd,td->ngt", qq.abs(), k[h].abs()) * scale).masked_fill(~see[:, None], 0.0)
            any_ = see.any(1)[:, None, None]
            p = torch.where(any_, torch.softmax(s, -1), torch.zeros_like(s))
            o = torch.einsum("ngt,td->ngd", p, v[h])
            size = torch.einsum("ngt,td->ngd", p, v[h].abs())
            # a score's error moves its weight by e^(2 ds) at most; the sums keep T roundings and ex2's
            ds = 2 * (D + 4) * 2.0 ** -24 * s_abs.amax(-1, keepdim=True)
            rel = 2 * ds + (k.shape[1] + 64) * 2.0 ** -23 + (half if q.dtype == torch.bfloat16 else 0.0)
            out[b, :, h * G:(h + 1) * G] = o
            tol[b, :, h * G:(h + 1) * G] = rel * size + half * o.abs() + 1e-30
    return out, tol


def attention_case(ops, dtype, B, N, hq, H, D, lens, seed, *, layers=1, extra_rows=0, empty=(), scale=None, k_size=1.0):
    g = torch.Generator().manual_seed(seed)
    cap = max(max(lens) // BLK * BLK, BLK)
    cache = ops.Kv8Cache.empty(layers, B + extra_rows, H, cap, D, max_nodes=N, dtype=dtype, device=DEV)
    shape = (layers * (B + extra_rows) * H * cap // BLK, BLK, D)
    for codes, sc in ((cache.k8, cache.k_scale), (cache.v8, cache.v_scale)):
        x = torch.randn(shape, generator=g) * torch.exp(0.7 * torch.randn(shape[0], 1, 1, generator=g)) * (
            k_size if codes is cache.k8 else 1.0)
        amax = x.abs().amax((1, 2))
        e = torch.ceil(torch.log2(amax / 448.0))
        sc.copy_(torch.exp2(e).view(sc.shape))
        codes.copy_((x * torch.exp2(-e)[:, None, None]).to(torch.float8_e4m3fn).view(codes.shape))
    # what lies behind the lengths is never read: make it visible if it is
    for b in range(B + extra_rows):
        n = lens[b % B] // BLK
        cache.k_scale[:, b, :, n:] = math.nan
        cache.v_scale[:, b, :, n:] = math.nan
    cache.k_tail.copy_(torch.randn(cache.k_tail.shape, generator=g) * k_size)
    cache.v_tail.copy_(torch.randn(cache.v_tail.shape, generator=g))
    for b in range(B):
        cache.k_tail[:, b, :, lens[b] % BLK + N:] = math.nan
        cache.v_tail[:, b, :, lens[b] % BLK + N:] = math.inf
    q = torch.randn(B, N, hq, D, generator=g).to(dtype).to(DEV)
    return cache, q, i32([n // BLK * BLK for n in lens]), i32([n % BLK for n in lens]), tree_bits(N, g, empty).to(
        DEV), scale or D ** -0.5


def run_attention(ops, cache, q, ql, tl, anc, scale, *, layer=0, splits=0, rows=None, ws_fill=None):
    B, N, hq, D = q.shape
    most = int(ql.max())
    need = ops.kv8_attention_workspace_bytes(B, N, hq, cache.n_kv_heads, D, num_splits=splits, max_q_len=most)
    ws = torch.full((need // 4 + 4,), 0x7fc00000, dtype=torch.int32, device=DEV) if need else None
    out = torch.full_like(q, math.nan)
    got = ops.tree_attention_kv8(q, cache, layer, ql, tl, anc, scale=scale, out=out, workspace=ws, num_splits=splits,
                                 max_q_len=most)
    assert got is out
    return out


CASES = [
    # B, N, hq, H, D, lens
    (1, 1, 1, 1, 128, [0]),
    (1, 1, 12, 2, 128, [45]),
    (2, 7, 8, 8, 128, [0, 31]),
    (3, 13, 12, 2, 128, [64, 127, 96]),
    (5, 13, 12, 2, 128, [1024, 1, 33, 515, 1000]),
    (2, 32, 28, 4, 128, [300, 255]),
    (1, 128, 7, 1, 128, [1000]),
    (2, 128, 4, 2, 128, [31, 500]),
    (1, 16, 32, 8, 128, [4100]),
    (9, 21, 6, 1, 128, [5, 95, 160, 32, 129, 63, 0, 224, 417]),
]


@pytest.mark.parametrize("splits", [0, 1, 3, 64])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])))
def test_attention_bf16(ops, case, splits):
    B, N, hq, H, D, lens = case
    cache, q, ql, tl, anc, scale = attention_case(ops, torch.bfloat16, B, N, hq, H, D, lens, B * 100 + N)
    out = run_attention(ops, cache, q, ql, tl, anc, scale, splits=splits)
    want, tol = attention_reference(q, cache, 0, range(B), ql, tl, anc, scale)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("splits", [0, 2])
@pytest.mark.parametrize("case", [(1, 1, 4, 2, 64, [0]), (3, 9, 4, 2, 64, [70, 31, 200]), (2, 16, 6, 3, 16, [333, 64]),
                                  (1, 5, 8, 1, 96, [2049]), (2, 128, 3, 3, 128, [40, 97])],
                         ids=lambda c: "x".join(map(str, c[:5])))
def test_attention_f32(ops, case, splits):
    B, N, hq, H, D, lens = case
    cache, q, ql, tl, anc, scale = attention_case(ops, torch.float32, B, N, hq, H, D, lens, B * 100 + N)
    out = run_attention(ops, cache, q, ql, tl, anc, scale, splits=splits)
    want, tol = attention_reference(q, cache, 0, range(B), ql, tl, anc, scale)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 112), (torch.bfloat16, 128),
                                     (torch.float32, 64)])
def test_attention_layers_row_map_and_empty_rows(ops, dtype, D):
    """The second layer, cache rows in another order, nodes that see no tree slot and (prefix empty) nothing at all."""
    lens = [0, 50, 200, 0]
    cache, q, ql, tl, anc, scale = attention_case(ops, dtype, 4, 6, 6, 2, D, lens, 17, layers=2, empty=(2, 5))
    rows = i32([0, 1, 2, 3])
    perm = torch.tensor([2, 0, 3, 1])
    out = run_attention(ops, cache.view(perm.to(torch.int32).to(DEV)), q, ql[perm], tl[perm], anc, scale, layer=1)
    want, tol = attention_reference(q, cache, 1, perm.tolist(), ql[perm], tl[perm], anc, scale)
    assert ((out.double() - want).abs() <= tol).all()
    nothing = (tl[perm] == 0) & (ql[perm] == 0)
    assert nothing.any() and (out[nothing][:, [2, 5]] == 0).all() and rows is not None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_large_scores_and_values(ops, dtype):
    """Scores of some hundreds (one slot takes all the weight) and blocks whose V differ by 2^40 in size."""
    cache, q, ql, tl, anc, scale = attention_case(ops, dtype, 2, 5, 4, 2, 128, [300, 128], 23, k_size=40.0)
    cache.v_scale[:, :, :, 1::2] *= 2.0 ** 40
    cache.v_scale[:, :, 1] *= 2.0 ** -60
    out = run_attention(ops, cache, q, ql, tl, anc, scale)
    want, tol = attention_reference(q, cache, 0, range(2), ql, tl, anc, scale)
    assert ((out.double() - want).abs() <= tol).all()


def test_attention_shows_a_poisoned_block(ops):
    cache, q, ql, tl, anc, scale = attention_case(ops, torch.bfloat16, 3, 4, 4, 2, 128, [100, 300, 64], 29)
    cache.k_scale[0, 0, 1, 2] = math.nan
    cache.v_scale[0, 1, 0, 5] = math.nan
    out = run_attention(ops, cache, q, ql, tl, anc, scale)
    assert out[0, :, 2:].isnan().all() and out[0, :, :2].isfinite().all()
    assert out[1, :, :2].isnan().all() and out[1, :, 2:].isfinite().all() and out[2].isfinite().all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("what", ["q", "k_tail", "v_tail"])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 128)])
def test_attention_shows_values_that_are_not_finite(ops, dtype, D, what, bad):
    """One entry of a query row, of a tail token (all nodes see it) or of a tree node's K or V (its descendants and
    itself do).  The rows that meet it show it, the others are what they are without it."""
    lens = [100, 40, 5]
    for splits in (1, 2):
        cache, q, ql, tl, anc, scale = attention_case(ops, dtype, 3, 6, 4, 2, D, lens, 47)
        want, tol = attention_reference(q, cache, 0, range(3), ql, tl, anc, scale)
        bits = torch.tensor([[(int(w) >> j) & 1 for j in range(6)] for w in anc[:, 0].tolist()]).bool()
        assert bits[:, 4].any() and not bits[:, 4].all()
        hit = torch.zeros(3, 6, 4, dtype=torch.bool)  # rows that meet a bad value
        if what == "q":
            q[0, 2, 1, 7], q[2, 5, 3, D - 1] = bad, bad
            hit[0, 2, 1] = hit[2, 5, 3] = True
        else:
            t = getattr(cache, what)
            t[0, 0, 1, 2, 9] = bad             # a tail token of row 0, second KV head
            t[0, 1, 0, int(tl[1]) + 4, D - 3] = bad  # node 4 of row 1, first KV head
            hit[0, :, 2:] = True
            hit[1, :, :2] = bits[:, 4:5]
        hit = hit.to(DEV)
        out = run_attention(ops, cache, q, ql, tl, anc, scale, splits=splits)
        assert ((out.double() - want).abs() <= tol)[~hit].all()
        if what == "v_tail" and not (dtype == torch.bfloat16 and D == 128):  # fp32 sums: in the dim it is in
            assert not out[0, :, 2:, 9].isfinite().any() and not out[1][hit[1]][:, D - 3].isfinite().any()
        else:
            assert out[hit].isnan().all()


def test_attention_bad_lengths_are_recorded(ops):
    from flashgrpo_b200 import _native as N

    cache, q, ql, tl, anc, scale = attention_case(ops, torch.bfloat16, 2, 4, 4, 2, 128, [96, 64], 31)
    good = run_attention(ops, cache, q, ql, tl, anc, scale)
    for bad in (dict(q=33), dict(q=-32), dict(q=128), dict(t=-1), dict(t=33)):
        q2, t2 = ql.clone(), tl.clone()
        q2[0], t2[0] = bad.get("q", 96), bad.get("t", 0)
        out = torch.empty_like(q)
        ops.tree_attention_kv8(q, cache, 0, q2, t2, anc, scale=scale, num_splits=1, out=out)
        assert N.read_device_error(clear=True) == N.FG_EINVAL
        assert torch.equal(out[1], good[1])
    ops.tree_attention_kv8(q, cache.view(i32([2, 1])), 0, ql, tl, anc, scale=scale, num_splits=1, out=out)
    assert N.read_device_error(clear=True) == N.FG_EINVAL and torch.equal(out[1], good[1])


def test_attention_refusals(ops):
    from flashgrpo_b200 import _native as N

    cache, q, ql, tl, anc, scale = attention_case(ops, torch.bfloat16, 2, 4, 4, 2, 128, [96, 64], 31)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(N.NativeError):
            ops.tree_attention_kv8(q, cache, 0, ql, tl, anc, scale=bad, num_splits=1)
    with pytest.raises(N.NativeError):
        ops.tree_attention_kv8(q, cache, 0, ql, tl, anc, scale=scale, num_splits=65)
    with pytest.raises(N.NativeError):  # needs a workspace
        ops.tree_attention_kv8(q, cache, 0, ql, tl, anc, scale=scale, num_splits=2)
    for layer in (-1, 1):
        with pytest.raises(N.NativeError):
            ops.tree_attention_kv8(q, cache, layer, ql, tl, anc, scale=scale, num_splits=1)
    with pytest.raises(ValueError):
        ops.tree_attention_kv8(q, cache, 0, ql[:1], tl, anc, scale=scale)
    with pytest.raises(ValueError):
        ops.tree_attention_kv8(q, cache, 0, ql, tl, anc[:3].contiguous(), scale=scale)
    with pytest.raises(TypeError):
        ops.tree_attention_kv8(q.float(), cache, 0, ql, tl, anc, scale=scale)
    with pytest.raises(N.NativeError):
        ops.tree_attention_kv8(q[:, :, :3].contiguous(), cache, 0, ql, tl, anc, scale=scale, num_splits=1)
    big = torch.randn(2, 37, 4, 128, device=DEV).bfloat16()  # more nodes than the tail holds
    with pytest.raises(N.NativeError):
        ops.tree_attention_kv8(big, cache, 0, ql, tl, torch.ones(37, 4, dtype=torch.int32, device=DEV), scale=scale,
                               num_splits=1)
    with pytest.raises(TypeError):
        ops.Kv8Cache.empty(1, 1, 1, 32, 128, max_nodes=1, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError):
        ops.Kv8Cache.empty(1, 1, 1, 32, 40, max_nodes=1, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(1, 2, 128, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(N.NativeError):  # 128 tokens in a cache of 96
        ops.kv8_load(cache, 0, k, k, i32([5]), i32([0]), i32([0]))
    with pytest.raises(ValueError):
        ops.kv8_load(cache, 0, k[:, :1], k[:, :1], i32([5]), i32([0]), i32([0]))
    with pytest.raises(ValueError):
        ops.kv8_commit(cache, i32([[0], [0]]), i32([1, 1]), ql, tl, q_len_out=ql)
    with pytest.raises(N.NativeError):  # lengths that are half in place
        ops.kv8_commit(cache, i32([[0], [0]]), i32([1, 1]), ql, tl, q_len_out=ql, tail_len_out=i32([0, 0]))
    with pytest.raises(N.NativeError):
        ops.kv8_commit(cache, torch.zeros(2, 17, dtype=torch.int32, device=DEV), i32([1, 1]), ql, tl)


def test_a_run_of_rounds(ops):
    """Prompts loaded, then rounds of RoPE / K and V write to the tail, attention and commit, captured into one graph
    and replayed on a side stream: the cache is what the plain form makes of the same tokens, and each round's
    attention matches the reference on it."""
    g = torch.Generator().manual_seed(41)
    B, H, hq, D, N, L = 4, 2, 6, 128, 5, 2
    cache = ops.Kv8Cache.empty(L, B, H, 192, D, max_nodes=N, dtype=torch.bfloat16, device=DEV)
    plain = Plain(cache)
    lens = [61, 30, 94, 1]
    ql, tl = i32([0] * B), i32([0] * B)
    for layer in range(L):
        k, v = (torch.randn(B, H, 94, D, generator=g).bfloat16() for _ in range(2))
        ops.kv8_load(cache, layer, k.to(DEV), v.to(DEV), i32(lens), ql, tl)
        for b in range(B):
            for kv, x in enumerate((k, v)):
                plain.put(kv, layer, b, 0, x[b, :, :lens[b]])
    plain.same(cache)
    anc = tree_bits(N, g).to(DEV)
    qkv = torch.zeros(B * N, (hq + 2 * H) * D, dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(B, N, dtype=torch.int32, device=DEV)
    inv = (1.0 / 1e4 ** (torch.arange(0, D, 2).float() / D)).to(DEV)
    path, acc = i32([[0, 0, 0]] * B), i32([0] * B)
    qs = [torch.zeros(B, N, hq, D, dtype=torch.bfloat16, device=DEV) for _ in range(L)]
    outs = [torch.zeros_like(qs[0]) for _ in range(L)]
    need = ops.kv8_attention_workspace_bytes(B, N, hq, H, D, num_splits=2, max_q_len=192)
    ws = torch.empty(need // 4, dtype=torch.int32, device=DEV)

    def round_():
        for layer in range(L):
            ops.rope_kv_write(qkv, pos, inv, 1.0, B=B, n_nodes=N, n_q_heads=hq, n_kv_heads=H, head_dim=D, kv_len=tl,
                              k_cache=None, v_cache=None, q_out=qs[layer], kv=cache.tail_layer(layer))
            ops.tree_attention_kv8(qs[layer], cache, layer, ql, tl, anc, scale=0.1, out=outs[layer], workspace=ws,
                                   num_splits=2, max_q_len=192)
        ops.kv8_commit(cache, path, acc, ql, tl)

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        round_()
    assert ql.tolist() == [32, 0, 64, 0]
    total = list(lens)
    for step in range(12):
        qkv.copy_(torch.randn(qkv.shape, generator=g).bfloat16())
        a = [int(torch.randint(0, 4, (1,), generator=g)) for _ in range(B)]
        pt = torch.full((B, 3), -1, dtype=torch.int32)
        for b in range(B):
            pt[b, :a[b]] = torch.randperm(N, generator=g)[:a[b]].sort().values.to(torch.int32)
        path.copy_(pt)
        acc.copy_(torch.tensor(a, dtype=torch.int32))
        before = ql.clone(), tl.clone()
        eager = step == 5
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            round_() if eager else graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        # the tree's K/V rows as written (RoPE at position 0 leaves them as they are), then the commit
        kv = qkv.view(B, N, hq + 2 * H, D).cpu()
        ref = Plain(cache)
        for b in range(B):
            q0, t0 = int(before[0][b]), int(before[1][b])
            for layer in range(L):
                for i in range(2):
                    x = kv[b, :, hq + i * H:hq + (i + 1) * H].permute(1, 0, 2).double()
                    plain.tail[i][layer, b][:, t0:t0 + N] = x
                    at = list(range(t0)) + [t0 + int(pt[b, j]) for j in range(a[b])]
                    new = plain.put(i, layer, b, q0, plain.tail[i][layer, b][:, at].clone())
            total[b] += a[b]
            assert new == (total[b] // BLK * BLK, total[b] % BLK) == (int(ql[b]), int(tl[b]))
        plain.same(cache)
        del ref
        if step % 4 == 3:  # the next attention, on the state that the plain form agrees with
            out = torch.empty_like(qs[0])
            ops.tree_attention_kv8(qs[0], cache, 1, ql, tl, anc, scale=0.1, out=out, workspace=ws, num_splits=2,
                                   max_q_len=192)
            want, tol = attention_reference(qs[0], cache, 1, range(B), ql, tl, anc, 0.1)
            assert ((out.double() - want).abs() <= tol).all()
