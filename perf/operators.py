"""Cases of the 8-bit KV cache and the token log probabilities: inputs, plain forms, exact values and work.

  load       a prefill's K/V into the 8-bit cache (whole blocks of 32 tokens in e4m3, the rest in the tail)
  commit     the end of a verify round: accepted path compacted in the tail, completed blocks quantised
  attention  tree attention of one layer over the 8-bit blocks, the tail and the round's tree
  logprobs   log probability, entropy and best alternatives of given tokens
  backward   the gradient of log probability and entropy with respect to the logits

The plain forms are torch operations in 32 bits; `exact` computes the definitions in 64 bits.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

own = False

BLOCK = 32
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _ops():
    root = str(Path(__file__).resolve().parents[1] / "ss-grpo_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from flashgrpo_b200 import ops

    return ops


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one rollout just after a short prompt, no tree: the smallest attention call, all latency
        dict(name="attention one row", op="attention", dtype="bf16", batch=1, nodes=1, hq=12, hkv=2, dim=128,
             length=45),
        # the 1.5B shape's verify round: 64 rollouts around 1024 tokens, trees of 13 nodes
        dict(name="attention 64x1024", op="attention", dtype="bf16", batch=64, nodes=13, hq=12, hkv=2, dim=128,
             length=1024),
        # the 7B shape's shard: 32-node trees, 224 query rows on each KV head
        dict(name="attention 16x2048 wide", op="attention", dtype="bf16", batch=16, nodes=32, hq=28, hkv=4, dim=128,
             length=2048),
        # long rollouts, 32/8 heads: 1.1 GB of cache per layer, the call the cache is made for
        dict(name="attention 32x16384", op="attention", dtype="bf16", batch=32, nodes=16, hq=32, hkv=8, dim=128,
             length=16384),
        # prompts of 256 tokens, 8 samples of each, into one layer's cache (the rollout's start)
        dict(name="load 8x8x256", op="load", dtype="bf16", prompts=8, repeats=8, hkv=2, dim=128, length=256),
        # long ragged prompts at the 8B shape, one sample each
        dict(name="load 16x4099", op="load", dtype="bf16", prompts=16, repeats=1, hkv=8, dim=128, length=4099),
        # the end of a round at the 1.5B shape: all 28 layers of 64 rows, a path of up to 4 tokens
        dict(name="commit 28x64", op="commit", dtype="bf16", layers=28, batch=64, hkv=2, dim=128, nodes=13, path=4,
             length=256),
        # the same at the 8B shape with chain trees of 53 nodes
        dict(name="commit 32x32", op="commit", dtype="bf16", layers=32, batch=32, hkv=8, dim=128, nodes=53, path=4,
             length=192),
        # a round's accepted tokens under the packed target logits, with the four best alternatives
        dict(name="logprobs round", op="logprobs", dtype="bf16", n=192, rows=160, vocab=151936, pad=0, k=4,
             temperature=1.0),
        # a training micro-batch of 4096 positions: log probability and entropy
        dict(name="logprobs batch", op="logprobs", dtype="bf16", n=4096, rows=0, vocab=151936, pad=0, k=0,
             temperature=1.0),
        # the fp32 configuration's vocabulary on a few positions: the smallest gradient
        dict(name="backward small", op="backward", dtype="f32", n=37, vocab=4096, pad=0, entropy=True,
             temperature=0.7),
        # the micro-batch's gradient with the entropy bonus
        dict(name="backward batch", op="backward", dtype="bf16", n=4096, vocab=151936, pad=0, entropy=True,
             temperature=1.0),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], uniform over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "load", "commit", "logprobs", "backward"])
    if op == "attention":
        if rng.random() < 0.25:  # the fp32 configuration's range
            c = dict(op=op, dtype="f32", batch=_spread(rng, 1, 16), nodes=_spread(rng, 1, 16), dim=rng.choice([16, 64, 96, 128]),
                     length=_spread(rng, 1, 2048))
            c["hq"], c["hkv"] = rng.choice([(4, 2), (6, 3), (8, 1)])
            return c
        c = dict(op=op, dtype="bf16", batch=_spread(rng, 1, 128), nodes=_spread(rng, 1, 128), dim=128)
        c["hq"], c["hkv"] = rng.choice([(12, 2), (28, 4), (32, 8), (8, 8), (7, 1)])
        most = 32 * 8 * 16384 // (c["batch"] * c["hkv"])  # the largest listed cache ...
        rows = 32 * 32 * 16 * 16384 // (c["batch"] * c["hq"] * c["nodes"])  # ... and its products
        c["length"] = _spread(rng, 1, max(1, min(most, rows, 32768)))
        return c
    if op == "load":
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), prompts=_spread(rng, 1, 32),
                 repeats=rng.choice([1, 1, 2, 8]), hkv=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128, 128]))
        most = 16 * 8 * 4099 // (c["prompts"] * c["repeats"] * c["hkv"])
        c["length"] = _spread(rng, 1, max(1, min(most, 8192)))
        return c
    if op == "commit":
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), layers=_spread(rng, 1, 32),
                    batch=_spread(rng, 1, 64), hkv=rng.choice([1, 2, 4]), dim=rng.choice([64, 128, 128]),
                    nodes=_spread(rng, 1, 64), path=rng.randint(1, 8), length=_spread(rng, 32, 256))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = _spread(rng, 97, 152064)
    c = dict(op=op, dtype=dtype, n=_spread(rng, 1, max(1, min(4096, (1 << 29) // vocab))), vocab=vocab,
             pad=rng.choice([0, 0, 5, 8]), temperature=rng.choice([0.6, 1.0, 1.0, 1.3]))
    if op == "backward":
        c["entropy"] = rng.random() < 0.7
        return c
    c["k"] = rng.choice([0, 0, 1, 5, 16])
    if c["k"]:
        c["n"] = max(1, min(c["n"], (1 << 26) // vocab))
    c["rows"] = rng.choice([0, 0, max(1, c["n"] * 3 // 4)])
    return c


# -------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _keys_values(shape, dtype, g):
    """K with a few strong channels and tokens of unequal size, V plain: what projections of hidden states look like."""
    chan = 1.0 + 6.0 * (torch.rand(shape[-1], generator=g, device="cuda") > 0.95)
    size = torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=g, device="cuda"))
    k = (torch.randn(shape, generator=g, device="cuda") * chan * size).to(dtype)
    v = (torch.randn(shape, generator=g, device="cuda") * size * 0.5).to(dtype)
    return k, v


def _block_scale(amax):
    """2^e with the smallest e >= -126 for which amax <= 448 * 2^e."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax == 0, torch.full_like(e, -126), e.clamp(min=-126))
    return torch.ldexp(torch.ones_like(amax), e)


def _quantise(x):
    """x [..., n * 32, D] -> e4m3 codes of the same shape and scales [..., n]."""
    b = x.float().unflatten(-2, (-1, BLOCK))
    scale = _block_scale(b.abs().amax((-1, -2)))
    q = (b / scale[..., None, None]).to(torch.float8_e4m3fn)
    return q.flatten(-3, -2), scale


def _tree_bits(nodes, g):
    """Ancestor-or-self bits [nodes, 4] of a random tree at most four levels below its root."""
    pick = torch.rand(nodes, generator=torch.Generator().manual_seed(int(torch.randint(1 << 30, (1,), generator=g,
                                                                                       device="cuda")))).tolist()
    words, depth = [], []
    for j in range(nodes):
        above = [i for i in range(j) if depth[i] < 4]
        p = above[int(pick[j] * len(above))] if above else -1
        w = list(words[p]) if p >= 0 else [0, 0, 0, 0]
        w[j >> 5] |= 1 << (j & 31)
        words.append(w)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return torch.tensor([[x - (1 << 32) if x >> 31 else x for x in w] for w in words], dtype=torch.int32,
                        device="cuda")


def _lengths(n, length, g):
    """n lengths in (length - 64, length], at least 0, the longest one among them."""
    d = torch.randint(0, min(64, length + 1), (n,), generator=g, device="cuda")
    d[0] = 0
    return (length - d).to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    dt = _TYPES[case["dtype"]]
    op = case["op"]
    if op == "attention":
        B, H, D, N = case["batch"], case["hkv"], case["dim"], case["nodes"]
        cap = -(-case["length"] // BLOCK) * BLOCK + BLOCK
        k, v = _keys_values((1, B, H, cap, D), dt, g)
        (k8, ks), (v8, vs) = _quantise(k), _quantise(v)
        del k, v
        kt, vt = _keys_values((1, B, H, BLOCK + N, D), dt, g)
        total = _lengths(B, case["length"], g)
        return dict(case=case, k8=k8, v8=v8, ks=ks, vs=vs, kt=kt, vt=vt, q_len=total // BLOCK * BLOCK,
                    tail_len=total % BLOCK, anc=_tree_bits(N, g), scale=D ** -0.5,
                    q=torch.randn(B, N, case["hq"], D, generator=g, device="cuda").to(dt))
    if op == "load":
        P, R, H, D, S = case["prompts"], case["repeats"], case["hkv"], case["dim"], case["length"]
        k, v = _keys_values((P, H, S, D), dt, g)
        cap = -(-S // BLOCK) * BLOCK
        return dict(case=case, k=k, v=v, lengths=_lengths(P, S, g),
                    q_len=torch.zeros(P * R, dtype=torch.int32, device="cuda"),
                    tail_len=torch.zeros(P * R, dtype=torch.int32, device="cuda"),
                    **_empty_cache(1, P * R, H, cap, D, BLOCK + 16, dt))
    if op == "commit":
        L, B, H, D, N = case["layers"], case["batch"], case["hkv"], case["dim"], case["nodes"]
        s = _empty_cache(L, B, H, case["length"] // BLOCK * BLOCK + BLOCK, D, BLOCK + N, dt)
        s["kt"], s["vt"] = _keys_values((L, B, H, BLOCK + N, D), dt, g)
        most = min(case["path"], N)
        acc_len = torch.randint(1, most + 1, (B,), generator=g, device="cuda")
        # a path through the tree: strictly increasing nodes from the root
        nodes = torch.rand(B, N, generator=g, device="cuda")
        nodes[:, 0] = 2.0
        nodes = nodes.topk(most, dim=1).indices.sort(dim=1).values
        nodes = torch.where(torch.arange(most, device="cuda") < acc_len[:, None], nodes, -1)
        # row lengths of a running batch: every (32 / mean path)-th round completes a block
        total = _lengths(B, case["length"], g)
        return dict(case=case, **s, acc_nodes=nodes.to(torch.int32), acc_len=acc_len.to(torch.int32),
                    q_len=total // BLOCK * BLOCK, tail_len=total % BLOCK,
                    q_out=torch.zeros(B, dtype=torch.int32, device="cuda"),
                    t_out=torch.zeros(B, dtype=torch.int32, device="cuda"))
    n, V = case["n"], case["vocab"]
    src = case.get("rows") or n
    wide = torch.empty(src, V + case["pad"], dtype=dt, device="cuda")
    for lo in range(0, src, 512):  # logits of a model that has learnt something: a few tokens stand out
        part = wide[lo:lo + 512]
        x = torch.randn(part.shape, generator=g, device="cuda").mul_(2.0)
        hot = torch.randint(0, V, (part.shape[0], 4), generator=g, device="cuda")
        part.copy_(x.scatter_add_(1, hot, 8.0 * torch.rand(hot.shape, generator=g, device="cuda")))
    logits = wide[:, :V]
    rows = torch.randint(0, src, (n,), generator=g, device="cuda").to(torch.int32) if case.get("rows") else None
    hit = logits if rows is None else logits[rows.long()]
    tokens = torch.where(torch.rand(n, generator=g, device="cuda") < 0.7, hit.argmax(1),
                         torch.randint(0, V, (n,), generator=g, device="cuda")).to(torch.int32)
    if n > 4:  # positions behind a sequence's end
        tokens[torch.rand(n, generator=g, device="cuda") < 0.1] = -1
    s = dict(case=case, logits=logits, tokens=tokens, rows=rows)
    if op == "backward":
        lse, ent = [], []
        for lo in range(0, n, 512):
            x = logits[lo:lo + 512].double() / case["temperature"]
            z = torch.logsumexp(x, 1)
            lse.append(z)
            ent.append(-(torch.exp(x - z[:, None]) * (x - z[:, None])).sum(1))
        s["lse"], s["ent"] = torch.cat(lse).float(), torch.cat(ent).float()
        s["g"] = torch.randn(n, generator=g, device="cuda")
        s["h"] = 0.1 * torch.randn(n, generator=g, device="cuda") if case["entropy"] else None
        s["out"] = torch.empty(n, V, dtype=dt, device="cuda")
    return s


def _empty_cache(L, B, H, cap, D, tail, dt):
    z = dict(device="cuda")
    return dict(k8=torch.zeros(L, B, H, cap, D, **z).to(torch.float8_e4m3fn),
                v8=torch.zeros(L, B, H, cap, D, **z).to(torch.float8_e4m3fn),
                ks=torch.zeros(L, B, H, cap // BLOCK, **z), vs=torch.zeros(L, B, H, cap // BLOCK, **z),
                kt=torch.zeros(L, B, H, tail, D, dtype=dt, **z), vt=torch.zeros(L, B, H, tail, D, dtype=dt, **z))


# --------------------------------------------------------------- plain forms
def _plain_attention(s):
    q, N = s["q"].float(), s["case"]["nodes"]
    B, _, hq, D = q.shape
    H = s["k8"].shape[2]
    qh = q.view(B, N, H, hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D)
    cap, tail = s["k8"].shape[3], s["kt"].shape[3]
    at, tt = torch.arange(cap, device="cuda"), torch.arange(tail, device="cuda")
    j = tt[None, :] - s["tail_len"][:, None].long()  # tree index of each tail slot
    jn = j.clamp(0, N - 1)
    word = s["anc"].long()[:, :, None]
    bits = (word >> torch.arange(32, device="cuda") & 1).flatten(1)[:, :N].bool()  # [node, node]
    seen = torch.where(j[:, None, :] < 0, True, bits[:, jn].transpose(0, 1) & (j < N)[:, None, :])  # [B, N, tail]
    kd = s["k8"][0].float() * s["ks"][0].repeat_interleave(BLOCK, -1)[..., None]
    x = torch.matmul(qh, kd.transpose(-1, -2))
    del kd
    x.masked_fill_((at[None, :] >= s["q_len"][:, None])[:, None, None, :], float("-inf"))
    y = torch.matmul(qh, s["kt"][0].float().transpose(-1, -2))
    y.masked_fill_(~seen.repeat(1, hq // H, 1)[:, None], float("-inf"))
    x.mul_(s["scale"])
    y.mul_(s["scale"])
    m = torch.maximum(x.amax(-1, True), y.amax(-1, True))
    x.sub_(m).exp_()
    y.sub_(m).exp_()
    total = x.sum(-1, True) + y.sum(-1, True)
    vd = s["v8"][0].float() * s["vs"][0].repeat_interleave(BLOCK, -1)[..., None]
    o = (torch.matmul(x, vd) + torch.matmul(y, s["vt"][0].float())) / total
    return o.view(B, H, hq // H, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, hq, D).to(s["q"].dtype)


def _plain_load(s):
    R = s["case"]["repeats"]
    S = s["k"].shape[2]
    nb = s["k8"].shape[3] // BLOCK
    lens = s["lengths"].long()
    q, r = lens // BLOCK * BLOCK, lens % BLOCK
    whole = (torch.arange(nb, device="cuda") < (q // BLOCK)[:, None]).repeat_interleave(R, 0)[:, None, :]
    at = (q[:, None] + torch.arange(BLOCK, device="cuda")).clamp(max=S - 1)
    rest = (torch.arange(BLOCK, device="cuda") < r[:, None]).repeat_interleave(R, 0)[:, None, :, None]

    def one(x, codes, scale, tail):
        x8, sc = _quantise(torch.nn.functional.pad(x, (0, 0, 0, nb * BLOCK - S)))
        x8, sc = x8.repeat_interleave(R, 0), sc.repeat_interleave(R, 0)
        keep = whole.repeat_interleave(BLOCK, -1)[..., None]
        codes[0].view(torch.uint8).copy_(torch.where(keep, x8.view(torch.uint8), codes[0].view(torch.uint8)))
        scale[0].copy_(torch.where(whole, sc, scale[0]))
        last = torch.gather(x, 2, at[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3])).repeat_interleave(R, 0)
        tail[0, :, :, :BLOCK].copy_(torch.where(rest, last, tail[0, :, :, :BLOCK]))

    one(s["k"], s["k8"], s["ks"], s["kt"])
    one(s["v"], s["v8"], s["vs"], s["vt"])
    s["q_len"].copy_(q.repeat_interleave(R))
    s["tail_len"].copy_(r.repeat_interleave(R))


def _plain_commit(s):
    q_len, tl, al = s["q_len"].long(), s["tail_len"].long(), s["acc_len"].long()
    tail, cap = s["kt"].shape[3], s["k8"].shape[3]
    p = torch.arange(tail, device="cuda")
    j = p[None, :] - tl[:, None]
    step = torch.gather(s["acc_nodes"].long(), 1, j.clamp(0, s["acc_nodes"].shape[1] - 1))
    src = torch.where((j >= 0) & (j < al[:, None]), tl[:, None] + step, p[None, :])  # compact slot -> tail slot
    nt = tl + al
    nb, r = nt // BLOCK, nt % BLOCK
    most = -(-(BLOCK - 1 + s["acc_nodes"].shape[1]) // BLOCK)  # blocks that a row can complete
    shift = torch.gather(src, 1, (p[None, :] + BLOCK * nb[:, None]).clamp(max=tail - 1))
    moved = (p[None, :] < r[:, None])[None, :, None, :, None]
    first = src[:, (torch.arange(most * BLOCK, device="cuda")).clamp(max=tail - 1)]
    # the slots that the blocks can take, wrapped at the capacity (a slot that is not written gets its own value back)
    slot = (q_len[:, None] + torch.arange(most * BLOCK, device="cuda")) % cap
    done = torch.arange(most * BLOCK, device="cuda") < (BLOCK * nb)[:, None]
    whole = lambda ix, like: ix[None, :, None, :].expand(like.shape[0], -1, like.shape[2], -1)  # noqa: E731

    def one(codes, scale, t):
        pick = lambda ix: torch.gather(t, 3, whole(ix, t)[..., None].expand(-1, -1, -1, -1, t.shape[4]))  # noqa: E731
        x8, sc = _quantise(pick(first))
        old = codes.view(torch.uint8)
        ix = whole(slot, old)[..., None].expand(-1, -1, -1, -1, old.shape[4])
        old.scatter_(3, ix, torch.where(done[None, :, None, :, None], x8.view(torch.uint8), torch.gather(old, 3, ix)))
        ix = whole(slot[:, ::BLOCK] // BLOCK, scale)
        scale.scatter_(3, ix, torch.where(done[None, :, None, ::BLOCK], sc, torch.gather(scale, 3, ix)))
        t.copy_(torch.where(moved, pick(shift), t))

    one(s["k8"], s["ks"], s["kt"])
    one(s["v8"], s["vs"], s["vt"])
    s["q_out"].copy_(q_len + BLOCK * nb)
    s["t_out"].copy_(r)


def _order(x):
    """Whole numbers in the order of x's values, ties by the lower index first; all different in a row."""
    b = (x + 0.0).view(torch.int32)
    b = b ^ ((b >> 31) & 0x7FFFFFFF)
    return (b.long() << 32) | (0x7FFFFFFF - torch.arange(x.shape[-1], device=x.device))


def _plain_logprobs(s):
    c = s["case"]
    raw = (s["logits"] if s["rows"] is None else s["logits"][s["rows"].long()]).float()
    pad = s["tokens"] < 0
    t = s["tokens"].clamp(min=0).long()[:, None]
    out = {}
    if c["k"]:
        best = torch.topk(_order(raw), c["k"], dim=1).values
        best = 0x7FFFFFFF - (best & 0xFFFFFFFF)
        out["top_idx"] = torch.where(pad[:, None], -1, best).to(torch.int32)
    x = raw if c["temperature"] == 1.0 else raw / c["temperature"]
    m = x.amax(1, True)
    z = x - m
    e = torch.exp(z)
    s0 = e.sum(1, True)
    ls = torch.log(s0)
    zero = torch.zeros((), device="cuda")
    out["logp"] = torch.where(pad, zero, (z.gather(1, t) - ls)[:, 0])
    out["lse"] = torch.where(pad, zero, (m + ls)[:, 0])
    if c["k"]:
        out["top_logp"] = torch.where(pad[:, None], zero, z.gather(1, best) - ls)
    out["entropy"] = torch.where(pad, zero, (ls - e.mul_(z).sum(1, True) / s0)[:, 0])
    return out


def _plain_backward(s):
    c = s["case"]
    pad = (s["tokens"] < 0)[:, None]
    t = s["tokens"].clamp(min=0).long()[:, None]
    z = s["logits"].float()
    z = z / c["temperature"] if c["temperature"] != 1.0 else z
    z = z - s["lse"][:, None]
    p = torch.exp(z)
    if s["h"] is not None:
        w = z.add_(s["ent"][:, None]).mul_(s["h"][:, None]).add_(s["g"][:, None])
    else:
        w = s["g"][:, None]
    d = p.mul_(w).neg_()
    d.scatter_add_(1, t, s["g"][:, None])
    if c["temperature"] != 1.0:
        d = d / c["temperature"]
    return s["out"].copy_(d.masked_fill_(pad, 0.0))


# ---------------------------------------------------------------- operators
def _handle(s):
    """The cache handle and workspace that a program keeps for its buffers."""
    if "cache" not in s:
        ops = _ops()
        s["cache"] = ops.Kv8Cache(s["k8"], s["v8"], s["ks"], s["vs"], s["kt"], s["vt"])
        if s["case"]["op"] == "attention":
            B, N, hq, D = s["q"].shape
            need = ops.kv8_attention_workspace_bytes(B, N, hq, s["k8"].shape[2], D, max_q_len=s["case"]["length"])
            s["ws"] = torch.zeros(need // 4 + 4, dtype=torch.int32, device="cuda") if need else None
            s["o"] = torch.empty_like(s["q"])
    return s["cache"]


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if op == "attention":
        if not own:
            return _plain_attention(s)
        cache = _handle(s)
        return _ops().tree_attention_kv8(s["q"], cache, 0, s["q_len"], s["tail_len"], s["anc"], scale=s["scale"],
                                         out=s["o"], workspace=s["ws"], max_q_len=c["length"])
    if op in ("load", "commit"):
        if own and op == "load":
            _ops().kv8_load(_handle(s), 0, s["k"], s["v"], s["lengths"], s["q_len"], s["tail_len"],
                            repeats=c["repeats"])
        elif own:
            _ops().kv8_commit(_handle(s), s["acc_nodes"], s["acc_len"], s["q_len"], s["tail_len"],
                              q_len_out=s["q_out"], tail_len_out=s["t_out"])
        else:
            _plain_load(s) if op == "load" else _plain_commit(s)
        q, t = (s["q_len"], s["tail_len"]) if op == "load" else (s["q_out"], s["t_out"])
        return dict(k8=s["k8"], v8=s["v8"], k_scale=s["ks"], v_scale=s["vs"], k_tail=s["kt"], v_tail=s["vt"],
                    q_len=q, tail_len=t)
    if op == "logprobs":
        if not own:
            return _plain_logprobs(s)
        r = _ops().token_logprobs(s["logits"], s["tokens"], rows=s["rows"], temperature=c["temperature"], k=c["k"])
        out = dict(logp=r.logp, entropy=r.entropy, lse=r.lse)
        return dict(out, top_idx=r.top_idx, top_logp=r.top_logp) if c["k"] else out
    if not own:
        return _plain_backward(s)
    return _ops().token_logprobs_backward(s["logits"], s["tokens"], s["lse"], s["ent"], s["g"], s["h"],
                                          temperature=c["temperature"], out=s["out"])


# -------------------------------------------------------------- exact values
def _e4m3(x):
    """x (64 bits, at most 448 in size) rounded to the nearest e4m3 value, ties to even."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    e = torch.where(x.abs() >= torch.exp2(e + 1), e + 1, torch.where((x.abs() < torch.exp2(e)) & (e > -6), e - 1, e))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_blocks(x):
    """x [m, 32, D] in 64 bits, all blocks at once: code values and scales [m]."""
    amax = x.abs().amax((1, 2))
    e = torch.floor(torch.log2((amax / 448.0).clamp(min=2.0 ** -126)))
    e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where((amax <= 448.0 * torch.exp2(e - 1)) & (e > -126), e - 1, e)
    return _e4m3(x * torch.exp2(-e)[:, None, None]), torch.exp2(e)


def _exact_attention(s):
    B, N, hq, D = s["q"].shape
    H = s["k8"].shape[2]
    G = hq // H
    bits = [[(int(w) >> j) & 1 for w in row for j in range(32)][:N] for row in s["anc"].tolist()]
    bits = torch.tensor(bits, dtype=torch.bool, device="cuda")
    out = torch.zeros(B, N, hq, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, t = int(s["q_len"][b]), int(s["tail_len"][b])
        blocks = lambda x, sc: (x[0, b, :, :n].double().view(H, -1, BLOCK, D)  # noqa: E731
                                * sc[0, b, :, :n // BLOCK].double()[..., None, None]).view(H, n, D)
        k = torch.cat([blocks(s["k8"], s["ks"]), s["kt"][0, b, :, :t + N].double()], 1)
        v = torch.cat([blocks(s["v8"], s["vs"]), s["vt"][0, b, :, :t + N].double()], 1)
        see = torch.cat([torch.ones(N, n + t, dtype=torch.bool, device="cuda"), bits], 1)
        for h in range(H):
            q = s["q"][b, :, h * G:(h + 1) * G].double()
            x = torch.einsum("ngd,td->ngt", q, k[h]) * s["scale"]
            x = x.masked_fill(~see[:, None, :], float("-inf")).softmax(-1)
            out[b, :, h * G:(h + 1) * G] = torch.einsum("ngt,td->ngd", x, v[h])
    return out


def _exact_cache(s, src, start, count, row_of):
    """The cache after whole blocks of src(row) went to slot start[row] on, in 64 bits. src: rows' tokens
    [layers, heads, tokens, D] for K or V; count[row]: tokens taken."""
    out = {}
    for x, name in (("k", "k8"), ("v", "v8")):
        codes, scale = s[name].double(), s[x + "s"].double()
        tail = s[x + "t"].double()
        for b in range(codes.shape[1]):
            rows = src(x, row_of(b))
            L, H, _, D = rows.shape
            whole, c0 = count[b] // BLOCK, start[b]
            if whole:
                w, sc = _exact_blocks(rows[:, :, :whole * BLOCK].reshape(-1, BLOCK, D))
                codes[:, b, :, c0:c0 + whole * BLOCK] = w.view(L, H, -1, D)
                scale[:, b, :, c0 // BLOCK:c0 // BLOCK + whole] = sc.view(L, H, whole)
            r = count[b] % BLOCK
            tail[:, b, :, :r] = rows[:, :, whole * BLOCK:whole * BLOCK + r]
        out.update({name: codes, x + "_scale": scale, x + "_tail": tail})
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "attention":
        return _exact_attention(s)
    if op == "load":
        lens = s["lengths"].tolist()
        R = case["repeats"]
        out = _exact_cache(s, lambda x, p: s[x][None, p].double(), [0] * (len(lens) * R),
                           [n for n in lens for _ in range(R)], lambda b: b // R)
        return dict(out, q_len=None, tail_len=None)
    if op == "commit":
        tl, al, ql = s["tail_len"].tolist(), s["acc_len"].tolist(), s["q_len"].tolist()
        path = s["acc_nodes"].tolist()

        def src(x, b):
            at = list(range(tl[b])) + [tl[b] + path[b][j] for j in range(al[b])]
            return s[x + "t"][:, b][:, :, at].double()

        out = _exact_cache(s, src, ql, [a + b for a, b in zip(tl, al)], lambda b: b)
        return dict(out, q_len=None, tail_len=None)
    T, t = case["temperature"], s["tokens"].long()
    got = {"logp": [], "entropy": [], "lse": [], "top_logp": [], "d": []}
    for lo in range(0, case["n"], 256):
        sel = slice(lo, lo + 256)
        x = (s["logits"][sel] if s["rows"] is None else s["logits"][s["rows"][sel].long()]).double() / T
        live = (t[sel] >= 0).double()[:, None]
        at = t[sel].clamp(min=0)[:, None]
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        if op == "backward":
            z = x - s["lse"][sel].double()[:, None]
            one_hot = torch.zeros_like(x).scatter_(1, at, 1.0)
            d = s["g"][sel].double()[:, None] * (one_hot - z.exp())
            if s["h"] is not None:
                d -= s["h"][sel].double()[:, None] * z.exp() * (z + s["ent"][sel].double()[:, None])
            got["d"].append((d / T * live).float())  # the gradient's type has at most 24 bits
            continue
        got["logp"].append((lp.gather(1, at) * live)[:, 0])
        got["lse"].append((torch.logsumexp(x, 1, True) * live)[:, 0])
        got["entropy"].append((-(p * lp).sum(1, True) * live)[:, 0])
        if case["k"]:
            got["top_logp"].append(lp.topk(case["k"], dim=1).values * live)
    if op == "backward":
        return torch.cat(got["d"])
    out = {k: torch.cat(got[k]) for k in ("logp", "entropy", "lse")}
    if case["k"]:
        out.update(top_logp=torch.cat(got["top_logp"]), top_idx=None)
    return out


# ---------------------------------------------------------------------- work
def work(case):
    op, D, w = case["op"], case.get("dim", 0), _BYTES[case["dtype"]]
    if op == "attention":
        B, H, N, T = case["batch"], case["hkv"], case["nodes"], case["length"] + case["nodes"]
        whole = case["length"] // BLOCK * BLOCK
        kv = B * H * 2 * (whole * D + whole // BLOCK * 4 + (T - whole) * D * w)
        return dict(bytes=kv + 2 * B * N * case["hq"] * D * w, flops=4.0 * B * case["hq"] * N * T * D)
    if op == "load":
        n = case["length"] * case["hkv"] * D * 2
        rows = case["prompts"] * case["repeats"]
        return dict(bytes=case["prompts"] * n * w + rows * n * (1 + 4 / BLOCK / D), flops=rows * n)
    if op == "commit":
        heads = case["layers"] * case["batch"] * case["hkv"] * 2
        mean = (1 + min(case["path"], case["nodes"])) / 2  # accepted tokens of a row
        # the moved path entries, and the rows (mean / 32 of them) that complete a block
        per = (mean - 1) * D * w * 2 + mean / BLOCK * (BLOCK * D * (w + 1) + 4)
        return dict(bytes=heads * max(per, 1.0), flops=heads * mean * D)
    n, V = case["n"], case["vocab"]
    if op == "logprobs":
        rows = min(case["rows"] or n, n)
        return dict(bytes=rows * V * w + n * (16 + 8 * case["k"]), flops=8.0 * n * V)
    return dict(bytes=2 * n * V * w, flops=8.0 * n * V)
