"""Measured cases of the serving-step operators: the fp8 KV cache (written, read back,
attended), decode attention over a shared prefix, and the verification of drafted tokens.

``run`` computes a case in its plain form (elementary torch operations in 32 or 64 bits),
or, with ``own``, by the framework's operators. Sizes are those of the framework's own
configurations: 16, 32 or 64 query heads over 8 KV heads of 128 dims (or one KV head, a
rank's share at 8-way tensor parallelism), blocks of 256 tokens, a vocabulary of 151,936.
"""
from __future__ import annotations

import math
import random
import sys

import torch

own = False  # set by the caller: False = plain form, True = the framework's operators

D = 128                 # head dim
E4M3_MAX = 448.0
MIN_EXP = -100          # smallest exponent a cache row is stored with
SCALE = D ** -0.5


def _ops():
    if "nano-vllm-x_b200" not in sys.path:
        sys.path.insert(0, "nano-vllm-x_b200")
    from nvattn import ops
    return ops


# ------------------------------------------------------------------------- cases

def listed():
    return [
        # one short prompt chunk written and its context read back: launch latency counts
        dict(name="kv8-chunk-1x33", kind="cache", seqs=1, new=33, ctx_lo=300, ctx_hi=300, kvh=8,
             block=256),
        # eight long prompts in chunks of 2048 at all 8 KV heads: a loaded prefill step
        dict(name="kv8-chunk-8x2048", kind="cache", seqs=8, new=2048, ctx_lo=2048, ctx_hi=14001,
             kvh=8, block=256),
        # a single user's decode step
        dict(name="kv8-decode-1x777", kind="decode", batch=1, heads=16, kvh=8, ctx_lo=777,
             ctx_hi=777, block=256, pad=0),
        # a full decode batch of a small model, contexts of 100 to 2048 tokens
        dict(name="kv8-decode-256", kind="decode", batch=256, heads=16, kvh=8, ctx_lo=100,
             ctx_hi=2048, block=256, pad=0),
        # long documents at 64 query heads over 8 KV heads
        dict(name="kv8-decode-32xlong", kind="decode", batch=32, heads=64, kvh=8, ctx_lo=4096,
             ctx_hi=32768, block=256, pad=1),
        # one very long context on a rank that holds one KV head with 16 query heads
        dict(name="kv8-decode-1x131071", kind="decode", batch=1, heads=16, kvh=1, ctx_lo=131071,
             ctx_hi=131071, block=256, pad=0),
        # a few conversations behind one system prompt
        dict(name="prefix-5x1024", kind="shared", batch=5, heads=16, kvh=8, shared=1024, own_lo=1,
             own_hi=200, block=256, pad=0, fp8=False),
        # many questions on one long document, 64 query heads
        dict(name="prefix-64x16384", kind="shared", batch=64, heads=64, kvh=8, shared=16384,
             own_lo=1, own_hi=1023, block=256, pad=2, fp8=False),
        # a large batch behind a few thousand shared tokens, cache in fp8
        dict(name="prefix-200x4096-kv8", kind="shared", batch=200, heads=32, kvh=8, shared=4096,
             own_lo=1, own_hi=600, block=256, pad=8, fp8=True),
        # one user, four drafted tokens without draft probabilities (n-gram drafting)
        dict(name="verify-chain-1x5", kind="verify", batch=1, nodes=5, vocab=151936, form="chain",
             noise=1.0),
        # a batch with seven drafted tokens and the draft model's logits
        dict(name="verify-draft-64x8", kind="verify", batch=64, nodes=8, vocab=151936,
             form="draft", noise=1.0),
        # draft trees of 64 nodes
        dict(name="verify-tree-16x64", kind="verify", batch=16, nodes=64, vocab=151936,
             form="tree", noise=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "decode", "decode", "shared", "shared", "verify", "verify"])
    kvh = rng.choice([1, 2, 4, 8])
    block = rng.choice([128, 256, 512])
    if kind == "cache":
        seqs = _log_int(rng, 1, 24)
        hi = _log_int(rng, 64, min(65536, 100000 // seqs))
        lo = rng.randint(1, hi)
        return dict(kind=kind, seqs=seqs, new=rng.randint(1, min(lo, max(1, 16000 // seqs))),
                    ctx_lo=lo, ctx_hi=hi, kvh=kvh, block=rng.choice([64, block]))
    if kind == "decode":
        batch = _log_int(rng, 1, 300)
        hi = _log_int(rng, 32, min(131071, 500000 // batch))
        return dict(kind=kind, batch=batch, heads=kvh * rng.choice([1, 2, 4, 5, 8, 16]), kvh=kvh,
                    ctx_lo=rng.randint(1, hi), ctx_hi=hi, block=rng.choice([64, block]),
                    pad=rng.randint(0, batch // 4))
    if kind == "shared":
        batch = _log_int(rng, 2, 220)
        group = rng.choice([1, 2, 4, 5, 8, 16])
        shared = block * rng.randint(1, max(1, min(64 * 256, 64 * 16384 // (batch * group)) // block))
        hi = _log_int(rng, 8, min(4096, 60000 // batch))
        return dict(kind=kind, batch=batch, heads=kvh * group, kvh=kvh, shared=shared,
                    own_lo=rng.randint(1, hi), own_hi=hi, block=block, pad=rng.randint(0, batch // 4),
                    fp8=rng.random() < 0.4)
    form = rng.choice(["chain", "draft", "tree"])
    nodes = rng.randint(2, 64) if form == "tree" else rng.randint(1, 12)
    rows = nodes * (2 if form == "draft" else 1)
    return dict(kind=kind, batch=_log_int(rng, 1, min(96, max(1, 1000 // rows))), nodes=nodes,
                vocab=_log_int(rng, 32000, 151936), form=form, noise=rng.choice([0.5, 1.0, 2.0]))


def _fixed(case):
    """A generator that depends on the case's sizes alone: lengths belong to the case."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    r = _fixed(case)
    if case["kind"] == "cache":
        return [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    live = case["batch"] - case["pad"]
    if case["kind"] == "decode":
        lens = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(live)]
    else:
        lens = [case["shared"] + r.randint(case["own_lo"], case["own_hi"]) for _ in range(live)]
    return lens + [0] * case["pad"]  # padding rows of a captured batch come last


def work(case):
    kind = case["kind"]
    if kind == "verify":
        # rows the walk needs: a fixed share of drafts is accepted (about 0.7 a step)
        v, b, n = case["vocab"], case["batch"], case["nodes"]
        depth = n - 1 if case["form"] != "tree" else 6
        rows = sum(0.7 ** i for i in range(min(depth, n - 1) + 1))
        if case["form"] == "draft":
            rows += sum(0.7 ** i for i in range(n - 1))
        return {"bytes": int(b * rows * v * 2 + b * n * 24), "flops": int(b * rows * v * 4)}
    lens, kvh = _lengths(case), case["kvh"]
    row8 = kvh * (D + 1) * 2  # one token's K and V in the fp8 cache
    row16 = kvh * D * 4       # the same in bf16
    if kind == "cache":
        new = case["seqs"] * case["new"]
        # new rows read and written, every context key read back
        return {"bytes": new * (row16 + row8) + sum(lens) * (row8 + row16),
                "flops": (new * 2 + sum(lens)) * kvh * D * 2}
    live = sum(n > 0 for n in lens)
    qo = case["batch"] * case["heads"] * D * 4
    if kind == "decode":
        return {"bytes": sum(lens) * row8 + live * row16 + qo,
                "flops": 4 * D * case["heads"] * sum(lens)}
    row = row8 if case["fp8"] else row16
    own_keys = sum(n - case["shared"] for n in lens if n)
    return {"bytes": (case["shared"] + own_keys) * row + qo, "flops": 4 * D * case["heads"] * sum(lens)}


# ------------------------------------------------------------------------ inputs

def _quantise(x):
    """bf16 rows (..., 128) -> e4m3 rows and one exponent byte a row: the smallest power of two
    that brings the row's largest magnitude to at most 448."""
    x = x.float()
    amax = x.abs().amax(-1)
    mant, exp = torch.frexp(amax)  # amax = mant * 2^exp, 448 = 0.875 * 2^9
    k = (exp - 9 + (mant > 0.875).to(exp.dtype)).clamp_min(MIN_EXP)
    k = torch.where(amax > 0, k, torch.full_like(k, MIN_EXP))
    finite = torch.isfinite(amax)
    q = torch.where(finite[..., None], x * torch.exp2(-k.float())[..., None],
                    torch.full_like(x, float("nan"))).to(torch.float8_e4m3fn)
    return q, torch.where(finite, k + 127, torch.full_like(k, 255)).to(torch.uint8)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _cache(g, blocks, block, kvh, fp8, spread):
    """Random cache pages: per-channel spread for keys, unit values; fp8 rows with exponents
    (blocks, kvh, block) or bf16."""
    shape = (blocks, block, kvh, D)
    out = torch.empty(shape, dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16, device="cuda")
    exps = torch.empty((blocks, kvh, block), dtype=torch.uint8, device="cuda") if fp8 else None
    step = max(1, (1 << 27) // (block * kvh * D))
    for i in range(0, blocks, step):
        n = min(step, blocks - i)
        x = (torch.randn((n, *shape[1:]), generator=g, device="cuda") * spread).to(torch.bfloat16)
        if fp8:
            out[i:i + n], e = _quantise(x)
            exps[i:i + n] = e.transpose(1, 2)
        else:
            out[i:i + n] = x
    return out, exps


def _tables(g, lens, block, shared=0):
    """Block tables over a permuted pool, rows padded with -1; the first shared / block columns
    of every row are the same pages."""
    ns = shared // block
    need = [max(0, -(-n // block) - ns) for n in lens]
    pages = ns + sum(need) + 2
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    width = max(1, ns + max(need))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    table[:, :ns] = ids[:ns]
    at = ns
    for i, n in enumerate(need):
        table[i, ns:ns + n] = ids[at:at + n]
        at += n
    return pages, table


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _qkv(g, n, heads, kvh, spread):
    """q, k, v as the views that a fused projection leaves."""
    qkv = torch.randn((n, (heads + 2 * kvh) * D), generator=g, device="cuda")
    qkv[:, heads * D:(heads + kvh) * D] *= spread.repeat(kvh)
    q, k, v = qkv.to(torch.bfloat16).split([heads * D, kvh * D, kvh * D], dim=-1)
    return q.view(n, heads, D), k.view(n, kvh, D), v.view(n, kvh, D)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "verify":
        return _prepare_verify(case, g)
    lens, kvh, block = _lengths(case), case["kvh"], case["block"]
    spread = 0.5 + 1.5 * torch.rand(D, generator=g, device="cuda") ** 4  # a few large key channels
    fp8 = kind != "shared" or case["fp8"]
    pages, table = _tables(g, lens, block, case.get("shared", 0))
    kc, ks = _cache(g, pages, block, kvh, fp8, spread)
    vc, vs = _cache(g, pages, block, kvh, fp8, torch.ones(D, device="cuda"))
    s = dict(kind=kind, block=block, kc=kc, vc=vc, ks=ks, vs=vs, table=table.cuda(), lens=_ints(lens),
             max_len=max(lens))
    if kind == "cache":
        new = [(i, p) for i, n in enumerate(lens) for p in range(n - case["new"], n)]
        _, s["k"], s["v"] = _qkv(g, len(new), kvh, kvh, spread)
        s["slots"] = _ints([int(table[i, p // block]) * block + p % block for i, p in new])
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s["cu"], s["total"] = _ints(cu), cu[-1]
        return s
    s["q"], s["k"], s["v"] = _qkv(g, len(lens), case["heads"], kvh, spread)
    s["q"] = (s["q"].float() * 1.5).to(torch.bfloat16)
    if kind == "decode":
        s["slots"] = _ints([int(table[i, (n - 1) // block]) * block + (n - 1) % block if n else -1
                            for i, n in enumerate(lens)])
    else:
        s["shared"] = case["shared"]
    return s


def _tree(case):
    """Parents of a draft tree whose nodes come after their parents, up to 4 children a node."""
    r, n = _fixed(case), case["nodes"]
    if case["form"] != "tree":
        return list(range(-1, n - 1))
    parents, kids = [-1], [0]
    for j in range(1, n):
        p = r.choice([c for c in range(max(0, j - 12), j) if kids[c] < 4] or [j - 1])
        kids[p] += 1
        kids.append(0)
        parents.append(p)
    return parents


def _prepare_verify(case, g):
    b, n, v = case["batch"], case["nodes"], case["vocab"]
    r = _fixed(case)
    parents = _tree(case)
    logits = 2.0 * torch.randn((b, n, v), generator=g, device="cuda")
    # a few likely tokens a row hold most of the mass, as after a trained model
    hot = torch.randint(0, v, (b, n, 12), generator=g, device="cuda")
    logits.scatter_add_(2, hot, 6 + 8 * torch.rand((b, n, 12), generator=g, device="cuda"))
    draft = logits + case["noise"] * torch.randn((b, n, v), generator=g, device="cuda")
    logits = logits.to(torch.bfloat16)
    temps = 0.6 + 0.5 * torch.rand(b, generator=g, device="cuda")
    temps[3::8] = 0.0  # greedy requests in the batch
    counts = [n if i % 5 or n < 3 else r.randint(1, n) for i in range(b)]  # some draft fewer
    u = torch.rand((b, max(0, n - 1)), generator=g, device="cuda")
    s = dict(kind="verify", logits=logits, temps=temps, u=u,
             pick=torch.rand(b, generator=g, device="cuda"), counts=_ints(counts), draft=None, parents=None)
    anc = [1]
    for j in range(1, n):
        anc.append(anc[parents[j]] | 1 << j)
    s["anc"] = torch.tensor([a - (1 << 64) if a >> 63 else a for a in anc], dtype=torch.int64).cuda()
    s["chain"] = case["form"] != "tree"
    if case["form"] == "draft":
        s["draft"] = draft[:, :n - 1].to(torch.bfloat16).contiguous()
        t = torch.where(temps > 0, temps, torch.full_like(temps, 1e-3))[:, None, None]
        e = torch.empty_like(draft[:, :n - 1]).exponential_(generator=g)
        s["tokens"] = (s["draft"].float() / t - e.log()).argmax(-1)
        return s
    ranks, seen = [], {}
    for p in parents[1:]:
        ranks.append(seen.get(p, 0))
        seen[p] = ranks[-1] + 1
    top = draft.topk(min(v, 4), dim=-1).indices  # children of a node: its likeliest tokens, in order
    if n > 1:
        s["tokens"] = top[:, torch.tensor(parents[1:]).cuda(), torch.tensor(ranks).cuda()].contiguous()
    else:
        s["tokens"] = torch.empty((b, 0), dtype=torch.int64, device="cuda")
    if case["form"] == "tree":
        s["parents"] = _ints(parents).expand(b, n)
    return s


# --------------------------------------------------------------------------- run

def run(s):
    kind = s["kind"]
    if own:
        return _own(s)
    if kind == "cache":
        _store(s)
        return _read_back(s)
    if kind == "decode":
        _store(s)
        return _attend(s)
    if kind == "shared":
        return _attend_shared(s)
    return _verify(s)


def _own(s):
    ops = _ops()
    kind = s["kind"]
    if kind == "cache":
        ops.store_kvcache_fp8(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
        return ops.load_kvcache_fp8(s["kc"], s["vc"], s["ks"], s["vs"], s["cu"], s["table"], s["total"])
    if kind == "decode":
        ops.store_kvcache_fp8(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
        return ops.paged_decode_fp8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["lens"], s["table"],
                                    softmax_scale=SCALE)
    if kind == "shared":
        return ops.shared_prefix_decode(s["q"], s["kc"], s["vc"], s["lens"], s["table"], s["shared"],
                                        softmax_scale=SCALE, k_scale=s["ks"], v_scale=s["vs"])
    return ops.verify_draft(s["logits"], s["tokens"], s["u"], s["pick"], temperatures=s["temps"],
                            draft_logits=s["draft"], parents=s["parents"], num_nodes=s["counts"])


def _store(s):
    """Rows of new tokens into the fp8 pages; slot -1 (a padding row) is skipped."""
    block = s["block"]
    keep = s["slots"] >= 0
    # a skipped row goes to where its first kept neighbour goes: with that row's own values
    rows = torch.where(keep, torch.arange(keep.numel(), device="cuda"), keep.to(torch.int32).argmax())
    slots = s["slots"][rows].long()
    for x, cache, exps in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        q, e = _quantise(x[rows])
        cache.view(torch.uint8).view(-1, *cache.shape[2:])[slots] = q.view(torch.uint8)
        exps[slots // block, :, slots % block] = e


def _values(cache, exps, pages, at):
    """float32 rows of the keys at (pages, at): e4m3 times a power of two, or bf16."""
    if exps is None:
        return cache[pages, at].float()
    e = exps[pages, :, at].float() - 127.0
    return cache.view(torch.uint8)[pages, at].view(torch.float8_e4m3fn).float() * torch.exp2(e)[..., None]


def _read_back(s):
    pos = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(s["cu"].long(), pos, right=True) - 1
    pos = pos - s["cu"][seq]
    pages, at = s["table"][seq, pos // s["block"]].long(), pos % s["block"]
    return tuple(_values(c, e, pages, at).to(torch.bfloat16) for c, e in ((s["kc"], s["ks"]),
                                                                         (s["vc"], s["vs"])))


def _own_keys(s, start):
    """Keys from `start` on of every row, padded to the longest: (B, L, KVH, 128) K and V and the mask."""
    pos = torch.arange(start, max(s["max_len"], start + 1), device="cuda")
    ok = pos[None, :] < s["lens"][:, None]
    col = (pos // s["block"]).clamp_max(s["table"].shape[1] - 1)
    pages = s["table"][:, col].long().clamp_min(0)
    at = (pos % s["block"])[None, :].expand_as(pages)
    return _values(s["kc"], s["ks"], pages, at), _values(s["vc"], s["vs"], pages, at), ok


def _softmax(scores, ok):
    scores = torch.where(ok, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))  # a row without keys: zeros


def _attend(s):
    k, v, ok = _own_keys(s, 0)
    b, h, kvh = s["q"].shape[0], s["q"].shape[1], k.shape[2]
    q = s["q"].float().view(b, kvh, h // kvh, D)
    p = _softmax(torch.einsum("bkgd,blkd->bkgl", q, k) * SCALE, ok[:, None, None, :])
    return torch.einsum("bkgl,blkd->bkgd", p, v).reshape(b, h, D).to(torch.bfloat16)


def _attend_shared(s):
    shared, block = s["shared"], s["block"]
    pos = torch.arange(shared, device="cuda")
    pages = s["table"][0, pos // block].long()
    k0, v0 = (_values(c, e, pages, pos % block) for c, e in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
    k, v, ok = _own_keys(s, shared)
    b, h, kvh = s["q"].shape[0], s["q"].shape[1], k.shape[2]
    q = s["q"].float().view(b, kvh, h // kvh, D)
    scores = torch.cat([torch.einsum("bkgd,lkd->bkgl", q, k0), torch.einsum("bkgd,blkd->bkgl", q, k)], -1)
    ok = torch.cat([pos[None, :] < s["lens"][:, None], ok], -1)
    p = _softmax(scores * SCALE, ok[:, None, None, :])
    o = torch.einsum("bkgl,lkd->bkgd", p[..., :shared], v0) + torch.einsum("bkgl,blkd->bkgd", p[..., shared:], v)
    return o.reshape(b, h, D).to(torch.bfloat16)


def _probabilities(logits, t):
    x = logits.double()
    x = torch.exp((x - x.amax(-1, keepdim=True)) / t.double()[:, None, None])
    return x / x.sum(-1, keepdim=True)


def _first_max(x):
    col = torch.arange(x.shape[-1], device="cuda")
    return torch.where(x == x.amax(-1, keepdim=True), col, x.shape[-1]).amin(-1)


def _verify(s):
    """Sums and comparisons in 64 bits: the answers are tokens, and a draw or an acceptance may lie
    next to a border."""
    logits, tokens, n = s["logits"], s["tokens"], s["logits"].shape[1]
    b, v = logits.shape[0], logits.shape[2]
    node = torch.arange(n, device="cuda")
    greedy = (s["temps"] <= 0)[:, None]
    t = torch.where(s["temps"] > 0, s["temps"], torch.ones_like(s["temps"]))
    p, best = _probabilities(logits, t), _first_max(logits)
    parent = (node - 1).expand(b, n) if s["chain"] else s["parents"].long()
    tok = torch.cat([tokens.new_full((b, 1), -1), tokens], 1)
    u = torch.cat([s["u"].new_zeros((b, 1)), s["u"]], 1).double()
    exists = (node[None, :] < s["counts"][:, None]) & (node > 0)
    up = parent.clamp_min(0)
    row = torch.arange(b, device="cuda")[:, None]
    here = p[row, up, tok.clamp_min(0)]
    older = (parent[:, :, None] == parent[:, None, :]) & exists[:, None, :] & (node[None, :] < node[:, None])
    twin = (older & (tok[:, :, None] == tok[:, None, :])).any(-1)
    here = torch.where(twin | ~exists, torch.zeros_like(here), here)
    if s["draft"] is not None:
        q = _probabilities(s["draft"], t) if n > 1 else p[:, :0]
        against = torch.cat([here[:, :1], q[row, up[:, 1:], tokens]], 1)
    else:
        against = 1.0 - (older * here[:, None, :]).sum(-1)
    taken = (u * against < here) & (here > 0)
    taken = torch.where(greedy, tok == best[row, up], taken) & exists
    taken = taken & ~(older & taken[:, None, :]).any(-1)
    above = (s["anc"][:, None] >> node[None, :] & 1).bool() & (node > 0)[None, :]
    reached = ~(above[None] & ~taken[:, None, :]).any(-1)
    count = reached.sum(-1) - 1
    last = torch.where(reached, node, 0).amax(-1)
    w = p[row[:, 0], last]
    child = exists & (parent == last[:, None])
    if s["draft"] is not None:
        if n > 1:
            rest = (w - q[row[:, 0], last.clamp_max(n - 2)]).clamp_min(0.0)
            w_left = torch.where(child.any(-1, keepdim=True), rest, w)
        else:
            w_left = w
    else:
        w_left = torch.cat([w, w.new_zeros((b, 1))], 1).scatter(1, torch.where(child, tok, v), 0.0)[:, :v]
    w = torch.where(w_left.sum(-1, keepdim=True) > 0, w_left, w)
    c = w.cumsum(-1)
    drawn = (c <= s["pick"].double()[:, None] * c[:, -1:]).sum(-1).clamp_max(v - 1)
    drawn = torch.where(greedy[:, 0], best[row[:, 0], last], drawn)
    order = torch.where(reached, node, n).sort(-1).values
    path = torch.where(order < n, order, -1)
    after = torch.cat([path[:, 1:], path.new_full((b, 1), -1)], 1)
    out = torch.where(after >= 0, tok[row, after.clamp_min(0)], -1)
    out = torch.where(node[None, :] == count[:, None], drawn[:, None], out)
    return out, path.to(torch.int32), count.to(torch.int32)


# -------------------------------------------------------------------- 64-bit answers

def _e4m3(y):
    """Nearest e4m3 value, ties to even: 3 fraction bits, spacing 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def _stored(x):
    """What a row written to the fp8 cache stands for."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    k = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -80) / E4M3_MAX))
    k = k + (amax > E4M3_MAX * torch.exp2(k)).double() - (amax <= E4M3_MAX * torch.exp2(k - 1)).double()
    return _e4m3(x * torch.exp2(-k)) * torch.exp2(k)


def _pages64(s, which):
    """The cache as 64-bit values, block after block, with the step's new rows in place."""
    c, e = s[which + "c"], s[which + "s"]
    x = c.double()
    if e is not None:
        x = x * torch.exp2(e.double() - 127).transpose(1, 2)[..., None]
    x = x.reshape(-1, *c.shape[2:])
    if "slots" in s:
        keep = s["slots"] >= 0
        x[s["slots"][keep].long()] = _stored(s[which][keep])
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "verify":
        return _exact_verify(s)
    k, v = _pages64(s, "k"), _pages64(s, "v")
    lens, block, table = _lengths(case), s["block"], s["table"].long()
    rows = []
    for i, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        rows.append(table[i, pos // block] * block + pos % block)
    if s["kind"] == "cache":
        at = torch.cat(rows)
        return k[at], v[at]
    b, h, kvh = s["q"].shape[0], s["q"].shape[1], k.shape[1]
    o = torch.zeros((b, h, D), dtype=torch.float64, device="cuda")
    for i, at in enumerate(rows):
        if at.numel():
            q = s["q"][i].double().view(kvh, h // kvh, D)
            a = torch.softmax(q @ k[at].permute(1, 2, 0) * SCALE, -1)
            o[i] = (a @ v[at].transpose(0, 1)).reshape(h, D)
    return o


def _exact_verify(s):
    """The walk as it is defined, one sequence after another, on the host in 64 bits."""
    import numpy as np
    b, n, _ = s["logits"].shape
    tokens, u, pick = s["tokens"].tolist(), s["u"].tolist(), s["pick"].tolist()
    temps, counts = s["temps"].tolist(), s["counts"].tolist()
    out, paths, num = np.full((b, n), -1, np.int64), np.full((b, n), -1, np.int32), np.zeros(b, np.int32)

    def law(x, t):
        x = x.double().cpu().numpy()
        if t <= 0:
            return (np.arange(x.size) == int(np.argmax(x))).astype(np.float64)
        x = np.exp((x - x.max()) / t)
        return x / x.sum()

    for i in range(b):
        parents = list(range(-1, n - 1)) if s["parents"] is None else s["parents"][i].tolist()
        t, node, step = temps[i], 0, 0
        paths[i, 0] = 0
        while True:
            p = law(s["logits"][i, node], t)
            rest, left, found = p, 1.0, None
            for c in range(node + 1, counts[i]):
                if parents[c] != node:
                    continue
                x = tokens[i][c - 1]
                if s["draft"] is not None and t > 0:
                    q = law(s["draft"][i, node], t)
                    rest = np.maximum(p - q, 0.0)
                    ok = u[i][c - 1] * q[x] < p[x]
                else:
                    ok = u[i][c - 1] * left < rest[x] and rest[x] > 0
                    if not ok:
                        left -= rest[x]
                        rest = np.where(np.arange(p.size) == x, 0.0, rest)
                if ok:
                    found = c
                    break
            if found is None:
                break
            out[i, step] = tokens[i][found - 1]
            node, step = found, step + 1
            paths[i, step] = node
        w = rest if rest.sum() > 0 else p
        c = np.cumsum(w)
        out[i, step] = int(np.searchsorted(c, pick[i] * c[-1], side="right")) if t > 0 else int(np.argmax(p))
        num[i] = step
    return torch.from_numpy(out), torch.from_numpy(paths), torch.from_numpy(num)
