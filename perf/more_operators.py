"""More serving operators over the paged cache and their measured cases: attention for rows that share a prefix (a
common system prompt, or the drafted tokens of a sequence), attention over the blocks that a cheap score selects, and
the verification of drafted tokens.

``own`` false computes the operators in elementary torch operations; true calls the framework's."""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_GOLDEN = 0.6180339887498949


def _package():
    """epure's paged and sampling modules (the package's folder is not on the path of a plain script)."""
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "epure-runtime_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from epure import paged, sampling
    return paged, sampling


# -- cases ----------------------------------------------------------------------------------------------------

def listed():
    return [
        # attention for rows that share a prefix
        # four answers to one short prompt: latency
        dict(name="shared-4x1k", op="shared", groups=1, rows=4, low=1024, prefix=1024, own=64, kind="prompts", heads=16,
             kv_heads=8, head_dim=128, page_size=16, format="same", dtype="bf16"),
        # four drafted tokens and the one before them of each of 16 sequences, quantised cache
        dict(name="shared-drafts-16x4k-int8", op="shared", groups=16, rows=5, low=1, prefix=4096, own=5, kind="drafts",
             heads=32, kv_heads=8, head_dim=128, page_size=64, format="int8", dtype="bf16"),
        # a batch of conversations behind one system prompt and its documents
        dict(name="shared-64x8k", op="shared", groups=1, rows=64, low=8192, prefix=8192, own=512, kind="prompts", heads=32,
             kv_heads=8, head_dim=128, page_size=64, format="same", dtype="bf16"),
        # a few prefixes of ragged lengths with ragged numbers of rows, odd heads and pages
        dict(name="shared-ragged-f16", op="shared", groups=7, rows=13, low=1, prefix=2500, own=100, kind="prompts",
             heads=12, kv_heads=4, head_dim=80, page_size=24, format="same", dtype="f16"),
        # many samples of one long context, eight query heads a key head, 8-bit floats
        dict(name="shared-256x32k-fp8", op="shared", groups=1, rows=256, low=32768, prefix=32768, own=1024, kind="prompts",
             heads=64, kv_heads=8, head_dim=128, page_size=32, format="fp8", dtype="bf16"),
        # attention over selected blocks: bounds of the newest page, selection, attention
        # one sequence with a very long context
        dict(name="sparse-1x128k", op="sparse", seqs=1, low=131072, high=131072, new=1, heads=32, kv_heads=8,
             head_dim=128, page_size=64, count=64, sinks=1, recent=2, format="same", dtype="bf16"),
        # a batch of ordinary lengths over a quantised cache; some shorter than what is selected
        dict(name="sparse-16x16k-int8", op="sparse", seqs=16, low=1, high=16384, new=1, heads=32, kv_heads=8, head_dim=128,
             page_size=64, count=32, sinks=1, recent=2, format="int8", dtype="bf16"),
        # the first step behind eight long prompts: the bounds of all their pages
        dict(name="sparse-prompts8x8k-f16", op="sparse", seqs=8, low=8191, high=8191, new=8191, heads=12, kv_heads=4,
             head_dim=80, page_size=48, count=21, sinks=0, recent=1, format="same", dtype="f16"),
        # a full batch of long contexts, eight query heads a key head, small pages of 8-bit floats
        dict(name="sparse-64x32k-fp8", op="sparse", seqs=64, low=1, high=32768, new=1, heads=64, kv_heads=8, head_dim=128,
             page_size=32, count=64, sinks=2, recent=4, format="fp8", dtype="bf16"),
        # verification of drafted tokens
        # one sequence: latency
        dict(name="verify-1x4", op="verify", batch=1, drafts=4, vocab=151936, draft="model", dtype="f32"),
        # drafts without probabilities (looked up in the text so far), 16-bit probabilities, an odd vocabulary
        dict(name="verify-33x7-lookup-bf16", op="verify", batch=33, drafts=7, vocab=32001, draft="lookup", dtype="bf16"),
        # a full batch with a draft model
        dict(name="verify-64x4", op="verify", batch=64, drafts=4, vocab=128256, draft="model", dtype="f32"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw(rng):
    op = rng.choice(("shared", "shared", "sparse", "sparse", "verify"))
    heads, kv_heads, head_dim = rng.choice(((32, 8, 128), (16, 8, 128), (64, 8, 128), (8, 2, 64), (4, 4, 128), (12, 4, 80),
                                            (28, 4, 128), (16, 1, 64), (6, 2, 256)))
    if op == "verify":
        return dict(op=op, batch=_log_int(rng, 1, 64), drafts=rng.randint(0, 8),
                    vocab=rng.choice((_log_int(rng, 2, 128256), 32001, 128256, 151936)),
                    draft=rng.choice(("model", "model", "lookup")), dtype=rng.choice(("f32", "f32", "bf16", "f16")))
    base = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=head_dim, format=rng.choice(("same", "int8", "fp8")),
                dtype=rng.choice(("bf16", "bf16", "f16")))
    if op == "shared":
        groups, high, drafts = _log_int(rng, 1, 16), _log_int(rng, 1, 32768), rng.random() < 0.3
        rows = rng.randint(1, 9) if drafts else _log_int(rng, 1, 256 // groups)
        return dict(base, groups=groups, rows=rows, low=rng.randint(1, high), prefix=high,
                    own=rows if drafts else rng.choice((1, 13, 77, 1024)), kind="drafts" if drafts else "prompts",
                    page_size=rng.choice((1, 16, 24, 48, 64, 128)))
    seqs, high = _log_int(rng, 1, 64), _log_int(rng, 1, 131072)
    page_size = rng.choice((8, 16, 24, 32, 48, 64, 128))
    high = max(1, min(high, 2097152 // seqs, 4096 * page_size))
    sinks, recent = rng.randint(0, 2), rng.randint(1, 4)
    return dict(base, seqs=seqs, low=rng.randint(1, high), high=high, new=rng.choice((1, 1, 1, 5, 513)), page_size=page_size,
                count=sinks + recent + rng.choice((0, 1, 10, 28, 60)), sinks=sinks, recent=recent)


def draw(rng):
    """A case of the listed ranges: 1 to 256 rows in up to 16 groups with prefixes of 1 to 32,768 tokens, 1 to 64 sequences
    of 1 to 131,072 tokens of which 1 to 67 blocks are selected, 1 to 64 sequences with up to 8 drafted tokens."""
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        case = _draw(rng)
        cost = work(case)
        if all(cost[k] <= most[k] for k in most):
            return case


# -- what a user's program has in hand -------------------------------------------------------------------------

def _spread(low, high, count):
    """`count` whole numbers from low to high in a scattered order."""
    return [low + int(round(((i + 1) * _GOLDEN % 1.0) * (high - low))) for i in range(count)]


def _rows(case):
    """Of a shared case: rows and prefix of every group, and the new tokens of every row (0: an idle row)."""
    counts = _spread(1, case["rows"], case["groups"]) if case["groups"] > 1 and case["kind"] == "prompts" \
        else [case["rows"]] * case["groups"]
    prefix = _spread(case["low"], case["prefix"], case["groups"])
    if case["kind"] == "drafts":
        return counts, prefix, [i + 1 for n in counts for i in range(n)]
    return counts, prefix, _spread(0, case["own"], sum(counts))


def _table(need, shared, page_size, total, g):
    """Page tables of rows of `need` tokens each, pages in a random order, -1 behind the last one; a row's first `shared[i]`
    tokens lie in whole pages of row first[i] (shared: a list of (first, tokens))."""
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
    most = max(1, max(-(-n // page_size) for n in need))
    table, at = torch.full((len(need), most), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        first, tokens = shared[i]
        have = min(tokens // page_size, -(-n // page_size)) if first != i else 0
        table[i, :have] = table[first, :have]
        more = -(-n // page_size) - have
        table[i, have:have + more] = order[at:at + more]
        at += more
    return table.cuda()


def _quantise(x, fmt):
    """Rows of float32 values to codes and scales."""
    top, dt = (127.0, torch.int8) if fmt == "int8" else (448.0, torch.float8_e4m3fn)
    a = x.abs().amax(-1, keepdim=True)
    inv = torch.where(a > 0, torch.full_like(a, top) / a, torch.zeros_like(a))
    c = x * inv
    return (c.round() if fmt == "int8" else c).to(dt), (a * (1.0 / top)).squeeze(-1)


def _pool(case, pages, g):
    """Filled key and value pools [pages, kv_heads, page_size, head_dim] and their scales; a few channels are large."""
    shape = (pages, case["kv_heads"], case["page_size"], case["head_dim"])
    gain = 0.4 + 2.0 * torch.rand(case["head_dim"], generator=g, device="cuda") ** 4
    got = {}
    for name in ("k", "v"):
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16) * gain.to(torch.bfloat16)
        if case["format"] == "same":
            got[name], got[name + "_scale"] = x.to(_DTYPES[case["dtype"]]), None
        else:
            got[name], got[name + "_scale"] = _quantise(x.float(), case["format"])
    return got


def _values(s, name, page, slot=slice(None)):
    """float32 values of cached rows: `page` any index tensor; all heads and slots of each page, or one slot each."""
    x, scale = s[name], s[name + "_scale"]
    at = (page,) if isinstance(slot, slice) else (page, slice(None), slot)
    x = x.view(torch.int8)[at].view(x.dtype).float() if x.element_size() == 1 else x[at].float()
    return x if scale is None else x * scale[at][..., None]


def _prepare_shared(case, g, dt):
    counts, prefix, new = _rows(case)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    group = [i for i, n in enumerate(counts) for _ in range(n)]
    drafts = case["kind"] == "drafts"
    lengths = [prefix[i] + n if n or drafts else 0 for i, n in zip(group, new)]
    if drafts:                                              # every group is one sequence
        need = [p + n for p, n in zip(prefix, counts)]
        shared, seq = [(i, 0) for i in range(len(need))], torch.tensor(group, dtype=torch.int32, device="cuda")
    else:                                                   # every row is one; the whole pages of a prefix are shared
        first = [starts[i] for i in group]
        need = [prefix[i] if r == starts[i] else 0 for r, i in enumerate(group)]
        need = [max(n, m) for n, m in zip(need, lengths)]
        shared, seq = list(zip(first, (prefix[i] for i in group))), None
    ps = case["page_size"]
    total = 3 + sum(-(-n // ps) - (min(t // ps, -(-n // ps)) if f != i else 0) for i, (n, (f, t)) in
                    enumerate(zip(need, shared)))
    s = dict(case=case, table=_table(need, shared, ps, total, g), seq=seq, **_pool(case, total, g))
    if not drafts:                                          # a prefix that ends inside a page: its rest is copied
        part = [(r, i) for r, i in enumerate(group) if prefix[i] % ps and lengths[r] > 0 and r != starts[i]]
        if part:
            r, i = (torch.tensor(x, device="cuda") for x in zip(*part))
            p, f = torch.tensor(prefix, device="cuda")[i], torch.tensor(starts, device="cuda")[i]
            src, dst = s["table"][f, p // ps].long(), s["table"][r, p // ps].long()
            keep = torch.arange(ps, device="cuda")[None, :] < (p % ps)[:, None]
            for name in ("k", "v", "k_scale", "v_scale"):
                if s[name] is not None:
                    x = s[name].view(torch.int8) if s[name].element_size() == 1 else s[name]
                    mask = keep[:, None, :, None] if x.dim() == 4 else keep[:, None, :]
                    x[dst] = torch.where(mask, x[src], x[dst])
    s["q"] = torch.randn((len(group), case["heads"], case["head_dim"]), generator=g, device="cuda").to(dt) * 2
    s["lengths"] = torch.tensor(lengths, device="cuda")
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["prefix"] = torch.tensor(prefix, device="cuda")
    return s


def _prepare_sparse(case, g, dt):
    lengths, ps = _spread(case["low"], case["high"], case["seqs"]), case["page_size"]
    total = sum(-(-n // ps) for n in lengths) + 3
    s = dict(case=case, table=_table(lengths, [(i, 0) for i in range(len(lengths))], ps, total, g), **_pool(case, total, g))
    s["q"] = torch.randn((len(lengths), case["heads"], case["head_dim"]), generator=g, device="cuda").to(dt) * 2
    s["lengths"] = torch.tensor(lengths, device="cuda")
    s["first"] = (s["lengths"] - case["new"]).clamp_(min=0)
    kind = dt if case["format"] == "same" else torch.bfloat16
    s["bounds"] = torch.zeros(total, case["kv_heads"], 2, case["head_dim"], dtype=kind, device="cuda")
    _bound(s, torch.zeros_like(s["first"]), s["first"])     # what earlier steps left: all but the new tokens
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "shared":
        return _prepare_shared(case, g, dt)
    if case["op"] == "sparse":
        return _prepare_sparse(case, g, dt)
    B, K, V = case["batch"], case["drafts"], case["vocab"]
    z = torch.randn(B, K + 1, V, generator=g, device="cuda") * 2.5
    draft = torch.softmax(z[:, :K], -1)
    target = torch.softmax(z + 0.7 * torch.randn(B, K + 1, V, generator=g, device="cuda"), -1).to(dt)
    s = dict(case=case, target=target, draft=draft.to(dt) if case["draft"] == "model" else None)
    if case["draft"] == "lookup":                           # likely tokens of the target; a row has up to K of them
        draft = torch.softmax(target[:, :K].float().clamp_min(1e-30).log() * 2, -1)
    tok = torch.multinomial(draft.reshape(B * K, V).clamp_min(1e-30), 1, generator=g).view(B, K) if K else \
        torch.zeros(B, 0, dtype=torch.long, device="cuda")
    if case["draft"] == "lookup":
        have = torch.tensor(_spread(0, K, B), device="cuda")
        tok = tok.masked_fill(torch.arange(K, device="cuda") >= have[:, None], -1)
    s["tokens"], s["uniforms"] = tok, torch.rand(B, K + 1, generator=g, device="cuda")
    return s


# -- the operators in their plain form -------------------------------------------------------------------------

def _shared_plain(s):
    case, q = s["case"], s["q"].float()
    B, H, hd = q.shape
    KV, ps, dt = case["kv_heads"], case["page_size"], s["q"].dtype
    scale = 1.0 / math.sqrt(hd)
    counts = (s["starts"][1:] - s["starts"][:-1]).long()
    G, R = counts.shape[0], case["rows"]
    at = s["starts"][:-1, None].long() + torch.arange(R, device="cuda")                 # rows of a group, padded
    on = torch.arange(R, device="cuda") < counts[:, None]
    at = torch.where(on, at, s["starts"][:-1, None].long())
    seq = torch.arange(B, device="cuda") if s["seq"] is None else s["seq"].long()
    group = torch.repeat_interleave(torch.arange(G, device="cuda"), counts)
    # the prefix, once a group
    cols = torch.arange(-(-case["prefix"] // ps), device="cuda").clamp(max=s["table"].shape[1] - 1)
    page = s["table"][seq[s["starts"][:-1].long()]][:, cols].long().clamp(min=0)        # [G, pages]
    L = cols.shape[0] * ps
    t = torch.arange(L, device="cuda")
    there = t < s["prefix"][:, None]

    def prefix(name):
        x = _values(s, name, page).transpose(1, 2).reshape(G, KV, L, hd)
        return x.masked_fill(~there[:, None, :, None], 0.0)

    seen = there[:, None, :] & (t < s["lengths"][at][..., None])                        # [G, R, L]
    qg = q[at].view(G, R, KV, H // KV, hd).transpose(1, 2).reshape(G, KV, R * (H // KV), hd)
    a = (qg @ prefix("k").transpose(-1, -2)).mul_(scale).view(G, KV, R, H // KV, L)
    a = a.masked_fill_(~seen[:, None, :, None, :], -math.inf).view(G, KV, R * (H // KV), L)
    # each row's own tokens: positions prefix .. length - 1 (the padding rows repeat a group's first)
    n = case["own"]
    mine = s["prefix"][:, None, None] + torch.arange(n, device="cuda")                  # [G, 1, n]
    mine = mine.expand(G, R, n)
    seen = mine < s["lengths"][at][..., None]
    col = torch.where(seen, mine // ps, 0)
    page2 = s["table"][seq[at][..., None], col].long().clamp(min=0)

    def owned(name):                                                                    # [G, KV, R, n, hd]
        x = _values(s, name, page2, mine % ps).permute(0, 3, 1, 2, 4)
        return x.masked_fill(~seen[:, None, :, :, None], 0.0)

    b = qg.view(G, KV, R, H // KV, hd) @ owned("k").transpose(-1, -2) * scale
    b = b.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = torch.maximum(a.amax(-1), b.amax(-1).flatten(2, 3)) if n else a.amax(-1)
    low = top.clamp(min=-3e38)[..., None]
    pa, pb = a.sub_(low).exp_(), torch.exp(b - low.view(G, KV, R, H // KV, 1))
    total = pa.sum(-1) + pb.sum(-1).flatten(2, 3)
    out = pa @ prefix("v") + (pb @ owned("v")).flatten(2, 3)
    out = out / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    out = out.view(G, KV, R, H // KV, hd).transpose(1, 2).reshape(G, R, H, hd)[on]
    lse = (top + torch.log(total)).view(G, KV, R, H // KV).transpose(1, 2).reshape(G, R, H)[on]
    return [out.to(dt), lse]


def _bound(s, first, lengths):
    """Bounds of the pages that hold tokens [first, lengths) of each sequence, over all their tokens below lengths."""
    ps = s["case"]["page_size"]
    cols = torch.arange(s["table"].shape[1], device="cuda")
    b, col = ((cols >= first[:, None] // ps) & (cols * ps < lengths[:, None]) & (first < lengths)[:, None]).nonzero().T
    page = s["table"][b, col].long()
    there = (col[:, None] * ps + torch.arange(ps, device="cuda") < lengths[b][:, None])[:, None, :, None]
    x = _values(s, "k", page)
    low = torch.where(there, x, torch.full_like(x[:1, :1, :1, :1], math.inf)).amin(2)
    high = torch.where(there, x, torch.full_like(x[:1, :1, :1, :1], -math.inf)).amax(2)
    s["bounds"][page] = torch.stack((low, high), 2).to(s["bounds"].dtype)


def _pairs(x):
    """Sums over the last dimension: neighbours first, then neighbours of those sums, each rounded to float32."""
    x = torch.nn.functional.pad(x, (0, (1 << (x.shape[-1] - 1).bit_length()) - x.shape[-1]))
    while x.shape[-1] > 1:
        x = x[..., 0::2] + x[..., 1::2]
    return x[..., 0]


def _choose(score, n, case):
    """[batch, kv_heads, count] int32: the first sinks and last recent of each row's n blocks and the best of the others, in
    ascending order, -1 behind the last; score [batch, kv_heads, blocks]."""
    j = torch.arange(score.shape[-1], device="cuda")
    n = n[:, None, None]
    key = score.masked_fill((j < case["sinks"]) | (j >= n - case["recent"]), math.inf).masked_fill(j >= n, -math.inf)
    # forced blocks come first of equal scores (a score can be infinite itself), then the lowest block
    forced = ((j < case["sinks"]) | (j >= n - case["recent"])) & (j < n)
    count = min(case["count"], score.shape[-1])
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    order = order.gather(-1, torch.argsort((~forced).expand_as(score).gather(-1, order).int(), dim=-1, stable=True))
    got = order[..., :count]
    got = got.masked_fill(got >= n, score.shape[-1]).sort(-1)[0]
    got = got.masked_fill(got == score.shape[-1], -1)
    return torch.nn.functional.pad(got, (0, case["count"] - count), value=-1).int()


def _sparse_plain(s):
    case, q = s["case"], s["q"].float()
    B, H, hd = q.shape
    KV, ps = case["kv_heads"], case["page_size"]
    _bound(s, s["first"], s["lengths"])
    page = s["table"].long().clamp(min=0)                                               # [B, blocks]
    bounds = s["bounds"].float()[page].transpose(1, 2)[:, :, None]                      # [B, KV, 1, blocks, 2, hd]
    qg = q.view(B, KV, H // KV, 1, hd)
    score = _pairs(torch.maximum(qg * bounds[..., 0, :], qg * bounds[..., 1, :])).amax(2)
    chosen = _choose(score, -(-s["lengths"] // ps), case)
    # attention over the chosen blocks
    col = chosen.long().clamp(min=0)
    at = page[torch.arange(B, device="cuda")[:, None, None], col]                       # [B, KV, count]
    head = torch.arange(KV, device="cuda")[None, :, None]
    seen = (chosen >= 0)[..., None] & (col[..., None] * ps + torch.arange(ps, device="cuda") < s["lengths"][:, None, None, None])

    def dense(name):                                                                    # [B, KV, count * ps, hd]
        x, scale = s[name], s[name + "_scale"]
        x = x.view(torch.int8)[at, head].view(x.dtype).float() if x.element_size() == 1 else x[at, head].float()
        x = x if scale is None else x * scale[at, head][..., None]
        return x.masked_fill(~seen[..., None], 0.0).flatten(2, 3)

    z = q.view(B, KV, H // KV, hd) @ dense("k").transpose(-1, -2) * (1.0 / math.sqrt(hd))
    z = z.masked_fill(~seen.flatten(2)[:, :, None, :], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - top.clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    out = (p @ dense("v")) / torch.where(total > 0, total, torch.ones_like(total))
    return [s["bounds"], chosen, out.reshape(B, H, hd).to(s["q"].dtype), (top + torch.log(total)).view(B, H)]


def _verify_plain(s):
    p, q, x, u = s["target"], s["draft"], s["tokens"], s["uniforms"].double()
    B, K = x.shape
    V = p.shape[-1]
    every = torch.arange(B, device="cuda")
    have = (x >= 0).int().cumprod(-1).sum(-1)                                           # drafts of a row
    at = x.clamp(min=0)[..., None]
    px = p[:, :K].gather(-1, at)[..., 0].double()
    qx = torch.ones_like(px) if q is None else q.gather(-1, at)[..., 0].double()
    ok = (u[:, :K] * qx < px) & (x >= 0)
    n = ok.int().cumprod(-1).sum(-1)                                                    # accepted
    row = p[every, n].double()
    less = torch.zeros_like(row)
    if K:
        i = n.clamp(max=K - 1)
        less = torch.nn.functional.one_hot(at[every, i, 0], V).double() if q is None else q[every, i].double()
        if q is None:                                                                   # all of a drafted token's weight
            less = less * math.inf
            less = torch.where(less.isnan(), 0.0, less)
        less = torch.where((n < have)[:, None], less, torch.zeros_like(less))
    rest = (row - less).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, row)
    c = rest.cumsum(-1)
    hit = (c > u[:, K:] * c[:, -1:]) & (rest > 0)
    last = (V - 1) - (rest > 0).flip(-1).int().argmax(-1)
    token = torch.where(hit.any(-1), hit.int().argmax(-1), last)
    j = torch.arange(K + 1, device="cuda")
    out = torch.where(j < n[:, None], torch.nn.functional.pad(x, (0, 1)), -1)
    return [torch.where(j == n[:, None], token[:, None], out), n.long()]


# -- one pass ---------------------------------------------------------------------------------------------------

def run(state):
    s, case = state, state["case"]
    if not own:
        return {"shared": _shared_plain, "sparse": _sparse_plain, "verify": _verify_plain}[case["op"]](s)
    paged, sampling = _package()
    if case["op"] == "verify":
        return list(sampling.verify(s["target"], s["draft"], s["tokens"], s["uniforms"]))
    pages = paged.KVPages(s["k"], s["v"], s["table"], s["k_scale"], s["v_scale"])
    if case["op"] == "shared":
        return list(paged.attend_shared(pages, s["q"], s["lengths"], s["starts"], s["prefix"], seq=s["seq"],
                                        return_lse=True))
    paged.summarise(pages, s["bounds"], s["lengths"], first=s["first"])
    chosen = paged.select(pages, s["bounds"], s["q"], s["lengths"], case["count"], sinks=case["sinks"],
                          recent=case["recent"])
    out, lse = paged.attend(pages, s["q"], s["lengths"], blocks=chosen, return_lse=True)
    return [s["bounds"], chosen, out, lse]


def work(case):
    """Bytes that the pass has to read and write once, and its operations."""
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "verify":
        B, K, V = case["batch"], case["drafts"], case["vocab"]
        rows = 2 if case["draft"] == "model" and K else 1   # of the target and the draft, at the first refusal
        return {"bytes": B * rows * V * e + B * (K * (8 + 2 * e) + (K + 1) * 12 + 8), "flops": B * 3 * V}
    H, KV, hd, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    c, extra = (e, 0) if case["format"] == "same" else (1, 4)
    row = 2 * KV * (hd * c + extra)                         # one cached token: key, value and their scales
    if case["op"] == "shared":
        counts, prefix, new = _rows(case)
        group = [i for i, n in enumerate(counts) for _ in range(n)]
        drafts = case["kind"] == "drafts"
        read = sum(prefix) + (sum(counts) if drafts else sum(new))
        seen = sum(prefix[i] + n for i, n in zip(group, new) if n or drafts)
        B = len(group)
        return {"bytes": read * row + 2 * B * H * hd * e + B * H * 4 + -(-read // ps) * 4 + B * 8, "flops": 4 * seen * H * hd}
    lengths, B = _spread(case["low"], case["high"], case["seqs"]), case["seqs"]
    blocks = [-(-n // ps) for n in lengths]
    new = [b - max(0, n - case["new"]) // ps for b, n in zip(blocks, lengths)]
    half = 2 * KV * hd * 2                                  # the bounds of one page
    tokens = sum(min(case["count"] * ps, n) for n in lengths)
    moved = sum(new) * (ps * row // 2 + half) + sum(blocks) * (half + 4) + tokens * row
    return {"bytes": moved + 2 * B * H * hd * e + B * H * 4 + B * KV * case["count"] * 4 + B * 16,
            "flops": 4 * tokens * H * hd + sum(blocks) * 4 * H * hd + sum(new) * ps * KV * hd * 2}


# -- the definition in 64 bits ----------------------------------------------------------------------------------

def _exact_rows(s, name, page, head, slot):
    """Cached rows of one head as 64-bit values."""
    x = s[name]
    x = x.view(torch.int8)[page, head, slot].view(x.dtype).double() if x.element_size() == 1 else x[page, head, slot].double()
    return x if s[name + "_scale"] is None else x * s[name + "_scale"][page, head, slot].double()[..., None]


def _exact_attention(s, seq, at, head, queries):
    """(sum, log-sum-exp) of query rows [n, hd] over tokens `at` of one sequence's head."""
    ps = s["case"]["page_size"]
    page = s["table"][seq, at // ps].long()
    z = queries.double() @ _exact_rows(s, "k", page, head, at % ps).T / math.sqrt(queries.shape[-1])
    return torch.softmax(z, -1) @ _exact_rows(s, "v", page, head, at % ps), torch.logsumexp(z, -1)


def _exact_shared(s):
    """Every row by itself, over its own page table."""
    case = s["case"]
    B, H, hd = s["q"].shape
    g = H // case["kv_heads"]
    out = torch.zeros(B, H, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        if n:
            seq = b if s["seq"] is None else int(s["seq"][b])
            for h in range(case["kv_heads"]):
                hs = slice(h * g, h * g + g)
                out[b, hs], lse[b, hs] = _exact_attention(s, seq, torch.arange(n, device="cuda"), h, s["q"][b, hs])
    return [out, lse]


def _exact_halves(x):
    """The float32 sum of neighbours, then of neighbours' sums: the order that the score is defined by."""
    if len(x) == 1:
        return x[0]
    return _exact_halves([x[i] + x[i + 1] if i + 1 < len(x) else x[i] + 0.0 for i in range(0, len(x), 2)])


def _exact_sparse(s):
    """Blocks one by one; what is chosen follows from the bounds as they are held and from sums of 32 bits, as defined."""
    case = s["case"]
    B, H, hd = s["q"].shape
    KV, ps = case["kv_heads"], case["page_size"]
    g = H // KV
    bounds, held = s["bounds"].double(), s["bounds"].clone()
    out = torch.zeros(B, H, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    chosen = torch.full((B, KV, case["count"]), -1, dtype=torch.int32, device="cuda")
    heads = torch.arange(KV, device="cuda")[:, None]
    for b, (n, first) in enumerate(zip(s["lengths"].tolist(), s["first"].tolist())):
        blocks = -(-n // ps)
        for j in range(first // ps, blocks):
            page, slot = int(s["table"][b, j]), torch.arange(min(ps, n - j * ps), device="cuda")
            x = _exact_rows(s, "k", page, heads, slot)
            bounds[page, :, 0], bounds[page, :, 1] = x.amin(1), x.amax(1)
            held[page] = bounds[page].float().to(held.dtype)
        edge = held[s["table"][b, :blocks].long()].float()
        for h in range(KV):
            score = []
            for i in range(h * g, h * g + g):
                t = torch.maximum(s["q"][b, i].float() * edge[:, h, 0], s["q"][b, i].float() * edge[:, h, 1])
                score.append(_exact_halves(list(t.unbind(-1))))
            score = torch.stack(score).amax(0).tolist()
            forced = set(range(min(case["sinks"], blocks))) | set(range(max(0, blocks - case["recent"]), blocks))
            rest = sorted((j for j in range(blocks) if j not in forced), key=lambda j: (-score[j], j))
            got = sorted(list(forced) + rest[:max(0, case["count"] - len(forced))])
            chosen[b, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
            at = torch.cat([torch.arange(j * ps, min(n, j * ps + ps)) for j in got]).cuda()
            hs = slice(h * g, h * g + g)
            out[b, hs], lse[b, hs] = _exact_attention(s, b, at, h, s["q"][b, hs])
    return [bounds, chosen, out, lse]


def _exact_verify(s):
    """Row by row, the cumulative weights in numpy's 64 bits."""
    p, x, u = s["target"], s["tokens"].tolist(), s["uniforms"].double().tolist()
    B, K = s["tokens"].shape
    out, count = [], []
    for b in range(B):
        n = 0
        while n < K and x[b][n] >= 0:
            q = 1.0 if s["draft"] is None else float(s["draft"][b, n, x[b][n]])
            if not u[b][n] * q < float(p[b, n, x[b][n]]):
                break
            n += 1
        w = p[b, n].cpu().double()
        if n < K and x[b][n] >= 0:
            less = w.clone()
            if s["draft"] is None:
                less[x[b][n]] = 0.0
            else:
                less = torch.relu(w - s["draft"][b, n].cpu().double())
            w = less if bool((less > 0).any()) else w
        c = torch.cumsum(w, 0)
        above = torch.nonzero((c > u[b][K] * float(c[-1])) & (w > 0))
        token = int(above[0]) if len(above) else int(torch.nonzero(w > 0)[-1])
        out.append(x[b][:n] + [token] + [-1] * (K - n))
        count.append(n)
    return [torch.tensor(out), torch.tensor(count)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verify(s)
    if case["op"] == "sparse":
        if case["seqs"] * case["kv_heads"] > 256 or work(case)["bytes"] > 1e9:
            return None                                     # too long block by block
        return _exact_sparse(s)
    return _exact_shared(s)


if __name__ == "__main__":
    for c in listed():
        print(c["name"], work(c))
    print(draw(random.Random(0)))
