"""The serving operators and their measured cases: rotary positions (with their gradient), the paged key-value
cache that is quantised as it is written and read back, and the attention of one new token a sequence over it.

``own`` false computes the operators in elementary torch operations in 32 bits; true calls the framework's."""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_GOLDEN = 0.6180339887498949


def _package():
    """epure's paged and rotary modules (the package's folder is not on the path of a plain script)."""
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "epure-runtime_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from epure import paged, rotary
    return paged, rotary


# -- cases ----------------------------------------------------------------------------------------------------

def listed():
    return [
        # rotary positions
        # the q and k of one decode step of 16 sequences deep in a long context
        dict(name="rope-step16", op="rope", tokens=16, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, dtype="bf16", scaling="bands", max_len=131072, train=False),
        # q and k of one layer of the fine-tune step (8 x 2048 tokens), forward and gradient
        dict(name="rope-train16k", op="rope", tokens=16384, heads=16, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, dtype="bf16", scaling="none", max_len=2048, train=True),
        # interleaved pairs over part of an odd-sized head, in float32, a ragged number of tokens
        dict(name="rope-part-f32", op="rope", tokens=5003, heads=12, kv_heads=4, head_dim=80, rotary_dim=32,
             interleaved=True, dtype="f32", scaling="yarn", max_len=32768, train=True),
        # the cache: rows rotated, quantised and written, and read back
        # one decode step of 16 sequences: 16 rows of q, k and v
        dict(name="write-step16-int8", op="write", seqs=16, new=1, past=2047, heads=32, kv_heads=8, head_dim=128,
             page_size=64, format="int8", dtype="bf16", rope=True, qk_norm=False, whole=False),
        # the prompt of one sequence with per-head norms of q and k
        dict(name="write-prompt2k-fp8", op="write", seqs=1, new=2048, past=0, heads=16, kv_heads=8, head_dim=128,
             page_size=16, format="fp8", dtype="bf16", rope=True, qk_norm=True, whole=False),
        # a prompt's next chunk: ragged rows behind a cached prefix, all of it read back for the chunk's attention
        dict(name="write-chunk-f16", op="write", seqs=4, new=509, past=1531, heads=0, kv_heads=2, head_dim=64,
             page_size=48, format="int8", dtype="f16", rope=False, qk_norm=False, whole=True),
        # eight long prompts at once
        dict(name="write-prompts64k-int8", op="write", seqs=8, new=8192, past=0, heads=32, kv_heads=8, head_dim=128,
             page_size=64, format="int8", dtype="bf16", rope=True, qk_norm=False, whole=False),
        # attention of one new token a sequence
        # a single sequence just after a short prompt: latency
        dict(name="attend-1x145", op="attend", seqs=1, low=145, high=145, empty=0, heads=32, kv_heads=8,
             head_dim=128, page_size=16, format="same", dtype="bf16", window=0),
        # a batch of ordinary lengths, quantised cache
        dict(name="attend-16x4k-int8", op="attend", seqs=16, low=1, high=4096, empty=0, heads=32, kv_heads=8,
             head_dim=128, page_size=64, format="int8", dtype="bf16", window=0),
        # one sequence with a very long context
        dict(name="attend-1x128k", op="attend", seqs=1, low=131072, high=131072, empty=0, heads=32, kv_heads=8,
             head_dim=128, page_size=64, format="same", dtype="bf16", window=0),
        # a full batch of ragged lengths, eight query heads a key head, 8-bit floats
        dict(name="attend-64x8k-fp8", op="attend", seqs=64, low=1, high=8192, empty=0, heads=64, kv_heads=8,
             head_dim=128, page_size=32, format="fp8", dtype="bf16", window=0),
        # small heads, a sliding window, slots without a sequence
        dict(name="attend-33x1k-window", op="attend", seqs=33, low=1, high=1000, empty=3, heads=8, kv_heads=2,
             head_dim=64, page_size=48, format="same", dtype="f16", window=300),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw(rng):
    op = rng.choice(("rope", "write", "attend", "attend"))
    heads, kv_heads, head_dim = rng.choice(((32, 8, 128), (16, 8, 128), (64, 8, 128), (8, 2, 64), (4, 4, 128),
                                            (12, 4, 80), (28, 4, 128), (16, 1, 64), (6, 2, 256)))
    if op == "rope":
        return dict(op=op, tokens=_log_int(rng, 1, 16384), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rng.choice((head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2))),
                    interleaved=rng.random() < 0.5, dtype=rng.choice(("bf16", "bf16", "f16", "f32")),
                    scaling=rng.choice(("none", "linear", "ntk", "bands", "yarn")),
                    max_len=rng.choice((2048, 32768, 131072)), train=rng.random() < 0.5)
    if op == "write":
        seqs = _log_int(rng, 1, 16)
        return dict(op=op, seqs=seqs, new=_log_int(rng, 1, 65536 // seqs // 8), past=rng.choice((0, 1, 777, 2000)),
                    heads=rng.choice((0, heads)), kv_heads=kv_heads, head_dim=head_dim,
                    page_size=rng.choice((1, 16, 24, 48, 64, 128)), format=rng.choice(("same", "int8", "fp8")),
                    dtype=rng.choice(("bf16", "bf16", "f16")), rope=rng.random() < 0.7, qk_norm=rng.random() < 0.3,
                    whole=rng.random() < 0.5)
    seqs, high = _log_int(rng, 1, 64), _log_int(rng, 1, 65536)
    high = max(1, min(high, 262144 // seqs))
    return dict(op=op, seqs=seqs, low=rng.randint(1, high), high=high, empty=rng.choice((0, 0, 5)), heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page_size=rng.choice((1, 16, 24, 48, 64, 128)),
                format=rng.choice(("same", "int8", "fp8")), dtype=rng.choice(("bf16", "bf16", "f16")),
                window=rng.choice((0, 0, 0, 1, 777)))


def draw(rng):
    """A case of the listed ranges: 1 to 16,384 rotated tokens, 1 to 8,192 rows written a sequence, caches of 1 to
    64 sequences and 1 to 65,536 tokens each."""
    most = max(work(c)["bytes"] for c in listed())
    while True:
        case = _draw(rng)
        if work(case)["bytes"] <= most:
            return case


# -- what a user's program has in hand -------------------------------------------------------------------------

def _lengths(case):
    """Cached tokens of every sequence of an attention case: spread from low to high; every `empty`-th slot is free."""
    span = case["high"] - case["low"]
    got = [case["low"] + int(round(((i + 1) * _GOLDEN % 1.0) * span)) for i in range(case["seqs"])]
    return [0 if case["empty"] and i % case["empty"] == case["empty"] - 1 else n for i, n in enumerate(got)]


def _tables(rotary_dim, max_len, scaling, device):
    """Float32 cos and sin [max_len, rotary_dim / 2], angles in 64 bits."""
    theta, factor, original = 5.0e5, 8.0, 8192
    j = torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64)
    if scaling == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    f, gain = theta ** (-j / rotary_dim), 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":        # long wavelengths divided by the factor, short ones kept, a ramp between them
        turns = original * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / factor
    elif scaling == "yarn":         # the same by the index of the pair, and a gain on both tables
        at = [rotary_dim * math.log(original / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
        ramp = ((j / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = (1 - ramp) * f + ramp * f / factor
        gain = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(max_len, device=device, dtype=torch.float64)[:, None] * f
    return (gain * angle.cos()).float(), (gain * angle.sin()).float()


def _pages(case, lengths, extra, g):
    """An allocated pool's page table [seqs, most pages]: pages in a random order, -1 behind the last one."""
    ps = case["page_size"]
    need = torch.tensor([-(-n // ps) for n in lengths])
    most, total = max(1, int(need.max())), int(need.sum()) + extra
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(most)[None, :] < need[:, None]
    table = torch.full((len(lengths), most), -1, dtype=torch.int32, device="cuda")
    table[at.cuda()] = order[: int(need.sum())]
    return table, total


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


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    H, KV, hd = case["heads"], case["kv_heads"], case["head_dim"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    if case["op"] == "rope":
        T = case["tokens"]
        qkv = randn(T, H + 2 * KV, hd)                      # one projection's rows: q and k are views of it
        cos, sin = _tables(case["rotary_dim"], case["max_len"], case["scaling"], "cuda")
        pos = torch.randint(0, case["max_len"], (T,), generator=g, device="cuda")
        if T > 256:                                         # whole sequences; a decode step has one token of each
            pos = torch.arange(T, device="cuda") % case["max_len"]
        return dict(case=case, q=qkv[:, :H], k=qkv[:, H:H + KV], pos=pos, cos=cos, sin=sin,
                    dq=randn(T, H, hd) if case["train"] else None, dk=randn(T, KV, hd) if case["train"] else None)
    if case["op"] == "write":
        n, past = case["new"], case["past"]
        table, pages = _pages(case, [past + n] * case["seqs"], 3, g)
        s = dict(case=case, table=table, **_pool(case, pages, g))
        qkv = randn(case["seqs"] * n, H + 2 * KV, hd) * (0.4 + 2.0 * torch.rand(hd, generator=g, device="cuda") ** 4
                                                       ).to(dt)
        s.update(q=qkv[:, :H] if H else None, k_new=qkv[:, H:H + KV], v_new=qkv[:, H + KV:])
        seq = torch.arange(case["seqs"], device="cuda", dtype=torch.int32)
        s["seq"] = seq.repeat_interleave(n)
        s["pos"] = torch.arange(past, past + n, device="cuda").repeat(case["seqs"])
        first = 0 if case["whole"] else past                # the rows that are read back
        s["read_seq"] = seq.repeat_interleave(past + n - first)
        s["read_pos"] = torch.arange(first, past + n, device="cuda").repeat(case["seqs"])
        s["cos"], s["sin"] = _tables(hd, past + n, "none", "cuda") if case["rope"] else (None, None)
        return s
    lengths = _lengths(case)
    table, pages = _pages(case, lengths, 3, g)
    s = dict(case=case, table=table, **_pool(case, pages, g))
    s["q"] = randn(case["seqs"], H, hd) * 2
    s["lengths"] = torch.tensor(lengths, device="cuda")
    return s


# -- the operators in their plain form -------------------------------------------------------------------------

def _rotate(x, pos, cos, sin, interleaved):
    """x [T, heads, head_dim] in float32."""
    r = 2 * cos.shape[1]
    c, s = cos[pos][:, None, :], sin[pos][:, None, :]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    ya, yb = a * c - b * s, b * c + a * s
    y = torch.stack((ya, yb), -1).flatten(-2) if interleaved else torch.cat((ya, yb), -1)
    return torch.cat((y, x[..., r:]), -1)


def _norm(x, dt):
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(dt).float()


def _rope_plain(s):
    dt, flip = s["q"].dtype, s["case"]["interleaved"]
    out = [_rotate(s[n].float(), s["pos"], s["cos"], s["sin"], flip).to(dt) for n in ("q", "k")]
    if s["case"]["train"]:
        out += [_rotate(s[n].float(), s["pos"], s["cos"], -s["sin"], flip).to(dt) for n in ("dq", "dk")]
    return out


def _write_plain(s):
    case, dt = s["case"], s["k_new"].dtype
    ps, fmt = case["page_size"], case["format"]
    q, k, v = s["q"], s["k_new"].float(), s["v_new"].float()
    q = None if q is None else q.float()
    if case["qk_norm"]:
        q, k = None if q is None else _norm(q, dt), _norm(k, dt)
    if case["rope"]:
        q = None if q is None else _rotate(q, s["pos"], s["cos"], s["sin"], False)
        k = _rotate(k, s["pos"], s["cos"], s["sin"], False).to(dt).float()
    page, slot = s["table"][s["seq"].long(), s["pos"] // ps].long(), s["pos"] % ps
    rpage, rslot = s["table"][s["read_seq"].long(), s["read_pos"] // ps].long(), s["read_pos"] % ps
    if fmt == "same":
        s["k"][page, :, slot], s["v"][page, :, slot] = k.to(dt), v.to(dt)
        rk, rv = s["k"][rpage, :, rslot], s["v"][rpage, :, rslot]
    else:
        raw = torch.int8                                    # 8-bit floats are moved as bytes
        (ck, sk), (cv, sv) = _quantise(k, fmt), _quantise(v, fmt)
        s["k"].view(raw)[page, :, slot], s["v"].view(raw)[page, :, slot] = ck.view(raw), cv.view(raw)
        s["k_scale"][page, :, slot], s["v_scale"][page, :, slot] = sk, sv
        kind = s["k"].dtype
        rk = (s["k"].view(raw)[rpage, :, rslot].view(kind).float() * s["k_scale"][rpage, :, rslot][..., None]).to(dt)
        rv = (s["v"].view(raw)[rpage, :, rslot].view(kind).float() * s["v_scale"][rpage, :, rslot][..., None]).to(dt)
    return [rk, rv] if q is None else [q.to(dt), rk, rv]


def _attend_plain(s):
    case, q = s["case"], s["q"].float()
    B, H, hd = q.shape
    KV, ps, most = case["kv_heads"], case["page_size"], s["table"].shape[1]
    raw = s["table"].long().clamp(min=0)
    t = torch.arange(most * ps, device="cuda")
    n = s["lengths"][:, None]
    seen = t < n
    if case["window"]:
        seen = seen & (t >= n - case["window"])

    def dense(name):                                        # [B, KV, tokens, hd] in float32, zero where not seen
        x = s[name].view(torch.int8)[raw].view(s[name].dtype).float() if s[name].element_size() == 1 \
            else s[name][raw].float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][raw][..., None]
        x = x.transpose(1, 2).reshape(B, KV, most * ps, hd)
        return x.masked_fill(~seen[:, None, :, None], 0.0)

    score = (q.view(B, KV, H // KV, hd) @ dense("k").transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    out = (p @ dense("v")) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total)).view(B, H)
    return [out.reshape(B, H, hd).to(s["q"].dtype), lse]


# -- one pass ---------------------------------------------------------------------------------------------------

def run(state):
    s, case = state, state["case"]
    if not own:
        return {"rope": _rope_plain, "write": _write_plain, "attend": _attend_plain}[case["op"]](s)
    paged, rotary = _package()
    if case["op"] == "rope":
        out = list(rotary.rope(s["q"], s["k"], s["pos"], s["cos"], s["sin"], interleaved=case["interleaved"]))
        if case["train"]:
            out += rotary.rope(s["dq"], s["dk"], s["pos"], s["cos"], s["sin"], interleaved=case["interleaved"],
                               inverse=True)
        return out
    pages = paged.KVPages(s["k"], s["v"], s["table"], s["k_scale"], s["v_scale"])
    if case["op"] == "write":
        q = paged.write(pages, s["k_new"], s["v_new"], s["seq"], s["pos"], q=s["q"], cos=s["cos"], sin=s["sin"],
                        qk_norm=case["qk_norm"], eps=1e-6)
        k, v = paged.read(pages, s["read_seq"], s["read_pos"], dtype=s["k_new"].dtype)
        return [k, v] if q is None else [q, k, v]
    return list(paged.attend(pages, s["q"], s["lengths"], window=case["window"], return_lse=True))


def work(case):
    """Bytes that the pass has to read and write once, and its operations."""
    e = 4 if case["dtype"] == "f32" else 2
    H, KV, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        T, r = case["tokens"], case["rotary_dim"]
        times = 2 if case["train"] else 1
        table = min(T, case["max_len"]) * r * 4
        return {"bytes": times * 2 * T * (H + KV) * hd * e + table + T * 8, "flops": times * 3 * T * (H + KV) * r}
    c, extra = (e, 0) if case["format"] == "same" else (1, 4)
    row = 2 * KV * (hd * c + extra)                         # one cached token: key, value and their scales
    if case["op"] == "write":
        n, read = case["seqs"] * case["new"], case["seqs"] * (case["new"] + (case["past"] if case["whole"] else 0))
        moved = n * (2 * H + 2 * KV) * hd * e + n * row + read * (row + 2 * KV * hd * e)
        if case["rope"]:
            moved += case["new"] * hd * 4
        return {"bytes": moved + n * 12 + read * 12, "flops": n * (3 * (H + KV) + 4 * KV) * hd + read * 2 * KV * hd}
    seen = sum(min(n, case["window"] or n) for n in _lengths(case))
    B, ps = case["seqs"], case["page_size"]
    return {"bytes": seen * row + 2 * B * H * hd * e + B * H * 4 + -(-seen // ps) * 4 + B * 8,
            "flops": 4 * seen * H * hd}


# -- the definition in 64 bits ----------------------------------------------------------------------------------

def _exact_turn(x, angles, interleaved):
    """Each pair (a, b) times the complex number cos + i sin."""
    r = 2 * angles.shape[1]
    head = x[..., :r].reshape(*x.shape[:-1], r // 2, 2) if interleaved else \
        x[..., :r].reshape(*x.shape[:-1], 2, r // 2).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * angles[:, None, :])
    y = z if interleaved else z.transpose(-1, -2)
    return torch.cat((y.reshape(*x.shape[:-1], r), x[..., r:]), -1)


def _exact_rows(x, fmt):
    """What the cache holds of the rows x, as the values that it stands for."""
    if fmt == "same":
        return x
    top = 127.0 if fmt == "int8" else 448.0
    scale = x.abs().amax(-1, keepdim=True) / top
    c = x / torch.where(scale > 0, scale, torch.ones_like(scale))
    c = torch.round(c) if fmt == "int8" else c.float().to(torch.float8_e4m3fn).double()
    return c * scale


def exact(case, seed):
    s = prepare(case, seed)
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "rope":
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"]]
        out = [_exact_turn(s[n].double(), turn, case["interleaved"]) for n in ("q", "k")]
        if case["train"]:
            out += [_exact_turn(s[n].double(), turn.conj(), case["interleaved"]) for n in ("dq", "dk")]
        return out
    if case["op"] == "write":
        out, kept = [], {}
        for name in ("q", "k_new", "v_new"):
            if s[name] is None:
                continue
            x = s[name].double()
            if name != "v_new":
                if case["qk_norm"]:
                    x = (x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()).to(dt).double()
                if case["rope"]:
                    x = _exact_turn(x, torch.complex(s["cos"].double(), s["sin"].double())[s["pos"]], False)
                if name == "k_new":
                    x = x.to(dt).double()
            if name == "q":
                out.append(x)
            else:
                kept[name] = _exact_rows(x, case["format"])
        for name, new in (("k", "k_new"), ("v", "v_new")):
            fresh = kept[new].view(case["seqs"], case["new"], *kept[new].shape[1:])
            if case["whole"] and case["past"]:
                ps = case["page_size"]
                at = torch.arange(case["past"], device="cuda")
                page = s["table"][:, at // ps].long()
                old = s[name].view(torch.int8)[page, :, at % ps].view(s[name].dtype).double() \
                    if s[name].element_size() == 1 else s[name][page, :, at % ps].double()
                if s[name + "_scale"] is not None:
                    old = old * s[name + "_scale"][page, :, at % ps].double()[..., None]
                fresh = torch.cat((old, fresh), 1)
            out.append(fresh.reshape(-1, *fresh.shape[2:]))
        return out
    H, KV, hd, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    out = torch.zeros(case["seqs"], H, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((case["seqs"], H), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n, device="cuda")
        page = s["table"][b, at // ps].long()
        for h in range(KV):
            kv = []
            for name in ("k", "v"):
                x = s[name].view(torch.int8)[page, h, at % ps].view(s[name].dtype).double() \
                    if s[name].element_size() == 1 else s[name][page, h, at % ps].double()
                if s[name + "_scale"] is not None:
                    x = x * s[name + "_scale"][page, h, at % ps].double()[:, None]
                kv.append(x)
            g = slice(h * (H // KV), (h + 1) * (H // KV))
            z = s["q"][b, g].double() @ kv[0].T / math.sqrt(hd)
            lse[b, g] = torch.logsumexp(z, -1)
            out[b, g] = torch.softmax(z, -1) @ kv[1]
    return [out, lse]


if __name__ == "__main__":
    for c in listed():
        print(c["name"], work(c))
    print(draw(random.Random(0)))
