"""The paged KV cache that is quantised as it is written, and the attention that reads it: what is measured, in which
sizes, and the operators' plain form.

A cache row's token t lies in page table[row, t // P], slot t % P. A page holds, for one layer, P rows of d elements per
kv head, of K and of V: bf16, or MX e4m3, codes of 8 bits and a scale byte s per 32 elements that stands for 2^(s - 127), the
smallest power of two, at least 2^-126, that holds the block's largest magnitude without saturation (448); codes are rounded to
nearest, ties to even.

  write      N projected tokens per sequence: rotary positions for q and k, K and V into the pages; read back
  attention  N new tokens per sequence attend to the committed tokens and, by a tree's ancestor masks or as a causal chain,
             to the new ones; a row that sees nothing is 0
  path       write, then the rows of the accepted tree nodes moved together behind the committed tokens; read back
  step       write, attention, the accepted path: what one layer does in a verify round

Sizes are those of this repository's model configurations and benchmark and what lies between them.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False  # True: run() calls the framework's operators

DEV = "cuda"
BLOCK = 32
HEADS = {"tiny": (8, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128), "8b": (32, 8, 128), "14b": (40, 8, 128)}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # One token of one sequence at 1.5B: a call of latency alone.
        dict(name="write-token-1.5b", kind="write", heads="1.5b", batch=1, new=1, length=700, span=0, page=64, ragged=False),
        # The tree nodes of a 7B verify round.
        dict(name="write-verify-7b", kind="write", heads="7b", batch=64, new=29, length=2048, span=500, page=64, ragged=False),
        # A prefill chunk of prompts of unequal length at 8B, positions beyond the first chunk.
        dict(name="write-chunk-8b", kind="write", heads="8b", batch=4, new=1024, length=9000, span=777, page=128, ragged=True),
        # One token of one sequence against a short cache: latency.
        dict(name="token-1.5b", kind="attention", heads="1.5b", fmt="e4m3", batch=1, new=1, length=700, span=0, page=64, chain=True),
        # Single tokens of 64 sequences of unequal length at 8B, as in plain decoding: the cache is streamed once.
        dict(name="tokens-64-8b", kind="attention", heads="8b", fmt="e4m3", batch=64, new=1, length=4096, span=3000, page=64, chain=True),
        # Single tokens over two very long caches: few rows, a long axis.
        dict(name="token-long-8b", kind="attention", heads="8b", fmt="e4m3", batch=2, new=1, length=131071, span=30001, page=256, chain=True),
        # One layer's attention of a 7B verify round; 8 repeats of a prompt share its pages.
        dict(name="verify-7b", kind="attention", heads="7b", fmt="e4m3", batch=64, new=29, length=2048, span=0, page=64, chain=False, share=8, prompt=1024),
        # A verify round at 14B on bf16 pages.
        dict(name="verify-14b-bf16", kind="attention", heads="14b", fmt="bf16", batch=32, new=29, length=4096, span=1000, page=128, chain=False),
        # A prefill chunk behind ragged prefixes at 8B, the prompts ending inside it.
        dict(name="chunk-8b", kind="attention", heads="8b", fmt="e4m3", batch=4, new=1024, length=1000, span=250, page=64, chain=True, ragged=True),
        # A small model with heads of 64 and pages that are shorter than a tile, one sequence without a prefix.
        dict(name="verify-tiny", kind="attention", heads="tiny", fmt="e4m3", batch=8, new=13, length=256, span=256, page=16, chain=False, empty=True),
        # The accepted path of a 7B verify round, behind the tree that was written for it.
        dict(name="path-7b", kind="path", heads="7b", batch=64, new=29, length=2048, span=100, page=64, depth=5),
        # One layer of a 1.5B verify round: write, attention, accepted path.
        dict(name="step-1.5b", kind="step", heads="1.5b", batch=32, new=13, length=512, span=200, page=64, depth=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one(rng):
    kind = rng.choice(["write", "write", "attention", "attention", "attention", "attention", "path", "step"])
    c = dict(kind=kind, heads=rng.choice(["tiny", "1.5b", "7b", "8b", "14b"]), page=rng.choice([16, 32, 64, 64, 128, 256]))
    if kind == "write":
        c |= dict(batch=_log(rng, 1, 128), new=_log(rng, 1, 1024), length=_log(rng, 1, 100000), ragged=rng.random() < 0.3)
        return c | dict(span=rng.randint(0, c["length"]))
    if kind == "attention":
        what = rng.choice(["token", "token", "tree", "tree", "chunk"])
        n = 1 if what == "token" else rng.randint(2, 64) if what == "tree" else _log(rng, 8, 2048)
        c |= dict(fmt=rng.choice(["e4m3", "e4m3", "bf16"]), batch=_log(rng, 1, 128), new=n, length=_log(rng, 1, 100000), chain=what != "tree")
        c |= dict(span=rng.randint(0, c["length"]))
        if what == "tree" and rng.random() < 0.3:
            c |= dict(empty=True)
        if what == "chunk" and rng.random() < 0.5:
            c |= dict(ragged=True)
        return c
    c |= dict(batch=_log(rng, 1, 128), new=rng.randint(2, 64), length=_log(rng, 1, 8192))
    return c | dict(span=rng.randint(0, c["length"]), depth=rng.randint(1, min(8, c["new"])))


_MOST = None


def draw(rng):
    global _MOST
    if _MOST is None:
        w = [work(c) for c in listed()]
        _MOST = max(x["bytes"] for x in w), max(x["flops"] for x in w)
    while True:
        c = _one(rng)
        w = work(c)
        # the plain form holds every row's keys, and a score for each row and key, as far as the longest sequence goes
        hq, hkv, d = HEADS[c["heads"]]
        held = c["batch"] * (c["length"] + c["new"])
        if w["bytes"] <= _MOST[0] and w["flops"] <= _MOST[1] and held * hkv * d <= 1.5e9 and held * hq * c["new"] <= 5e8:
            return c


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """The committed tokens of each sequence (a long one first), and how many of its new tokens count."""
    b, n, span = case["batch"], case["new"], case["span"]
    lens = [case["length"] - (i * 7919 + 13 * i * i) % (span + 1) for i in range(b)]
    if case.get("empty"):
        lens[-1] = 0
    counts = [n - (i * 5 % 7) * n // 8 for i in range(b)] if case.get("ragged") else [n] * b
    return lens, counts


def _pages_of(case):
    """Rows of page numbers (before they are mixed) and how many there are: the sequences of a group share the prompt's."""
    page, rows, count, common = case["page"], [], 0, []
    lens, _ = _lengths(case)
    share, whole = case.get("share", 1), case.get("prompt", 0) // page
    for i, length in enumerate(lens):
        if i % share == 0:
            common = list(range(count, count + whole))
            count += whole
        mine = -(-(length + case["new"]) // page) - whole
        rows.append(common + list(range(count, count + mine)))
        count += mine
    return rows, count


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _tree(rng, n, empty):
    """Ancestor-or-self masks of a random tree; with `empty`, of its last node none at all."""
    bits = [1]
    for i in range(1, n):
        bits.append(bits[rng.randrange(max(0, i - 8), i)] | 1 << i)
    if empty:
        bits[-1] = 0
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def _channels(g, hkv, d):
    """K's spread over its channels: a few far larger than the others, as a decoder's K has."""
    c = torch.exp(0.3 * _normal(g, hkv, 1, d))
    return torch.where(torch.rand(hkv, 1, d, device=DEV, generator=g) < 0.02, 6.0 * c, c)


def prepare(case, seed):
    g, rng = _gen(seed), random.Random(int(seed))
    hq, hkv, d = HEADS[case["heads"]]
    b, n, page = case["batch"], case["new"], case["page"]
    rows, count = _pages_of(case)
    mixed = list(range(count))
    rng.shuffle(mixed)
    wide = max(len(r) for r in rows) + 1
    table = torch.tensor([[mixed[p] for p in r] + [-1] * (wide - len(r)) for r in rows], dtype=torch.int32, device=DEV)
    lens, counts = _lengths(case)
    s = dict(case=dict(case), table=table, seq=torch.tensor(lens, dtype=torch.int32, device=DEV),
             new_len=torch.tensor(counts, dtype=torch.int32, device=DEV) if case.get("ragged") else None, scale=d ** -0.5)
    spread = _channels(g, hkv, d)
    k = (_normal(g, count, hkv, page, d) * spread).to(torch.bfloat16)
    v = _normal(g, count, hkv, page, d).to(torch.bfloat16)
    if case.get("fmt") == "bf16":
        s["k"], s["v"], s["ks"], s["vs"] = k, v, None, None
    else:
        s["k"], s["ks"] = _quantize(k)
        s["v"], s["vs"] = _quantize(v)
    del k, v
    if case["kind"] == "attention":
        s["q"] = (_normal(g, b, n, hq, d) / spread.repeat_interleave(hq // hkv, 0).reshape(1, 1, hq, d).clamp_min(1.0)).to(torch.bfloat16)
        s["out"] = torch.zeros(b, n, hq, d, dtype=torch.bfloat16, device=DEV)
    else:
        qkv = _normal(g, b, n, (hq + 2 * hkv) * d)
        qkv[..., hq * d:(hq + hkv) * d] *= spread.reshape(-1)
        s["qkv"] = qkv.reshape(b * n, -1).to(torch.bfloat16)
        s["inv_freq"] = 1.0 / (1.0e6 ** (torch.arange(0, d, 2, device=DEV).float() / d))
        s["q"] = torch.zeros(b, n, hq, d, dtype=torch.bfloat16, device=DEV)
    s["offset"] = torch.arange(n, dtype=torch.int32, device=DEV)
    s["anc"] = None
    if case["kind"] in ("path", "step") or not case.get("chain", True):
        s["anc"] = torch.tensor([_tree(rng, n, case.get("empty")) for _ in range(b)], dtype=torch.int64, device=DEV)
    if "depth" in case:  # accepted nodes: the root, then ever later ones; paths of unequal length
        nodes = [[0] + sorted(rng.sample(range(1, n), case["depth"] - 1)) for _ in range(b)]
        s["nodes"] = torch.tensor(nodes, dtype=torch.int32, device=DEV)
        s["taken"] = torch.tensor([rng.randint(1, case["depth"]) for _ in range(b)], dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------ the plain form, in 32 bits
def _quantize(x):
    """(codes, scales) of the rows of x, blocks of 32 along the last axis."""
    v = x.float().unflatten(-1, (-1, BLOCK))
    amax = v.abs().amax(-1)
    # The exponent field of the largest magnitude, one more where its fraction is over that of 448 (1.75: the addition
    # carries into the exponent), less the exponent of 448.
    e = (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp_min(1)
    y = v * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)
    bad = ~torch.isfinite(amax)
    codes = torch.where(bad.unsqueeze(-1), 0.0, y).flatten(-2).to(torch.float8_e4m3fn)
    return codes, torch.where(bad, 255, e).to(torch.uint8)


def _values(codes, scales):
    if scales is None:
        return codes.float()
    x = torch.where(scales == 255, math.nan, (scales.to(torch.int32) << 23).view(torch.float32))
    return (codes.float().unflatten(-1, (-1, BLOCK)) * x.unsqueeze(-1)).flatten(-2)


def _bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _at(s, tokens):
    """Page and slot of tokens [batch, any] of each sequence."""
    page = s["case"]["page"]
    return s["table"].long().gather(1, tokens // page), tokens % page


def _read(s, tokens):
    """The values of K and V at tokens [batch, any]: [batch, kv heads, any, d]."""
    p, i = _at(s, tokens)
    got = []
    for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        c = _bits(codes)[p, :, i].view(codes.dtype)
        got.append(_values(c, None if scales is None else scales[p, :, i]).transpose(1, 2))
    return got


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _put(s, name, tokens, rows, counts):
    """rows [batch, any, kv heads, d] into the pages, where a token counts."""
    p, i = _at(s, tokens)
    c, e = _quantize(rows)
    _bits(s[name])[p[counts], :, i[counts]] = _bits(c)[counts]
    s[name + "s"][p[counts], :, i[counts]] = e[counts]


def _new_tokens(s):
    n = s["case"]["new"]
    tokens = s["seq"].long().unsqueeze(1) + torch.arange(n, device=DEV)
    counts = torch.arange(n, device=DEV) < (s["new_len"].unsqueeze(1) if s["new_len"] is not None else n)
    return tokens, counts.expand(tokens.shape)


def _write(s):
    hq, hkv, d = HEADS[s["case"]["heads"]]
    tokens, counts = _new_tokens(s)
    position = s["seq"].long().unsqueeze(1) + s["offset"].long()
    angle = position.double().unsqueeze(-1) * s["inv_freq"].double()
    cos, sin = (f(angle).float().unsqueeze(2) for f in (torch.cos, torch.sin))
    q, k, v = s["qkv"].float().reshape(*tokens.shape, hq + 2 * hkv, d).split((hq, hkv, hkv), 2)
    s["q"].copy_(torch.where(counts[..., None, None], _rotate(q, cos, sin).to(torch.bfloat16), s["q"]))
    _put(s, "k", tokens, _rotate(k, cos, sin), counts)
    _put(s, "v", tokens, v, counts)
    return tokens


def _attention(s):
    hq, hkv, d = HEADS[s["case"]["heads"]]
    b, n = s["q"].shape[:2]
    tokens, counts = _new_tokens(s)
    top = s["case"]["length"] + n
    every = torch.arange(top, device=DEV)
    held = s["seq"].long() + counts.sum(1)
    k, v = _read(s, torch.where(every < held.unsqueeze(1), every, 0))
    m = every - s["seq"].long().unsqueeze(1)  # which new token a key is
    if s["anc"] is None:
        sees = m.unsqueeze(1) <= torch.arange(n, device=DEV).unsqueeze(1)
    else:
        sees = (m < 0).unsqueeze(1) | ((s["anc"].unsqueeze(2) >> m.clamp(0, 63).unsqueeze(1)) & 1).bool()
    sees = (sees & (every < held.unsqueeze(1)).unsqueeze(1)).repeat_interleave(hq // hkv, 1)
    q = s["q"].float().reshape(b, n, hkv, -1, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    score = q @ k.transpose(2, 3).contiguous() * s["scale"]
    sees = sees.reshape(b, n, -1, top).permute(0, 2, 1, 3).reshape(b, 1, -1, top)
    score = torch.where(sees, score, -math.inf)
    high = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(high == -math.inf, 0.0, high))
    total = p.sum(-1, keepdim=True)
    o = p @ v / torch.where(total == 0, 1.0, total)
    o = o.reshape(b, hkv, -1, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).to(torch.bfloat16)
    return torch.where(counts[..., None, None], o, 0.0)


def _compact(s):
    """The accepted nodes' rows moved together."""
    j = torch.arange(s["case"]["depth"], device=DEV)
    taken = j < s["taken"].unsqueeze(1)
    seq = s["seq"].long().unsqueeze(1)
    p, i = _at(s, seq + s["nodes"])
    to, at = _at(s, seq + j)
    for name in ("k", "ks", "v", "vs"):
        t = _bits(s[name])
        t[to[taken], :, at[taken]] = t[p[taken], :, i[taken]]


def _back(s, tokens):
    k, v = _read(s, tokens)
    return dict(k=k.to(torch.bfloat16), v=v.to(torch.bfloat16))


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "attention":
        return _attention(s)
    tokens = _write(s)
    if kind == "write":
        return dict(q=s["q"], **_back(s, tokens))
    out = dict(out=_attention(s)) if kind == "step" else {}
    _compact(s)
    return out | _back(s, tokens[:, :s["case"]["depth"]])


# ------------------------------------------------------------------ the framework's operators
_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ss-grpo_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)


def _framework(s):
    from flashgrpo_amd import kernels as K

    c = s["case"]
    hq, hkv, d = HEADS[c["heads"]]
    pages = K.KVPages(s["k"], s["v"], s["ks"], s["vs"], s["table"])
    sizes = dict(num_nodes=c["new"], q_heads=hq, kv_heads=hkv, head_dim=d)
    if c["kind"] == "attention":
        return K.paged_attention(s["q"], pages, seq_len=s["seq"], anc=s["anc"], out=s["out"], new_len=s["new_len"], scale=s["scale"], **sizes)
    K.rope_kv_write_paged(s["qkv"], pages, batch=c["batch"], seq_len=s["seq"], pos_offset=s["offset"], inv_freq=s["inv_freq"], q_out=s["q"],
                          new_len=s["new_len"], **sizes)
    if c["kind"] == "write":
        k, v = K.kv_read_paged(pages, start=s["seq"], count=c["new"])
        return dict(q=s["q"], k=k, v=v)
    out = {}
    if c["kind"] == "step":
        out["out"] = K.paged_attention(s["q"], pages, seq_len=s["seq"], anc=s["anc"], scale=s["scale"], **sizes)
    K.kv_path_gather_paged(pages, seq_len=s["seq"], acc_nodes=s["nodes"], acc_len=s["taken"], tree_nodes=c["new"])
    k, v = K.kv_read_paged(pages, start=s["seq"], count=c["depth"])
    return out | dict(k=k, v=v)


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------ the least work of one pass
def work(case):
    hq, hkv, d = HEADS[case["heads"]]
    lens, counts = _lengths(case)
    row = 2 * hkv * (2 * d if case.get("fmt") == "bf16" else d + d // BLOCK)  # K and V of a token as they are held
    value = 2 * hkv * 2 * d                                                   # and as bf16 values
    new = sum(counts)
    written = new * (2 * (hq + 2 * hkv) * d + 2 * hq * d + row)
    if case["kind"] == "write":  # projected rows in, q and K and V out; what was written in, its values out
        return dict(bytes=written + case["batch"] * case["new"] * (row + value), flops=6.0 * new * (hq + hkv) * d)
    # the tokens that some sequence sees: a shared prompt's once
    held = sum(lens) + new - sum(case["prompt"] // case["page"] * case["page"] for i in range(case["batch"]) if i % case["share"]) if "share" in case else sum(lens) + new
    seen = sum(c * (l + ((c + 1) / 2 if case.get("chain") else min(c, 6))) for l, c in zip(lens, counts))
    flops = 4.0 * hq * d * seen
    if case["kind"] == "attention":
        return dict(bytes=held * row + 2 * 2 * new * hq * d, flops=flops)
    moved = case["batch"] * case["depth"]
    path = dict(bytes=written + 2 * moved * row + moved * (row + value), flops=6.0 * new * (hq + hkv) * d)
    if case["kind"] == "path":
        return path
    return dict(bytes=path["bytes"] + held * row + 2 * new * hq * d, flops=path["flops"] + flops)


# ------------------------------------------------------------------ from the definition, in 64 bits
def _two64(e):
    """2^e, from its bits: a power function may be off by its last one."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _through64(x):
    """The values that x's e4m3 blocks stand for: steps of 2^-3 of a value's power of two, of 2^-9 at least."""
    b = x.double().reshape(-1, BLOCK)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True) / 448.0)  # the least power of two not below m 2^e
    f = _two64(torch.where(m == 0.5, e - 1, e).clamp_min(-126))
    step = _two64((torch.frexp(b / f)[1] - 1).clamp_min(-6) - 3)
    return (torch.round(b / f / step) * step * f).reshape(x.shape)


def _cache64(s, i, tokens):
    """K and V of tokens of sequence i, [kv heads, tokens, d]."""
    at = s["table"][i].long()[tokens // s["case"]["page"]] * s["case"]["page"] + tokens % s["case"]["page"]
    got = []
    for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        raw = codes if scales is None else codes.view(torch.uint8)
        x = raw.transpose(1, 2).reshape(-1, raw.shape[1], raw.shape[3])[at]
        if scales is None:
            x = x.double()
        else:
            f = scales.transpose(1, 2).reshape(-1, scales.shape[1], scales.shape[3])[at]
            x = x.view(torch.float8_e4m3fn).double() * _two64(f.to(torch.int64) - 127).repeat_interleave(BLOCK, -1)
        got.append(x.transpose(0, 1))
    return got


def _turn64(x, position, inv_freq):
    z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), position.double().unsqueeze(-1) * inv_freq.double()).unsqueeze(-2)
    h = x.shape[-1] // 2
    y = torch.complex(x[..., :h].double(), x[..., h:].double()) * z
    return torch.cat([y.real, y.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d = HEADS[case["heads"]]
    lens, counts = _lengths(case)
    n, kind, got = case["new"], case["kind"], dict(q=[], k=[], v=[], out=[])
    for i, (length, count) in enumerate(zip(lens, counts)):
        held = torch.arange(length + n, device=DEV)
        k, v = _cache64(s, i, held)
        if kind == "attention":
            q = s["q"][i].double()
        else:
            x = s["qkv"].reshape(case["batch"], n, hq + 2 * hkv, d)[i]
            position = length + s["offset"].long()
            q = _turn64(x[:, :hq], position, s["inv_freq"])
            k[:, length:length + count] = _through64(_turn64(x[:count, hq:hq + hkv], position[:count], s["inv_freq"])).transpose(0, 1)
            v[:, length:length + count] = _through64(x[:count, hq + hkv:]).transpose(0, 1)
        q[count:] = 0.0
        if kind in ("attention", "step"):
            if kind == "step":
                q = q.to(torch.bfloat16).double()  # the queries as the operator hands them on
            new = torch.arange(n, device=DEV)
            sees = new.unsqueeze(1) >= new if s["anc"] is None else ((s["anc"][i].unsqueeze(1) >> new) & 1).bool()
            sees = torch.cat([torch.ones(n, length, dtype=torch.bool, device=DEV), sees & (new < count)], 1)
            o = torch.zeros(n, hq, d, dtype=torch.float64, device=DEV)
            for h in range(hkv):
                rows = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                score = (q[:, rows].reshape(-1, d) @ k[h].T * s["scale"]).reshape(n, -1, length + n)
                score = score.masked_fill(~sees.unsqueeze(1), -math.inf)
                o[:, rows] = torch.nan_to_num(torch.softmax(score, -1)) @ v[h]
            o[count:] = 0.0
            got["out"].append(o)
        if "depth" in case:
            node = length + s["nodes"][i].long()
            taken = torch.arange(case["depth"], device=DEV) < s["taken"][i]
            for x in (k, v):
                x[:, length:length + case["depth"]] = torch.where(taken[:, None], x[:, node], x[:, length:length + case["depth"]])
        until = length + case.get("depth", n)
        got["q"].append(q)
        got["k"].append(k[:, length:until].clone())
        got["v"].append(v[:, length:until].clone())
    if kind == "attention":
        return torch.stack(got["out"])
    names = dict(write="q k v", path="k v", step="out k v")[kind].split()
    return {x: torch.stack(got[x]) for x in names}
