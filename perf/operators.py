"""The decode-side operators over a 4-bit KV cache, as they are measured.

Four operators that one generation loop uses together:

  attn     grouped-query attention of one new token per sequence over a cache
           held in 4 bits; with `track`, every slot's attention weight is
           accumulated as well
  put      RoPE on the q and k heads of new tokens, their k and v quantized
           into the cache, and the written rows read back as values
  evict    every (layer, sequence, kv head) cut down to `budget` slots: the
           `recent` newest positions and the slots of largest accumulated
           weight stay, moved into the freed slots
  beam     one beam-search selection over beams x vocabulary
  reorder  the beams' cache rows moved to follow the selection

A cache layer is codes uint8 [blocks, kv heads, block size, bytes] (element e of
a head in nibble e & 1 of byte e / 2, heads padded to 32, 64, 96, 128, 192 or
256 elements) and a grid bf16 [blocks, kv heads, block size, 2] = (step, base)
per row; the value is base + step * code.  put returns what it wrote as values.
evict and reorder compute no value: they return the rows' bytes where they moved
them to, which have to be equal.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

THETA = 10000.0
EOS = 2


def _fw():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forge-llm_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import forgellm
    return forgellm


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the latency of one chat turn's step: a short context in a small preallocated cache
        dict(name="attn one short sequence", op="attn", B=1, n=37, cap=1024, nH=12, nKV=4, dH=64, block=0,
             ragged=False, track=False),
        # a serving batch in steady state, grouped heads
        dict(name="attn batch 64 x 4096", op="attn", B=64, n=4096, cap=4352, nH=32, nKV=8, dH=128, block=0,
             ragged=False, track=False),
        # a server's mixed batch on pages, weights kept for the eviction
        dict(name="attn ragged pages tracked", op="attn", B=48, n=9001, cap=9024, nH=16, nKV=2, dH=96, block=48,
             ragged=True, track=True),
        # one very long document, nothing but the long axis to split
        dict(name="attn one sequence of 262000", op="attn", B=1, n=262000, cap=262144, nH=12, nKV=4, dH=64, block=0,
             ragged=False, track=False),
        # every head with its own cache, an odd length and a head of 80, weights kept
        dict(name="attn heads of 80 tracked", op="attn", B=16, n=2047, cap=2048, nH=16, nKV=16, dH=80, block=64,
             ragged=False, track=True),
        # one decode step of a batch: latency
        dict(name="put step of 32", op="put", B=32, T=1, start=700, cap=1024, nH=12, nKV=4, dH=64, block=64),
        # a prompt chunk of several sequences: bandwidth
        dict(name="put chunk 4 x 2048", op="put", B=4, T=2048, start=2049, cap=4352, nH=32, nKV=8, dH=128, block=0),
        # steady state: a slot freed for every token
        dict(name="evict one of 1025", op="evict", L=12, B=8, n=1025, cap=1088, budget=1024, recent=256, nKV=4, dH=64,
             block=64, fresh=False),
        # a long prompt cut down before generation starts
        dict(name="evict 16001 to 2048", op="evict", L=4, B=16, n=16001, cap=16384, budget=2048, recent=511, nKV=8,
             dH=128, block=0, fresh=True),
        # one request's search
        dict(name="beam 1 x 4", op="beam", B=1, W=4, V=32000, done=0.0, first=True),
        # a batch of searches over a large odd vocabulary, some beams finished
        dict(name="beam 32 x 8", op="beam", B=32, W=8, V=100003, done=0.15, first=False),
        # the caches of a batch of searches after a selection
        dict(name="reorder 16 x 4", op="reorder", L=12, B=16, W=4, n=1003, cap=1024, nKV=4, dH=64, block=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    c = _drawn(rng)
    most = max(work(x)["bytes"] for x in listed() if x["op"] == c["op"])
    while work(c)["bytes"] > most and c["B"] > 1:
        c["B"] = max(1, int(c["B"] * 0.8))
    return c


def _drawn(rng):
    op = rng.choice(["attn", "attn", "attn", "put", "evict", "beam", "reorder"])
    dH = rng.choice([16, 32, 48, 64, 72, 80, 96, 112, 128, 128, 160, 192, 256])
    nKV = rng.choice([1, 2, 3, 4, 8])
    g = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    block = rng.choice([0, 0, 16, 48, 64, 100, 128])

    def cap_of(n):
        cap = n + rng.randrange(0, 200)
        return -(-cap // block) * block if block else cap

    if op == "attn":
        n = _log(rng, 1, 65536)
        room = 64 * 4096 * 8 * 128
        B = max(1, min(_log(rng, 1, 128), room // (n * nKV * dH)))
        return dict(op=op, B=B, n=n, cap=cap_of(n), nH=nKV * g, nKV=nKV, dH=dH, block=block,
                    ragged=rng.random() < 0.5, track=rng.random() < 0.4)
    if op == "put":
        T = rng.choice([1, 1, _log(rng, 2, 2048)])
        B = max(1, min(_log(rng, 1, 256), 4 * 2048 * 64 * 64 // (T * nKV * (g + 2) * dH)))
        start = _log(rng, 1, 20000)
        return dict(op=op, B=B, T=T, start=start, cap=cap_of(start + T), nH=nKV * g, nKV=nKV, dH=dH, block=block)
    if op == "evict":
        n = _log(rng, 8, 30000)
        budget = max(1, int(n * rng.uniform(0.05, 1.05)))
        recent = rng.randrange(0, budget + 1)
        L = rng.choice([1, 2, 6, 12])
        B = max(1, min(_log(rng, 1, 64), 4 * 16 * 8 * 16000 * 128 // (L * nKV * n * dH)))
        return dict(op=op, L=L, B=B, n=n, cap=cap_of(n), budget=budget, recent=recent, nKV=nKV, dH=dH, block=block,
                    fresh=rng.random() < 0.5)
    if op == "beam":
        W = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        V = _log(rng, 64, 130000)
        B = max(1, min(_log(rng, 1, 64), 32 * 8 * 100003 // (W * V)))
        return dict(op=op, B=B, W=W, V=V, done=rng.choice([0.0, 0.2]), first=rng.random() < 0.3)
    n = _log(rng, 1, 8192)
    W = rng.choice([2, 3, 4, 5, 8])
    L = rng.choice([1, 4, 12])
    B = max(1, min(_log(rng, 1, 32), 12 * 16 * 4 * 1003 * 4 * 64 * 4 // (L * W * n * nKV * dH)))
    return dict(op=op, L=L, B=B, W=W, n=n, cap=cap_of(n), nKV=nKV, dH=dH, block=block)


# ------------------------------------------------------------------ inputs
def _row_bytes(dH):
    return next(p for p in (32, 64, 96, 128, 192, 256) if p >= dH) // 2


def _blocks(c):
    bs = c["block"] or c["cap"]
    return bs, c["cap"] // bs


def _lens_of(c):
    if not c["ragged"]:
        return [c["n"]] * c["B"]
    return [round(c["n"] * (b + 1) / c["B"]) for b in range(c["B"])]


def _quantize(x, rb):
    """(codes uint8 [..., rb], grid bf16 [..., 2]) of rows x [..., dH] fp32."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    base = lo.to(torch.bfloat16)
    step = ((hi.double() - base.double()) / 15).clamp_(min=0).float().to(torch.bfloat16)
    b, s = base.double(), step.double()
    code = torch.where(s > 0, ((x.double() - b) / torch.where(s > 0, s, 1.0)).round_(), 0.0).clamp_(0, 15)
    code = torch.nn.functional.pad(code.to(torch.uint8), (0, 2 * rb - x.shape[-1]))
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([step, base], -1)


def _cache(gen, lead, nKV, bs, dH):
    """A filled cache's (codes, grid): rows of normal values with a part that
    the positions share, quantized row by row (the last dimension)."""
    shape = (*lead, nKV, bs)
    rb = _row_bytes(dH)
    codes = torch.empty(*shape, rb, dtype=torch.uint8, device="cuda")
    grid = torch.empty(*shape, 2, dtype=torch.bfloat16, device="cuda")
    fc, fg = codes.view(-1, rb), grid.view(-1, 2)
    common = torch.randn(dH, generator=gen, device="cuda")
    chunk = max(1, (1 << 26) // dH)
    for a in range(0, fc.shape[0], chunk):
        m = min(chunk, fc.shape[0] - a)
        x = torch.randn(m, dH, generator=gen, device="cuda") + 0.5 * common
        fc[a:a + m], fg[a:a + m] = _quantize(x, rb)
    return codes, grid


def _table(gen, c, B):
    """A shuffled block table, as a server's allocator leaves it; none for a contiguous cache."""
    _, mb = _blocks(c)
    if not c["block"]:
        return None
    return torch.randperm(B * mb, generator=gen, device="cuda").to(torch.int32).view(B, mb)


def prepare(case, seed):
    c = case
    gen = torch.Generator("cuda").manual_seed(seed)
    dev = "cuda"
    s = {"case": c}
    if c["op"] == "attn":
        bs, mb = _blocks(c)
        B = c["B"]
        s["k"], s["kg"] = _cache(gen, (B * mb,), c["nKV"], bs, c["dH"])
        s["v"], s["vg"] = _cache(gen, (B * mb,), c["nKV"], bs, c["dH"])
        s["table"] = _table(gen, c, B)
        lens = torch.tensor(_lens_of(c), dtype=torch.int32, device=dev)
        s["lens"] = lens[torch.randperm(B, generator=gen, device=dev)].contiguous()
        s["q"] = torch.randn(B, c["nH"], c["dH"], generator=gen, device=dev) * 1.5
        if c["track"]:
            s["weight"] = torch.rand(B * mb, c["nKV"], bs, generator=gen, device=dev)
    elif c["op"] == "put":
        bs, mb = _blocks(c)
        B, rb = c["B"], _row_bytes(c["dH"])
        s["k"] = torch.zeros(B * mb, c["nKV"], bs, rb, dtype=torch.uint8, device=dev)
        s["kg"] = torch.zeros(B * mb, c["nKV"], bs, 2, dtype=torch.bfloat16, device=dev)
        s["v"], s["vg"] = torch.zeros_like(s["k"]), torch.zeros_like(s["kg"])
        s["table"] = _table(gen, c, B)
        s["qkv"] = torch.randn(B * c["T"], (c["nH"] + 2 * c["nKV"]) * c["dH"], generator=gen, device=dev)
        # sequences of different lengths; the rotary position runs ahead of the slot where slots were freed
        back = torch.randint(0, min(c["start"], 64) + 1, (B,), generator=gen, device=dev)
        s["slots"] = (c["start"] - back).to(torch.int32)
        s["positions"] = (s["slots"] + torch.randint(0, 1000, (B,), generator=gen, device=dev)).to(torch.int32)
    elif c["op"] == "evict":
        bs, mb = _blocks(c)
        L, B, nKV, n = c["L"], c["B"], c["nKV"], c["n"]
        s["k"], s["kg"] = _cache(gen, (L, B * mb), nKV, bs, c["dH"])
        s["v"], s["vg"] = _cache(gen, (L, B * mb), nKV, bs, c["dH"])
        s["table"] = _table(gen, c, B)
        s["lens"] = torch.full((B,), n, dtype=torch.int32, device=dev)
        # few slots hold most of the weight
        s["weight0"] = torch.randn(L, B * mb, nKV, bs, generator=gen, device=dev).mul_(2).exp_()
        order = torch.arange(mb * bs, device=dev).expand(L, B, nKV, mb * bs)
        if not c["fresh"]:  # slots already refilled many times: positions in no order, with gaps
            order = torch.rand(L, B, nKV, mb * bs, generator=gen, device=dev).argsort(-1) * 3
        pos = torch.empty(L, B * mb, nKV, bs, dtype=torch.int32, device=dev)
        at = s["table"].long().view(-1) if s["table"] is not None else torch.arange(B * mb, device=dev)
        pos[:, at] = order.reshape(L, B, nKV, mb, bs).transpose(2, 3).reshape(L, B * mb, nKV, bs).to(torch.int32)
        s["pos0"] = pos
        s["weight"], s["pos"] = torch.empty_like(s["weight0"]), torch.empty_like(pos)
    elif c["op"] == "beam":
        R = c["B"] * c["W"]
        x = torch.randn(R, c["V"], generator=gen, device=dev)
        s["logits"] = x * 2 + torch.randn(c["V"], generator=gen, device=dev)  # the beams agree in part
        s["logits"][:, torch.randint(0, c["V"], (3,), generator=gen, device=dev)] = -math.inf  # banned tokens
        s["scores"] = -10 * torch.rand(R, generator=gen, device=dev)
        if c["first"]:  # the first step of a search: one live beam
            s["scores"].view(c["B"], c["W"])[:, 1:] = -math.inf
        s["done"] = torch.rand(R, generator=gen, device=dev) < c["done"]
    else:
        bs, mb = _blocks(c)
        L, B, W = c["L"], c["B"], c["W"]
        R = B * W
        s["k"], s["kg"] = _cache(gen, (L, R * mb), c["nKV"], bs, c["dH"])
        s["v"], s["vg"] = _cache(gen, (L, R * mb), c["nKV"], bs, c["dH"])
        s["table"] = _table(gen, c, R)
        s["lens"] = torch.full((R,), c["n"], dtype=torch.int32, device=dev)
        s["parents"] = torch.randint(0, W, (B, W), generator=gen, device=dev, dtype=torch.int32)
    return s


# ------------------------------------------------------------------ the plain forms
def _by_sequence(x, table, B):
    """[blocks, nKV, bs, ...] as [B, nKV, slots, ...]."""
    mb = x.shape[0] // B
    x = x[table.long()] if table is not None else x.view(B, mb, *x.shape[1:])
    return x.transpose(1, 2).reshape(B, x.shape[2], mb * x.shape[3], *x.shape[4:])


def _values(codes, grid, dH):
    x = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :dH].float()
    return x.mul_(grid[..., :1].float()).add_(grid[..., 1:].float())


def _places(c, table, B, device):
    """Flat (block * bs + slot in block) index [B, slots] of every slot."""
    bs, mb = _blocks(c)
    blocks = table.long() if table is not None else torch.arange(B * mb, device=device).view(B, mb)
    j = torch.arange(mb * bs, device=device)
    return blocks[:, j // bs], j % bs


def _plain_attn(s):
    c = s["case"]
    B, nKV, dH = c["B"], c["nKV"], c["dH"]
    g = c["nH"] // nKV
    k = _values(_by_sequence(s["k"], s["table"], B), _by_sequence(s["kg"], s["table"], B), dH)
    q = s["q"].view(B, nKV, g, dH) * (1 / math.sqrt(dH))
    p = q @ k.transpose(-1, -2)
    del k
    alive = torch.arange(p.shape[-1], device=p.device) < s["lens"].view(B, 1, 1, 1)
    p = torch.where(alive, p, -math.inf)
    m = p.amax(-1, keepdim=True)
    p = torch.where(alive, torch.exp(p - m), 0.0)
    p = p / p.sum(-1, keepdim=True)
    p = torch.where(alive, p, 0.0)
    v = _values(_by_sequence(s["v"], s["table"], B), _by_sequence(s["vg"], s["table"], B), dH)
    out = (p @ v).reshape(B, c["nH"], dH)
    if not c["track"]:
        return out
    blk, off = _places(c, s["table"], B, p.device)
    s["weight"][blk[:, None], torch.arange(nKV, device=p.device)[None, :, None], off] += p.sum(2)
    return out, s["weight"]


def _plain_put(s):
    c = s["case"]
    B, T, nH, nKV, dH = c["B"], c["T"], c["nH"], c["nKV"], c["dH"]
    x = s["qkv"].view(B, T, nH + 2 * nKV, dH)
    t = torch.arange(T, device=x.device)
    freq = 1.0 / torch.pow(THETA, torch.arange(0, dH, 2, device=x.device, dtype=torch.float64) / dH)
    ang = (s["positions"].double()[:, None] + t)[..., None, None] * freq
    co, si = ang.cos().float().double(), ang.sin().float().double()
    r = x[:, :, :nH + nKV].double()
    u, w = r[..., 0::2], r[..., 1::2]
    r = torch.stack([u * co - w * si, u * si + w * co], -1).flatten(-2).float()
    x[:, :, :nH] = r[:, :, :nH]
    slot = s["slots"].long()[:, None] + t
    blk, off = _places(c, s["table"], B, x.device)
    b = torch.arange(B, device=x.device)[:, None]
    blk, off = blk[b, slot], off[slot]
    rb = _row_bytes(dH)
    for codes, grid, rows in ((s["k"], s["kg"], r[:, :, nH:]), (s["v"], s["vg"], x[:, :, nH + nKV:])):
        codes[blk, :, off], grid[blk, :, off] = _quantize(rows, rb)
    q = s["qkv"][:, :nH * dH]
    return q, _values(s["k"][blk, :, off], s["kg"][blk, :, off], dH), _values(s["v"][blk, :, off], s["vg"][blk, :, off], dH)


def _ordered(x):
    """int64 that orders as the fp32 values do."""
    i = (x + 0.0).view(torch.int32).long()
    return torch.where(i < 0, -(i & 0x7FFFFFFF), i)


def _plain_evict(s):
    c = s["case"]
    L, B, nKV, n, budget = c["L"], c["B"], c["nKV"], c["n"], c["budget"]
    s["weight"].copy_(s["weight0"])
    s["pos"].copy_(s["pos0"])
    state = [s[x] for x in ("k", "kg", "v", "vg", "weight", "pos")]
    new = s["lens"].clamp(max=budget)
    if n > budget:
        blk, off = _places(c, s["table"], B, new.device)
        blk, off = blk[None, :, None, :n], off[:n]
        l = torch.arange(L, device=new.device)[:, None, None, None]
        h = torch.arange(nKV, device=new.device)[:, None]
        w, pos = s["weight"][l, blk, h, off], s["pos"][l, blk, h, off]
        key = torch.where(pos > pos.amax(-1, keepdim=True) - c["recent"], 1 << 33, _ordered(w))
        key = key * (1 << 20) + (n - 1 - torch.arange(n, device=new.device))   # ties to the lowest slot
        kept = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, key.topk(budget, -1).indices, True)
        hole, mover = ~kept[..., :budget], kept[..., budget:]
        at = hole.nonzero(as_tuple=True)           # per head as many holes as movers, both in slot order
        fr = mover.nonzero(as_tuple=True)
        li, bi, hi = at[:3]
        dst, src = at[3], fr[3] + budget
        bd, bs_ = blk[0, bi, 0, dst], blk[0, bi, 0, src]
        for x in state:
            x[li, bd, hi, off[dst]] = x[li, bs_, hi, off[src]]
    return new, *state


def _plain_beam(s):
    c = s["case"]
    B, W, V = c["B"], c["W"], c["V"]
    x, cum, done = s["logits"], s["scores"].double(), s["done"]
    m = x.amax(-1, keepdim=True).double()
    lse = m.squeeze(-1) + (x.double() - m).exp().sum(-1).log()
    # the row's best tokens: by logit, ties to the lowest token
    k = min(W, V)
    key = _ordered(x) * (1 << 20) + (V - 1 - torch.arange(V, device=x.device))
    tok = key.topk(k, -1).indices
    val = cum[:, None] + (x.gather(-1, tok).double() - lse[:, None])
    # a finished beam goes on as itself; a dead one offers its first tokens
    first = torch.arange(k, device=x.device).expand(B * W, k)
    only = torch.where(first == 0, EOS, first - (first <= EOS).long())
    tok = torch.where(done[:, None], only, tok)
    val = torch.where(done[:, None], torch.where(first == 0, cum[:, None], -math.inf), val)
    dead = ~torch.isfinite(val).any(-1, keepdim=True)
    tok = torch.where(dead, first, tok)
    val = torch.where(torch.isfinite(val), val, -math.inf).view(B, W * k)
    flat = (tok.view(B, W, k) + V * torch.arange(W, device=x.device)[:, None]).view(B, W * k)
    flat, by = flat.sort(-1)
    val, order = val.gather(-1, by).sort(dim=-1, descending=True, stable=True)
    flat = flat.gather(-1, order)[:, :W]
    parent, token = flat // V, flat % V
    ended = done.view(B, W).gather(-1, parent) | (token == EOS)
    return val[:, :W].float(), token.int(), parent.int(), ended


def _plain_reorder(s):
    c = s["case"]
    B, W, n = c["B"], c["W"], c["n"]
    state = [s[x] for x in ("k", "kg", "v", "vg")]
    blk, off = _places(c, s["table"], B * W, s["k"].device)
    blk, off = blk[:, :n], off[:n]
    src = (s["parents"].long() + W * torch.arange(B, device=blk.device)[:, None]).view(-1)
    for x in state:
        x[:, blk, :, off] = x[:, blk[src], :, off]
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    c = s["case"]
    op = c["op"]
    if not own:
        return {"attn": _plain_attn, "put": _plain_put, "evict": _plain_evict, "beam": _plain_beam,
                "reorder": _plain_reorder}[op](s)
    F = _fw()
    if op == "attn":
        weight = s.get("weight")
        out = F.kv4Attention(s["q"], s["k"], s["kg"], s["v"], s["vg"], s["lens"], table=s["table"], weight=weight)
        return (out, weight) if c["track"] else out
    if op == "put":
        F.kv4Put(s["qkv"], c["nH"], s["positions"], s["slots"], s["k"], s["kg"], s["v"], s["vg"], T=c["T"],
                 theta=THETA, table=s["table"])
        k, v = F.kv4Values(s["k"], s["kg"], s["v"], s["vg"], c["dH"], s["slots"], c["T"], table=s["table"])
        return s["qkv"][:, :c["nH"] * c["dH"]], k, v
    if op == "evict":
        s["weight"].copy_(s["weight0"])
        s["pos"].copy_(s["pos0"])
        new = F.kv4Evict(s["k"], s["kg"], s["v"], s["vg"], s["weight"], s["pos"], s["lens"], c["budget"], c["recent"],
                         table=s["table"])
        return new, s["k"], s["kg"], s["v"], s["vg"], s["weight"], s["pos"]
    if op == "beam":
        return F.beamStep(s["logits"], s["scores"], s["done"], c["W"], EOS)
    state = [s["k"], s["kg"], s["v"], s["vg"]]
    F.cacheReorder(state, s["parents"], s["lens"], table=s["table"])
    return state


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    op = c["op"]
    if op == "beam":
        n = c["B"] * c["W"] * c["V"]
        return {"bytes": 4 * n + 22 * c["B"] * c["W"], "flops": 3 * n}
    row = 2 * (c["dH"] / 2 + 4) * c["nKV"]     # a slot's codes and grids, k and v, all kv heads
    if op == "attn":
        slots = sum(_lens_of(c))
        io = 8 * c["B"] * c["nH"] * c["dH"]
        return {"bytes": slots * (row + 8 * c["nKV"] * c["track"]) + io, "flops": 4 * slots * c["nH"] * c["dH"]}
    if op == "put":
        rows = c["B"] * c["T"]
        moved = 4 * c["dH"] * (2 * c["nH"] + 2 * c["nKV"] + 2 * c["nKV"]) + row   # q both ways, k and v in, their values out
        return {"bytes": rows * moved, "flops": rows * c["dH"] * (3 * c["nH"] + 13 * c["nKV"])}
    if op == "evict":
        n, m, r = c["n"], c["budget"], c["recent"]
        heads = c["L"] * c["B"] * c["nKV"]
        if n <= m:
            moves = 0.0
        elif c["fresh"]:   # the recent slots are the last ones, the others anywhere
            tail = min(r, n - m)
            moves = tail + (m - r) * max(0, n - r - m) / max(1, n - r)
        else:
            moves = m * (n - m) / n
        # both inputs are read whole and kept; the moved slots' rows move
        return {"bytes": heads * (16 * n + moves * 2 * (row / c["nKV"] + 8)), "flops": heads * n}
    W = c["W"]
    moved = W - 1                                       # of W beams, for independent parents
    read = W * (1 - (1 - 1 / W) ** (W - 1))             # different beams that some other beam copies
    return {"bytes": c["L"] * c["B"] * c["n"] * row * (moved + read), "flops": 0}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def _np(x):
    return x.cpu().numpy() if x.dtype != torch.bfloat16 else x.float().cpu().numpy()


def _slots64(codes, grid, blocks, n, dH):
    """Values [nKV, n, dH] in 64 bits of one sequence whose blocks are given."""
    cd = codes[blocks].movedim(1, 0).flatten(1, 2)[:, :n]
    gr = grid[blocks].movedim(1, 0).flatten(1, 2)[:, :n].double()
    x = torch.empty(*cd.shape[:2], 2 * cd.shape[2], dtype=torch.float64, device=cd.device)
    x[..., 0::2], x[..., 1::2] = (cd % 16).double(), (cd // 16).double()
    return gr[..., 1:2] + gr[..., 0:1] * x[..., :dH]


def _sequence_blocks(s, c, B):
    _, mb = _blocks(c)
    if s["table"] is not None:
        return s["table"].long()
    return torch.arange(B * mb, device=s["k"].device).view(B, mb)


def _exact_attn(c, s):
    g = c["nH"] // c["nKV"]
    bs, _ = _blocks(c)
    out = torch.zeros(c["B"], c["nH"], c["dH"], dtype=torch.float64, device="cuda")
    weight = s["weight"].double() if c["track"] else None
    for b, blocks in enumerate(_sequence_blocks(s, c, c["B"])):
        n = int(s["lens"][b])
        if n == 0:
            continue
        blocks = blocks[:-(-n // bs)]
        kk = _slots64(s["k"], s["kg"], blocks, n, c["dH"])
        vv = _slots64(s["v"], s["vg"], blocks, n, c["dH"])
        for h in range(c["nH"]):
            p = torch.softmax(kk[h // g] @ s["q"][b, h].double() / math.sqrt(c["dH"]), 0)
            out[b, h] = p @ vv[h // g]
            if c["track"]:
                weight[blocks, h // g] += torch.cat([p, p.new_zeros(len(blocks) * bs - n)]).view(-1, bs)
    return (out, weight) if c["track"] else out


def _exact_put(c, s):
    B, T, nH, nKV, dH = c["B"], c["T"], c["nH"], c["nKV"], c["dH"]
    x = s["qkv"].view(B, T, nH + 2 * nKV, dH).double()
    # the rotation as a product of complex numbers, with the angles' cosine and sine held in 32 bits
    place = (s["positions"].view(B, 1) + torch.arange(T, device="cuda")).double()
    e = torch.arange(dH // 2, device="cuda", dtype=torch.float64)
    angle = place[..., None] / THETA ** (2 * e / dH)
    turn = torch.complex(torch.cos(angle).float().double(), torch.sin(angle).float().double())
    z = torch.view_as_complex(x[:, :, :nH + nKV].reshape(B, T, nH + nKV, dH // 2, 2).contiguous())
    x[:, :, :nH + nKV] = torch.view_as_real(z * turn[:, :, None]).flatten(-2)
    q = x[:, :, :nH].reshape(B * T, nH * dH)

    def nearest(rows):
        rows = rows.float().double()                      # what is quantized is held in 32 bits
        base = rows.min(-1, keepdim=True).values.bfloat16().double()
        step = ((rows.max(-1, keepdim=True).values - base).clamp(min=0) / 15).float().bfloat16().double()
        t = (rows - base) / step
        low = torch.floor(t)
        up = (t - low > 0.5) | ((t - low == 0.5) & (low % 2 == 1))
        t = torch.clamp(low + up, 0, 15)
        return base + step * torch.where(step > 0, t, torch.zeros_like(t))

    return q, nearest(x[:, :, nH:nH + nKV]), nearest(x[:, :, nH + nKV:])


def _exact_evict(c, s):
    L, B, nKV, n, m = c["L"], c["B"], c["nKV"], c["n"], c["budget"]
    bs, _ = _blocks(c)
    names = ("k", "kg", "v", "vg", "weight0", "pos0")
    new = np.minimum(_np(s["lens"]), m)
    st = [s[x].clone() for x in names]
    w, pos = _np(s["weight0"]).astype(np.float64), _np(s["pos0"])
    blocks = _np(_sequence_blocks(s, c, B))
    j = np.arange(n)
    moves = []
    if n > m:
        for l in range(L):
            for b in range(B):
                for h in range(nKV):
                    pl = (blocks[b, j // bs], j % bs)
                    ww, pp = w[l, pl[0], h, pl[1]], pos[l, pl[0], h, pl[1]]
                    ww = np.where(pp > pp.max() - c["recent"], np.inf, ww)
                    stay = np.sort(np.lexsort((j, -ww))[:m])
                    come = stay[stay >= m]
                    free = np.setdiff1d(j[:m], stay[stay < m], assume_unique=True)
                    moves.append(np.stack([np.full(len(come), l), np.full(len(come), h), blocks[b, free // bs], free % bs,
                                           blocks[b, come // bs], come % bs]))
        l, h, db, do, sb, so = (torch.from_numpy(x).cuda() for x in np.concatenate(moves, 1))
        for x in st:
            x[l, db, h, do] = x[l, sb, h, so].clone()
    return torch.from_numpy(new), *(x.double() if x.is_floating_point() else x for x in st)


def _exact_beam(c, s):
    B, W, V = c["B"], c["W"], c["V"]
    lp = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[:, None]
    alone = torch.full_like(lp, -math.inf)
    alone[:, EOS] = s["scores"].double()
    lp = torch.where(s["done"][:, None], alone, lp)
    lp = torch.where(torch.isfinite(lp), lp, torch.full_like(lp, -math.inf)).view(B, W * V)
    best, at = torch.sort(lp, dim=-1, descending=True, stable=True)
    best, at = best[:, :W], at[:, :W]
    ended = torch.gather(s["done"].view(B, W), 1, at // V) | (at % V == EOS)
    return best, (at % V).int(), (at // V).int(), ended


def _exact_reorder(c, s):
    bs, _ = _blocks(c)
    blocks = _sequence_blocks(s, c, c["B"] * c["W"])
    got = []
    for x in (s["k"], s["kg"], s["v"], s["vg"]):
        y = x.clone()
        for r in range(c["B"] * c["W"]):
            src = r // c["W"] * c["W"] + int(s["parents"].view(-1)[r])
            for i in range(-(-c["n"] // bs)):
                upto = min(bs, c["n"] - i * bs)
                y[:, blocks[r, i], :, :upto] = x[:, blocks[src, i], :, :upto]
        got.append(y.double() if y.is_floating_point() else y)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "put": _exact_put, "evict": _exact_evict, "beam": _exact_beam,
            "reorder": _exact_reorder}[case["op"]](case, s)
