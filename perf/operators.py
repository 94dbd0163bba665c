"""Operators of paged beam-search decoding: what is measured, on which sizes.

Five operators make one decoding step over a paged key-value cache:

  resize   request lengths -> block tables, slot map and positions (ce.paged_resize)
  append   rotary positions on q and k, k and v into their slots     (ce.paged_append)
  attend   attention of one new token per sequence over its pages    (ce.paged_attention)
  select   the best beams x tokens of a beam search                  (ce.beam_select)
  reorder  sequences follow their parent beam, partly filled pages
           are copied                                                (ce.paged_reorder)

`run` computes a case in its plain form (elementary torch operations in 32
bits) or, where `own` is true, by the library's entry point on the same inputs.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
NEG = float("-inf")


def _ce():
    from __graft_entry__ import load_package
    return load_package()


# ---------------------------------------------------------------------------
# Cases

def listed():
    return [
        # One user of the 110M-shaped model (12 heads of 64): the call is all latency.
        dict(name="attend one user", op="attend", seqs=1, top=512, kv_heads=12, group=1, dim=64, page=16,
             cache="bf16", io="bf16", layout="hnd"),
        # The 7B-shaped decode batch (64 sequences, 32 heads of 128), lengths up to 1024.
        dict(name="attend 7B batch", op="attend", seqs=64, top=1024, kv_heads=32, group=1, dim=128, page=16,
             cache="bf16", io="bf16", layout="hnd"),
        # A few long documents with grouped heads; the longest has an odd length past 100,000.
        dict(name="attend long documents", op="attend", seqs=6, top=100003, kv_heads=8, group=4, dim=128, page=64,
             cache="bf16", io="bf16", layout="hnd"),
        # An 8-bit cache in token-major pages, an odd group and a head size that is no power of two.
        dict(name="attend 8-bit cache", op="attend", seqs=96, top=3001, kv_heads=3, group=5, dim=96, page=32,
             cache="e4m3", io="f16", layout="nhd"),
        # One decoded token for each of 64 sequences, from the fp32 rows of a QKV product.
        dict(name="append one token each", op="append", tokens=64, heads=32, kv_heads=32, dim=128, page=16,
             io="f32", out="bf16", cache="bf16", layout="hnd"),
        # Prompts of a prefill, 16-bit rows into an 8-bit cache.
        dict(name="append prompts", op="append", tokens=8190, heads=32, kv_heads=8, dim=128, page=16,
             io="bf16", out="bf16", cache="e4m3", layout="nhd"),
        # A decode step of 64 sequences: each one token longer.
        dict(name="resize decode step", op="resize", seqs=64, top=1024, page=16, pages=4096, admit=0, ended=0),
        # A busy server: 1021 requests, most decoding, some ended, 60 prompts let in.
        dict(name="resize admission", op="resize", seqs=1021, top=2000, page=16, pages=98304, admit=60, ended=48),
        # The four beams of one user over the Llama-2 vocabulary.
        dict(name="select 4 beams", op="select", batch=1, beams=4, vocab=32000, io="f32"),
        # 64 users with eight beams each.
        dict(name="select batch", op="select", batch=64, beams=8, vocab=32000, io="f32"),
        # The four beams of one user of the 110M-shaped model, prompt shared.
        dict(name="reorder 4 beams", op="reorder", batch=1, beams=4, prompt=301, grown=37, page=16, layers=12,
             kv_heads=12, dim=64, cache="bf16", layout="hnd"),
        # 16 users with eight beams each, 32 layers of grouped heads.
        dict(name="reorder batch", op="reorder", batch=16, beams=8, prompt=511, grown=130, page=16, layers=32,
             kv_heads=8, dim=128, cache="bf16", layout="hnd"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "append", "resize", "select", "reorder"))
    if op == "attend":
        dim, group = rng.choice((32, 48, 64, 80, 96, 112, 128)), rng.choice((1, 1, 2, 3, 4, 4, 5, 7, 8, 12, 16))
        cache, kv_heads = rng.choice(("bf16", "bf16", "f16", "e4m3")), rng.choice((1, 2, 3, 4, 5, 8, 12, 32))
        top = _log(rng, 1, 131072)
        room = 1 << 30  # bytes of keys and values at most, by this bound on the number of sequences
        seqs = _log(rng, 1, max(1, min(512, room // (top * kv_heads * dim * 4))))
        return dict(op=op, seqs=seqs, top=top, kv_heads=kv_heads, group=group, dim=dim,
                    page=rng.choice((8, 16, 32, 64, 128)), cache=cache,
                    io=cache if cache != "e4m3" else rng.choice(("bf16", "f16")), layout=rng.choice(("hnd", "nhd")))
    if op == "append":
        kv_heads = rng.choice((1, 2, 4, 8, 12))
        cache = rng.choice(("bf16", "f16", "e4m3"))
        return dict(op=op, tokens=_log(rng, 1, 8000), heads=kv_heads * rng.choice((1, 2, 3, 4)), kv_heads=kv_heads,
                    dim=rng.choice((32, 48, 64, 96, 128)), page=rng.choice((8, 16, 32, 64)), io=rng.choice(("f32", "bf16", "f16")),
                    out=cache if cache != "e4m3" else rng.choice(("bf16", "f16")), cache=cache,
                    layout=rng.choice(("hnd", "nhd")))
    if op == "resize":
        seqs, page = _log(rng, 1, 2000), rng.choice((8, 16, 32, 64))
        top = _log(rng, 2, 4000)
        return dict(op=op, seqs=seqs, top=top, page=page, pages=seqs * (-(-top // page) + 1) + _log(rng, 1, 2000),
                    admit=rng.randrange(0, seqs // 4 + 1), ended=rng.randrange(0, seqs // 4 + 1))
    if op == "select":
        beams, vocab = rng.choice((1, 2, 3, 4, 5, 8, 16, 32)), _log(rng, 100, 130000)
        return dict(op=op, batch=_log(rng, 1, max(1, min(256, (64 << 20) // (beams * vocab * 4)))), beams=beams, vocab=vocab,
                    io=rng.choice(("f32", "bf16", "f16")))
    return dict(op=op, batch=_log(rng, 1, 12), beams=rng.choice((2, 3, 4, 5, 8)), prompt=_log(rng, 1, 600),
                grown=_log(rng, 1, 130), page=rng.choice((8, 16, 32)), layers=_log(rng, 1, 24),
                kv_heads=rng.choice((1, 2, 5, 8)), dim=rng.choice((48, 64, 128)), cache=rng.choice(("bf16", "f16", "e4m3")),
                layout=rng.choice(("hnd", "nhd")))


def _pages(tokens, page):
    return -(-tokens // page)


def _lengths(c):
    """Sequence lengths of an attention case: the longest is `top`, the others spread over
    (top / 2, top]; where there are eight or more, one is empty and one has a single token."""
    n, top = c["seqs"], c["top"]
    lens = [top - int(top * 0.5 * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]
    if n >= 8:
        lens[3], lens[5] = 0, 1
    return lens


def _sizes(c):
    """Old and new lengths of a resize case."""
    n, top = c["seqs"], c["top"]
    old = [1 + int((top - 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]
    new = [x + 1 for x in old]
    for i in range(c["admit"]):  # an empty row that a prompt comes into
        old[i], new[i] = 0, 1 + int((top - 1) * ((i * 0.7548776662466927) % 1.0))
    for i in range(c["admit"], c["admit"] + c["ended"]):
        new[i] = 0
    return old, new


def _survivors(c):
    """How many of a group's beams have children, and the parents before they are shuffled."""
    beams = c["beams"]
    kept = max(1, (beams * 5) // 8)
    return kept, [i % kept for i in range(beams)]


def work(c):
    if c["op"] == "attend":
        n = sum(_lengths(c))
        item = 1 if c["cache"] == "e4m3" else 2
        rows = c["seqs"] * c["kv_heads"] * c["group"]
        return dict(bytes=2 * n * c["kv_heads"] * c["dim"] * item + rows * c["dim"] * 4 + rows * 4 +
                    4 * sum(_pages(x, c["page"]) for x in _lengths(c)),
                    flops=4 * n * c["kv_heads"] * c["group"] * c["dim"])
    if c["op"] == "append":
        size = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
        q, kv = c["tokens"] * c["heads"] * c["dim"], 2 * c["tokens"] * c["kv_heads"] * c["dim"]
        return dict(bytes=q * (size[c["io"]] + 2) + kv * (size[c["io"]] + size[c["cache"]]) +
                    c["tokens"] * (12 + 4 * c["dim"]), flops=3 * (q + kv / 2))
    if c["op"] == "resize":
        old, new = _sizes(c)
        taken = sum(_pages(b, c["page"]) - _pages(a, c["page"]) for a, b in zip(old, new) if b > a)
        given = sum(_pages(a, c["page"]) - _pages(b, c["page"]) for a, b in zip(old, new) if b < a)
        tokens = sum(max(0, b - a) for a, b in zip(old, new))
        return dict(bytes=12 * c["seqs"] + 8 * c["pages"] + 4 * taken + 4 * given + 12 * tokens,
                    flops=c["pages"] + 2 * c["seqs"] + 4 * tokens)
    if c["op"] == "select":
        n = c["batch"] * c["beams"] * c["vocab"]
        return dict(bytes=n * (4 if c["io"] == "f32" else 2) + c["batch"] * c["beams"] * 19, flops=4 * n)
    kept, _ = _survivors(c)
    n, length = c["batch"] * c["beams"], c["prompt"] + c["grown"]
    copied = c["batch"] * (c["beams"] - kept) * (length % c["page"])
    item = 1 if c["cache"] == "e4m3" else 2
    return dict(bytes=4 * copied * c["layers"] * c["kv_heads"] * c["dim"] * item + 8 * n * _pages(length, c["page"]) +
                20 * n, flops=n * _pages(length, c["page"]))


# ---------------------------------------------------------------------------
# Inputs

def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    """Normal values rounded to dtype; made in pieces, so that no large fp32 copy is held."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        m = min(1 << 27, flat.numel() - i)
        flat[i:i + m] = (torch.randn(m, generator=g, device="cuda") * scale).to(dtype)
    return out


def _pool(g, c, layers, pages):
    """One K or V pool [layers][pages][kv_heads][page][dim]; token-major pages are a permuted view."""
    inner = (c["kv_heads"], c["page"]) if c["layout"] == "hnd" else (c["page"], c["kv_heads"])
    p = _randn(g, layers, pages, *inner, c["dim"], dtype=DT[c["cache"]], scale=16.0 if c["cache"] == "e4m3" else 1.0)
    return p if c["layout"] == "hnd" else p.transpose(2, 3)


def _scales(g, c):
    """Decode scales of an 8-bit cache, one per head, such that the values are about N(0, 1)."""
    if c["cache"] != "e4m3":
        return None, None
    return tuple((0.75 + 0.5 * torch.rand(c["kv_heads"], generator=g, device="cuda")) / 16.0 for _ in range(2))


def _shuffled(g, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")[torch.randperm(len(values), generator=g, device="cuda")]


def prepare(c, seed):
    s = {"case": c}
    g = _gen(seed)
    dev = "cuda"
    if c["op"] == "attend":
        lens = _shuffled(g, _lengths(c))
        P = max(1, _pages(c["top"], c["page"]))
        used = sum(_pages(x, c["page"]) for x in _lengths(c))
        pages = used + used // 16 + 1
        perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        col = torch.arange(P, device=dev)[None]
        held = (lens[:, None] + c["page"] - 1) // c["page"]
        at = torch.cumsum(held.view(-1), 0)[:, None] - held + col
        s["table"] = torch.where(col < held, perm[at.clamp(max=pages - 1)], 0).to(torch.int32).contiguous()
        s["lens"] = lens
        s["k"], s["v"] = _pool(g, c, 1, pages), _pool(g, c, 1, pages)
        s["ks"], s["vs"] = _scales(g, c)
        s["q"] = _randn(g, c["seqs"], c["kv_heads"] * c["group"], c["dim"], dtype=DT[c["io"]], scale=1.5)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(c["seqs"], c["kv_heads"] * c["group"], device=dev)
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device=dev)
        if own:
            ce = _ce()
            s["pt"] = ce.PageTable(s["table"], s["lens"], s["refs"], c["page"])
            s["kv"] = ce.PagedKV(s["k"], s["v"], s["ks"], s["vs"])
    elif c["op"] == "append":
        T, H, Hk, D = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        pages = _pages(T, c["page"]) + 3
        s["k"], s["v"] = _pool(g, c, 1, pages), _pool(g, c, 1, pages)
        s["ks"], s["vs"] = _scales(g, c)
        s["qkv"] = _randn(g, T, (H + 2 * Hk) * D, dtype=DT[c["io"]])
        s["q"] = s["qkv"][:, :H * D].view(T, H, D)
        s["kn"] = s["qkv"][:, H * D:(H + Hk) * D].view(T, Hk, D)
        s["vn"] = s["qkv"][:, (H + Hk) * D:].view(T, Hk, D)
        slots = torch.randperm(pages * c["page"], generator=g, device=dev)[:T]
        slots[T // 2] = -1 if T > 1 else slots[0]  # a token that is left out
        s["slots"] = slots.contiguous()
        s["pos"] = torch.randint(0, 4096, (T,), generator=g, device=dev, dtype=torch.int32)
        angle = torch.arange(4096, device=dev, dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)[None]
        s["rope"] = torch.stack((angle.cos(), angle.sin()), -1).float().contiguous()
        s["q_out"] = torch.empty(T, H, D, dtype=DT[c["out"]], device=dev)
        if own:
            s["kv"] = _ce().PagedKV(s["k"], s["v"], s["ks"], s["vs"])
    elif c["op"] == "resize":
        old, new = _sizes(c)
        order = torch.randperm(c["seqs"], generator=g, device=dev)
        old = torch.tensor(old, dtype=torch.int32, device=dev)[order]
        s["lens"], s["new"] = old, torch.tensor(new, dtype=torch.int32, device=dev)[order]
        P = _pages(c["top"] + 1, c["page"])
        perm = torch.randperm(c["pages"], generator=g, device=dev).to(torch.int32)
        held = (old[:, None] + c["page"] - 1) // c["page"]
        col = torch.arange(P, device=dev)[None]
        at = torch.cumsum(held.view(-1), 0)[:, None] - held + col
        s["table"] = torch.where(col < held, perm[at.clamp(max=c["pages"] - 1)], 0).to(torch.int32).contiguous()
        s["refs"] = torch.zeros(c["pages"], dtype=torch.int32, device=dev)
        s["refs"][perm[:int(held.sum())].long()] = 1
        a, b = _sizes(c)
        T = sum(max(0, y - x) for x, y in zip(a, b))
        s["slots"] = torch.empty(max(1, T), dtype=torch.int64, device=dev)
        s["pos"] = torch.empty(max(1, T), dtype=torch.int32, device=dev)
        s["starts"] = torch.empty(c["seqs"] + 1, dtype=torch.int32, device=dev)
        s["status"] = torch.empty(4, dtype=torch.int32, device=dev)
        s["lens_out"], s["refs_out"] = torch.empty_like(s["lens"]), torch.empty_like(s["refs"])
        if own:
            ce = _ce()
            s["pt"] = ce.PageTable(s["table"], s["lens"], s["refs"], c["page"])
            s["to"] = ce.PageTable(s["table"], s["lens_out"], s["refs_out"], c["page"])
    elif c["op"] == "select":
        B, K, V = c["batch"], c["beams"], c["vocab"]
        s["logits"] = _randn(g, B * K, V, dtype=DT[c["io"]], scale=2.5)
        s["logits"][:, 2::97] = NEG  # banned tokens
        s["scores"] = -20.0 * torch.rand(B, K, generator=g, device=dev)
        s["scores"][::5, 1:] = NEG  # prompts whose beams have not parted yet
        s["finished"] = torch.rand(B, K, generator=g, device=dev) < 0.15
        s["o"] = (torch.empty(B, K, device=dev), torch.empty(B, K, dtype=torch.int32, device=dev),
                  torch.empty(B, K, dtype=torch.int32, device=dev), torch.empty(B, K, dtype=torch.bool, device=dev))
        if own:
            s["ws"] = _ce().beam_workspace(B, K, V)
    else:
        B, K, ps = c["batch"], c["beams"], c["page"]
        n, length = B * K, c["prompt"] + c["grown"]
        P, shared = _pages(length, ps), c["prompt"] // ps
        pages = B * shared + n * (P - shared) + n + 5
        perm = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        row, col = torch.arange(n, device=dev)[:, None], torch.arange(P, device=dev)[None]
        at = torch.where(col < shared, row // K * shared + col, B * shared + row * (P - shared) + col - shared)
        s["table"] = perm[at].contiguous()
        s["lens"] = torch.full((n,), length, dtype=torch.int32, device=dev)
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device=dev)
        s["refs"].index_add_(0, s["table"].view(-1).long(), torch.ones(n * P, dtype=torch.int32, device=dev))
        _, parents = _survivors(c)
        relabel = torch.argsort(torch.rand(B, K, generator=g, device=dev), 1)
        spots = torch.argsort(torch.rand(B, K, generator=g, device=dev), 1)
        p = torch.tensor(parents, device=dev).expand(B, K).gather(1, spots)
        s["parents"] = relabel.gather(1, p).to(torch.int32).view(-1).contiguous()
        s["k"], s["v"] = _pool(g, c, c["layers"], pages), _pool(g, c, c["layers"], pages)
        s["table_out"] = torch.zeros_like(s["table"])
        s["lens_out"], s["refs_out"] = torch.empty_like(s["lens"]), torch.empty_like(s["refs"])
        s["copies"] = torch.empty(n, 2, dtype=torch.int32, device=dev)
        s["status"] = torch.empty(4, dtype=torch.int32, device=dev)
        if own:
            ce = _ce()
            s["pt"] = ce.PageTable(s["table"], s["lens"], s["refs"], ps)
            s["to"] = ce.PageTable(s["table_out"], s["lens_out"], s["refs_out"], ps)
            s["kv"] = ce.PagedKV(s["k"], s["v"], *_scales(g, c))
    return s


# ---------------------------------------------------------------------------
# The operators' plain forms

def _bytes_of(t):
    """8-bit floating point tensors are indexed as bytes."""
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _plain_attend(s):
    c = s["case"]
    B, Hk, G, D = c["seqs"], c["kv_heads"], c["group"], c["dim"]
    L = s["table"].shape[1] * c["page"]

    def rows(pool, scale):
        x = _bytes_of(pool)[0][s["table"].long()].view(pool.dtype)  # [B][P][Hk][page][D]
        x = x.permute(0, 2, 1, 3, 4).reshape(B, Hk, L, D).float()
        return x if scale is None else x * scale[None, :, None, None]

    q = s["q"].float().view(B, Hk, G, D)
    w = q @ rows(s["k"], s["ks"]).transpose(-1, -2) * (1.0 / math.sqrt(D))
    w = w.masked_fill(torch.arange(L, device=w.device) >= s["lens"][:, None, None, None], NEG)
    m = w.amax(-1, keepdim=True)
    w = torch.exp(w - m.masked_fill(m == NEG, 0.0))
    l = w.sum(-1, keepdim=True)
    o = w @ rows(s["v"], s["vs"]) / l.masked_fill(l == 0, 1.0)
    return {"out": o.view(B, Hk * G, D).to(DT[c["io"]]), "lse": (m + l.log()).view(B, Hk * G)}


def _plain_append(s):
    c = s["case"]
    keep = s["slots"] >= 0
    page, off = s["slots"][keep] // c["page"], s["slots"][keep] % c["page"]
    cs = s["rope"][s["pos"].long()]  # [T][D / 2][2]

    def turned(x):
        a, b = x.float().unflatten(-1, (-1, 2)).unbind(-1)
        cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)

    def stored(x, scale):
        x = x if scale is None else (x / scale[None, :, None]).clamp(-448.0, 448.0)
        return _bytes_of(x[keep].to(DT[c["cache"]]))

    _bytes_of(s["k"])[0][page, :, off] = stored(turned(s["kn"]), s["ks"])
    _bytes_of(s["v"])[0][page, :, off] = stored(s["vn"].float(), s["vs"])
    q = turned(s["q"]) * keep[:, None, None]
    return {"q": q.to(DT[c["out"]]), "k": s["k"], "v": s["v"]}


def _plain_resize(s):
    c = s["case"]
    ps, table, refs = c["page"], s["table"], s["refs"].clone()
    old, new = s["lens"], torch.where(s["new"] < 0, s["lens"], s["new"])
    P, cap = table.shape[1], s["slots"].numel()
    col = torch.arange(P, device=table.device)[None]
    have, want = (old + ps - 1) // ps, (new + ps - 1) // ps
    back = (col >= want[:, None]) & (col < have[:, None])
    refs.index_add_(0, table[back].long(), -torch.ones_like(table[back]))
    grow = new > old
    tail = refs[table.gather(1, (old // ps).clamp(max=P - 1).long()[:, None])[:, 0].long()]
    fits = grow & (want <= P) & ((old % ps == 0) | (tail == 1))
    need, more = torch.where(fits, want - have, 0), torch.where(fits, new - old, 0)
    free = torch.nonzero(refs == 0)[:, 0].to(torch.int32)
    given = fits & (need.cumsum(0) <= free.numel()) & (more.cumsum(0) <= cap)
    need, more = torch.where(given, need, 0), torch.where(given, more, 0)
    lens = torch.where(given | (new < old), new, old).to(torch.int32)
    first = need.cumsum(0) - need
    mine = (col >= have[:, None]) & (col < (have + need)[:, None])
    taken = free[(first[:, None] + col - have[:, None])[mine]]
    table[mine] = taken
    refs[taken.long()] = 1
    ends = more.cumsum(0)
    starts = torch.cat((ends.new_zeros(1), ends)).to(torch.int32)
    j = torch.arange(cap, device=table.device)
    r = torch.searchsorted(ends, j, right=True).clamp(max=old.numel() - 1)
    pos = old[r] + j - starts[r]
    page = table[r, (pos // ps).clamp(0, P - 1)].long()
    live = j < ends[-1]
    status = torch.stack((need.sum(), (grow & ~given).sum(), free.numel() - need.sum(), ends[-1])).to(torch.int32)
    return {"table": table, "lens": lens, "refs": refs, "slots": torch.where(live, page * ps + pos % ps, -1),
            "pos": torch.where(live, pos, -1).to(torch.int32), "starts": starts, "status": status}


def _plain_select(s):
    c = s["case"]
    B, K, V = c["batch"], c["beams"], c["vocab"]
    x = torch.nan_to_num(s["logits"].float(), nan=NEG, posinf=torch.finfo(torch.float32).max, neginf=NEG)
    m = x.amax(-1, keepdim=True)
    lse = m + torch.exp(x - m.masked_fill(m == NEG, 0.0)).sum(-1, keepdim=True).log()
    n = min(K, V)
    best, token = torch.sort(x, dim=-1, descending=True, stable=True)
    best, token = best[:, :n], token[:, :n]  # of each beam, ties to the lowest token
    step = (best - lse).masked_fill(best == NEG, NEG).view(B, K, n)
    token, done = token.view(B, K, n), s["finished"][..., None]
    score = torch.where(done, torch.where(torch.arange(n, device=x.device) == 0, s["scores"][..., None], math.nan),
                        s["scores"][..., None] + step).view(B, K * n)
    token = torch.where(done, 0, token).view(B, K * n)
    order = torch.nan_to_num(score, nan=NEG, posinf=math.inf, neginf=NEG)
    rank = torch.sort(torch.where(torch.isnan(score), 1, 0), dim=-1, stable=True).indices  # a finished beam's empty places last
    pick = rank.gather(1, torch.sort(order.gather(1, rank), dim=-1, descending=True, stable=True).indices[:, :K])
    parent, token = (pick // n).to(torch.int32), token.gather(1, pick).to(torch.int32)
    over = s["finished"].gather(1, parent.long())
    return {"scores": score.gather(1, pick), "parents": parent, "tokens": token, "finished": over | (token == 2)}


def _plain_reorder(s):
    c = s["case"]
    B, K, ps = c["batch"], c["beams"], c["page"]
    n, P = s["table"].shape
    col = torch.arange(P, device=s["table"].device)[None]
    row = torch.arange(n, device=col.device)
    parent = row // K * K + s["parents"]
    lens, rows = s["lens"][parent], s["table"][parent]
    refs = s["refs"].clone()
    held = col < ((s["lens"] + ps - 1) // ps)[:, None]
    mine = col < ((lens + ps - 1) // ps)[:, None]
    refs.index_add_(0, s["table"][held].long(), -torch.ones_like(s["table"][held]))
    refs.index_add_(0, rows[mine].long(), torch.ones_like(rows[mine]))
    at = (lens // ps).clamp(max=P - 1).long()[:, None]
    tail, part = rows.gather(1, at)[:, 0], lens % ps != 0
    t, f = tail.view(B, K), part.view(B, K)
    same = (t[:, :, None] == t[:, None, :]) & f[:, :, None] & f[:, None, :]
    alone = refs[t.long()] == same.sum(-1)  # held by this group only: its first beam keeps the page
    first = torch.argmax(same.int(), -1) == torch.arange(K, device=col.device)
    copy = (f & ~(alone & first)).view(-1)
    free = torch.nonzero(refs == 0)[:, 0].to(torch.int32)
    copy_ok = copy & (copy.cumsum(0) <= free.numel())
    dst = torch.where(copy_ok, free[(copy_ok.cumsum(0) - 1).clamp(0, free.numel() - 1)], -1)
    src = torch.where(copy_ok, tail, -1)
    a, b = src[copy_ok].long(), dst[copy_ok].long()
    refs.index_add_(0, a, -torch.ones_like(src[copy_ok]))
    refs[b] = 1
    rows = torch.where((col == at) & copy_ok[:, None], dst[:, None], rows)
    live = torch.arange(ps, device=col.device)[None] < (lens % ps)[copy_ok][:, None]
    for pool in (s["k"], s["v"]):
        x = _bytes_of(pool)
        x[:, b] = torch.where(live[None, :, None, :, None], x[:, a], x[:, b])
    s["table_out"].copy_(torch.where(mine, rows, s["table_out"]))
    status = torch.stack((copy_ok.sum(), (copy & ~copy_ok).sum(), free.numel() - copy_ok.sum(), copy_ok.sum()))
    return {"table": s["table_out"], "lens": lens, "refs": refs, "copies": torch.stack((src, dst), 1).to(torch.int32),
            "status": status.to(torch.int32), "k": s["k"], "v": s["v"]}


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "resize": _plain_resize, "select": _plain_select,
                "reorder": _plain_reorder}[op](s)
    ce = _ce()
    if op == "attend":
        ce.paged_attention(s["kv"], s["out"], s["q"], s["pt"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "append":
        ce.paged_append(s["kv"], s["q_out"], s["q"], s["kn"], s["vn"], s["slots"], s["pos"], s["rope"])
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if op == "resize":
        ce.paged_resize(s["pt"], s["new"], s["slots"], s["pos"], starts=s["starts"], status=s["status"], out=s["to"])
        return {"table": s["table"], "lens": s["lens_out"], "refs": s["refs_out"], "slots": s["slots"],
                "pos": s["pos"], "starts": s["starts"], "status": s["status"]}
    if op == "select":
        scores, parents, tokens, over = s["o"]
        ce.beam_select(scores, parents, tokens, over, s["logits"], s["scores"], s["finished"], eos=2, pad=0, workspace=s["ws"])
        return {"scores": scores, "parents": parents, "tokens": tokens, "finished": over}
    ce.paged_reorder(s["pt"], s["parents"], s["case"]["beams"], s["to"], kv=s["kv"], copies=s["copies"], status=s["status"])
    return {"table": s["table_out"], "lens": s["lens_out"], "refs": s["refs_out"], "copies": s["copies"],
            "status": s["status"], "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------------------
# The definitions in 64 bits

def exact(c, seed):
    if c["op"] in ("resize", "reorder"):  # whole numbers, and values that are only moved
        return None
    s = prepare(c, seed)
    if c["op"] == "attend":
        H, G, D, ps = c["kv_heads"] * c["group"], c["group"], c["dim"], c["page"]
        out = torch.zeros(c["seqs"], H, D, dtype=torch.float64, device="cuda")
        lse = torch.full((c["seqs"], H), NEG, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            ids = s["table"][b, :_pages(n, ps)].long()
            for h in range(c["kv_heads"] if n else 0):
                k = _bytes_of(s["k"])[0][ids, h].view(DT[c["cache"]]).double().reshape(-1, D)[:n]
                v = _bytes_of(s["v"])[0][ids, h].view(DT[c["cache"]]).double().reshape(-1, D)[:n]
                if s["ks"] is not None:
                    k, v = k * s["ks"][h].double(), v * s["vs"][h].double()
                w = s["q"][b, h * G:(h + 1) * G].double() @ k.T / D ** 0.5
                out[b, h * G:(h + 1) * G] = torch.softmax(w, -1) @ v
                lse[b, h * G:(h + 1) * G] = torch.logsumexp(w, -1)
        return {"out": out, "lse": lse}
    if c["op"] == "append":
        cos, sin = s["rope"].double()[s["pos"].long()].unbind(-1)
        whole = torch.complex(cos, sin)[:, None]

        def turn(x):
            return torch.view_as_real(torch.view_as_complex(x.double().reshape(*x.shape[:-1], -1, 2)) * whole).flatten(-2)

        res = {"q": turn(s["q"])}
        res["q"][s["slots"] < 0] = 0
        for name, new, scale in (("k", turn(s["kn"]), s["ks"]), ("v", s["vn"].double(), s["vs"])):
            pool = s[name].double()
            new = new if scale is None else new / scale.double()[None, :, None]
            t = torch.nonzero(s["slots"] >= 0)[:, 0]
            pool[0, s["slots"][t] // c["page"], :, s["slots"][t] % c["page"]] = new[t]
            res[name] = pool
        return res
    B, K, V = c["batch"], c["beams"], c["vocab"]
    scores = torch.empty(B, K, dtype=torch.float64, device="cuda")
    for b in range(B):
        step = torch.log_softmax(s["logits"][b * K:(b + 1) * K].double(), -1)
        done = s["finished"][b]
        step[done] = NEG
        step[done, 0] = 0.0
        scores[b] = torch.topk((s["scores"][b].double()[:, None] + step).view(-1), K).values
    return {"scores": scores, "parents": None, "tokens": None, "finished": None}
