"""Plain numpy definitions (64-bit where they compute) of the paged cache and
beam search operators, one loop per row: the oracle of their tests."""
import numpy as np


def pages_of(tokens, page):
    return -(-int(tokens) // page)


def attention(q, k, v, table, lens, page, scale):
    """q [n][H][D], k and v [pages][Hk][page][D] (already decoded, float64).
    Returns out, lse and, per (row, head), the largest sum_i |q_i k_i| scale
    and sum_j p_j |v_j| (for error bounds)."""
    n, H, D = q.shape
    G = H // k.shape[1]
    out, lse = np.zeros((n, H, D)), np.full((n, H), -np.inf)
    mag, spread = np.zeros((n, H)), np.zeros((n, H, D))
    for i in range(n):
        L = int(lens[i])
        if L == 0:
            continue
        ids = table[i, :pages_of(L, page)]
        for h in range(H):
            kk = k[ids, h // G].reshape(-1, D)[:L]
            vv = v[ids, h // G].reshape(-1, D)[:L]
            with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
                s = (kk * q[i, h]).sum(-1) * scale
                m = s.max()
                p = np.exp(s - (m if np.isfinite(m) else 0.0))
                lse[i, h] = (m if np.isfinite(m) else 0.0) + np.log(p.sum())
                out[i, h] = p @ vv / p.sum()
                mag[i, h] = (np.abs(kk * q[i, h])).sum(-1).max() * scale
                spread[i, h] = p @ np.abs(vv) / p.sum()
    return out, lse, mag, spread


def resize(table, lens, refs, new_lens, page, capacity):
    """In place on copies; returns table, lens, refs, slots, pos, starts, status."""
    table, lens, refs = table.copy(), lens.copy(), refs.copy()
    n, P = table.shape
    for i in range(n):
        if 0 <= new_lens[i] < lens[i]:
            for j in range(pages_of(new_lens[i], page), pages_of(lens[i], page)):
                refs[table[i, j]] -= 1
    free = [p for p in range(len(refs)) if refs[p] == 0]
    had = len(free)
    tails = refs.copy()
    out_lens = lens.copy()
    slots, pos, starts = [], [], []
    need = tokens = refused = taken = 0
    for i in range(n):
        starts.append(len(slots))
        old, new = int(lens[i]), int(new_lens[i])
        if 0 <= new < old:
            out_lens[i] = new
        if new <= old:
            continue
        bad = pages_of(new, page) > P or (old % page and tails[table[i, old // page]] != 1)
        if not bad:
            need += pages_of(new, page) - pages_of(old, page)
            tokens += new - old
        if bad or need > had or tokens > capacity:
            refused += 1
            continue
        for j in range(pages_of(old, page), pages_of(new, page)):
            table[i, j] = free.pop(0)
            refs[table[i, j]] = 1
            taken += 1
        out_lens[i] = new
        for t in range(old, new):
            slots.append(int(table[i, t // page]) * page + t % page)
            pos.append(t)
    starts.append(len(slots))
    status = np.array([taken, refused, had - taken, len(slots)], np.int32)
    pad = [-1] * (capacity - len(slots))
    return (table, out_lens, refs, np.array(slots + pad, np.int64), np.array(pos + pad, np.int32),
            np.array(starts, np.int32), status)


def reorder(table, lens, refs, parents, beams, page):
    """Returns table, lens, refs, copies, status; table entries past a row's
    pages are -1."""
    n, P = table.shape
    refs = refs.copy()
    out, out_lens = np.full((n, P), -1, np.int32), np.zeros(n, np.int32)
    for i in range(n):
        for j in range(pages_of(lens[i], page)):
            refs[table[i, j]] -= 1
    for i in range(n):
        if 0 <= parents[i] < beams:
            src = i // beams * beams + parents[i]
            out_lens[i] = lens[src]
            for j in range(pages_of(lens[src], page)):
                out[i, j] = table[src, j]
                refs[out[i, j]] += 1
    part = [int(out[i, out_lens[i] // page]) if out_lens[i] % page else -1 for i in range(n)]
    want = []
    for i in range(n):
        if part[i] >= 0:
            g = i // beams * beams
            same = [k for k in range(g, g + beams) if part[k] == part[i]]
            if not (refs[part[i]] == len(same) and same[0] == i):
                want.append(i)
    free = [p for p in range(len(refs)) if refs[p] == 0]
    copies = np.full((n, 2), -1, np.int32)
    for i, p in zip(want, free):
        out[i, out_lens[i] // page] = p
        refs[p] = 1
        refs[part[i]] -= 1
        copies[i] = part[i], p
    done = min(len(want), len(free))
    return out, out_lens, refs, copies, np.array([done, len(want) - done, len(free) - done, done], np.int32)


def append(x, pos, rope):
    """Rotary turn of x [T][H][D] (float64) by rope [positions][D / 2][2]."""
    if rope is None:
        return x
    c, s = rope[pos, :, 0][:, None], rope[pos, :, 1][:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    out = np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = a * c - b * s, a * s + b * c
    return out


def beam_offers(logits, beams):
    """(tokens, logits, lse) of one beam: its best tokens by logit, ties to the lowest."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
    order = np.lexsort((np.arange(len(x)), -x))[:beams]
    m = x.max()
    lse = m + np.log(np.exp(x - m).sum()) if np.isfinite(m) else 0.0
    return order, x[order], lse


def beam_select(logits, scores, finished, eos, pad):
    """logits [B * K][V]; returns scores (float64), parents, tokens, finished."""
    B, K = scores.shape
    o = [np.zeros((B, K)), np.zeros((B, K), np.int32), np.zeros((B, K), np.int32), np.zeros((B, K), bool)]
    for b in range(B):
        offers = []
        for k in range(K):
            base = float(scores[b, k])
            if finished[b, k]:
                offers.append((base, k, 0, pad))
                continue
            tok, x, lse = beam_offers(logits[b * K + k], K)
            for r in range(len(tok)):
                offers.append((base + (x[r] - lse) if np.isfinite(x[r]) else -np.inf, k, r, int(tok[r])))
        offers = [(-np.inf if np.isnan(s) else s, k, r, t) for s, k, r, t in offers]
        offers.sort(key=lambda e: (-e[0], e[1], e[2]))
        for r, (s, k, _, t) in enumerate(offers[:K]):
            o[0][b, r], o[1][b, r], o[2][b, r] = s, k, t
            o[3][b, r] = finished[b, k] or t == eos
    return o
