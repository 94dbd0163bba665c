"""Refusals of the paged cache and beam search entry points (no GPU: every
argument error is found before any device work), and the oracle's own ground."""
import ctypes

import numpy as np
import pytest

from oracle import paged_ref as R

PTR = 256  # a non-null, aligned pointer that is never followed


def kv(ce, **change):
    c = ce._PagedKVStruct(PTR, PTR, None, None, ce.TYPE_BF16, 2, 10, 4, 16, 64, 40960, 4096, 1024, 64)
    for n, x in change.items():
        setattr(c, n, x)
    return ctypes.byref(c)


def pt(ce, **change):
    c = ce._PageTableStruct(PTR, PTR, PTR, 8, 5, 10, 16)
    for n, x in change.items():
        setattr(c, n, x)
    return ctypes.byref(c)


def refused(ce, rc, word):
    assert rc == ce.ERR_USAGE
    assert word in ce.last_error()[1], ce.last_error()


BAD_TABLES = [(dict(table=None), "null buffer"), (dict(lens=None), "null buffer"), (dict(refs=None), "null buffer"),
              (dict(seqs=0), "seqs"), (dict(seqs=8193), "seqs"), (dict(max_pages=0), "max_pages"),
              (dict(pages=0), "pages"), (dict(pages=(1 << 20) + 1), "pages"), (dict(page_size=24), "power of two"),
              (dict(page_size=0), "power of two"), (dict(page_size=2048), "power of two"),
              (dict(max_pages=1 << 28), "2^31")]
BAD_CACHES = [(dict(k=None), "null k or v"), (dict(v=None), "null k or v"), (dict(type=0), "cache type"), (dict(type=9), "cache type"), (dict(k_scale=PTR), "no scales"),
              (dict(layers=0), "layers"), (dict(pages=0), "pages"), (dict(kv_heads=0), "kv_heads"),
              (dict(page_size=12), "power of two"), (dict(head_dim=72), "head_dim"), (dict(head_dim=144), "head_dim"),
              (dict(head_dim=0), "head_dim"), (dict(k=PTR + 8), "16 bytes"), (dict(token_stride=68), "16 bytes"),
              (dict(page_stride=4097), "16 bytes")]


@pytest.mark.parametrize("change,word", BAD_TABLES)
def test_bad_tables(ce, change, word):
    L = ce.lib()
    refused(ce, L.ce_paged_resize(pt(ce), pt(ce, **change), PTR, PTR, PTR, 4, None, None, None), word)
    refused(ce, L.ce_paged_reorder(pt(ce, **change), pt(ce), PTR, 4, None, PTR, None, None), word)
    refused(ce, L.ce_paged_attention(kv(ce), 0, pt(ce, **change), PTR, None, PTR, ce.TYPE_BF16, 4, 256, 256, 1.0, PTR,
                                     1 << 30, None), word)


@pytest.mark.parametrize("change,word", BAD_CACHES)
def test_bad_caches(ce, change, word):
    L = ce.lib()
    refused(ce, L.ce_paged_attention(kv(ce, **change), 0, pt(ce), PTR, None, PTR, ce.TYPE_BF16, 4, 256, 256, 1.0, PTR,
                                     1 << 30, None), word)
    refused(ce, L.ce_paged_append(kv(ce, **change), 0, PTR, ce.TYPE_BF16, PTR, PTR, PTR, ce.TYPE_F32, 256, 256, 256, PTR,
                                  None, 3, 4, None, 0, None), word)
    other = ce._PageTableStruct(PTR + 256, PTR, PTR, 8, 5, 10, 16)
    refused(ce, L.ce_paged_reorder(ctypes.byref(other), pt(ce), PTR, 4, kv(ce, **change), PTR, None, None), word)


def test_resize_refusals(ce):
    f = ce.lib().ce_paged_resize
    refused(ce, f(None, pt(ce), PTR, PTR, PTR, 4, None, None, None), "null page table")
    refused(ce, f(pt(ce), None, PTR, PTR, PTR, 4, None, None, None), "null page table")
    refused(ce, f(pt(ce), pt(ce, seqs=9), PTR, PTR, PTR, 4, None, None, None), "same rows")
    refused(ce, f(pt(ce), pt(ce), None, PTR, PTR, 4, None, None, None), "new lengths")
    refused(ce, f(pt(ce), pt(ce), PTR, None, PTR, 4, None, None, None), "slots")
    refused(ce, f(pt(ce), pt(ce), PTR, PTR, None, 4, None, None, None), "slots")
    refused(ce, f(pt(ce), pt(ce), PTR, PTR, PTR, -1, None, None, None), "slots")


def test_reorder_refusals(ce):
    f = ce.lib().ce_paged_reorder
    other = ctypes.byref(ce._PageTableStruct(PTR + 256, PTR, PTR, 8, 5, 10, 16))
    refused(ce, f(pt(ce), pt(ce), PTR, 4, None, PTR, None, None), "must differ")
    refused(ce, f(other, pt(ce), None, 4, None, PTR, None, None), "null parents")
    refused(ce, f(other, pt(ce), PTR, 4, None, None, None, None), "null parents")
    refused(ce, f(other, pt(ce), PTR, 3, None, PTR, None, None), "whole number of groups")
    refused(ce, f(other, pt(ce), PTR, 0, None, PTR, None, None), "groups")
    refused(ce, f(other, pt(ce), PTR, 4, kv(ce, pages=11), PTR, None, None), "the block table")
    refused(ce, f(other, pt(ce), PTR, 4, kv(ce, page_size=8), PTR, None, None), "the block table")


def test_append_refusals(ce):
    f, b, w = ce.lib().ce_paged_append, ce.TYPE_BF16, ce.TYPE_F32

    def call(layer=0, qo=PTR, qt=b, q=PTR, k=PTR, v=PTR, it=w, ql=256, kl=256, vl=256, slots=PTR, pos=PTR, T=3, heads=4,
             rope=None, rl=0):
        return f(kv(ce), layer, qo, qt, q, k, v, it, ql, kl, vl, slots, pos, T, heads, rope, rl, None)

    for change, word in ((dict(layer=2), "layer 2 of 2"), (dict(layer=-1), "layer"), (dict(T=-1), "tokens"),
                         (dict(k=None), "null k"), (dict(v=None), "null k"), (dict(slots=None), "null k"),
                         (dict(q=None), "come together"), (dict(qo=None), "come together"), (dict(it=3), "q, k, v must"),
                         (dict(qt=0), "q_out must"), (dict(qt=3), "q_out must"), (dict(heads=0), "heads"),
                         (dict(rope=PTR, rl=0), "rope_len"), (dict(rope=PTR, rl=9, pos=None), "positions"),
                         (dict(q=PTR + 4), "aligned"), (dict(kl=258), "multiples of 16 bytes"),
                         (dict(vl=252), "shorter"), (dict(ql=128), "shorter")):
        refused(ce, call(**change), word)
    assert call(T=0) == ce.OK


def test_attention_refusals(ce):
    f, b = ce.lib().ce_paged_attention, ce.TYPE_BF16

    def call(cache=None, layer=0, table=None, out=PTR, q=PTR, io=b, heads=4, ql=256, ol=256, ws=PTR, wb=1 << 30):
        return f(cache or kv(ce), layer, table or pt(ce), out, None, q, io, heads, ql, ol, 1.0, ws, wb, None)

    for change, word in ((dict(layer=2), "layer"), (dict(table=pt(ce, pages=9)), "the block table"),
                         (dict(table=pt(ce, page_size=32)), "the block table"), (dict(q=None), "null q"),
                         (dict(out=None), "null q"), (dict(io=ce.TYPE_F16), "cache's type"),
                         (dict(io=ce.TYPE_F32), "cache's type"), (dict(io=ce.TYPE_E4M3), "cache's type"),
                         (dict(heads=6), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"),
                         (dict(q=PTR + 2), "aligned"), (dict(ql=260), "multiples of 8"), (dict(ol=128), "at least"),
                         (dict(ws=None), "workspace"), (dict(wb=0), "workspace"), (dict(ws=PTR + 1), "workspace")):
        refused(ce, call(**change), word)


def test_beam_refusals(ce):
    L = ce.lib()
    n = ctypes.c_size_t()
    for shape in ((0, 4, 100), (1, 0, 100), (1, 33, 100), (1, 4, 0)):
        refused(ce, L.ce_beam_workspace(*shape, ctypes.byref(n)), "beams in [1, 32]")
    refused(ce, L.ce_beam_workspace(1, 4, 100, None), "null")

    def call(so=PTR, pa=PTR, to=PTR, fo=PTR, lg=PTR, ty=ce.TYPE_F32, ld=100, sc=PTR, fi=PTR, B=1, K=4, V=100, ws=PTR,
             wb=1 << 30):
        return L.ce_beam_select(so, pa, to, fo, lg, ty, ld, sc, fi, B, K, V, 2, 0, ws, wb, None)

    for change, word in ((dict(so=None), "null"), (dict(pa=None), "null"), (dict(to=None), "null"), (dict(fo=None), "null"),
                         (dict(lg=None), "null"), (dict(sc=None), "null"), (dict(fi=None), "null"), (dict(ty=3), "logits"),
                         (dict(ld=99), "row stride"), (dict(K=33), "beams"), (dict(B=16385), "batch"),
                         (dict(ws=None), "workspace"), (dict(wb=8), "workspace"), (dict(ws=PTR + 4), "workspace")):
        refused(ce, call(**change), word)


def test_oracle_attention_is_a_mean_of_the_values():
    """Equal keys weigh equally: the output is the mean of the values, lse the
    score plus log n; the result does not depend on which pages hold the row."""
    rng = np.random.default_rng(0)
    k, v = np.ones((5, 1, 4, 8)), rng.standard_normal((5, 1, 4, 8))
    q = np.ones((1, 2, 8))
    out, lse, _, _ = R.attention(q, k, v, np.array([[3, 1, 4]]), [10], 4, 0.5)
    rows = np.concatenate([v[3, 0], v[1, 0], v[4, 0]])[:10]
    assert np.allclose(out, rows.mean(0)) and np.allclose(lse, 4.0 + np.log(10))


def test_oracle_beam_search_finds_the_best_sequences():
    """Over a first-order chain, beams as wide as the vocabulary squared find
    the exhaustive best sequences of three tokens."""
    rng = np.random.default_rng(1)
    V, K = 3, 9
    table = rng.standard_normal((V, V))
    logp = table - np.log(np.exp(table).sum(-1, keepdims=True))
    scores = np.full((1, K), -np.inf)
    scores[0, 0] = 0.0
    last, hist = np.zeros(K, int), [[] for _ in range(K)]
    for _ in range(3):
        s, parents, tokens, _ = R.beam_select(table[last], scores.astype(np.float32), np.zeros((1, K), bool), -1, 0)
        hist = [hist[p] + [t] for p, t in zip(parents[0], tokens[0])]
        scores, last = s, tokens[0]
    best = sorted(((logp[0, a] + logp[a, b] + logp[b, c], [a, b, c]) for a in range(V) for b in range(V) for c in range(V)),
                  reverse=True)[:K]
    assert [h for _, h in best] == hist
    assert np.allclose([s for s, _ in best], scores[0], atol=1e-5)


def test_resize_refuses_a_capacity_whose_numbers_would_overflow(ce):
    """A warp numbers 128 tokens at once: from 2^31 - 127 on the last ones
    would be negative and index before the outputs."""
    f = ce.lib().ce_paged_resize
    for capacity in (2 ** 31 - 127, 2 ** 31 - 1):
        refused(ce, f(pt(ce), pt(ce), PTR, PTR, PTR, capacity, None, None, None), "capacity")


def test_reorder_refuses_too_large_a_page_before_any_launch(ce):
    """1,023 tokens of 2^18 heads are more 16-byte pieces than the copy counts;
    the tables must not have changed by then."""
    table = dict(page_size=1024, max_pages=5)
    other = ce._PageTableStruct(PTR + 256, PTR, PTR, 8, 5, 10, 1024)
    cache = kv(ce, page_size=1024, kv_heads=1 << 18, head_stride=65536, page_stride=1 << 34, layer_stride=1 << 35)
    refused(ce, ce.lib().ce_paged_reorder(ctypes.byref(other), pt(ce, **table), PTR, 4, cache, PTR, None, None),
            "too large")


def test_beam_selection_refuses_outputs_over_inputs(ce):
    """Scores or flags in place, or one element into the other's memory."""
    f, n = ce.lib().ce_beam_select, 12  # 3 x 4 beams
    at = dict(so=0x1000, pa=0x2000, to=0x3000, fo=0x4000, sc=0x5000, fi=0x6000, lg=0x10000, ws=0x80000)

    def call(**change):
        a = dict(at, **change)
        return f(a["so"], a["pa"], a["to"], a["fo"], a["lg"], ce.TYPE_F32, 128, a["sc"], a["fi"], 3, 4, 100, 2, 0, a["ws"],
                 1 << 30, None)

    end = 0x10000 + 4 * (11 * 128 + 100)  # of the logits
    for change in (dict(so=at["sc"]), dict(so=at["sc"] + 4 * n - 4), dict(so=at["sc"] - 4 * n + 4), dict(fo=at["fi"]),
                   dict(fo=at["fi"] + n - 1), dict(fi=at["to"] + 3), dict(pa=at["sc"]), dict(to=0x10000), dict(so=end - 4)):
        refused(ce, call(**change), "over an input")
