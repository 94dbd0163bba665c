"""The paged beam search program (cuda-elastic_b200/paged_beam.py): logits over
the paged cache against the library's contiguous-cache model on the same
weights, greedy decoding as one beam, and beam scores against a plain fp32
forward of the returned sequences."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CFG = dict(dim=256, hidden_dim=512, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, seq_len=128)


@pytest.fixture(scope="module")
def pb(ce):
    from cuda_elastic_b200 import paged_beam
    return paged_beam


def plain_logits(w, cfg, tokens, cache=None):
    """fp32 forward of one sequence, every position's logits; `cache`: the
    keys (turned) and values [layers][T][kv_heads][hs] to attend to in the
    place of its own."""
    f = {k: [m.float().cpu() for m in v] if isinstance(v, list) else v.float().cpu() for k, v in w.items()}
    D, H, Hk, T = cfg["dim"], cfg["n_heads"], cfg["n_kv_heads"], len(tokens)
    hs = D // H
    ang = torch.arange(T)[:, None].double() * 10000.0 ** (-torch.arange(0, hs, 2).double() / hs)
    c, s = ang.cos().float()[:, None], ang.sin().float()[:, None]

    def norm(x, g):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * g

    def rope(x):
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)

    x = f["tok_emb"][torch.tensor(tokens)]
    for l in range(cfg["n_layers"]):
        q, k, v = (norm(x, f["rms_att"][l]) @ f["wqkv"][l].T).view(T, H + 2 * Hk, hs).split((H, Hk, Hk), 1)
        k, v = (rope(k), v) if cache is None else (cache[0][l], cache[1][l])
        k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
        a = torch.einsum("qhd,khd->hqk", rope(q), k) / hs ** 0.5
        a = a.masked_fill(torch.ones(T, T).triu(1).bool(), float("-inf")).softmax(-1)
        x = x + torch.einsum("hqk,khd->qhd", a, v).reshape(T, D) @ f["wo"][l].T
        g, u = (norm(x, f["rms_ffn"][l]) @ f["w13"][l].T).unflatten(1, (-1, 2)).unbind(-1)
        x = x + (torch.nn.functional.silu(g) * u) @ f["w2"][l].T
    return norm(x, f["rms_final"]) @ f["wcls"].T


def rel(a, b):
    return float((a - b).norm() / b.norm())


def cached(m, row):
    """A row's keys and values as they stand in the cache, decoded."""
    n, page = int(m.pt.lens[row]), m.pt.page_size
    ids = m.pt.table[row, :-(-n // page)].long()
    out = []
    for pool, scale in ((m.kv.k, m.kv.k_scale), (m.kv.v, m.kv.v_scale)):
        x = pool.float()[:, ids]  # [layers][pages][kv_heads][page][hs]
        x = x if scale is None else x * scale[:, None, None]
        out.append(x.permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :n].cpu())
    return out


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_prefill_logits_of_ragged_prompts(pb, dev, cache):
    """Against an fp32 forward that attends to the cache as it is stored, so
    that only the bf16 operands of two layers' products differ: the library's
    own bound for a bf16 GEMM, 1e-2, for each layer. The bf16 cache agrees
    with the forward's own keys and values within the same bound."""
    w = pb.PagedLlama.random_weights(CFG, 1, std=0.08)
    m = pb.PagedLlama(CFG, w, 5, 64, page_size=8, cache=cache)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 512, n).tolist() for n in (1, 7, 8, 9, 40)]
    rows = [3, 0, 4, 1, 2]
    got = m.prefill(prompts, rows)
    m.ce.device_status()
    for i, p in enumerate(prompts):
        assert rel(got[i].cpu(), plain_logits(w, CFG, p, cached(m, rows[i]))[-1]) <= 2e-2
        if cache == "bf16":
            assert rel(got[i].cpu(), plain_logits(w, CFG, p)[-1]) <= 2e-2
    assert m.pt.lens.tolist() == [7, 9, 40, 1, 8]
    m.release()
    assert int(m.pt.refs.abs().sum()) == 0 and int(m.pt.lens.sum()) == 0


def test_logits_match_the_contiguous_cache_model(ce, pb, dev, tmp_path):
    """One token a step through ce_llama (its own cache and attention) and
    through the pages, from one llama2.c checkpoint."""
    from cuda_elastic_b200 import convert_weights as cw
    cfg = dict(CFG)
    rng = np.random.default_rng(2)
    D, F, V, L, kvd = cfg["dim"], cfg["hidden_dim"], cfg["vocab_size"], cfg["n_layers"], 128

    def r(*s):
        return (rng.standard_normal(s) * 0.06).astype(np.float32)

    t = dict(tok_emb=r(V, D), rms_att=np.ones((L, D), np.float32), wq=r(L, D, D), wk=r(L, kvd, D), wv=r(L, kvd, D),
             wo=r(L, D, D), rms_ffn=np.ones((L, D), np.float32), w1=r(L, F, D), w2=r(L, D, F), w3=r(L, F, D),
             rms_final=np.ones(D, np.float32), wcls=r(V, D))
    path = str(tmp_path / "m.bin")
    cw.write_llama2c(path, cfg, t, shared=False)
    B, steps = 3, 12
    first = rng.integers(0, V, B).astype(np.int32)
    model = ce.Llama(cfg, B, steps)
    model.load_llama2c(path)
    model.start(first, 0)
    pcfg, w = pb.PagedLlama.read_weights(path)
    m = pb.PagedLlama(pcfg, w, B, 64, page_size=4)
    tokens = torch.from_numpy(first).to(dev)
    for step in range(steps):
        model.step()
        slots, pos = m.grow(m.pt.lens + 1, B)
        logits = m.forward(tokens, slots, pos, m.pt)
        want = torch.from_numpy(model.logits())
        assert rel(logits.cpu(), want) <= 1e-2
        tokens = torch.from_numpy(model.generated()[:, step].copy()).to(dev)
    ce.llama_status()
    m.ce.device_status()
    model.close()


def test_one_beam_is_greedy(pb, dev):
    w = pb.PagedLlama.random_weights(CFG, 3, std=0.08)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 512, n).tolist() for n in (5, 17)]
    m = pb.PagedLlama(CFG, w, 2, 64, page_size=4)
    out, _ = m.beam_search(prompts, 1, 10, eos=-1)
    g = pb.PagedLlama(CFG, w, 2, 64, page_size=16)
    logits = g.prefill(prompts, [0, 1])
    for step in range(10):
        tok = logits.argmax(-1)
        assert tok.tolist() == out[:, 0, step].tolist()
        slots, pos = g.grow(g.pt.lens + 1, 2)
        logits = g.forward(tok, slots, pos, g.pt)


@pytest.mark.parametrize("page", [1, 8])
def test_beam_scores_are_the_sequences_log_probabilities(pb, dev, page):
    """Each returned score is the log probability of its sequence under a
    plain fp32 forward: bf16 products put each token's log probability off by
    at most 0.05 at these sizes (logits of order 1, 1e-2 relative), 8 tokens.
    Sequences of a group differ, scores descend, and the cache ends with
    exactly the pages of the beams."""
    w = pb.PagedLlama.random_weights(CFG, 4, std=0.08)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 512, n).tolist() for n in (3, 24, 11)]
    K, steps = 4, 8
    m = pb.PagedLlama(CFG, w, 3 * K, 64, page_size=page)
    out, scores = m.beam_search(prompts, K, steps, eos=-1)
    for b, p in enumerate(prompts):
        seqs = [tuple(s) for s in out[b].tolist()]
        assert len(set(seqs)) == K
        assert all(x >= y for x, y in zip(scores[b].tolist(), scores[b].tolist()[1:]))
        for k in range(K):
            lp = plain_logits(w, CFG, p + list(seqs[k])).log_softmax(-1)
            want = sum(float(lp[len(p) - 1 + i, t]) for i, t in enumerate(seqs[k]))
            assert abs(want - scores[b, k].item()) <= 0.05 * steps
    lens = m.pt.lens.tolist()
    assert lens == [len(p) + steps - 1 for p in prompts for _ in range(K)]
    held = {x for i, n in enumerate(lens) for x in m.pt.table[i, :-(-n // page)].tolist()}
    assert held == set(torch.nonzero(m.pt.refs).view(-1).tolist())


def test_eos_freezes_a_beam(pb, dev):
    """With every token an end token, each beam ends with its first token and
    keeps its score while padding follows."""
    w = pb.PagedLlama.random_weights(CFG, 5, std=0.08)
    prompts = [[7, 8, 9]]
    m = pb.PagedLlama(CFG, w, 4, 32, page_size=8)
    first, s1 = m.beam_search(prompts, 4, 1)
    eos = int(first[0, 0, 0])
    m = pb.PagedLlama(CFG, w, 4, 32, page_size=8)
    out, s = m.beam_search(prompts, 4, 6, eos=eos, pad=99)
    done = [k for k in range(4) if out[0, k, 0].item() == eos]
    assert done and all(out[0, k, 1:].tolist() == [99] * 5 for k in done)
    assert abs(s[0, done[0]].item() - s1[0, 0].item()) < 1e-5


def test_program(dev):
    r = subprocess.run([sys.executable, os.path.join(ROOT, "cuda-elastic_b200", "paged_beam.py"), "--batch", "2", "--steps",
                        "4", "--cache", "e4m3"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert len(r.stdout.strip().splitlines()) == 2 and "log p" in r.stdout


def test_a_pool_too_small_is_reported(pb, dev):
    w = pb.PagedLlama.random_weights(CFG, 6)
    m = pb.PagedLlama(CFG, w, 4, 64, pages=3, page_size=8)
    with pytest.raises(RuntimeError, match="pool is too small"):
        m.beam_search([[1, 2, 3, 4, 5]], 4, 12, eos=-1)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_searches_one_after_the_other_on_one_model(pb, dev, cache):
    """Each as on a model of its own, whatever the cache still holds: after
    longer, shorter and equally long sequences, in a pool with room for one
    search only."""
    w = pb.PagedLlama.random_weights(CFG, 7, std=0.08)
    rng = np.random.default_rng(7)
    K, page, top = 3, 8, 48

    def model():
        return pb.PagedLlama(CFG, w, 2 * K, top, pages=2 * K * (top // page), page_size=page, cache=cache)

    m = model()
    for lengths, steps in (((5, 12), 6), ((3, 2), 20), ((40, 33), 8), ((40, 33), 8), ((23, 4), 3)):
        prompts = [rng.integers(0, 512, n).tolist() for n in lengths]
        out, scores = m.beam_search(prompts, K, steps, eos=-1)
        want, wscores = model().beam_search(prompts, K, steps, eos=-1)
        assert torch.equal(out, want) and torch.equal(scores, wscores)
        assert m.pt.lens.tolist() == [n + steps - 1 for n in lengths for _ in range(K)]


def test_prompts_into_rows_that_hold_a_sequence(pb, dev):
    """A longer, a shorter and an equally long one; the row between keeps its own."""
    w = pb.PagedLlama.random_weights(CFG, 8, std=0.08)
    rng = np.random.default_rng(8)
    m, fresh = (pb.PagedLlama(CFG, w, 4, 64, page_size=8) for _ in range(2))
    m.prefill([rng.integers(0, 512, n).tolist() for n in (10, 30, 9, 21)], [0, 1, 2, 3])
    kept = cached(m, 2)
    prompts = [rng.integers(0, 512, n).tolist() for n in (24, 7, 21)]
    got, want = m.prefill(prompts, [0, 1, 3]), fresh.prefill(prompts, [0, 1, 3])
    m.ce.device_status()
    assert torch.equal(got, want) and m.pt.lens.tolist() == [24, 7, 9, 21]
    assert all(torch.equal(a, b) for a, b in zip(kept, cached(m, 2)))
    for r in (0, 1, 3):
        assert all(torch.equal(a, b) for a, b in zip(cached(m, r), cached(fresh, r)))
    assert int(m.refused) == 0 and int(m.pt.refs.sum()) == 3 + 1 + 2 + 3


def test_a_search_after_one_that_found_no_page(pb, dev):
    w = pb.PagedLlama.random_weights(CFG, 6)
    m = pb.PagedLlama(CFG, w, 4, 64, pages=6, page_size=8)
    with pytest.raises(RuntimeError, match="pool is too small"):
        m.beam_search([[1, 2, 3, 4, 5]], 4, 30, eos=-1)
    out, scores = m.beam_search([[1, 2, 3]], 4, 5, eos=-1)
    want, wscores = pb.PagedLlama(CFG, w, 4, 64, page_size=8).beam_search([[1, 2, 3]], 4, 5, eos=-1)
    assert torch.equal(out, want) and torch.equal(scores, wscores)


def test_prompts_that_cannot_be_read_are_refused(pb, dev):
    """Before any device work: an empty prompt has no last token, a token past
    the vocabulary would be looked up outside the embedding."""
    m = pb.PagedLlama(CFG, pb.PagedLlama.random_weights(CFG, 9), 2, 20, page_size=8)
    m.prefill([[4, 5, 6]], [1])
    for prompts, rows, word in (([[1], []], [0, 1], "1 .. 20"), ([[1] * 21], [0], "1 .. 20"), ([], [], "a row each"),
                                ([[1], [2]], [0], "a row each"), ([[1], [2]], [0, 0], "a row each"),
                                ([[1]], [2], "a row each"), ([[1]], [-1], "a row each"), ([[1, 512]], [0], "tokens"),
                                ([[-1]], [0], "tokens")):
        with pytest.raises(ValueError, match=word):
            m.prefill(prompts, rows)
    with pytest.raises(ValueError, match="pad"):
        m.beam_search([[1], [2]], 1, 3, pad=512)
    assert m.pt.lens.tolist() == [0, 3]
    out, _ = m.beam_search([[1], [2]], 1, 3, pad=-1)
    assert out.shape == (2, 1, 3)


def test_prompts_of_more_tokens_than_a_table_has_rows(pb, dev):
    """8,192 tokens are the rows of one block table: longer prompts, and several
    that are longer together, go in parts, each of which attends to what the
    parts before have cached. Against each prompt by itself, fed in two steps
    of which neither reaches the limit, and the fp32 forward."""
    cfg = dict(CFG, n_layers=1, dim=64, hidden_dim=64, n_heads=1, n_kv_heads=1)
    w = pb.PagedLlama.random_weights(cfg, 10, std=0.1)
    rng = np.random.default_rng(10)
    prompts = [rng.integers(0, 512, n).tolist() for n in (8193, 3, 8190, 2)]
    m = pb.PagedLlama(cfg, w, 4, 8200, page_size=16)
    got = m.prefill(prompts, [1, 0, 3, 2])
    m.ce.device_status()
    assert m.pt.lens.tolist() == [3, 8193, 2, 8190]
    for p, row, logits in zip(prompts, [1, 0, 3, 2], got):
        f = pb.PagedLlama(cfg, w, 1, 8200, page_size=16)
        alone = f.prefill([p[:-1]], [0])
        slots, pos = f.grow(f.pt.lens + 1, 1)
        alone = f.forward(torch.tensor(p[-1:], device=dev), slots, pos, f.pt)[0]
        assert all(torch.equal(a, b) for a, b in zip(cached(m, row), cached(f, 0)))
        assert rel(logits, alone) <= 1e-2
        if len(p) < 8193:
            assert rel(logits.cpu(), plain_logits(w, cfg, p)[-1]) <= 1e-2
