#!/usr/bin/env python3
"""Beam search over a Llama-2-shaped model with a paged key-value cache.

Usage: paged_beam.py [MODEL.bin] [--batch 4] [--beams 4] [--steps 32]
                     [--cache bf16|e4m3] [--page-size 16] [--seed 0]

Runs the paged operators together as a server would: prompts of different
lengths share one pool of pages, every beam group forks from its prompt, and
each step grows every row by a token (paged_resize), writes the new keys and
values (paged_append), attends (paged_attention), selects (beam_select) and
lets the rows follow their parents (paged_reorder). Lengths, pages, slots and
beams stay on the device; the host reads the sequences once, at the end. The
GEMMs and norms are the library's (gemm_bf16, rmsnorm_bf16); the embedding
lookup, the SwiGLU product and the residual sums are single torch operations.

With a llama2.c checkpoint the weights are its own, without one random
(110M-shaped).
"""
import argparse
import importlib.util
import os
import sys

import numpy as np
import torch


def _ce():
    """The package, also when this file is run as a program."""
    if "cuda_elastic_b200" in sys.modules:
        return sys.modules["cuda_elastic_b200"]
    here = os.path.dirname(os.path.abspath(__file__))
    spec = importlib.util.spec_from_file_location("cuda_elastic_b200", os.path.join(here, "__init__.py"),
                                                  submodule_search_locations=[here])
    mod = importlib.util.module_from_spec(spec)
    sys.modules["cuda_elastic_b200"] = mod
    spec.loader.exec_module(mod)
    return mod


NAMES = ("wqkv", "wo", "w13", "w2")
TABLE_ROWS = 8192  # rows of a block table at most


class PagedLlama:
    """bf16 weights of a Llama-2-shaped model and a paged cache for `rows`
    sequences of at most max_len tokens in `pages` pages."""

    def __init__(self, cfg, weights, rows, max_len, pages=None, page_size=16, cache="bf16", device="cuda"):
        self.ce, self.cfg, self.rows, self.max_len = _ce(), cfg, rows, max_len
        ce = self.ce
        D, H, L = cfg["dim"], cfg["n_heads"], cfg["n_layers"]
        self.hs, self.heads, self.kv_heads, self.layers = D // H, H, cfg["n_kv_heads"], L
        self.w = {k: [m.to(device) for m in v] if isinstance(v, list) else v.to(device) for k, v in weights.items()}
        cols = -(-max_len // page_size)
        pages = rows * cols if pages is None else pages
        dtype = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}[cache]
        k, v = (torch.zeros(L, pages, self.kv_heads, page_size, self.hs, device=device).to(dtype) for _ in "kv")
        scale = None
        if cache == "e4m3":  # keys and values of a normalized model are of order 1: 1/16 leaves room to 28
            scale = torch.full((self.kv_heads,), 1.0 / 16, device=device)
        self.kv = ce.PagedKV(k, v, scale, scale)
        self.pt = ce.PageTable.empty(rows, cols, pages, page_size, device)
        # the other table of paged_reorder; lengths and references are the same ones
        self.spare = ce.PageTable(torch.zeros_like(self.pt.table), self.pt.lens, self.pt.refs, page_size)
        angle = np.arange(max_len)[:, None] * 10000.0 ** (-np.arange(0, self.hs, 2) / self.hs)
        self.rope = torch.from_numpy(np.stack((np.cos(angle), np.sin(angle)), -1).astype(np.float32)).to(device)
        self.status = torch.zeros(4, dtype=torch.int32, device=device)
        self.refused = torch.zeros((), dtype=torch.int32, device=device)

    @staticmethod
    def random_weights(cfg, seed=0, std=0.02):
        g = torch.Generator().manual_seed(seed)
        D, F, V, L = cfg["dim"], cfg["hidden_dim"], cfg["vocab_size"], cfg["n_layers"]
        kvd = D // cfg["n_heads"] * cfg["n_kv_heads"]

        def m(r, c):
            return (torch.randn(r, c, generator=g) * std).to(torch.bfloat16)

        return {"tok_emb": m(V, D), "wcls": m(V, D), "rms_final": torch.ones(D), "rms_att": [torch.ones(D)] * L,
                "rms_ffn": [torch.ones(D)] * L, "wqkv": [m(D + 2 * kvd, D) for _ in range(L)],
                "wo": [m(D, D) for _ in range(L)], "w13": [m(2 * F, D) for _ in range(L)],
                "w2": [m(D, F) for _ in range(L)]}

    @staticmethod
    def read_weights(path):
        """(config, weights) of a llama2.c checkpoint (w13: w1 and w3 rows interleaved)."""
        _ce()
        from cuda_elastic_b200 import convert_weights as cw
        cfg, t, _ = cw.read_llama2c(path)

        def m(a):
            return torch.from_numpy(np.array(a, dtype=np.float32)).to(torch.bfloat16)

        L = cfg["n_layers"]
        w = {k: [m(cw.model_matrix(t, k, l)) for l in range(L)] for k in NAMES}
        w["tok_emb"], w["wcls"] = m(t["tok_emb"]), m(cw.model_matrix(t, "wcls", 0))
        for k in ("rms_att", "rms_ffn"):
            w[k] = [torch.from_numpy(np.array(t[k][l], np.float32)) for l in range(L)]
        w["rms_final"] = torch.from_numpy(np.array(t["rms_final"], np.float32))
        return cfg, w

    def _gemm(self, a, w):
        out = torch.empty(a.shape[0], w.shape[0], device=a.device)
        return self.ce.gemm_bf16(out, a, w)

    def _norm(self, x, w):
        return self.ce.rmsnorm_bf16(None, torch.empty_like(x, dtype=torch.bfloat16), x, w)

    def grow(self, new_lens, capacity):
        """Gives the rows their new lengths; slots and positions of the new tokens."""
        dev = self.rope.device
        slots = torch.empty(capacity, dtype=torch.int64, device=dev)
        pos = torch.empty(capacity, dtype=torch.int32, device=dev)
        self.ce.paged_resize(self.pt, new_lens, slots, pos, status=self.status)
        self.refused += self.status[1]
        return slots, pos

    def forward(self, tokens, slots, pos, pt):
        """Logits [tokens][vocab] of new tokens whose cache places are `slots`;
        pt: one row per token, its length ending with that token."""
        ce, w, T = self.ce, self.w, tokens.numel()
        H, Hk, hs = self.heads, self.kv_heads, self.hs
        x = w["tok_emb"][tokens.long()].float()
        q = torch.empty(T, H, hs, dtype=torch.bfloat16, device=x.device)
        att = torch.empty_like(q)
        for l in range(self.layers):
            qkv = self._gemm(self._norm(x, w["rms_att"][l]), w["wqkv"][l]).view(T, H + 2 * Hk, hs)
            ce.paged_append(self.kv, q, qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:], slots, pos, self.rope, layer=l)
            ce.paged_attention(self.kv, att, q, pt, layer=l)
            x = x + self._gemm(att.view(T, H * hs), w["wo"][l])
            gate, up = self._gemm(self._norm(x, w["rms_ffn"][l]), w["w13"][l]).unflatten(1, (-1, 2)).unbind(-1)
            x = x + self._gemm((torch.nn.functional.silu(gate) * up).to(torch.bfloat16), w["w2"][l])
        return self._gemm(self._norm(x, w["rms_final"]), w["wcls"])

    def prefill(self, prompts, rows):
        """Writes the prompts (lists of tokens) into the cache rows `rows`,
        whose old sequences end; the last token's logits of each. Every prompt
        token attends as a row of its own, with the block table of its prompt
        and the length up to it."""
        dev = self.rope.device
        lens = [len(p) for p in prompts]
        if not prompts or len(rows) != len(prompts) or len(set(rows)) != len(rows) or not all(0 <= r < self.rows for r in rows):
            raise ValueError(f"prompts need a row each of 0 .. {self.rows - 1} (got {len(prompts)} for rows {list(rows)})")
        if not all(0 < n <= self.max_len for n in lens):
            raise ValueError(f"prompts must have 1 .. {self.max_len} tokens (got {lens})")
        if not all(0 <= t < self.cfg["vocab_size"] for p in prompts for t in p):
            raise ValueError(f"prompt tokens must be in 0 .. {self.cfg['vocab_size'] - 1}")
        new = torch.full((self.rows,), -1, dtype=torch.int32)
        new[torch.tensor(rows)] = 0
        self.grow(new.to(dev), 0)
        new[torch.tensor(rows)] = torch.tensor(lens, dtype=torch.int32)
        order = sorted(range(len(rows)), key=lambda i: rows[i])  # tokens are numbered row by row
        tokens = torch.tensor([t for i in order for t in prompts[i]], device=dev)
        slots, pos = self.grow(new.to(dev), tokens.numel())
        owner = torch.tensor([rows[i] for i in order for _ in prompts[i]], device=dev)
        last = np.cumsum([lens[i] for i in order]) - 1  # the tokens whose logits are wanted
        logits = []
        for a in range(0, tokens.numel(), TABLE_ROWS):
            part = slice(a, a + TABLE_ROWS)
            pt = self.ce.PageTable(self.pt.table[owner[part]].contiguous(), pos[part] + 1, self.pt.refs, self.pt.page_size)
            wanted = torch.tensor(last[(last >= a) & (last < part.stop)] - a, device=dev)
            logits.append(self.forward(tokens[part], slots[part], pos[part], pt)[wanted])
        back = torch.empty(len(rows), dtype=torch.long, device=dev)
        back[torch.tensor(order, device=dev)] = torch.arange(len(rows), device=dev)
        return torch.cat(logits)[back]

    def beam_search(self, prompts, beams, steps, eos=2, pad=0):
        """Generates `steps` tokens for every prompt: (sequences int32
        [batch][beams][steps], log probabilities [batch][beams]), best first.
        What the cache held before ends; the new sequences stay in it."""
        ce, dev, B, V = self.ce, self.rope.device, len(prompts), self.cfg["vocab_size"]
        if B * beams != self.rows:
            raise ValueError(f"{B} prompts x {beams} beams need a cache of {B * beams} rows (has {self.rows})")
        if not -V <= pad < V:  # a finished beam's next tokens, looked up in the embedding like any
            raise ValueError(f"pad must be a token of the vocabulary of {V} (got {pad})")
        self.release()
        self.refused.zero_()
        logits = self.prefill(prompts, list(range(0, self.rows, beams))).repeat_interleave(beams, 0)
        scores = torch.full((B, beams), float("-inf"), device=dev)
        scores[:, 0] = 0.0  # the other beams part from the first
        finished = torch.zeros(B, beams, dtype=torch.bool, device=dev)
        scores2, finished2 = torch.empty_like(scores), torch.empty_like(finished)
        parents, tokens = (torch.empty(B, beams, dtype=torch.int32, device=dev) for _ in "pt")
        ws = ce.beam_workspace(B, beams, V, dev)
        out = torch.empty(B, beams, 0, dtype=torch.int32, device=dev)
        for step in range(steps):
            ce.beam_select(scores2, parents, tokens, finished2, logits, scores, finished, eos, pad, ws)
            scores, scores2, finished, finished2 = scores2, scores, finished2, finished
            out = torch.cat((out.gather(1, parents.long()[..., None].expand(-1, -1, step)), tokens[..., None]), 2)
            if step + 1 == steps:
                break
            ce.paged_reorder(self.pt, parents.view(-1), beams, self.spare, kv=self.kv, status=self.status)
            self.refused += self.status[1]
            self.pt, self.spare = self.spare, self.pt
            slots, pos = self.grow(self.pt.lens + 1, self.rows)
            logits = self.forward(tokens.view(-1), slots, pos, self.pt)
        ce.device_status()
        if int(self.refused):
            raise RuntimeError(f"the pool is too small: {int(self.refused)} rows found no page")
        return out, scores

    def release(self):
        """Ends every sequence: its pages are free again."""
        z = torch.zeros(self.rows, dtype=torch.int32, device=self.rope.device)
        self.grow(z, 0)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("model", nargs="?")
    for name, default in (("batch", 4), ("beams", 4), ("steps", 32), ("page-size", 16), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--cache", choices=("bf16", "e4m3"), default="bf16")
    a = ap.parse_args(argv)
    if a.model:
        cfg, w = PagedLlama.read_weights(a.model)
    else:
        cfg = dict(dim=768, hidden_dim=2048, n_layers=12, n_heads=12, n_kv_heads=12, vocab_size=32000, seq_len=1024)
        w = PagedLlama.random_weights(cfg, a.seed)
    rng = np.random.default_rng(a.seed)
    prompts = [rng.integers(3, cfg["vocab_size"], 5 + 11 * i % 40).tolist() for i in range(a.batch)]
    longest = max(map(len, prompts)) + a.steps
    m = PagedLlama(cfg, w, a.batch * a.beams, longest, page_size=a.page_size, cache=a.cache)
    out, scores = m.beam_search(prompts, a.beams, a.steps)
    for b in range(a.batch):
        print(f"prompt {b} ({len(prompts[b])} tokens): log p {scores[b, 0].item():.3f}: "
              f"{' '.join(map(str, out[b, 0].tolist()))}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
