"""Beam search selection on the GPU against oracle/paged_ref.py."""
import numpy as np
import pytest
import torch

from oracle import paged_ref as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def run(ce, dev, logits, scores, finished, eos=2, pad=0, ws=None):
    B, K = scores.shape
    o = [torch.full((B, K), float("nan"), device=dev)] + [torch.full((B, K), -7, dtype=torch.int32, device=dev)
                                                         for _ in range(2)] + [torch.zeros(B, K, dtype=torch.bool, device=dev)]
    ws = ce.beam_workspace(B, K, logits.shape[1]) if ws is None else ws
    ce.beam_select(*o, logits, torch.from_numpy(scores).to(dev), torch.from_numpy(finished).to(dev), eos, pad, ws)
    ce.device_status()
    return [x.cpu().numpy() for x in o]


def check(got, want, V):
    """Scores: a logit and a base exact in fp32, the log of a sum of V fp32
    exponentials (relative error of the sum below V 2^-24 taken pairwise or
    in pieces, 2^-18 is ample for V <= 2^17), two rounded additions."""
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3])
    fin = np.isfinite(want[0])
    assert np.array_equal(got[0][~fin], want[0][~fin].astype(np.float32))
    tol = 2.0 ** -18 + 2.0 ** -21 * np.abs(want[0][fin])
    assert (np.abs(got[0][fin] - want[0][fin]) <= tol).all()


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 2), (2, 3, 31), (3, 8, 257), (2, 5, 4097), (1, 32, 9001),
                                  (9, 4, 32000), (1, 2, 128256), (40, 16, 1000)])
def test_select(ce, dev, io, B, K, V):
    rng = np.random.default_rng(V + K)
    logits = torch.from_numpy(rng.standard_normal((B * K, V)).astype(np.float32) * 2.5).to(dev).to(DT[io])
    scores = (-20 * rng.random((B, K))).astype(np.float32)
    finished = rng.random((B, K)) < 0.2
    got = run(ce, dev, logits, scores, finished)
    check(got, R.beam_select(logits.float().cpu().numpy(), scores, finished, 2, 0), V)


def test_ties_go_to_the_lowest_token_and_beam(ce, dev):
    B, K, V = 2, 6, 20000
    logits = torch.zeros(B * K, V, device=dev)  # all equal
    scores, finished = np.zeros((B, K), np.float32), np.zeros((B, K), bool)
    got = run(ce, dev, logits, scores, finished, eos=-1)
    assert (got[1] == 0).all() and (got[2] == np.arange(K)).all() and not got[3].any()
    logits[:, [17, 4095, 4096, 19999, 11]] = 3.0  # five ties, across any split of the row
    logits[0, 5] = -0.0
    got = run(ce, dev, logits, scores, finished, eos=4095)
    assert (got[1] == [0, 0, 0, 0, 0, 1]).all() and (got[2] == [11, 17, 4095, 4096, 19999, 11]).all()
    assert (got[3] == [False, False, True, False, False, False]).all()


def test_ties_across_tiles_of_long_rows(ce, dev):
    """So many rows that each is one CTA's: ties between the first tile, later
    ones and the row's last elements (odd vocabulary) go to the lowest token;
    16-bit logits are full of them."""
    rng = np.random.default_rng(8)
    B, K, V = 100, 6, 12007
    x = torch.from_numpy((rng.standard_normal((B * K, V)) * 2).astype(np.float32)).to(dev).to(torch.bfloat16)
    x[::3, [5, 4100, 8200, V - 1, V - 2]] = 9.0
    x[1::3] = x[1::3].clamp(max=5.0)  # a plateau of the largest value
    x[2::12] = -1.5  # nothing but ties: 12,007 candidates
    scores, finished = -rng.random((B, K)).astype(np.float32), rng.random((B, K)) < 0.1
    check(run(ce, dev, x, scores, finished), R.beam_select(x.float().cpu().numpy(), scores, finished, 2, 0), V)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("B,K,V", [(3, 16, 50001), (2, 24, 128256), (1, 32, 95351), (4, 9, 70003), (32, 32, 20011)])
def test_many_beams(ce, dev, io, B, K, V):
    """Rows of several slices, and slices of several tiles, with many offers."""
    rng = np.random.default_rng(V)
    logits = torch.from_numpy(rng.standard_normal((B * K, V)).astype(np.float32) * 2.5).to(dev).to(DT[io])
    logits[1::5, ::3] = logits[1::5, 1:2]  # a third of the row equal
    scores = (-20 * rng.random((B, K))).astype(np.float32)
    finished = rng.random((B, K)) < 0.2
    got = run(ce, dev, logits, scores, finished)
    check(got, R.beam_select(logits.float().cpu().numpy(), scores, finished, 2, 0), V)


def test_very_long_rows_of_one_cta(ce, dev):
    """So many rows that each is one CTA's, 74 tiles long: random, with ties,
    ascending, descending. The other rows are finished and not read. (A sum is
    one of at most 74 + 16 + 13 additions in sequence: 2^-17.3 of it.)"""
    rng = np.random.default_rng(3)
    B, K, V = 56, 8, 300001
    x = torch.empty(B * K, V, dtype=torch.bfloat16, device=dev)
    finished = np.ones((B, K), bool)
    finished[[0, 55]] = False
    rows = np.flatnonzero(finished.ravel() == 0)
    part = (rng.standard_normal((len(rows), V)) * 2).astype(np.float32)
    part[2] = np.linspace(-9, 9, V)
    part[3] = part[2, ::-1]
    part[4, [7, 5000, 13000, 29000, 60000, 130000, 270000, V - 1]] = 12
    part[5, 257 * 1000:] += 6
    x[torch.from_numpy(rows).to(dev)] = torch.from_numpy(part).to(dev).to(torch.bfloat16)
    scores = -rng.random((B, K)).astype(np.float32)
    got = run(ce, dev, x, scores, finished)
    part = torch.from_numpy(part).to(torch.bfloat16).float().numpy()
    check([g[[0, 55]] for g in got], R.beam_select(part, scores[[0, 55]], finished[[0, 55]], 2, 0), V)
    assert (got[2][1:55] == 0).all() and got[3][1:55].all()


@pytest.mark.parametrize("V", [50, 9000])
def test_infinities_and_nan(ce, dev, V):
    """Banned (-inf) and NaN logits are never taken before a finite one; a row
    of them alone offers its lowest tokens at -inf; +inf is the largest value."""
    rng = np.random.default_rng(V)
    B, K = 3, 3
    x = rng.standard_normal((B * K, V)).astype(np.float32)
    x[0] = -np.inf
    x[1, 2:] = np.nan
    x[2, ::3] = -np.inf
    x[3:6] = np.nan
    x[6, 7] = np.inf
    x[7, [8, V - 1]] = np.inf
    x[8] = -3.4e38
    scores = np.array([[-1, -2, -3], [0, -np.inf, np.nan], [-np.inf, -1, -np.inf]], np.float32)
    finished = np.zeros((B, K), bool)
    got = run(ce, dev, torch.from_numpy(x).to(dev), scores, finished)
    check(got, R.beam_select(x, scores, finished, 2, 0), V)


def test_finished_beams_keep_their_score(ce, dev):
    B, K, V = 2, 4, 300
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((B * K, V)).astype(np.float32)).to(dev)
    scores = np.array([[-1, -50, -60, -70], [-3, -1, -2, -4]], np.float32)
    finished = np.array([[True, False, False, True], [True] * 4])
    got = run(ce, dev, x, scores, finished, eos=2, pad=99)
    check(got, R.beam_select(x.cpu().numpy(), scores, finished, 2, 99), V)
    assert (got[0][0, 0], got[1][0, 0], got[2][0, 0], got[3][0, 0]) == (-1.0, 0, 99, True)
    assert got[0][1].tolist() == [-1, -2, -3, -4] and got[1][1].tolist() == [1, 2, 0, 3] and got[3][1].all()


def test_rows_apart_and_odd(ce, dev):
    """A row stride larger than the vocabulary, rows that are not 16-byte aligned."""
    rng = np.random.default_rng(6)
    for dt, V, ld in ((torch.float32, 1001, 1003), (torch.bfloat16, 777, 781), (torch.float16, 4099, 8200)):
        wide = torch.full((6, ld), 1e4, device=dev).to(dt)
        wide[:, :V] = torch.from_numpy(rng.standard_normal((6, V)).astype(np.float32)).to(dev).to(dt)
        x = wide[:, :V]
        scores, finished = -rng.random((2, 3)).astype(np.float32), np.zeros((2, 3), bool)
        check(run(ce, dev, x, scores, finished), R.beam_select(x.float().cpu().numpy(), scores, finished, 2, 0), V)
        shifted = wide.view(-1)[1:1 + 5 * ld].view(5, ld)[:2, :V]  # base off the 16-byte grid
        s1, f1 = scores[:1, :2].copy(), finished[:1, :2].copy()
        check(run(ce, dev, shifted, s1, f1), R.beam_select(shifted.float().cpu().numpy(), s1, f1, 2, 0), V)


def test_select_repeats_bit_for_bit_and_in_a_graph(ce, dev):
    rng = np.random.default_rng(7)
    B, K, V = 5, 4, 32000
    x = torch.from_numpy(rng.standard_normal((B * K, V)).astype(np.float32) * 2).to(dev)
    scores, finished = -rng.random((B, K)).astype(np.float32), rng.random((B, K)) < 0.3
    ws = ce.beam_workspace(B, K, V)
    first = run(ce, dev, x, scores, finished, ws=ws)
    for _ in range(4):
        for a, b in zip(first, run(ce, dev, x, scores, finished, ws=ws)):
            assert np.array_equal(a, b)
    ds, df = torch.from_numpy(scores).to(dev), torch.from_numpy(finished).to(dev)
    o = [torch.empty(B, K, device=dev), torch.empty(B, K, dtype=torch.int32, device=dev),
         torch.empty(B, K, dtype=torch.int32, device=dev), torch.empty(B, K, dtype=torch.bool, device=dev)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ce.beam_select(*o, x, ds, df, 2, 0, ws)
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, o):
        assert np.array_equal(a, b.cpu().numpy())


def test_select_refuses_a_workspace_that_is_not_on_the_device(ce, dev):
    """Before any launch: the kernel would follow the host pointer."""
    x = torch.zeros(2, 50, device=dev)
    scores, finished = np.zeros((1, 2), np.float32), np.zeros((1, 2), bool)
    ws = ce.beam_workspace(1, 2, 50)
    for bad in (ws.cpu(), torch.zeros(2 * ws.numel(), dtype=torch.uint8, device=dev)[::2]):
        with pytest.raises(TypeError, match="workspace"):
            run(ce, dev, x, scores, finished, ws=bad)


def test_very_large_logits(ce, dev):
    """Where the product of the largest logit and log2 e is rounded by more than
    the exponents that e^x has (1,580,999,936: by -127), and all the way up to
    the largest float, of either sign. All others lie further below than e^x
    reaches, so that the best token's score is its beam's own."""
    rng = np.random.default_rng(17)
    B, K, V = 64, 8, 5000
    x = rng.standard_normal((B * K, V)).astype(np.float32)
    top = np.exp2(rng.uniform(20, 127.9, B * K)).astype(np.float32)
    top[:200] = rng.uniform(1.5e9, 2.9e9, 200)
    top[0], top[1], top[2], top[3] = 1580999936.0, 3.4028234e38, 1048576.0, 1048577.0
    x[np.arange(B * K), rng.integers(0, V, B * K)] = top
    for r in range(0, B * K, 3):  # large negative ones
        x[r] = np.where(x[r] == top[r], -top[r], max(-2.0 * float(top[r]), -3.4e38))
    scores, finished = -rng.random((B, K)).astype(np.float32), np.zeros((B, K), bool)
    got = run(ce, dev, torch.from_numpy(x).to(dev), scores, finished)
    want = R.beam_select(x, scores, finished, 2, 0)
    assert np.isfinite(got[0]).all()
    check(got, want, V)


def test_outputs_beside_inputs(ce, dev):
    """In one allocation, next to each other, they are no overlap; in place they are refused."""
    rng = np.random.default_rng(18)
    B, K, V = 3, 4, 100
    x = torch.from_numpy(rng.standard_normal((B * K, V)).astype(np.float32)).to(dev)
    scores, finished = -rng.random((B, K)).astype(np.float32), rng.random((B, K)) < 0.3
    want = run(ce, dev, x, scores, finished)
    n = B * K
    words = torch.zeros(3 * n, device=dev)  # scores out, scores, parents' words
    flags = torch.zeros(2 * n, dtype=torch.bool, device=dev)
    so, sc, pa = (words[i * n:(i + 1) * n].view(B, K) for i in range(3))
    fi, fo = flags[:n].view(B, K), flags[n:].view(B, K)
    sc.copy_(torch.from_numpy(scores))
    fi.copy_(torch.from_numpy(finished))
    to = torch.empty(B, K, dtype=torch.int32, device=dev)
    ws = ce.beam_workspace(B, K, V)
    ce.beam_select(so, pa.view(torch.int32), to, fo, x, sc, fi, 2, 0, ws)
    for a, b in zip((so, pa.view(torch.int32), to, fo), want):
        assert np.array_equal(a.cpu().numpy(), b)
    for o in ((sc, pa.view(torch.int32), to, fo), (so, pa.view(torch.int32), to, fi), (so, sc.view(torch.int32), to, fo)):
        with pytest.raises(ce.CeError, match="over an input"):
            ce.beam_select(*o, x, sc, fi, 2, 0, ws)
