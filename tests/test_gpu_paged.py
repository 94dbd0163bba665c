"""Paged cache operators (resize, append, attention, reorder) on the GPU
against the plain numpy definitions of oracle/paged_ref.py, in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import paged_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn, "f32": torch.float32}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half the spacing at 1: one rounding's relative error


def pool(rng, dev, dtype, layers, pages, heads, page, dim, layout, scale=1.0):
    shape = (layers, pages, heads, page, dim) if layout == "hnd" else (layers, pages, page, heads, dim)
    x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * np.float32(scale)).to(dev).to(DT[dtype])
    return x if layout == "hnd" else x.transpose(2, 3)


def host(x):
    return x.float().cpu().numpy().astype(np.float64)


def tables(rng, lens, page, extra=3, max_pages=None):
    """Random disjoint pages; what stands behind a row's pages is garbage."""
    held = [R.pages_of(x, page) for x in lens]
    pages = sum(held) + extra
    P = max(max(held), 1) if max_pages is None else max_pages
    ids = rng.permutation(pages)
    table = rng.integers(-2 ** 31, 2 ** 31 - 1, (len(lens), P)).astype(np.int32)
    refs = np.zeros(pages, np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = ids[at:at + h]
        refs[table[i, :h]] = 1
        at += h
    return table, refs


def poison(kv, table, lens, page):
    """NaN in every place of the pool that no token stands in."""
    live = torch.zeros(kv.shape[1], page, dtype=torch.bool)
    for i, n in enumerate(lens):
        for j in range(R.pages_of(n, page)):
            live[table[i, j], :min(page, n - j * page)] = True
    dead = ~live.to(kv.device)[None, :, None, :, None]
    if kv.dtype == torch.float8_e4m3fn:
        kv.view(torch.uint8).masked_fill_(dead, 0x7f)
    else:
        kv.masked_fill_(dead, float("nan"))


def attention_case(ce, dev, seed, lens, kv_heads, group, dim, page, cache, io, layout, q_scale=1.5, layers=1, layer=0,
                   strided=False, edit=None):
    rng = np.random.default_rng(seed)
    table, refs = tables(rng, lens, page)
    s8 = 16.0 if cache == "e4m3" else 1.0
    k = pool(rng, dev, cache, layers, len(refs), kv_heads, page, dim, layout, s8)
    v = pool(rng, dev, cache, layers, len(refs), kv_heads, page, dim, layout, s8)
    if edit is not None:
        edit(k, v, table)
    poison(k, table, lens, page)
    poison(v, table, lens, page)
    ks = vs = None
    if cache == "e4m3":
        ks, vs = (torch.from_numpy((rng.uniform(0.75, 1.25, kv_heads) / 16).astype(np.float32)).to(dev) for _ in "kv")
    n, H = len(lens), kv_heads * group
    wide = H * dim * 3 if strided else H * dim
    qb = torch.from_numpy(rng.standard_normal((n, wide)).astype(np.float32) * np.float32(q_scale)).to(dev).to(DT[io])
    ob = torch.full((n, wide), float("nan"), dtype=DT[io], device=dev)
    q, out = qb[:, :H * dim].view(n, H, dim), ob[:, :H * dim].view(n, H, dim)
    lse = torch.full((n, H), float("nan"), device=dev)
    dl = torch.tensor(lens, dtype=torch.int32, device=dev)
    pt = ce.PageTable(torch.from_numpy(table).to(dev), dl, torch.from_numpy(refs).to(dev), page)
    kv = ce.PagedKV(k, v, ks, vs)
    ce.paged_attention(kv, out, q, pt, lse=lse, layer=layer)
    ce.device_status()
    hk, hv = host(k[layer]), host(v[layer])
    if ks is not None:
        hk *= host(ks)[None, :, None, None]
        hv *= host(vs)[None, :, None, None]
    want, wlse, mag, spread = R.attention(host(q), hk, hv, table, lens, page, dim ** -0.5)
    if strided:
        assert torch.isnan(ob[:, H * dim:]).all()
    return out, lse, want, wlse, mag, spread, (kv, pt, q)


def check_attention(io, dim, lens, out, lse, want, wlse, mag, spread):
    """Bounds, from the arithmetic: a score is a dot product of dim exact
    products summed in fp32 and scaled, |error| <= (dim + 16) 2^-22 mag (four
    times the unit roundoff per term, the tensor core's sum included); e^s
    then is off by that relative amount plus 2^-16 (weights enter the product
    with the values in two 16-bit parts), twice over for numerator and
    denominator, plus the sums' own n 2^-24; the output is rounded once."""
    n = np.array([max(1, x) for x in lens])[:, None]
    score = (dim + 16) * 2.0 ** -22 * mag + 2.0 ** -22
    rel = 2.0 * (score + 2.0 ** -16) + n * 2.0 ** -22
    tol = rel[..., None] * (spread + np.abs(want)) + UNIT[io] * np.abs(want) * (1 + rel[..., None]) + 2.0 ** -25
    err = np.abs(host(out) - want)
    assert (err <= tol).all(), (err / np.maximum(tol, 1e-30)).max()
    live = np.array(lens) > 0
    lerr = np.abs(host(lse)[live] - wlse[live])
    ltol = (score + n * 2.0 ** -22 + 2.0 ** -16 + 2.0 ** -22 * np.abs(wlse))[live]
    assert (lerr <= ltol).all(), (lerr / ltol).max()
    assert (host(lse)[~live] == -np.inf).all() and (host(out)[~live] == 0).all()


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("e4m3", "bf16"), ("e4m3", "f16")]


@pytest.mark.parametrize("cache,io", TYPES)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 128])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_attention_types_and_dims(ce, dev, cache, io, dim, layout):
    lens = [0, 1, 15, 16, 17, 33, 130, 0, 257]
    r = attention_case(ce, dev, dim, lens, 2, 3, dim, 16, cache, io, layout)
    check_attention(io, dim, lens, *r[:6])


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (3, 1), (1, 7), (2, 8), (2, 9), (1, 16), (1, 17), (2, 40)])
@pytest.mark.parametrize("cache,io,dim", [("bf16", "bf16", 128), ("e4m3", "f16", 64)])
def test_attention_head_groups(ce, dev, kv_heads, group, cache, io, dim):
    lens = [40, 3, 0, 100]
    r = attention_case(ce, dev, group, lens, kv_heads, group, dim, 16, cache, io, "hnd")
    check_attention(io, dim, lens, *r[:6])


@pytest.mark.parametrize("page", [1, 2, 8, 16, 32, 256, 1024])
def test_attention_page_sizes(ce, dev, page):
    lens = [1, 2, page, page + 1, max(1, page - 1), 70]
    r = attention_case(ce, dev, page, lens, 2, 2, 64, page, "bf16", "bf16", "nhd")
    check_attention("bf16", 64, lens, *r[:6])


@pytest.mark.parametrize("lens", [[5001], [4096, 0, 0, 1], [3000, 2999, 17], [1] * 300, [0, 0, 0]])
@pytest.mark.parametrize("group,dim", [(1, 128), (4, 64), (12, 128)])
def test_attention_split_and_joined(ce, dev, lens, group, dim):
    """One long row is shared by many warps and CTAs, short rows share one."""
    r = attention_case(ce, dev, len(lens), lens, 2, group, dim, 16, "f16", "f16", "hnd")
    check_attention("f16", dim, lens, *r[:6])


def test_attention_many_rows(ce, dev):
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 40, 1500).tolist()
    r = attention_case(ce, dev, 1, lens, 1, 2, 32, 8, "bf16", "bf16", "hnd")
    check_attention("bf16", 32, lens, *r[:6])


def test_attention_layers_and_strides(ce, dev):
    """A middle layer; q and out as slices of wider rows."""
    lens = [9, 0, 250, 31]
    r = attention_case(ce, dev, 3, lens, 2, 2, 64, 16, "bf16", "bf16", "nhd", layers=3, layer=1, strided=True)
    check_attention("bf16", 64, lens, *r[:6])


def test_attention_large_scores(ce, dev):
    """Scores of several hundred: the running maximum keeps e^s in range."""
    lens = [700, 33, 2]
    r = attention_case(ce, dev, 4, lens, 2, 4, 128, 16, "f16", "f16", "hnd", q_scale=60.0)
    check_attention("f16", 128, lens, *r[:6])


def test_attention_minus_infinity_scores(ce, dev):
    """Keys whose score is -inf weigh nothing, a whole leading tile of them
    included; a row that has only such keys is 0 / 0, as the formula says."""
    lens = [100, 20]

    def edit(k, v, table):
        for j in range(3):
            k[0, int(table[0, j]), :, :, 0] = float("-inf")  # positions 0 .. 47 of row 0
        for j in range(2):
            k[0, int(table[1, j]), :, :, 0] = float("-inf")  # all of row 1

    rng = np.random.default_rng(9)
    table, refs = tables(rng, lens, 16)
    k, v = (pool(rng, dev, "bf16", 1, len(refs), 1, 16, 64, "hnd") for _ in "kv")
    edit(k, v, table)
    q = torch.from_numpy(rng.standard_normal((2, 2, 64)).astype(np.float32)).to(dev).to(torch.bfloat16)
    q[:, :, 0] = 1.0
    out, lse = torch.empty_like(q), torch.empty(2, 2, device=dev)
    pt = ce.PageTable(torch.from_numpy(table).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                      torch.from_numpy(refs).to(dev), 16)
    ce.paged_attention(ce.PagedKV(k, v), out, q, pt, lse=lse)
    ce.device_status()
    hk = host(k[0])
    hk[np.isinf(hk)] = -1e30  # weight 0 in 64 bits, without inf * 0
    want, wlse, mag, spread = R.attention(host(q), hk, host(v[0]), table, lens, 16, 0.125)
    mag = np.full_like(mag, 40.0)
    check_attention("bf16", 64, lens[:1], out[:1], lse[:1], want[:1], wlse[:1], mag[:1], spread[:1])
    assert torch.isnan(out[1]).all() and (lse[1] == float("-inf")).all()


def test_attention_repeats_bit_for_bit(ce, dev):
    """The join adds the parts in their order, whichever CTA comes last; the
    workspace is ready for the next call of another shape."""
    lens = [6000, 100, 1, 2500]
    out, lse, *_, (kv, pt, q) = attention_case(ce, dev, 5, lens, 2, 4, 128, 16, "bf16", "bf16", "hnd")
    first, first_lse = out.clone(), lse.clone()
    short = torch.tensor([7, 0, 1, 300], dtype=torch.int32, device=dev)
    pt2 = ce.PageTable(pt.table, short, pt.refs, pt.page_size)
    for _ in range(5):
        ce.paged_attention(kv, out, q, pt2, lse=lse)
        ce.paged_attention(kv, out, q, pt, lse=lse)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)
    ce.device_status()


def test_attention_on_a_side_stream_and_in_a_graph(ce, dev):
    lens = [600, 31, 0, 90]
    out, lse, *_, (kv, pt, q) = attention_case(ce, dev, 6, lens, 2, 4, 64, 16, "bf16", "bf16", "hnd")
    want = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = torch.full_like(out, float("nan"))
    with torch.cuda.stream(side):
        ce.paged_attention(kv, other, q, pt, workspace=ce.paged_attention_workspace())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ce.paged_attention(kv, other, q, pt)
    for _ in range(3):
        other.fill_(float("nan"))
        g.replay()
        assert torch.equal(other, want)
    pt.lens.copy_(torch.tensor([0, 31, 0, 12], dtype=torch.int32))  # the graph reads lengths on the device
    g.replay()
    assert (other[0] == 0).all() and torch.equal(other[1], want[1]) and not torch.equal(other[3], want[3])


def test_attention_reports_bad_tables(ce, dev):
    """A page outside the pool reads as zeros, a length past the row is cut;
    both are reported, neither faults, and the other rows are right."""
    lens = [40, 64, 20]
    rng = np.random.default_rng(7)
    out, lse, want, wlse, mag, spread, (kv, pt, q) = attention_case(ce, dev, 7, lens, 2, 2, 64, 16, "bf16", "bf16", "hnd")
    good = out.clone()
    pt.table[2, 1] = pt.pages  # one past the end
    ce.paged_attention(kv, out, q, pt, lse=lse)
    with pytest.raises(ce.CeError) as e:
        ce.device_status()
    assert e.value.status == ce.ERR_USAGE and "page id" in str(e.value)
    assert torch.equal(out[:2], good[:2]) and torch.isfinite(out[2].float()).all()
    pt.table[2, 1] = pt.table[0, 0]
    pt.lens[1] = 2 ** 31 - 1
    ce.paged_attention(kv, out, q, pt, lse=lse)
    with pytest.raises(ce.CeError) as e:
        ce.device_status()
    assert e.value.status == ce.ERR_USAGE and "length" in str(e.value)
    assert torch.equal(out[:2], good[:2])  # row 1 holds max_pages pages: cut to the 64 it has
    pt.lens[1] = -5
    ce.paged_attention(kv, out, q, pt, lse=lse)
    with pytest.raises(ce.CeError):
        ce.device_status()
    assert (out[1] == 0).all() and torch.equal(out[0], good[0])
    ce.device_status()


def test_attention_offsets_past_32_bits(ce, dev):
    """Pages whose byte and element offsets pass 2^32: 33,000 pages of
    16 x 64 x 128 elements are 4.3 G elements (8.6 GB) per pool."""
    pages, heads, page, dim = 33000, 64, 16, 128
    k = torch.zeros(1, pages, heads, page, dim, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    rng = np.random.default_rng(8)
    ids = [32990, 5, 32999]
    for p in ids:
        for x in (k, v):
            x[0, p] = torch.from_numpy(rng.standard_normal((heads, page, dim)).astype(np.float32)).to(dev).to(torch.bfloat16)
    table = torch.tensor([ids], dtype=torch.int32, device=dev)
    lens = [45]
    pt = ce.PageTable(table, torch.tensor(lens, dtype=torch.int32, device=dev),
                      torch.zeros(pages, dtype=torch.int32, device=dev), page)
    q = torch.from_numpy(rng.standard_normal((1, heads, dim)).astype(np.float32)).to(dev).to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(1, heads, device=dev)
    kv = ce.PagedKV(k, v)
    ce.paged_attention(kv, out, q, pt, lse=lse)
    r = R.attention(host(q), host(k[0, ids]), host(v[0, ids]), np.array([[0, 1, 2]]), lens, page, dim ** -0.5)
    check_attention("bf16", dim, lens, out, lse, *r)
    slot = torch.tensor([32999 * 16 + 13], dtype=torch.int64, device=dev)
    new = torch.ones(1, heads, dim, device=dev)
    ce.paged_append(kv, None, None, new, 2 * new, slot)
    ce.device_status()
    assert (k[0, 32999, :, 13] == 1).all() and (v[0, 32999, :, 13] == 2).all() and (k[0, 32999, :, 14] != 1).any()


# ---------------------------------------------------------------------------
# append

@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cache,out", [("bf16", "bf16"), ("f16", "f16"), ("e4m3", "f16"), ("bf16", "f16")])
@pytest.mark.parametrize("dim,heads,kv_heads,layout", [(64, 6, 3, "hnd"), (16, 1, 1, "nhd"), (128, 8, 1, "nhd")])
def test_append(ce, dev, io, cache, out, dim, heads, kv_heads, layout):
    check_append(ce, dev, io, cache, out, dim, heads, kv_heads, layout, 37, 9)


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cache,out", [("bf16", "bf16"), ("f16", "bf16"), ("e4m3", "f16")])
@pytest.mark.parametrize("dim,heads,kv_heads,layout", [(128, 33, 8, "hnd"), (80, 40, 11, "nhd"), (128, 46, 1, "nhd")])
def test_append_of_many_tokens(ce, dev, io, cache, out, dim, heads, kv_heads, layout):
    """Enough tokens and heads for a thread to take several heads, with and
    without a remainder."""
    check_append(ce, dev, io, cache, out, dim, heads, kv_heads, layout, 901, 115)


def check_append(ce, dev, io, cache, out, dim, heads, kv_heads, layout, T, pages):
    rng = np.random.default_rng(dim + heads)
    page, layers = 8, 2
    k, v = (pool(rng, dev, cache, layers, pages, kv_heads, page, dim, layout) for _ in "kv")
    before = [host(x) for x in (k, v)]
    qkv = torch.from_numpy(rng.standard_normal((T, (heads + 2 * kv_heads) * dim)).astype(np.float32) * 3).to(dev).to(DT[io])
    q = qkv[:, :heads * dim].view(T, heads, dim)
    kn = qkv[:, heads * dim:(heads + kv_heads) * dim].view(T, kv_heads, dim)
    vn = qkv[:, (heads + kv_heads) * dim:].view(T, kv_heads, dim)
    slots = rng.permutation(pages * page)[:T].astype(np.int64)
    slots[[3, T - 1]] = -1
    pos = rng.integers(0, 50, T).astype(np.int32)
    ang = np.arange(50)[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)
    rope = torch.from_numpy(np.stack((np.cos(ang), np.sin(ang)), -1).astype(np.float32)).to(dev)
    scales = [None, None]
    if cache == "e4m3":
        scales = [torch.from_numpy(rng.uniform(0.01, 0.05, kv_heads).astype(np.float32)).to(dev) for _ in "kv"]
    q_out = torch.full((T, heads, dim), float("nan"), dtype=DT[out], device=dev)
    kv = ce.PagedKV(k, v, *scales)
    ce.paged_append(kv, q_out, q, kn, vn, torch.from_numpy(slots).to(dev), torch.from_numpy(pos).to(dev), rope, layer=1)
    ce.device_status()
    live = slots >= 0
    hr = host(rope)
    # fp32: two products and a sum, each rounded (3 x 2^-24 of |a c| + |b s|
    # <= 1.5 |pair|), then one rounding to the output type
    wq = R.append(host(q), pos, hr)
    pair = np.repeat(np.abs(host(q)).reshape(T, heads, -1, 2).max(-1), 2, -1).reshape(wq.shape)
    tol = UNIT[out] * np.abs(wq) + 2.0 ** -21 * pair + 2.0 ** -25
    assert (np.abs(host(q_out)[live] - wq[live]) <= tol[live]).all()
    assert (host(q_out)[~live] == 0).all()
    for x, new, was, turn, scale in ((k, kn, before[0], True, scales[0]), (v, vn, before[1], False, scales[1])):
        w = R.append(host(new), pos, hr if turn else None)
        mag = np.repeat(np.abs(host(new)).reshape(T, kv_heads, -1, 2).max(-1), 2, -1).reshape(w.shape)
        if scale is not None:
            w, mag = w / host(scale)[None, :, None], mag / host(scale)[None, :, None]
            w = np.clip(w, -448, 448)
        unit = 2.0 ** -4 if cache == "e4m3" else UNIT[cache]
        floor = 2.0 ** -10 if cache == "e4m3" else 2.0 ** -25  # half the smallest subnormal
        got, want = host(x), was.copy()
        tolx = np.zeros_like(was)
        for t in np.flatnonzero(live):
            p, o = divmod(int(slots[t]), page)
            want[1, p, :, o] = w[t]
            tolx[1, p, :, o] = unit * np.abs(w[t]) * (1 + 2.0 ** -20) + 2.0 ** -21 * mag[t] + floor
        assert (np.abs(got - want) <= tolx).all()  # exact where nothing was written


def test_append_without_q_and_rope_and_tokens(ce, dev):
    rng = np.random.default_rng(1)
    k, v = (pool(rng, dev, "f16", 1, 4, 2, 16, 32, "hnd") for _ in "kv")
    kn, vn = (torch.from_numpy(rng.standard_normal((3, 2, 32)).astype(np.float16)).to(dev) for _ in "kv")
    slots = torch.tensor([63, 0, 17], dtype=torch.int64, device=dev)
    kv = ce.PagedKV(k, v)
    ce.paged_append(kv, None, None, kn, vn, slots)
    ce.paged_append(kv, None, None, kn[:0], vn[:0], slots[:0])
    ce.device_status()
    assert torch.equal(k[0, 3, :, 15], kn[0]) and torch.equal(v[0, 1, :, 1], vn[2])


def test_append_reports_bad_slots_and_positions(ce, dev):
    rng = np.random.default_rng(2)
    k, v = (pool(rng, dev, "bf16", 1, 4, 1, 16, 64, "hnd") for _ in "kv")
    was = k.clone()
    new = torch.ones(2, 1, 64, device=dev)
    kv = ce.PagedKV(k, v)
    q_out = torch.full((2, 1, 64), float("nan"), dtype=torch.bfloat16, device=dev)
    rope = torch.ones(10, 32, 2, device=dev)
    pos = torch.tensor([0, 0], dtype=torch.int32, device=dev)
    ce.paged_append(kv, q_out, new, new, new, torch.tensor([64, 2 ** 40], dtype=torch.int64, device=dev), pos, rope)
    with pytest.raises(ce.CeError) as e:
        ce.device_status()
    assert e.value.status == ce.ERR_USAGE and "slot" in str(e.value)
    ce.paged_append(kv, q_out, new, new, new, torch.tensor([0, 1], dtype=torch.int64, device=dev),
                    torch.tensor([10, -1], dtype=torch.int32, device=dev), rope)
    with pytest.raises(ce.CeError) as e:
        ce.device_status()
    assert "position" in str(e.value)
    assert torch.equal(k, was) and (q_out == 0).all()
    ce.device_status()


# ---------------------------------------------------------------------------
# resize and reorder

def state(rng, n, P, pages, page, top, share=None):
    """Rows of random lengths in a pool with holes; `share`: rows of a group
    of that size hold the same full pages in front."""
    lens = rng.integers(0, top + 1, n).astype(np.int32)
    table = rng.integers(-2 ** 31, 2 ** 31 - 1, (n, P)).astype(np.int32)
    refs = np.zeros(pages, np.int32)
    free = rng.permutation(pages).tolist()
    for i in range(n):
        head = i // share * share if share else i
        for j in range(R.pages_of(lens[i], page)):
            if share and head != i and (j + 1) * page <= min(lens[i], lens[head]) and j < 2:
                table[i, j] = table[head, j]
            else:
                table[i, j] = free.pop()
            refs[table[i, j]] += 1
    return table, lens, refs


def same_rows(table, want, lens, page):
    return all(np.array_equal(table[i, :R.pages_of(lens[i], page)], want[i, :R.pages_of(lens[i], page)])
               for i in range(len(lens)))


def run_resize(ce, dev, table, lens, refs, new, page, cap, in_place, other_table):
    dt, dl, dr, dn = (torch.from_numpy(x).to(dev) for x in (table, lens, refs, new))
    pt = ce.PageTable(dt, dl, dr, page)
    out = pt
    if not in_place:
        out = ce.PageTable(torch.full_like(dt, -7) if other_table else dt, torch.full_like(dl, -7),
                           torch.full_like(dr, -7), page)
    slots, pos = torch.full((cap,), -7, dtype=torch.int64, device=dev), torch.full((cap,), -7, dtype=torch.int32, device=dev)
    starts, status = (torch.full((m,), -7, dtype=torch.int32, device=dev) for m in (len(lens) + 1, 4))
    ce.paged_resize(pt, dn, slots, pos, starts=starts, status=status, out=out)
    ce.device_status()
    if not in_place:
        assert np.array_equal(dl.cpu().numpy(), lens) and np.array_equal(dr.cpu().numpy(), refs)
    return [x.cpu().numpy() for x in (out.table, out.lens, out.refs, slots, pos, starts, status)]


@pytest.mark.parametrize("n,P,pages,page,top", [(1, 4, 5, 16, 60), (7, 9, 70, 8, 70), (64, 12, 900, 4, 40),
                                               (300, 6, 2100, 1, 6), (1500, 5, 40000, 16, 70),
                                               (5000, 3, 9000, 16, 40), (33, 80, 300000, 16, 1000)])
@pytest.mark.parametrize("mode", ["in place", "other lens", "other table"])
def test_resize(ce, dev, n, P, pages, page, top, mode):
    rng = np.random.default_rng(n)
    table, lens, refs = state(rng, n, P, pages, page, min(top, P * page))
    new = np.clip(lens + rng.integers(-2 * page, 2 * page + 1, n), 0, None).astype(np.int32)
    new[rng.random(n) < 0.2] = 0
    new[rng.random(n) < 0.1] = -1
    if n > 2:
        new[n // 2] = P * page + 1  # more than its row can hold
    cap = int(np.maximum(new - lens, 0).sum()) + 5
    want = R.resize(table, lens, refs, new, page, cap)
    got = run_resize(ce, dev, table, lens, refs, new, page, cap, mode == "in place", mode == "other table")
    for name, g, w in zip(("lens", "refs", "slots", "pos", "starts", "status"), got[1:], want[1:]):
        assert np.array_equal(g, w), name
    assert same_rows(got[0], want[0], want[1], page)


@pytest.mark.parametrize("short", ["pages", "capacity", "both", "no capacity"])
def test_resize_refuses_from_the_first_that_does_not_fit(ce, dev, short):
    rng = np.random.default_rng(3)
    n, P, page = 40, 10, 8
    table, lens, refs = state(rng, n, P, 220, page, 40)
    new = (lens + rng.integers(0, 40, n)).astype(np.int32)
    if short in ("pages", "both"):
        refs[np.flatnonzero(refs == 0)[30:]] = 5  # pinned by the caller
    cap = {"pages": 2000, "capacity": 300, "both": 200, "no capacity": 0}[short]
    want = R.resize(table, lens, refs, new, page, cap)
    assert want[-1][1] > 0
    got = run_resize(ce, dev, table, lens, refs, new, page, cap, True, False)
    for g, w in zip(got[1:], want[1:]):
        assert np.array_equal(g, w)
    assert same_rows(got[0], want[0], want[1], page)


def test_resize_refuses_a_shared_last_page(ce, dev):
    page = 8
    table = np.array([[3, 1, 0], [3, 1, 0], [4, 2, 0], [5, 0, 0]], np.int32)
    lens = np.array([12, 12, 16, 3], np.int32)
    refs = np.array([0, 2, 1, 2, 1, 1, 0, 0], np.int32)
    new = np.array([13, 12, 17, 4], np.int32)
    want = R.resize(table, lens, refs, new, page, 4)
    assert want[-1].tolist() == [1, 1, 2, 2]  # pages 0, 6 and 7 are free
    got = run_resize(ce, dev, table, lens, refs, new, page, 4, True, False)
    for g, w in zip(got[1:], want[1:]):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("n,beams,P,pages,page,top", [(4, 4, 5, 30, 8, 40), (1, 1, 3, 4, 16, 40), (64, 8, 12, 1100, 4, 40),
                                                     (99, 3, 9, 1200, 16, 140), (1200, 4, 4, 50000, 16, 60),
                                                     (6, 6, 30, 200000, 1, 30), (5120, 32, 3, 16000, 16, 48)])
@pytest.mark.parametrize("in_place", [True, False])
def test_reorder_tables(ce, dev, n, beams, P, pages, page, top, in_place):
    rng = np.random.default_rng(n)
    table, lens, refs = state(rng, n, P, pages, page, min(top, P * page), share=beams)
    parents = rng.integers(0, beams, n).astype(np.int32)
    parents[rng.random(n) < 0.1] = -1
    if n > 3:
        parents[3] = beams  # also out of range: the row is dropped
        refs[table[0, 0] if lens[0] else 0] += 1  # pinned by the caller
    dt, dl, dr, dp = (torch.from_numpy(x).to(dev) for x in (table, lens, refs, parents))
    pt = ce.PageTable(dt, dl, dr, page)
    out = ce.PageTable(torch.full_like(dt, -1), dl if in_place else torch.full_like(dl, -7),
                       dr if in_place else torch.full_like(dr, -7), page)
    status = torch.full((4,), -7, dtype=torch.int32, device=dev)
    copies = ce.paged_reorder(pt, dp, beams, out, status=status)
    ce.device_status()
    want = R.reorder(table, lens, refs, parents, beams, page)
    for g, w in zip((out.lens, out.refs, copies, status), want[1:]):
        assert np.array_equal(g.cpu().numpy(), w)
    got = out.table.cpu().numpy()
    assert np.array_equal(got, want[0])  # entries past a row's pages are untouched
    assert np.array_equal(dt.cpu().numpy(), table)


def test_reorder_without_enough_pages(ce, dev):
    page, beams = 8, 4
    table = np.array([[0, 1]] * 4, np.int32)
    lens = np.full(4, 11, np.int32)
    refs = np.array([4, 4, 0, 9], np.int32)  # one page is free, three are wanted
    args = [torch.from_numpy(x).to(dev) for x in (table, lens, refs)]
    pt, out = ce.PageTable(*args, page), ce.PageTable(torch.full_like(args[0], -1), args[1], args[2], page)
    status = torch.zeros(4, dtype=torch.int32, device=dev)
    parents = np.array([2, 0, 1, 3], np.int32)
    copies = ce.paged_reorder(pt, torch.from_numpy(parents).to(dev), beams, out, status=status)
    want = R.reorder(table, lens, refs, parents, beams, page)
    assert want[-1].tolist() == [1, 2, 0, 1]
    for g, w in zip((out.table, out.lens, out.refs, copies, status), want):
        assert np.array_equal(g.cpu().numpy(), w)
    grow = run_resize(ce, dev, want[0], want[1], want[2], want[1] + 1, page, 4, True, False)
    assert grow[-1].tolist() == [0, 3, 0, 1]  # only the row with a page of its own grows


@pytest.mark.parametrize("cache,layout,page,dim", [("bf16", "hnd", 8, 64), ("e4m3", "nhd", 16, 48), ("f16", "nhd", 1, 32),
                                                   ("f16", "hnd", 32, 128)])
def test_beam_histories_survive(ce, dev, cache, layout, page, dim):
    """A beam search's life: prompts come in, fork into beams, grow and are
    reordered at random. Every token's key and value carry a number of its
    own (in base 8, exact in 8 bits); after every step each row must read
    back its own history from its pages, and refs must count the rows."""
    rng = np.random.default_rng(page)
    B, K, layers, heads, P = 3, 4, 2, 2, R.pages_of(60, page) + 1
    n = B * K
    pages = n * P
    kv = ce.PagedKV(*(pool(rng, dev, cache, layers, pages, heads, page, dim, layout) for _ in "kv"))
    pt, spare = (ce.PageTable.empty(n, P, pages, page) for _ in range(2))
    spare = ce.PageTable(spare.table, pt.lens, pt.refs, page)
    histories = [[] for _ in range(n)]
    serial = 0

    def grow(new_lens):
        nonlocal serial, pt
        more = [max(0, int(x) - len(h)) for x, h in zip(new_lens, histories)]
        cap = sum(more) + 3
        slots = torch.empty(cap, dtype=torch.int64, device=dev)
        pos = torch.empty(cap, dtype=torch.int32, device=dev)
        status = torch.empty(4, dtype=torch.int32, device=dev)
        ce.paged_resize(pt, torch.tensor(new_lens, dtype=torch.int32, device=dev), slots, pos, status=status)
        assert status.tolist()[1] == 0 and status.tolist()[3] == sum(more)
        rows = np.zeros((cap, heads, dim), np.float32)
        j = 0
        for i, m in enumerate(more):
            for _ in range(m):
                histories[i].append(serial)
                rows[j, 0, :6] = [serial // 8 ** e % 8 for e in range(6)]
                rows[j, 1, -6:] = rows[j, 0, :6]
                serial, j = serial + 1, j + 1
        x = torch.from_numpy(rows).to(dev)
        for layer in range(layers):
            ce.paged_append(kv, None, None, x + layer, 2 * x + layer, slots, pos, layer=layer)

    def verify():
        ce.device_status()
        table, lens, refs = pt.table.cpu().numpy(), pt.lens.cpu().numpy(), pt.refs.cpu().numpy()
        count = np.zeros(pages, np.int32)
        hk, hv = host(kv.k), host(kv.v)
        for i, h in enumerate(histories):
            assert lens[i] == len(h)
            np.add.at(count, table[i, :R.pages_of(len(h), page)], 1)
            for t, num in enumerate(h):
                digits = np.array([num // 8 ** e % 8 for e in range(6)], np.float64)
                for layer in range(layers):
                    p, o = table[i, t // page], t % page
                    assert np.array_equal(hk[layer, p, 0, o, :6], digits + layer)
                    assert np.array_equal(hv[layer, p, 1, o, -6:], 2 * digits + layer)
        assert np.array_equal(count, refs)

    lens = np.zeros(n, np.int64)
    lens[::K] = [13, 16, 1]
    grow(lens.tolist())
    verify()
    for step in range(7):
        parents = np.zeros(n, np.int64) if step == 0 else rng.integers(0, K, n)
        ce.paged_reorder(pt, torch.tensor(parents, dtype=torch.int32, device=dev), K, spare, kv=kv)
        pt, spare = spare, pt
        histories = [list(histories[i // K * K + parents[i]]) for i in range(n)]
        verify()
        grow([len(h) + 1 + (i // K == 2) for i, h in enumerate(histories)])
        verify()


# ---------------------------------------------------------------------------
# the Python side's refusals

def test_wrappers_refuse_wrong_tensors(ce, dev):
    rng = np.random.default_rng(11)
    k, v = (pool(rng, dev, "bf16", 1, 6, 2, 16, 64, "hnd") for _ in "kv")
    with pytest.raises(ValueError):
        ce.PagedKV(k, v[:, :5])
    with pytest.raises(ValueError):
        ce.PagedKV(k.cpu(), v.cpu())
    with pytest.raises(TypeError):
        ce.PagedKV(k.double(), v.double())
    with pytest.raises(ValueError):  # head rows apart
        ce.PagedKV(k.transpose(3, 4), v.transpose(3, 4))
    kv = ce.PagedKV(k, v)
    pt = ce.PageTable.empty(3, 4, 6, 16)
    with pytest.raises(TypeError):
        ce.PageTable(pt.table.long(), pt.lens, pt.refs, 16)
    with pytest.raises(ValueError):
        ce.PageTable(pt.table, pt.lens[:2], pt.refs, 16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=dev)
    out = torch.empty_like(q)
    for bad in (q[:2], q[:, :, :32], q.transpose(0, 1), q.cpu()):
        with pytest.raises(ValueError):
            ce.paged_attention(kv, out, bad, pt)
    with pytest.raises(TypeError):
        ce.paged_attention(kv, out, q.half(), pt)
    with pytest.raises(ce.CeError):  # f16 queries over a bf16 cache
        ce.paged_attention(kv, out.half(), q.half(), pt)
    with pytest.raises(ce.CeError):
        ce.paged_attention(kv, out, q, pt, layer=1)
    with pytest.raises(ValueError):
        ce.paged_attention(kv, out, q, pt, lse=torch.empty(3, 3, device=dev))
    slots, pos = torch.zeros(3, dtype=torch.int64, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    n = torch.zeros(3, 2, 64, device=dev)
    with pytest.raises(TypeError):
        ce.paged_append(kv, None, None, n, n.half(), slots, pos)
    with pytest.raises(TypeError):
        ce.paged_append(kv, None, None, n, n, slots.int(), pos)
    with pytest.raises(ValueError):
        ce.paged_append(kv, None, None, n, n, slots, pos, torch.zeros(4, 16, 2, device=dev))
    with pytest.raises(ValueError):
        ce.paged_append(kv, None, None, n[:2], n[:2], slots, pos)
    with pytest.raises(TypeError):
        ce.paged_resize(pt, torch.zeros(3, device=dev), slots, pos)
    with pytest.raises(ValueError):
        ce.paged_resize(pt, pos[:2], slots, pos)
    with pytest.raises(ce.CeError, match="must differ"):
        ce.paged_reorder(pt, pos, 3, pt)
    ce.device_status()


def test_one_row_with_any_stride(ce, dev):
    """The stride between tokens means nothing where there is one."""
    rng = np.random.default_rng(12)
    k, v = (pool(rng, dev, "f16", 1, 2, 1, 16, 32, "hnd") for _ in "kv")
    pt = ce.PageTable(torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.full((1,), 7, dtype=torch.int32, device=dev),
                      torch.zeros(2, dtype=torch.int32, device=dev), 16)
    q = torch.randn(2 * 32 * 3, device=dev).half()
    a = q.as_strided((1, 2, 32), (33, 32, 1))
    out, want = torch.empty(1, 2, 32, dtype=torch.float16, device=dev), torch.empty(1, 2, 32, dtype=torch.float16, device=dev)
    kv = ce.PagedKV(k, v)
    ce.paged_attention(kv, out, a, pt)
    ce.paged_attention(kv, want, a.clone().contiguous(), pt)
    ce.device_status()
    assert torch.equal(out, want)


def test_attention_refuses_a_workspace_that_is_not_on_the_device(ce, dev):
    """Before any launch: the kernels would follow the host pointer."""
    rng = np.random.default_rng(13)
    k, v = (pool(rng, dev, "bf16", 1, 2, 1, 16, 32, "hnd") for _ in "kv")
    kv, pt = ce.PagedKV(k, v), ce.PageTable.empty(1, 1, 2, 16)
    q = torch.zeros(1, 1, 32, dtype=torch.bfloat16, device=dev)
    ws = ce.paged_attention_workspace()
    for bad in (ws.cpu(), torch.zeros(2 * ws.numel(), dtype=torch.uint8, device=dev)[::2]):
        with pytest.raises(TypeError, match="workspace"):
            ce.paged_attention(kv, torch.empty_like(q), q, pt, workspace=bad)
    with pytest.raises(ce.CeError, match="workspace"):
        ce.paged_attention(kv, torch.empty_like(q), q, pt, workspace=ws[:-16])
    out = torch.full_like(q, float("nan"))
    ce.paged_attention(kv, out, q, pt, workspace=ws.view(torch.int32))  # bytes count, not elements
    ce.device_status()
    assert (out == 0).all()


def test_attention_of_the_longest_row(ce, dev):
    """2^31 - 16 tokens, as many as 16-token pages allow: one page 2^27 - 1
    times over, so that its 16 tokens weigh as they would alone and the log
    sum is larger by log(2^27 - 1). A warp (12 on each SM at this head size)
    adds at most ceil(2^26 / (12 SMs)) units, of two halves in two 16-bit
    parts each, one after the other, every sum off by at most 2^-23 of it."""
    page, columns = 16, 2 ** 27 - 1
    rng = np.random.default_rng(14)
    k, v = (pool(rng, dev, "bf16", 1, 1, 1, page, 16, "hnd") for _ in "kv")
    pt = ce.PageTable(torch.zeros(1, columns, dtype=torch.int32, device=dev),
                      torch.tensor([columns * page], dtype=torch.int32, device=dev),
                      torch.ones(1, dtype=torch.int32, device=dev), page)
    q = torch.from_numpy(rng.standard_normal((1, 2, 16)).astype(np.float32)).to(dev).to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(1, 2, device=dev)
    ce.paged_attention(ce.PagedKV(k, v), out, q, pt, lse=lse)
    ce.device_status()
    want, wlse, _, spread = R.attention(host(q), host(k[0]), host(v[0]), np.zeros((1, 1), np.int32), [page], page, 0.25)
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    rel = 4 * -(-2 ** 26 // (12 * sms)) * 2.0 ** -23
    assert rel < 0.02
    assert (np.abs(host(out) - want) <= 2 * rel * spread + UNIT["bf16"] * np.abs(want)).all()
    assert (np.abs(host(lse) - wlse - np.log(columns)) <= 2 * rel).all()


def first_attention(ce, dev):
    """A cache that no call has used, its answer by another object, and a call on it."""
    lens = [6000, 31, 0, 90]  # the first row is split over CTAs: it needs the workspace's counters
    out, *_, (kv, pt, q) = attention_case(ce, dev, 15, lens, 2, 4, 64, 16, "bf16", "bf16", "hnd")
    return out, pt, q, kv.k, kv.v


def keep_busy(dev):
    """Work of some 50 ms at least on the current stream."""
    x = torch.randn(8192, 8192, device=dev)
    for _ in range(5):
        x = x @ x * 1e-4
    return x


def test_a_first_call_on_another_stream(ce, dev):
    """The workspace is zeroed before a stream other than the current one,
    which is busy, uses it: the attention's and the beam selection's."""
    want, pt, q, k, v = first_attention(ce, dev)
    # what the workspaces will be made from is not zero: one block of each size, among others of the size
    sizes = [x.numel() for x in (ce.paged_attention_workspace(), ce.beam_workspace(1, 2, 128256))]
    dirt = [[torch.full((n,), 0x55, dtype=torch.uint8, device=dev) for _ in range(65)] for n in sizes]
    side = torch.cuda.Stream()
    other = torch.full_like(want, float("nan"))
    x, scores = torch.randn(2, 128256, device=dev), torch.zeros(1, 2, device=dev)
    done = torch.zeros(1, 2, dtype=torch.bool, device=dev)

    def select(ws, **stream):
        o = [torch.full((1, 2), -7, dtype=t, device=dev) for t in (torch.float32, torch.int32, torch.int32, torch.uint8)]
        torch.cuda.synchronize()
        return lambda: ce.beam_select(*o[:3], o[3].view(torch.bool), x, scores, done, -1, 0, ws(), **stream) or o

    best = select(lambda: ce.beam_workspace(1, 2, 128256))()
    go = select(lambda: ce.beam_workspace(1, 2, 128256), stream=side)
    busy = keep_busy(dev)
    torch.cuda.synchronize()
    for blocks in dirt:
        del blocks[32]
    busy = keep_busy(dev)
    ce.paged_attention(ce.PagedKV(k, v), other, q, pt, stream=side)
    busy = keep_busy(dev)
    got = go()
    side.synchronize()
    assert torch.equal(other, want)
    assert all(torch.equal(a, b) for a, b in zip(got, best))
    ce.device_status()


def test_a_captured_first_call_and_an_eager_one_before_its_replay(ce, dev):
    want, pt, q, k, v = first_attention(ce, dev)
    kv = ce.PagedKV(k, v)
    a, b = torch.full_like(want, float("nan")), torch.full_like(want, float("nan"))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ce.paged_attention(kv, a, q, pt)
    at = kv.workspace().data_ptr()  # not of the graph's memory, which only a replay would zero
    pools = [x["segment_pool_id"] for x in torch.cuda.memory_snapshot() if x["address"] <= at < x["address"] + x["total_size"]]
    assert pools == [(0, 0)]
    ce.paged_attention(kv, b, q, pt)
    assert torch.equal(b, want)
    for _ in range(2):
        a.fill_(float("nan"))
        g.replay()
        assert torch.equal(a, want)
    ce.device_status()


def test_a_cache_made_during_a_capture_has_no_workspace(ce, dev):
    want, pt, q, k, v = first_attention(ce, dev)
    out, ws = torch.full_like(want, float("nan")), ce.paged_attention_workspace()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv = ce.PagedKV(k, v)
        with pytest.raises(RuntimeError, match="capture"):
            ce.paged_attention(kv, out, q, pt)
        ce.paged_attention(kv, out, q, pt, workspace=ws)
    g.replay()
    assert torch.equal(out, want)


def sink_case(ce, dev, seed, n, kv_heads, group, dim, cache, io, gap, sinks):
    """Requests of n tokens with keys (`sinks`) that score `gap` nats above
    all others and have values of 0, so that what the others add is all there
    is. The first dimension carries the gap, the others a small spread."""
    rng = np.random.default_rng(seed)
    page, rows = 16, len(sinks)
    table, refs = tables(rng, [n] * rows, page)
    s8 = 16.0 if cache == "e4m3" else 1.0
    k = torch.from_numpy((rng.standard_normal((1, len(refs), kv_heads, page, dim)) * 0.2 * s8).astype(np.float32))
    v = torch.from_numpy(((1 + 0.2 * rng.standard_normal(k.shape)) * s8).astype(np.float32))
    k[..., 0] = 0
    high = (gap * dim ** 0.5) ** 0.5
    for i, places in enumerate(sinks):
        for p in places:
            k[0, table[i, p // page], :, p % page] = 0
            k[0, table[i, p // page], :, p % page, 0] = high * s8
            v[0, table[i, p // page], :, p % page] = 0
    k, v = k.to(dev).to(DT[cache]), v.to(dev).to(DT[cache])
    poison(k, table, [n] * rows, page)
    poison(v, table, [n] * rows, page)
    ks = vs = None
    if cache == "e4m3":
        ks, vs = (torch.full((kv_heads,), 1.0 / 16, device=dev) for _ in "kv")
    H = kv_heads * group
    q = torch.from_numpy((rng.standard_normal((rows, H, dim)) * 0.4).astype(np.float32))
    q[:, :, 0] = high
    q = q.to(dev).to(DT[io])
    out, lse = torch.full_like(q, float("nan")), torch.full((rows, H), float("nan"), device=dev)
    pt = ce.PageTable(torch.from_numpy(table).to(dev), torch.full((rows,), n, dtype=torch.int32, device=dev),
                      torch.from_numpy(refs).to(dev), page)
    ce.paged_attention(ce.PagedKV(k, v, ks, vs), out, q, pt, lse=lse)
    ce.device_status()
    hk, hv = host(k[0]) / s8, host(v[0]) / s8
    return host(out), host(lse), host(q), hk, hv, table, page


def check_sinks(r, n, group, dim, cache, io, sinks):
    """Every weight enters the product as two 16-bit parts. In bf16 they hold
    2^-16 of it; in f16 2^-22 of it and, where it is small, 2^-25. There the
    largest weight of its unit (16 keys, 32 where a head's row has at most 128
    bytes) is 2^11 when the reference is set; the sinks leave the window, the
    others differ by less than e, so 2^9 is the least: 2^-34 of that weight.
    `extra` adds these up with the values. The rest as in check_attention,
    with the spread of each key alone: |q k| of the sinks for the sum, of the
    others for what they add; sums of at most 256 numbers in sequence (a
    warp's units in two halves and parts, then 12 warps and 148 CTAs), 2^-23
    each; e^x by 2^x, 2^-18 with its argument's rounding; the output rounded
    once, in f16 with its least spacing."""
    out, lse, q, hk, hv, table, page = r
    unit = 16 if dim > 64 and cache != "e4m3" else 32
    for i in range(len(sinks)):
        ids = table[i, :R.pages_of(n, page)]
        for h in range(q.shape[1]):
            kk, vv = (x[ids, h // group].reshape(-1, dim)[:n] for x in (hk, hv))
            s = kk @ q[i, h] * dim ** -0.5
            mag = np.abs(kk) @ np.abs(q[i, h]) * dim ** -0.5
            w = np.exp(s - s.max())
            total = w.sum()
            want = w @ vv / total
            other = np.ones(n, bool)
            other[sinks[i]] = False
            spread = w @ np.abs(vv) / total
            starts = np.arange(0, n, unit)
            top = np.repeat(np.maximum.reduceat(w, starts), np.diff(np.append(starts, n)))
            assert np.ptp(s[other]) < 1
            extra = (2.0 ** -16 * spread if cache == "bf16" else
                     2.0 ** -22 * spread + 2.0 ** -34 * (top @ np.abs(vv)) / total)
            score = (dim + 16) * 2.0 ** -22 * (mag.max() + mag[other].max()) + 2 * 2.0 ** -18
            rel = score + 2 * 256 * 2.0 ** -23
            tol = rel * spread + extra + UNIT[io] * np.abs(want) * (1 + rel) + (2.0 ** -25 if io == "f16" else 0)
            err = np.abs(out[i, h] - want)
            assert (err <= tol).all(), (i, h, (err / tol).max(), want[:4], out[i, h, :4])
            wlse = s.max() + np.log(total)
            assert abs(lse[i, h] - wlse) <= score + 256 * 2.0 ** -23 + 2.0 ** -22 * abs(wlse)


@pytest.mark.parametrize("cache,io", TYPES)
@pytest.mark.parametrize("gap", [12, 18, 30])
@pytest.mark.parametrize("group,dim", [(2, 64), (3, 128), (12, 128)])
def test_attention_sinks_in_short_rows(ce, dev, cache, io, gap, group, dim):
    """First, last, in the middle, several apart, in one unit with others only."""
    sinks = [[0], [999], [500], [3, 17, 400, 996], [31, 32]]
    r = sink_case(ce, dev, gap + dim, 1000, 1, group, dim, cache, io, gap, sinks)
    check_sinks(r, 1000, group, dim, cache, io, sinks)


@pytest.mark.parametrize("cache,io", TYPES)
@pytest.mark.parametrize("gap", [15, 18, 40])
def test_attention_sinks_in_long_rows(ce, dev, cache, io, gap):
    """Split over all CTAs; far below (e^-40) only the sums' exponents hold the rest."""
    sinks = [[0], [70001]]
    r = sink_case(ce, dev, gap, 100003, 1, 2, 64, cache, io, gap, sinks)
    check_sinks(r, 100003, 2, 64, cache, io, sinks)


def test_a_wait_that_gave_up_is_reported_before_a_bad_slot(ce, dev):
    """Both since the last look: the status and the message are the wait's, an
    exchange with a rank that never came."""
    x = ce.RowExchange(4, 64, 2, 0)
    kv = ce.PagedKV(*(torch.zeros(1, 2, 1, 16, 32, dtype=torch.bfloat16, device=dev) for _ in "kv"))
    try:
        ce.set_wait_limit(0.05)
        ce.paged_append(kv, None, None, *(torch.zeros(1, 1, 32, device=dev) for _ in "kv"),
                        torch.tensor([32], dtype=torch.int64, device=dev))
        torch.cuda.synchronize()
        x.wait()
        with pytest.raises(ce.CeError) as e:
            ce.device_status()
        assert e.value.status == ce.ERR_TIMEOUT and "row-shard exchange wait" in str(e.value)
        ce.device_status()
    finally:
        ce.set_wait_limit(2.0)
        x.close()


@pytest.mark.parametrize("cache,io", TYPES)
@pytest.mark.parametrize("kv_heads,group,dim", [(1, 16, 128), (2, 4, 64)])
@pytest.mark.parametrize("at", [0, 31, 63])
def test_attention_one_long_row_among_many_short_ones(ce, dev, cache, io, kv_heads, group, dim, at):
    """Most of the CTAs share one request, the other 63 a few: both joins and
    rows that no CTA shares, in one call; the long row first, inside, last."""
    lens = np.random.default_rng(at).integers(1, 300, 64).tolist()
    lens[at] = 20011
    r = attention_case(ce, dev, at, lens, kv_heads, group, dim, 16, cache, io, "hnd")
    check_attention(io, dim, lens, *r[:6])


@pytest.mark.parametrize("cache,io", TYPES)
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_attention_of_rows_that_share_pages(ce, dev, cache, io, layout):
    """Beams of two prompts: rows that share all pages, all but the last, the
    prompt's only, and none; the same page twice in one row. Each is what it
    is with pages of its own, bit for bit, and the oracle's."""
    page, lens = 16, [70, 70, 75, 48, 33, 130, 130, 160, 20, 64]
    share = [None, (0, 5), (0, 4), (0, 3), None, None, (5, 9), (5, 8), (4, 1), None]  # (row, leading pages taken over)
    own = attention_case(ce, dev, 21, lens, 2, 3, 64, page, cache, io, layout)
    out, lse, _, _, _, _, (kv, pt, q) = own
    table = pt.table.cpu().numpy().copy()
    for i, s in enumerate(share):
        if s is not None:
            table[i, :s[1]] = table[s[0], :s[1]]
    table[9, 2] = table[9, 0]
    # a pool in which every row has copies of these pages to itself
    k, v, apart = torch.zeros_like(kv.k), torch.zeros_like(kv.v), pt.table.cpu().numpy()
    for i, n in enumerate(lens):
        for j in range(R.pages_of(n, page)):
            k[:, apart[i, j]] = kv.k[:, table[i, j]]
            v[:, apart[i, j]] = kv.v[:, table[i, j]]
    # a row's last page may be another's with more tokens in it: what lies past each length stays out
    ce.paged_attention(ce.PagedKV(k, v, kv.k_scale, kv.v_scale), out, q, pt, lse=lse)
    pt2 = ce.PageTable(torch.from_numpy(table).to(dev), pt.lens, pt.refs, page)
    out2, lse2 = torch.full_like(out, float("nan")), torch.full_like(lse, float("nan"))
    ce.paged_attention(kv, out2, q, pt2, lse=lse2)
    ce.device_status()
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    hk, hv = host(kv.k[0]), host(kv.v[0])
    if kv.k_scale is not None:
        hk, hv = hk * host(kv.k_scale)[None, :, None, None], hv * host(kv.v_scale)[None, :, None, None]
    check_attention(io, 64, lens, out2, lse2, *R.attention(host(q), hk, hv, table, lens, page, 64 ** -0.5))


@pytest.mark.parametrize("cache,io", TYPES)
def test_attention_of_values_and_keys_that_are_not_finite(ce, dev, cache, io):
    """A value that is not finite stays in its element of the heads that attend
    to it, a NaN key in its head; the rest is what it is without, bit for bit."""
    lens = [100, 700]
    out, _, _, _, _, _, (kv, pt, q) = attention_case(ce, dev, 23, lens, 2, 3, 64, 16, cache, io, "hnd")
    bad = 0x7f if cache == "e4m3" else float("inf")  # E4M3 has NaN alone
    at = int(pt.table[1, 20])
    x = kv.v.view(torch.uint8) if cache == "e4m3" else kv.v
    x[0, at, 1, 3, 5] = bad
    got = torch.empty_like(out)
    ce.paged_attention(kv, got, q, pt)
    ce.device_status()
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[1, 3:, 5] = True  # the second kv head's query heads
    assert not torch.isfinite(got[hit].float()).any() and torch.equal(got[~hit], out[~hit])
    x[0, at, 1, 3, 5] = 0
    k = kv.k.view(torch.uint8) if cache == "e4m3" else kv.k
    k[0, at, 0, 3, 5] = 0x7f if cache == "e4m3" else float("nan")
    ce.paged_attention(kv, got, q, pt)
    ce.device_status()
    assert torch.isnan(got[1, :3].float()).all() and torch.equal(got[0], out[0]) and torch.isfinite(got[1, 3:].float()).all()


def test_reorder_of_a_last_page_that_two_groups_share(ce, dev):
    """Every row of both copies it; it is free after the call, but not in its count."""
    page, beams = 8, 2
    table, lens = np.array([[0, 1, -1]] * 4, np.int32), np.full(4, 11, np.int32)
    refs = np.array([4, 4] + [0] * 6, np.int32)
    args = [torch.from_numpy(x).to(dev) for x in (table, lens, refs)]
    pt, out = ce.PageTable(*args, page), ce.PageTable(torch.full_like(args[0], -1), args[1], args[2], page)
    status = torch.zeros(4, dtype=torch.int32, device=dev)
    parents = np.array([0, 1, 1, 1], np.int32)
    copies = ce.paged_reorder(pt, torch.from_numpy(parents).to(dev), beams, out, status=status)
    for g, w in zip((out.table, out.lens, out.refs, copies, status), R.reorder(table, lens, refs, parents, beams, page)):
        assert np.array_equal(g.cpu().numpy(), w)
    assert out.refs.tolist() == [4, 0, 1, 1, 1, 1, 0, 0] and status.tolist() == [4, 0, 2, 4]
    slots, pos = (torch.zeros(32, dtype=t, device=dev) for t in (torch.int64, torch.int32))
    ce.paged_resize(out, torch.tensor([17, -1, -1, -1], dtype=torch.int32, device=dev), slots, pos, status=status)
    assert status.tolist() == [1, 0, 2, 6] and out.table[0].tolist() == [0, 2, 1]
