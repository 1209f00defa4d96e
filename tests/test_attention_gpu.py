"""Attention of prompts and of single tokens over a paged cache, storing and copying pages: against 64 bits, at the sizes
and masks where they can go wrong."""
import pytest
import torch

import flashoverlap_b200  # noqa: F401
from attention_oracle import attend, check
from flashoverlap_b200 import ops

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16


def randn(*shape, dtype, seed=0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(seed))


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Paged:
    """Sequences of given lengths in a cache whose pages lie in no order; everything that belongs to nobody is `filler`."""

    def __init__(self, lengths, kv, dim, page, dtype, seed=0, filler=float("nan"), spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        used = [-(-n // page) for n in lengths]
        order = torch.randperm(sum(used) + spare, generator=g).tolist()
        self.cache = torch.full((len(order), 2, kv, page, dim), filler, dtype=dtype, device="cuda")
        width = max(used + [1]) if width is None else width
        table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        self.k = [randn(n, kv, dim, dtype=dtype, seed=seed + 2 * s) for s, n in enumerate(lengths)]
        self.v = [randn(n, kv, dim, dtype=dtype, seed=seed + 2 * s + 1) for s, n in enumerate(lengths)]
        at = 0
        for s, n in enumerate(lengths):
            for i in range(used[s]):
                table[s, i] = order[at]
                m = min(page, n - i * page)
                for which, x in ((0, self.k[s]), (1, self.v[s])):
                    self.cache[order[at], which, :, :m] = x[i * page:i * page + m].transpose(0, 1)
                at += 1
        self.table, self.lengths, self.n = table.cuda(), ints(*lengths), lengths
        self.spare = order[at:]

    def check(self, q, got, window=0, sinks=0, scale=None, only=None):
        group = q.shape[1] // self.cache.shape[2]
        for s, n in enumerate(self.n):
            if only is not None and s not in only:
                continue
            for h in range(q.shape[1]):
                want, tol = attend(q[s, h][None], self.k[s][:, h // group], self.v[s][:, h // group], n - 1, n, window,
                                   sinks, scale)
                check(got[s, h][None], want, tol, f"sequence {s} of {n} tokens, head {h}")


# ---- one token over pages ------------------------------------------------------
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,page,window,sinks", [
    (4, 4, 16, 0, 0), (8, 1, 64, 0, 0), (12, 4, 24, 0, 0), (5, 1, 1, 0, 0), (16, 1, 7, 100, 3), (34, 2, 100, 0, 0),
    (40, 1, 16, 64, 0), (32, 8, 50, 1, 0), (14, 2, 128, 65, 64), (6, 2, 256, 17, 1000), (2, 1, 16, 0, 5)])
def test_single_tokens(dtype, dim, heads, kv, page, window, sinks):
    lengths = [0, 1, 2, 15, 16, 17, 63, 64, 65, 129, 300, 0, 777]
    p = Paged(lengths, kv, dim, page, dtype, seed=heads)
    q = randn(len(lengths), heads, dim, dtype=dtype, seed=99)
    got = ops.paged_attention(q, p.cache, p.table, p.lengths, window=window, sinks=sinks)
    p.check(q, got, window, sinks)
    assert not got[0].any() and not got[11].any()


@pytest.mark.parametrize("lengths", [[1], [40000], [5, 30011], [0], [0, 0, 0], [64] * 300, list(range(257)), [20000] + [3] * 40])
def test_work_is_cut_whatever_the_lengths(lengths):
    p = Paged(lengths, 1, 64, 32, BF16, seed=len(lengths))
    q = randn(len(lengths), 4, 64, dtype=BF16, seed=5)
    got = ops.paged_attention(q, p.cache, p.table, p.lengths)
    p.check(q, got)
    assert torch.equal(got, ops.paged_attention(q, p.cache, p.table, p.lengths))   # the same bits every time


@pytest.mark.parametrize("window,sinks", [(4096, 4), (100, 200), (1, 1), (63, 0)])
def test_long_windows_read_nothing_hidden(window, sinks):
    # tokens that are not visible hold NaN, in keys and in values
    lengths = [10007, 4101, 300, 1]
    p = Paged(lengths, 2, 128, 24, FP16, seed=3)
    for s, n in enumerate(lengths):
        for j in range(min(sinks, n), n - window):
            p.cache[p.table[s, j // 24], :, :, j % 24] = float("inf") if j % 2 else float("nan")
    q = randn(len(lengths), 10, 128, dtype=FP16, seed=8)
    p.check(q, ops.paged_attention(q, p.cache, p.table, p.lengths, window=window, sinks=sinks), window, sinks)


def test_entries_that_name_no_page_spoil_their_own_sequence():
    # (the kernel checks each entry: nothing outside the cache is read)
    lengths = [50, 200, 31, 64, 90]
    p = Paged(lengths, 2, 64, 16, BF16)
    q = randn(5, 4, 64, dtype=BF16, seed=1)
    table = p.table.clone()
    table[1, 5] = p.cache.shape[0]
    table[3, 0] = -7
    table[0, 4:] = 2 ** 31 - 1            # behind the length: not looked at
    lens = p.lengths.clone()
    lens[4] = 16 * table.shape[1] + 1     # longer than its row of the table
    got = ops.paged_attention(q, p.cache, table, lens)
    p.check(q, got, only=(0, 2))
    for s in (1, 3, 4):
        assert got[s].isnan().all()
    # outside the window a bad entry does not matter; a negative length is an empty sequence
    lens = p.lengths.clone()
    lens[2] = -5
    got = ops.paged_attention(q, p.cache, table, lens, window=64)
    p.check(q, got, 64, only=(0, 4))
    assert not got[2].any() and got[3].isnan().all()
    table[1, 5] = -1
    got = ops.paged_attention(q, p.cache, table, p.lengths, window=100, sinks=2)
    p.check(q, got, 100, 2, only=(0, 1, 2, 4))


def test_values_that_are_not_finite_stay_in_their_sequence():
    p = Paged([100, 100, 100], 1, 64, 16, BF16)
    p.cache[p.table[1, 2], 1, 0, 3] = float("inf")
    q = randn(3, 2, 64, dtype=BF16)
    got = ops.paged_attention(q, p.cache, p.table, p.lengths)
    p.check(q, got, only=(0, 2))
    assert not got[1].isfinite().any()


def test_strided_arguments_and_layers():
    layers, kv, dim, page = 3, 2, 64, 16
    lengths = [33, 100, 7]
    p = Paged(lengths, kv, dim, page, FP16)
    whole = torch.full((p.cache.shape[0], layers, 2, kv, page, dim), float("nan"), dtype=FP16, device="cuda")
    whole[:, 1] = p.cache
    qkv = randn(3, 6 + 2 * kv, dim, dtype=FP16, seed=4)
    table = torch.full((6, p.table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    table[::2, 2:2 + p.table.shape[1]] = p.table
    q = qkv[:, 1:7]
    out = torch.full((3, 6, dim), 7.0, dtype=FP16, device="cuda")
    assert ops.paged_attention(q, whole[:, 1], table[::2, 2:], p.lengths, out=out, scale=0.3) is out
    p.check(q, out, scale=0.3)
    # heads in an order of their own
    q = randn(6, 3, dim, dtype=FP16, seed=6).transpose(0, 1)
    p.check(q, ops.paged_attention(q, whole[:, 1], p.table, p.lengths))


def test_offsets_beyond_32_bits():
    # 5 GB of cache, sequences in its last pages; the table's rows are broadcast
    kv, page, dim = 8, 64, 128
    pages = 20000
    cache = torch.zeros(pages, 2, kv, page, dim, dtype=BF16, device="cuda")
    p = Paged([130, 190], kv, dim, page, BF16, filler=0.0)
    n = p.cache.shape[0]
    moves = torch.tensor([[i, pages - n + i] for i in range(n)])
    cache[:n] = p.cache
    ops.copy_pages(cache, moves)
    cache[:n] = float("nan")
    assert torch.equal(cache[pages - n:], p.cache)
    table = torch.where(p.table >= 0, p.table + (pages - n), -1)
    q = randn(2, 16, dim, dtype=BF16)
    p.check(q, ops.paged_attention(q, cache, table, p.lengths))
    ops.cache_append(p.k[1][None, 100:], p.v[1][None, 100:], cache, table[1:].expand(1, -1), ints(100))
    assert torch.equal(cache[pages - n:], p.cache)


def test_streams_and_graphs_do_not_share_anything():
    sets = []
    for seed in range(2):
        p = Paged([3000, 700, 50 + seed], 2, 128, 16, BF16, seed=seed * 10)
        sets.append((p, randn(3, 8, 128, dtype=BF16, seed=seed)))
    want = [ops.paged_attention(q, p.cache, p.table, p.lengths, window=1000, sinks=4) for p, q in sets]
    graphs, outs = [], []
    for p, q in sets:
        g = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=side):
            outs.append(ops.paged_attention(q, p.cache, p.table, p.lengths, window=1000, sinks=4))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    # another length, other queries: a replay reads them where they are
    p, q = sets[0]
    p.lengths[0] = 2000
    p.n = [2000, 700, 50]
    q.copy_(randn(3, 8, 128, dtype=BF16, seed=77))
    graphs[0].replay()
    torch.cuda.synchronize()
    p.check(q, outs[0], 1000, 4)


# ---- storing --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("kv,dim,page,tokens", [(1, 64, 16, 1), (8, 128, 64, 1), (3, 64, 7, 50), (2, 128, 24, 333),
                                                (40, 128, 16, 5), (2, 8, 4, 9)])
def test_storing_tokens(dtype, kv, dim, page, tokens):
    starts = [0, 3, page, 2 * page - 1, 100]
    counts = [tokens, 0, max(1, tokens - 3), tokens, 1]
    seqs, width = len(starts), -(-(100 + tokens) // page)
    g = torch.Generator().manual_seed(1)
    table = torch.randperm(seqs * width + 4, generator=g)[:seqs * width].to(torch.int32).reshape(seqs, width)
    new = randn(seqs, tokens, 2 * kv, dim, dtype=dtype, seed=2)
    k, v = new[:, :, :kv], new[:, :, kv:]
    for some in (None, counts):
        cache = randn(seqs * width + 4, 2, kv, page, dim, dtype=dtype, seed=3)
        want = cache.clone()
        for s in range(seqs):
            for i in range(tokens if some is None else some[s]):
                at = starts[s] + i
                want[table[s, at // page], 0, :, at % page] = k[s, i]
                want[table[s, at // page], 1, :, at % page] = v[s, i]
        ops.cache_append(k, v, cache, table.cuda(), ints(*starts), None if some is None else ints(*some))
        assert torch.equal(cache, want)


def test_tokens_without_a_place_are_left_out():
    cache = torch.zeros(6, 2, 2, 8, 64, dtype=FP16, device="cuda")
    table = torch.tensor([[1, -1, 2], [6, 3, 2 ** 31 - 1], [4, 5, 0]], dtype=torch.int32, device="cuda")
    x = torch.ones(3, 24, 2, 64, dtype=FP16, device="cuda")
    ops.cache_append(x, x, cache, table, ints(0, 0, -1))
    want = torch.zeros_like(cache)
    want[[1, 2, 3]] = 1
    assert torch.equal(cache, want)
    ops.cache_append(x, x, cache, table, ints(24, 2 ** 31 - 1, 20), ints(24, 24, 4))
    want[0, :, :, 4:] = 1
    assert torch.equal(cache, want)
    ops.cache_append(x[:0], x[:0], cache, table[:0], ints())
    ops.cache_append(x[:, :0], x[:, :0], cache, table, ints(0, 0, 0))
    assert torch.equal(cache, want)


# ---- copying --------------------------------------------------------------------
@pytest.mark.parametrize("shape,n", [((40, 2, 2, 8, 64), 20), ((9, 8), 4), ((9001, 2, 1, 1, 64), 4500), ((3, 1000008), 1),
                                     ((1200, 2, 1, 3, 8), 481), ((5, 24), 0)])
def test_copying_pages(shape, n):
    cache = torch.randint(-30000, 30000, shape, dtype=torch.int16, device="cuda")
    order = torch.randperm(shape[0])
    moves = torch.stack([order[:n], order[n:2 * n]], 1)
    for dtype in (torch.int32, torch.int64):
        want = cache.clone()
        want[moves[:, 1].cuda()] = cache[moves[:, 0].cuda()]
        ops.copy_pages(cache, moves.to(dtype))
        assert torch.equal(cache, want)
        cache.copy_(cache.flip(0))


def test_copying_one_page_to_many_and_of_one_layer():
    whole = randn(50, 3, 2, 2, 4, 64, dtype=BF16)
    want = whole.clone()
    want[10:40, 1] = whole[7, 1]
    moves = torch.tensor([[7, i] for i in range(10, 40)])
    ops.copy_pages(whole[:, 1], moves)
    assert torch.equal(whole, want)
    # a captured copy keeps the moves of its capture
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.copy_pages(whole, moves)
    moves.fill_(0)
    whole.copy_(randn(50, 3, 2, 2, 4, 64, dtype=BF16, seed=9))
    want = whole.clone()
    want[10:40] = whole[7]
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(whole, want)


# ---- prompts --------------------------------------------------------------------
def check_prompt(q, k, v, got, window=0, sinks=0, lengths=None, scale=None, heads=None):
    batch, sq, H, _ = q.shape
    sk, group = k.shape[1], H // k.shape[2]
    for b in range(batch):
        for h in range(H) if heads is None else heads:
            n = sk if lengths is None else lengths[b]
            want, tol = attend(q[b, :, h], k[b, :, h // group], v[b, :, h // group], sk - sq, n, window, sinks, scale)
            check(got[b, :, h], want, tol, f"sequence {b}, head {h}")


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,sq,sk,heads,kv,window,sinks", [
    (1, 1, 1, 1, 1, 0, 0), (2, 1, 300, 8, 2, 0, 0), (1, 127, 127, 2, 2, 0, 0), (1, 128, 128, 4, 1, 0, 0),
    (2, 129, 129, 3, 1, 0, 0), (1, 300, 300, 8, 8, 100, 3), (1, 65, 500, 6, 2, 64, 0), (1, 33, 33, 40, 1, 0, 0),
    (1, 257, 400, 16, 2, 1, 0), (2, 200, 456, 5, 1, 129, 130), (1, 40, 40, 7, 1, 3, 1000), (1, 3, 260, 128, 1, 0, 0),
    (1, 513, 513, 2, 1, 2, 1)])
def test_prompts(dtype, dim, batch, sq, sk, heads, kv, window, sinks):
    q = randn(batch, sq, heads, dim, dtype=dtype, seed=1)
    k, v = randn(batch, sk, kv, dim, dtype=dtype, seed=2), randn(batch, sk, kv, dim, dtype=dtype, seed=3)
    got = ops.prompt_attention(q, k, v, window=window, sinks=sinks)
    check_prompt(q, k, v, got, window, sinks, heads=range(0, heads, max(1, heads // 8)))
    assert torch.equal(got, ops.prompt_attention(q, k, v, window=window, sinks=sinks))


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 2), (200, 70)])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_of_different_lengths(dim, window, sinks):
    # padding holds NaN and infinities; its rows are zero, and so is all of an empty sequence
    lengths = [300, 0, 1, 299, 150, 128, 129, 173]
    batch, sq, sk = len(lengths), 200, 300
    qkv = randn(batch, sq, 8, dim, dtype=BF16, seed=1)
    k, v = randn(batch, sk, 2, dim, dtype=BF16, seed=2), randn(batch, sk, 2, dim, dtype=BF16, seed=3)
    q = qkv[:, :, 1:7]
    for b, n in enumerate(lengths):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
        v[b, n + 1::2] = float("nan")
        q[b, max(0, n - (sk - sq)):] = float("nan")
    out = torch.full((batch, sq, 6, dim), 5.0, dtype=BF16, device="cuda")
    assert ops.prompt_attention(q, k, v, window=window, sinks=sinks, lengths=ints(*lengths), out=out) is out
    check_prompt(q, k, v, out, window, sinks, lengths, heads=(0, 2, 5))
    for b, n in enumerate(lengths):
        assert not out[b, max(0, n - (sk - sq)):].any()
    # a length beyond the keys means all of them, one below zero none
    lens = ints(*[400, -1] + lengths[2:])
    assert torch.equal(ops.prompt_attention(q, k, v, window=window, sinks=sinks, lengths=lens), out)


@pytest.mark.parametrize("dim", [64, 128])
def test_hidden_tokens_that_are_not_finite(dim):
    # a token is seen by itself and later ones only, in the window or as a sink
    sq, window, sinks = 400, 70, 2
    q, k, v = (randn(1, sq, 2, dim, dtype=FP16, seed=i) for i in range(3))
    bad = 150
    v[0, bad] = float("inf")
    for w, s in ((0, 0), (window, sinks)):
        got = ops.prompt_attention(q, k, v, window=w, sinks=s)
        hit = torch.zeros(sq, dtype=torch.bool)
        hit[bad:bad + window if w else sq] = True
        clean = v.clone()
        clean[0, bad] = 0
        for h in range(2):
            want, tol = attend(q[0, :, h], k[0, :, h], clean[0, :, h], 0, sq, w, s)
            check(got[0, ~hit, h], want[~hit], tol[~hit])
            assert not got[0, hit, h].isfinite().any()
    v[0, bad], k[0, bad] = 0.5, float("nan")
    got = ops.prompt_attention(q, k, v, window=window, sinks=sinks)
    assert torch.equal(got.isnan().any(-1).any(-1)[0].cpu(), torch.arange(sq).ge(bad) & torch.arange(sq).lt(bad + window))


def test_large_scores_and_steep_changes():
    # rows whose largest score comes first, last, or rises from tile to tile by more than 16 bits hold
    for dtype, size in ((FP16, 6.0), (BF16, 30.0)):
        q, k, v = (randn(1, 700, 2, 64, dtype=dtype, seed=i) for i in range(3))
        ramp = torch.linspace(0, size, 700, device="cuda")[None, :, None, None]
        for factor in (ramp, ramp.flip(1), torch.full_like(ramp, size)):
            kk = (k * factor).to(dtype)
            check_prompt(q, kk, v, ops.prompt_attention(q, kk, v))
            check_prompt(q, kk, v, ops.prompt_attention(q, kk, v, scale=-0.2), scale=-0.2)
            check_prompt(q, kk, v, ops.prompt_attention(q, kk, v, scale=0.0), scale=0.0)


def test_layouts_of_prompts():
    # [batch, heads, tokens, dim] views, packed QKV, keys and values of different layouts, one sequence of a padded buffer
    q = randn(2, 6, 150, 128, dtype=BF16, seed=1).transpose(1, 2)
    k = randn(2, 180, 5, 128, dtype=BF16, seed=2)[:, :, 2:4]
    v = randn(2, 2, 200, 128, dtype=BF16, seed=3)[:, :, :180].transpose(1, 2)
    check_prompt(q, k, v, ops.prompt_attention(q, k, v, window=60, sinks=5), 60, 5)
    check_prompt(q[1:], k[1:], v[:1], ops.prompt_attention(q[1:], k[1:], v[:1]))
    # keys and values that a batch shares
    k1, v1 = k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)
    check_prompt(q, k1, v1, ops.prompt_attention(q, k1, v1))


def test_prompt_in_a_graph_and_on_a_side_stream():
    q, k, v = (randn(1, 700, h, 128, dtype=BF16, seed=h) for h in (8, 2, 2))
    want = ops.prompt_attention(q, k, v, window=300, sinks=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.prompt_attention(q, k, v, window=300, sinks=1)
    side.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.prompt_attention(q, k, v, window=300, sinks=1)
    q.copy_(randn(1, 700, 8, 128, dtype=BF16, seed=50))
    g.replay()
    torch.cuda.synchronize()
    check_prompt(q, k, v, out, 300, 1, heads=(0, 7))


# ---- together, and what is refused ------------------------------------------------
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
def test_prompt_then_tokens_one_by_one(window, sinks):
    # the cache filled by prompts of two lengths and by single tokens answers as one long prompt does
    heads, kv, dim, page, total = 8, 2, 64, 16, 230
    first = [200, 131]
    q, k, v = (randn(2, total, h, dim, dtype=BF16, seed=h + i) for i, h in enumerate((heads, kv, kv)))
    want = ops.prompt_attention(q, k, v, window=window, sinks=sinks)
    check_prompt(q, k, v, want, window, sinks, heads=(0, 5))
    width = -(-total // page)
    table = torch.randperm(2 * width, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(2, width).cuda()
    cache = torch.full((2 * width, 2, kv, page, dim), float("nan"), dtype=BF16, device="cuda")
    ops.cache_append(k[:, :200], v[:, :200], cache, table, ints(0, 0), ints(*first))
    at = list(first)
    for _ in range(25):
        now = torch.arange(2, device="cuda"), torch.tensor(at, device="cuda")
        ops.cache_append(k[now][:, None], v[now][:, None], cache, table, ints(*at))
        got = ops.paged_attention(q[now], cache, table, ints(*[n + 1 for n in at]), window=window, sinks=sinks)
        for s in range(2):
            for h in range(heads):
                ref, tol = attend(q[s, at[s], h][None], k[s, :at[s] + 1, h // 4], v[s, :at[s] + 1, h // 4], at[s],
                                  at[s] + 1, window, sinks)
                check(got[s, h][None], ref, tol)
                assert ((got[s, h].double() - want[s, at[s], h].double()).abs() <= 2 * tol[0]).all()
        at = [n + 1 for n in at]


def test_refusals():
    q, k = randn(2, 8, 4, 64, dtype=FP16), randn(2, 16, 2, 64, dtype=FP16)
    cache = randn(6, 2, 2, 8, 64, dtype=FP16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ints(1, 1)
    one = q[:, 0]
    dense = one.contiguous()
    buf = randn(2 * 8 * 4 * 64 * 3, dtype=FP16)

    def prompt(q=q, k=k, v=None, **kw):
        return lambda: ops.prompt_attention(q, k, k if v is None else v, **kw)

    def paged(q=one, cache=cache, table=table, lens=lens, **kw):
        return lambda: ops.paged_attention(q, cache, table, lens, **kw)

    def append(k=k[:, :4], v=None, cache=cache, table=table, starts=lens, counts=None):
        return lambda: ops.cache_append(k, k if v is None else v, cache, table, starts, counts)

    odd = torch.empty(q.numel() + 1, dtype=FP16, device="cuda")[1:].view_as(q)
    bad = {
        "dtype": prompt(q=q.float()), "mixed": prompt(k=k.bfloat16()), "mixed values": prompt(v=k.bfloat16()),
        "head_dim": prompt(q=randn(2, 8, 4, 96, dtype=FP16), k=randn(2, 16, 2, 96, dtype=FP16)),
        "groups": prompt(q=q[:, :, :3]), "more queries than keys": prompt(k=k[:, :7]), "batch": prompt(k=k[:1]),
        "shape of values": prompt(v=k[:, 1:]), "rank": prompt(q=q[0]), "alignment": prompt(q=odd),
        "strides": prompt(q=randn(2, 8, 4, 68, dtype=FP16)[..., :64]), "columns": prompt(q=q.transpose(2, 3)[:, :, :4].contiguous().transpose(2, 3)),
        "window": prompt(window=-1), "sinks": prompt(sinks=-1), "scale": prompt(scale=float("nan")),
        "lengths type": prompt(lengths=lens.long()), "lengths size": prompt(lengths=ints(1)), "lengths on CPU": prompt(lengths=lens.cpu()),
        "out shape": prompt(out=torch.empty_like(q[:, 1:])), "out dtype": prompt(out=torch.empty_like(q).float()),
        "out strides": prompt(out=torch.empty(2, 4, 8, 64, dtype=FP16, device="cuda").transpose(1, 2)), "out is q": prompt(out=q),
        "out in k": prompt(q=buf[:4096].view(2, 8, 4, 64), k=buf[4096:8192].view(2, 16, 2, 64), out=buf[6144:10240].view(2, 8, 4, 64)),
        "gradient": prompt(q=q.clone().requires_grad_()),
        "too many heads": prompt(q=randn(2, 8, 258, 64, dtype=FP16)),
        "cache dtype": paged(cache=cache.bfloat16()), "cache shape": paged(cache=cache[:, :1]), "cache rank": paged(cache=cache[:, 0]),
        "cache head_dim": paged(cache=randn(6, 2, 2, 8, 128, dtype=FP16)), "page strides": paged(cache=cache.transpose(2, 3)),
        "pages overlap": paged(cache=cache[:1].expand(6, -1, -1, -1, -1)), "table type": paged(table=table.long()),
        "table rows": paged(table=table[:1]), "table columns": paged(table=table.t().contiguous().t()), "table on CPU": paged(table=table.cpu()),
        "paged lengths": paged(lens=ints(1, 1, 1)), "paged lengths type": paged(lens=lens.long()), "paged groups": paged(q=one[:, :3]),
        "paged out": paged(out=torch.empty(2, 4, 128, dtype=FP16, device="cuda")), "paged out is q": paged(q=dense, out=dense),
        "paged window": paged(window=-2), "paged out in cache": paged(out=cache[0, 0, 0].reshape(-1)[:512].view(2, 4, 64)),
        "append heads": append(k=randn(2, 4, 3, 64, dtype=FP16)), "append dtype": append(k=k[:, :4].bfloat16()),
        "append values": append(v=k[:, :3]), "append starts": append(starts=ints(1)), "append counts": append(counts=ints(1, 2, 3)),
        "append out of the cache": append(k=cache.view(-1)[:1024].view(2, 4, 2, 64)),
        "copy on odd boundaries": lambda: ops.copy_pages(torch.empty(4, 7, dtype=FP16, device="cuda"), torch.tensor([[0, 1]])),
        "copy of columns": lambda: ops.copy_pages(cache.transpose(1, 4), torch.tensor([[0, 1]])),
        "copy into itself": lambda: ops.copy_pages(cache[:1].expand(6, -1, -1, -1, -1), torch.tensor([[0, 1]])),
        "moves on the GPU": lambda: ops.copy_pages(cache, torch.tensor([[0, 1]], device="cuda")),
    }
    for what, call in bad.items():
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"accepted: {what}")
    torch.cuda.synchronize()
    # what is no refusal: nothing to do, gradients off
    assert ops.prompt_attention(q[:, :0], k, k).shape == (2, 0, 4, 64)
    assert ops.prompt_attention(q[:0], k[:0], k[:0]).shape == (0, 8, 4, 64)
    assert ops.paged_attention(one[:0], cache, table[:0], lens[:0]).shape == (0, 4, 64)
    assert not ops.paged_attention(one, cache, table[:, :0], ints(0, 0)).any()
    assert ops.paged_attention(one, cache, table[:, :0], lens).isnan().all()
    assert ops.paged_attention(one, cache[:0], table, lens).isnan().all()
    ops.copy_pages(cache, torch.empty(0, 2, dtype=torch.int64))
    with torch.no_grad():
        ops.prompt_attention(q.clone().requires_grad_(), k, k)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_tensors_on_another_device_than_the_current_one():
    p = Paged([500, 3], 2, 64, 16, BF16)
    q = randn(2, 4, 64, dtype=BF16)
    want = ops.paged_attention(q, p.cache, p.table, p.lengths)
    dev = torch.device("cuda", 1)
    got = ops.paged_attention(q.to(dev), p.cache.to(dev), p.table.to(dev), p.lengths.to(dev))
    assert torch.equal(got.cpu(), want.cpu())


# ---- a cache with its pool, and the decoder block on it ---------------------------
def test_cache_of_sequences_that_fork_and_move():
    from flashoverlap_b200.models import PagedKVCache

    kv, dim, heads, page = 2, 64, 6, 16
    cache = PagedKVCache(60, page, kv, dim, dtype=BF16)
    tokens = {}

    def put(seqs, n, seed, counts=None):
        k, v = (randn(len(seqs), n, kv, dim, dtype=BF16, seed=seed + i) for i in (0, 1))
        cache.append(seqs, k, v, counts)
        for i, s in enumerate(seqs):
            m = n if counts is None else counts[i]
            old = tokens.get(s, (k[0, :0], v[0, :0]))
            tokens[s] = (torch.cat([old[0], k[i, :m]]), torch.cat([old[1], v[i, :m]]))

    def look(window=0, sinks=0):
        seqs = sorted(tokens)
        q = randn(len(seqs), heads, dim, dtype=BF16, seed=len(seqs))
        got = cache.attend(seqs, q, window=window, sinks=sinks)
        for i, s in enumerate(seqs):
            n = len(tokens[s][0])
            assert cache.length(s) == n
            for h in range(heads):
                want, tol = attend(q[i, h][None], tokens[s][0][:, h // 3], tokens[s][1][:, h // 3], n - 1, n, window, sinks)
                check(got[i, h][None], want, tol, f"sequence {s}")

    a, b, c = (cache.add() for _ in range(3))
    put([a, b, c], 50, 1, counts=[50, 32, 7])
    look()
    d, e = cache.fork(a), cache.fork(b)      # 50 tokens: a page is copied; 32: none is
    tokens[d], tokens[e] = tokens[a], tokens[b]
    put([a, d, e, b], 1, 10)                 # each goes on by itself
    put([d], 40, 20)
    look()
    cache.free(a)
    del tokens[a]
    look(window=20, sinks=3)
    assert cache.compact() > 0 and cache.compact() == 0
    look()
    put([c, e], 100, 30, counts=[100, 0])
    look()
    # what is refused leaves everything as it was
    free = cache.pool.free_pages()
    x = randn(1, 2000, kv, dim, dtype=BF16)
    for call in (lambda: cache.append([c], x, x), lambda: cache.append([c, c], x[:, :2].expand(2, -1, -1, -1), x[:, :2].expand(2, -1, -1, -1)),
                 lambda: cache.append([c], x[:, :2], x[:, :3]), lambda: cache.append([c], x[:, :2].half(), x[:, :2].half()),
                 lambda: cache.append([c], x[:, :2], x[:, :2], [3]), lambda: cache.append([99], x[:, :2], x[:, :2]),
                 lambda: cache.append([c], x[:, :2].cpu(), x[:, :2].cpu())):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    assert cache.pool.free_pages() == free
    look()
    y = randn(1, 3, kv, dim + 3, dtype=BF16)[..., 3:]      # rows off 16-byte boundaries are copied first
    cache.append([c], y, y)
    tokens[c] = tuple(torch.cat([t, y[0]]) for t in tokens[c])
    look()


@pytest.mark.parametrize("hidden,heads,kv_heads,window,sinks", [(512, 8, 2, 0, 0), (1024, 8, 8, 50, 3), (512, 4, 1, 0, 0)])
def test_decoder_block_token_by_token(hidden, heads, kv_heads, window, sinks):
    # prompts of 128 tokens, then single tokens: as a prompt of all of them
    from flashoverlap_b200.models import PagedKVCache
    from flashoverlap_b200.models.decoder_block import TPDecoderBlock

    impl = torch.classes.flashoverlap_class.OverlapImpl()
    impl.nccl_init(0, 1, [0] * 16)
    impl.cutlass_init()
    impl.overlap_init()
    block = TPDecoderBlock(impl, hidden, 512, heads, kv_heads, 1e-5, 3, dtype=BF16, window=window, sinks=sinks)
    batch, first, total = 2, 128, 192
    resid = randn(batch, total, hidden, dtype=BF16, seed=5)
    h = (resid.float() * torch.rsqrt(resid.float().pow(2).mean(-1, keepdim=True) + 1e-5)).to(BF16)
    want_q, want_r = (x.view(batch, total, -1) for x in block.forward_reference(h.view(-1, hidden), resid.view(-1, hidden), batch, total))
    cache = PagedKVCache(40, 16, kv_heads, hidden // heads, dtype=BF16)
    seqs = [cache.add() for _ in range(batch)]
    q, r = block(h[:, :first].reshape(-1, hidden), resid[:, :first].reshape(-1, hidden), batch, first, cache=cache, seqs=seqs)

    def close(got, want):
        # five products of 16-bit values in a row, each rounded: 2^-8 of the largest value and as much for what follows from it
        assert (got.float() - want.float()).abs().max() <= 2 ** -5 * want.float().abs().max()

    close(q.view(batch, first, -1), want_q[:, :first])
    close(r.view(batch, first, -1), want_r[:, :first])
    for t in range(first, first + 20):
        q, r = block.decode(h[:, t], resid[:, t], cache, seqs)
        assert q.shape[0] == batch
        close(q, want_q[:, t])
        close(r[:batch], want_r[:, t])
    assert [cache.length(s) for s in seqs] == [first + 20] * batch
    with pytest.raises(ValueError, match="empty"):
        block(h[:, :first].reshape(-1, hidden), resid[:, :first].reshape(-1, hidden), batch, first, cache=cache, seqs=seqs)
    torch.cuda.synchronize()
    impl.check_status()


# ---- forms that the sizes above do not take -----------------------------------------
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,page,window,sinks", [(16, 1, 24, 0, 0), (40, 1, 64, 0, 0), (10, 2, 16, 3500, 17), (8, 1, 128, 0, 0)])
def test_single_tokens_of_long_sequences(dtype, dim, heads, kv, page, window, sinks):
    # more tiles than a cluster takes: stretches that begin and end anywhere, joined by the second kernel
    lengths = [5000, 0, 4999, 1, 777, 4097]
    p = Paged(lengths, kv, dim, page, dtype, seed=heads)
    q = randn(len(lengths), heads, dim, dtype=dtype, seed=9)
    got = ops.paged_attention(q, p.cache, p.table, p.lengths, window=window, sinks=sinks)
    p.check(q, got, window, sinks)
    assert torch.equal(got, ops.paged_attention(q, p.cache, p.table, p.lengths, window=window, sinks=sinks))
    table = p.table.clone()
    table[2, 3] = -1                     # visible, or hidden by the window
    got = ops.paged_attention(q, p.cache, table, p.lengths, window=window, sinks=sinks)
    p.check(q, got, window, sinks, only=(0, 1, 3, 4, 5) + ((2,) if window else ()))
    assert window or got[2].isnan().all()


@pytest.mark.parametrize("scale", [-0.07, 0.0, 3.0])
def test_scales_of_single_tokens(scale):
    for lengths, dim in (([40, 300, 5], 128), ([9000, 33], 64)):
        p = Paged(lengths, 1, dim, 16, BF16)
        q = randn(len(lengths), 5, dim, dtype=BF16)
        p.check(q, ops.paged_attention(q, p.cache, p.table, p.lengths, scale=scale), scale=scale)


def test_sequences_in_the_hundreds():
    # more sequences than a warp looks at together, most of them short or empty; the table is wider than any needs
    lengths = [(i * 37) % 61 if i % 3 else 0 for i in range(333)] + [2900]
    p = Paged(lengths, 2, 64, 16, FP16, width=200)
    q = randn(len(lengths), 6, 64, dtype=FP16)
    got = ops.paged_attention(q, p.cache, p.table, p.lengths)
    p.check(q, got, only=list(range(0, 334, 7)) + [333, 332, 331])
    assert not got[::3][:111].any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,sq,sk,heads,kv,window,sinks", [(3, 1500, 1500, 16, 4, 300, 5), (40, 300, 300, 8, 8, 0, 0),
                                                               (2, 30, 2000, 8, 1, 0, 0), (1, 100, 1700, 6, 2, 900, 130)])
def test_many_and_few_pairs_with_values_that_are_not_finite(dim, batch, sq, sk, heads, kv, window, sinks):
    # more pairs of tiles than SMs, and so few that their keys are divided; lengths that leave pairs without keys
    q = randn(batch, sq, heads, dim, dtype=BF16, seed=1)
    k, v = randn(batch, sk, kv, dim, dtype=BF16, seed=2), randn(batch, sk, kv, dim, dtype=BF16, seed=3)
    lengths = [(sk * (b + 1)) // batch - 3 * b for b in range(batch)]
    lengths[-1] = sk
    clean = v.clone()
    for b, n in enumerate(lengths):
        v[b, n:], k[b, n:] = float("inf"), float("nan")
    bad = sk - sq // 2
    v[0, bad, :, 5] = float("nan")
    v[-1, bad, 0, 3] = float("-inf")
    got = ops.prompt_attention(q, k, v, window=window, sinks=sinks, lengths=ints(*lengths))
    group = heads // kv
    pos = torch.arange(sk - sq, sk)
    for b in {0, batch // 2, batch - 1}:
        for h in {0, heads - 1}:
            want, tol = attend(q[b, :, h], k[b, :, h // group], clean[b, :, h // group], sk - sq, lengths[b], window, sinks)
            hit = (pos >= bad) & (pos < lengths[b]) & (bad < lengths[b])
            if window:
                hit &= pos < bad + window
            if b not in (0, batch - 1) or (b == batch - 1 and b != 0 and h // group != 0):
                hit &= False
            check(got[b, ~hit, h], want[~hit], tol[~hit], f"sequence {b}, head {h}")
            col = 5 if b == 0 else 3
            if hit.any():
                assert not got[b, hit, h, col].isfinite().any()


def test_prompts_on_two_streams():
    sets = [[randn(1, n, h, 128, dtype=FP16, seed=n + h) for h in (8, 2, 2)] for n in (1900, 1901)]
    want = [ops.prompt_attention(*x, window=500, sinks=2) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for x, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(ops.prompt_attention(*x, window=500, sinks=2))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_a_split_prompt_in_two_graphs():
    # each graph has partial results of its own
    sets = [[randn(1, n, h, 64, dtype=BF16, seed=n + h) for n, h in ((20, 8), (3000, 1), (3000, 1))] for _ in range(2)]
    sets[1] = [x + 1 for x in sets[1]]
    want = [ops.prompt_attention(*x) for x in sets]
    graphs, outs = [], []
    for x in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.prompt_attention(*x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_decoder_block_refuses_heads_that_the_kernels_do_not_take():
    from flashoverlap_b200.models import PagedKVCache
    from flashoverlap_b200.models.decoder_block import TPDecoderBlock

    with pytest.raises(ValueError, match="heads of 64 or 128"):
        TPDecoderBlock(None, 512, 256, 2, 2, window=10)
    block = TPDecoderBlock(None, 512, 256, 2, 2)      # heads of 256: prompts as before, no cache
    cache = PagedKVCache(4, 16, 2, 256)
    x = torch.zeros(1, 512, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="heads of 64 or 128"):
        block.decode(x, x, cache, [cache.add()])
    assert cache.pool.free_pages() == 4
