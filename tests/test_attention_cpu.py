"""Attention operators without a GPU: where tokens lie, which tiles a position looks at (the host build of the functions
the kernels use), and what is refused before anything is launched."""
import random

import pytest
import torch

import flashoverlap_b200  # noqa: F401  (loads the native library)

OPS = torch.ops.flashoverlap_op


def test_operators_are_registered():
    for name in ("prompt_attention", "paged_attention", "cache_append", "copy_pages", "prompt_attention_new",
                 "paged_attention_new", "page_place", "seen_tiles"):
        assert hasattr(OPS, name), name


@pytest.mark.parametrize("page", [1, 2, 3, 7, 8, 16, 24, 50, 64, 100, 256, 4096])
def test_places_of_tokens(page):
    rng = random.Random(page)
    pages, kv, dim = 1000, 3, 64
    row = [rng.randrange(pages) for _ in range(17)]
    for pos in [0, 1, page - 1, page, page + 1, 5 * page + page // 2, 17 * page - 1]:
        got = OPS.page_place(row, pos, pages, kv, page, dim, 2)
        at = row[pos // page]
        assert got == [at, pos % page, ((at * 2 * kv + 2) * page + pos % page) * dim]


def test_offsets_pass_32_bits():
    pages, kv, page, dim = 2_000_000, 8, 64, 128
    row = [0] * 20 + [pages - 1]
    _, place, offset = OPS.page_place(row, 20 * page + 63, pages, kv, page, dim, 7)
    assert place == 63 and offset == ((pages - 1) * 2 * kv + 7) * page * dim + 63 * dim and offset > 2 ** 37


def test_pages_that_are_not_there():
    for bad in (-1, -(2 ** 31), 10, 2 ** 31 - 1):
        assert OPS.page_place([3, bad, 4], 16 + 5, 10, 2, 16, 64, 0)[0] == -1
        assert OPS.page_place([3, bad, 4], 5, 10, 2, 16, 64, 0)[0] == 3
    assert OPS.page_place([3, 4], 32, 10, 2, 16, 64, 0)[0] == -1            # behind the row
    assert OPS.page_place([3, 4], 2 ** 31 - 1, 10, 2, 16, 64, 0)[0] == -1
    assert OPS.page_place([], 0, 10, 2, 16, 64, 0)[0] == -1
    assert OPS.page_place([0], 0, 0, 2, 16, 64, 0)[0] == -1                 # a cache without pages


def test_division_by_the_page_size_is_exact():
    rng = random.Random(5)
    for page in list(range(1, 70)) + [127, 129, 1000, 4095, 4097, 65535, 1 << 20]:
        for pos in [0, page - 1, page, 2 ** 31 - 1] + [rng.randrange(2 ** 31) for _ in range(20)]:
            # a row long enough would not fit: what counts is the place
            got = OPS.page_place([0], pos, 1, 1, page, 8, 0)
            assert got[1] == pos % page, (page, pos)


@pytest.mark.parametrize("tile,align", [(16, 1), (64, 16), (128, 32), (128, 1), (64, 64)])
def test_tiles_hold_all_visible_tokens_once(tile, align):
    rng = random.Random(tile)
    for _ in range(2000):
        length = rng.choice([0, 1, rng.randrange(1, 40), rng.randrange(1, 900)])
        p0 = rng.randrange(0, 900)
        p1 = p0 + rng.choice([0, 1, 31, 127])
        window, sinks = rng.choice([0, 1, 2, 63, 64, 65, 300, 2 ** 31 - 1]), rng.choice([0, 1, 4, 63, 64, 65, 500, 2 ** 31 - 1])
        starts = OPS.seen_tiles(p0, p1, length, window, sinks, tile, align)
        assert all(b - a >= tile for a, b in zip(starts, starts[1:])) and all(0 <= a < length for a in starts)
        held = {j for a in starts for j in range(a, a + tile)}
        need = {j for i in range(p0, p1 + 1) for j in range(min(i + 1, length))
                if window == 0 or j > i - window or j < sinks}
        assert need <= held
        if p1 < length:     # no more tiles than the sinks and the rest take
            lo = max(0, p0 - window + 1) if window else 0
            front = min(sinks, lo)
            assert len(starts) <= -(-front // tile) + -(-(p1 + 1 - lo // align * align) // tile)
        assert all(a % align == 0 or a % tile == 0 for a in starts)


def test_tiles_of_the_longest_sequences():
    top = 2 ** 31 - 1025
    assert len(OPS.seen_tiles(top - 1, top - 1, top, 100, 2 ** 20, 64, 1)) == 2 ** 14 + 2
    assert OPS.seen_tiles(top - 1, top - 1, top, 100, 3, 64, 1) == [0, top - 100, top - 36]
    assert OPS.seen_tiles(top - 1, top - 1, top, 2 ** 31 - 1, 3, 1024, 1)[0] == 0


def test_operators_refuse_tensors_on_the_cpu():
    from flashoverlap_b200 import ops

    x = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    cache = torch.zeros(4, 2, 2, 8, 64, dtype=torch.float16)
    ints = torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    for call in (lambda: ops.prompt_attention(x, x, x), lambda: ops.paged_attention(x[0, :1], cache, table, ints),
                 lambda: ops.cache_append(x, x, cache, table, ints),
                 lambda: ops.copy_pages(cache, torch.tensor([[0, 1]])),
                 lambda: OPS.prompt_attention_new(x, x, x, 0, 0, None, None),
                 lambda: OPS.paged_attention_new(x[0, :1], cache, table, ints, 0, 0, None),
                 lambda: OPS.cache_append(x, x, cache, table, ints, None),
                 lambda: OPS.copy_pages(cache, torch.tensor([[0, 1]]))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_moves_are_checked_before_anything_is_copied():
    cache = torch.zeros(8, 2, 2, 8, 64, dtype=torch.float16)
    for moves, why in (([[0, 8]], "outside"), ([[-1, 2]], "outside"), ([[8, 2]], "outside"), ([[0, 2], [1, 2]], "twice"),
                       ([[0, 1], [1, 2]], "reads page 1"), ([[3, 3]], "reads page 3"), ([[2 ** 40, 0]], "outside")):
        with pytest.raises(RuntimeError, match=why):
            OPS.copy_pages(cache, torch.tensor(moves))
    with pytest.raises(RuntimeError, match=r"\[n, 2\]"):
        OPS.copy_pages(cache, torch.tensor([0, 1]))
    with pytest.raises(RuntimeError, match="int32 or int64"):
        OPS.copy_pages(cache, torch.tensor([[0.0, 1.0]]))
    # one page may go to several; a list in any order and of any layout is read as it stands
    with pytest.raises(RuntimeError, match="CUDA"):
        OPS.copy_pages(cache, torch.tensor([[0, 0], [5, 6]]).t())
