"""The pool of a paged cache takes tokens back: what a refused operation had been given, and no page that others read."""
import random

import pytest
import torch

import flashoverlap_b200  # noqa: F401

Pool = torch.classes.flashoverlap_class.PagePool


def state(pool, seqs):
    return [(pool.length(s), pool.pages(s)) for s in seqs], pool.free_pages(), pool.num_sequences()


@pytest.mark.parametrize("size,seed", [(1, 0), (4, 1), (16, 2)])
def test_growing_is_undone_to_the_last_free_page(size, seed):
    rng = random.Random(seed)
    pool, twin = Pool(300, size), Pool(300, size)
    seqs = []
    for step in range(400):
        what = rng.choice(["add", "grow", "undone", "undone", "fork", "free"])
        some = rng.sample(seqs, rng.randrange(0, len(seqs) + 1))
        counts = [rng.randrange(0, 3 * size) for _ in some]
        if what == "undone":
            before = state(pool, seqs)
            try:
                pool.grow(some, counts)
            except RuntimeError:
                continue
            pool.shrink(some, counts)
            assert state(pool, seqs) == before
            continue
        n, s = rng.randrange(0, 2 * size), rng.choice(seqs) if seqs else None
        results = []
        for p in (pool, twin):
            try:
                if what == "add":
                    results.append(p.add(n))
                elif what == "grow":
                    p.grow(some, counts)
                elif s is not None:
                    results.append(p.fork(s)[0] if what == "fork" else p.free(s))
            except RuntimeError:
                results.append(None)
        if what in ("add", "fork") and results and results[0] is not None:
            assert results[0] == results[1]
            seqs.append(results[0])
        elif what == "free" and s is not None:
            seqs.remove(s)
        assert state(pool, seqs) == state(twin, seqs)    # as if nothing had been tried


def test_shared_pages_are_not_opened_again():
    pool = Pool(10, 4)
    a = pool.add(8)
    b, moves = pool.fork(a)
    assert moves.shape[0] == 0 and pool.free_pages() == 8
    with pytest.raises(RuntimeError, match="shares"):
        pool.shrink([b], [1])
    assert pool.length(b) == 8 and pool.pages(b) == pool.pages(a)
    pool.shrink([b], [4])                   # to a page's end: the page is the other's alone
    assert pool.length(b) == 4 and pool.pages(b) == pool.pages(a)[:1] and pool.free_pages() == 8
    pool.shrink([a], [3])
    assert pool.length(a) == 5 and pool.free_pages() == 8
    pool.shrink([a, b], [1, 0])
    assert pool.free_pages() == 9
    pool.shrink([b], [4])
    assert pool.length(b) == 0 and pool.pages(b) == [] and pool.free_pages() == 9


def test_what_shrinking_refuses():
    pool = Pool(10, 4)
    a, b = pool.add(6), pool.add(4)
    c, _ = pool.fork(b)
    before = state(pool, [a, b, c])
    for seqs, counts in (([a], [7]), ([a], [-1]), ([a, a], [1, 1]), ([a], [1, 1]), ([9], [0]), ([a, b], [1, 1]), ([a], [2 ** 62])):
        with pytest.raises(RuntimeError):
            pool.shrink(seqs, counts)
        assert state(pool, [a, b, c]) == before


def test_a_cache_of_other_types_is_refused():
    from flashoverlap_b200.models import PagedKVCache

    for dtype in (torch.float32, torch.float8_e4m3fn, torch.int16):
        with pytest.raises(ValueError, match="float16 or bfloat16"):
            PagedKVCache(4, 16, 2, 64, dtype=dtype, device="cuda:0")
