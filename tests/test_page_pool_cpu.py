"""The pool of a paged cache: sequences grow, fork, end and move, against a model of what every page holds."""
import random

import pytest
import torch

import flashoverlap_b200  # noqa: F401

Pool = torch.classes.flashoverlap_class.PagePool


def contents(pool, memory, seq):
    size, n = pool.page_size(), pool.length(seq)
    pages = pool.pages(seq)
    assert len(pages) == -(-n // size)
    return [memory[pages[i // size]][i % size] for i in range(n)]


@pytest.mark.parametrize("pages,size,seed", [(40, 4, 0), (40, 1, 1), (12, 7, 2), (200, 16, 3)])
def test_random_life_of_a_cache(pages, size, seed):
    rng = random.Random(seed)
    pool = Pool(pages, size)
    memory = [[None] * size for _ in range(pages)]
    want, token = {}, 0

    def put(seq, new):
        nonlocal token
        for _ in range(new):
            i = len(want[seq])
            memory[pool.pages(seq)[i // size]][i % size] = token
            want[seq].append(token)
            token += 1

    def move(moves):
        old = [list(p) for p in memory]
        assert len({int(t) for _, t in moves}) == len(moves) and not ({int(f) for f, _ in moves} & {int(t) for _, t in moves})
        for f, t in moves.tolist():
            memory[t] = list(old[f])

    for _ in range(1500):
        what = rng.choice(["add", "grow", "grow", "grow", "fork", "free", "compact", "check"])
        seqs = sorted(want)
        before = pool.free_pages()
        try:
            if what == "add":
                n = rng.randrange(0, 3 * size)
                s = pool.add(n)
                want[s] = []
                put(s, n)
            elif what == "grow" and seqs:
                some = rng.sample(seqs, rng.randrange(1, len(seqs) + 1))
                counts = [rng.choice([0, 1, size, rng.randrange(0, 2 * size + 1)]) for _ in some]
                pool.grow(some, counts)
                for s, n in zip(some, counts):
                    put(s, n)
            elif what == "fork" and seqs:
                s = rng.choice(seqs)
                new, moves = pool.fork(s)
                assert moves.shape == ((1 if len(want[s]) % size else 0), 2) and moves.dtype == torch.int32
                move(moves)
                want[new] = list(want[s])
            elif what == "free" and seqs:
                s = rng.choice(seqs)
                pool.free(s)
                del want[s]
            elif what == "compact":
                move(pool.compact())
                used = {p for s in want for p in pool.pages(s)}
                assert used == set(range(len(used)))
        except RuntimeError as e:
            assert "out of pages" in str(e) and pool.free_pages() == before
        assert pool.num_sequences() == len(want)
        used = {p for s in want for p in pool.pages(s)}
        assert len(used) + pool.free_pages() == pages and all(0 <= p < pages for p in used)
        for s in want:
            assert pool.length(s) == len(want[s]) and contents(pool, memory, s) == want[s]


def test_tables_and_lengths():
    pool = Pool(10, 4)
    a, b, c = pool.add(9), pool.add(0), pool.add(4)
    t = pool.table([c, a, b], 0)
    assert t.dtype == torch.int32 and t.tolist() == [pool.pages(c) + [-1, -1], pool.pages(a), [-1, -1, -1]]
    assert pool.table([b], 0).tolist() == [[-1]] and pool.table([a], 5).shape == (1, 5) and pool.table([], 0).shape == (0, 1)
    assert pool.lengths([b, a]).tolist() == [0, 9] and pool.lengths([]).dtype == torch.int32
    with pytest.raises(RuntimeError, match="too narrow"):
        pool.table([a], 2)


def test_what_a_pool_refuses():
    pool = Pool(3, 4)
    a = pool.add(5)
    for call in (lambda: pool.add(-1), lambda: pool.add(5), lambda: pool.grow([a, a], [1, 1]), lambda: pool.grow([a], [-1]),
                 lambda: pool.grow([a], [1, 2]), lambda: pool.grow([a], [9]), lambda: pool.grow([a], [2 ** 62]),
                 lambda: pool.length(7), lambda: pool.free(7), lambda: pool.fork(7), lambda: pool.table([7], 0),
                 lambda: pool.lengths([-1]), lambda: pool.pages(7), lambda: Pool(-1, 4), lambda: Pool(4, 0), lambda: Pool(2 ** 40, 1),
                 lambda: pool.add(2 ** 40)):
        with pytest.raises(RuntimeError):
            call()
    assert pool.length(a) == 5 and pool.free_pages() == 1 and pool.num_sequences() == 1
    b, _ = pool.fork(a)
    with pytest.raises(RuntimeError, match="out of pages"):
        pool.fork(a)
    pool.free(a)
    assert pool.free_pages() == 1 and pool.pages(b)[0] not in (pool.pages(pool.add(1)),)
    with pytest.raises(RuntimeError):
        pool.free(a)


def test_what_a_cache_refuses_before_it_takes_memory():
    from flashoverlap_b200.models import PagedKVCache

    for kw in (dict(device="cpu"), dict(head_dim=12), dict(head_dim=0), dict(kv_heads=0), dict(page_size=0)):
        args = dict(pages=4, page_size=16, kv_heads=2, head_dim=64, device="cuda:0")
        args.update(kw)
        with pytest.raises(ValueError):
            PagedKVCache(**args)


def test_pages_of_a_forked_tree():
    # a page lives until the last sequence that holds it has ended, in whatever order they end
    pool = Pool(20, 4)
    root = pool.add(8)
    leaves = [pool.fork(root)[0] for _ in range(5)]
    assert pool.free_pages() == 18 and all(pool.pages(s) == pool.pages(root) for s in leaves)
    pool.grow(leaves, [1] * 5)
    assert pool.free_pages() == 13 and len({pool.pages(s)[-1] for s in leaves}) == 5
    pool.free(root)
    assert pool.free_pages() == 13
    moves = pool.compact()
    assert moves.shape[0] == 0
    for s in leaves[:-1]:
        pool.free(s)
    assert pool.free_pages() == 17
    moves = pool.compact().tolist()
    assert all(t < 3 <= f for f, t in moves) and sorted(pool.pages(leaves[-1])) == [0, 1, 2]
    again, copied = pool.fork(leaves[-1])
    assert copied.tolist() == [[pool.pages(leaves[-1])[2], pool.pages(again)[2]]]
