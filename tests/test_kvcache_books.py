"""CPU tests of the page bookkeeping behind the paged key/value cache.

A model of the pool's contents (one value per token) is driven through random
adds, forks, appends, truncations, frees and compactions: after each, every
sequence must read back exactly what was written to it.
"""

from __future__ import annotations

import random

import pytest

from mxwave_b200.kvcache import PageBooks


class Pool:
    """Token values by page, and what each sequence should hold."""

    def __init__(self, pages: int, page: int) -> None:
        self.books = PageBooks(pages, page)
        self.page = page
        self.data = [[None] * page for _ in range(pages)]
        self.want: dict[int, list[int]] = {}
        self.clock = 0

    def copy(self, moves: list[tuple[int, int]]) -> None:
        sources, targets = [s for s, _ in moves], [t for _, t in moves]
        assert len(set(targets)) == len(targets) and not set(targets) & set(sources)
        for s, t in moves:
            self.data[t] = list(self.data[s])

    def grow(self, seqs: list[int], tokens: list[int]) -> None:
        self.copy(self.books.grow(seqs, tokens))
        for seq, n in zip(seqs, tokens):
            pages, length = self.books.pages_of(seq), self.books.length(seq)
            for at in range(length - n, length):
                self.clock += 1
                self.data[pages[at // self.page]][at % self.page] = self.clock
                self.want[seq].append(self.clock)

    def check(self) -> None:
        for seq, want in self.want.items():
            pages = self.books.pages_of(seq)
            assert self.books.length(seq) == len(want) and len(pages) == -(-len(want) // self.page)
            assert [self.data[pages[i // self.page]][i % self.page] for i in range(len(want))] == want
        held = {p for seq in self.want for p in self.books.pages_of(seq)}
        assert self.books.free_pages == self.books.pages - len(held)


@pytest.mark.parametrize("page", [1, 3, 16])
@pytest.mark.parametrize("seed", range(6))
def test_random_histories(page: int, seed: int) -> None:
    rng = random.Random(seed)
    pool = Pool(40, page)
    full = 0
    for _ in range(400):
        seqs = list(pool.want)
        op = rng.choice(("add", "fork", "grow", "grow", "grow", "truncate", "free", "compact"))
        if op == "add" and len(seqs) < 8:
            pool.want[pool.books.add()] = []
        elif op == "fork" and seqs and len(seqs) < 8:
            seq = rng.choice(seqs)
            pool.want[pool.books.fork(seq)] = list(pool.want[seq])
        elif op == "grow" and seqs:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            before = [(pool.books.length(s), pool.books.pages_of(s)) for s in seqs]
            try:
                pool.grow(some, [rng.randint(1, 2 * page + 1) for _ in some])
            except RuntimeError as err:
                assert "full" in str(err)
                assert before == [(pool.books.length(s), pool.books.pages_of(s)) for s in seqs]
                full += 1
                seq = rng.choice(seqs)
                pool.books.free(seq)
                del pool.want[seq]
        elif op == "truncate" and seqs:
            seq = rng.choice(seqs)
            n = rng.randint(0, len(pool.want[seq]))
            pool.books.truncate(seq, n)
            del pool.want[seq][n:]
        elif op == "free" and len(seqs) > 3:
            seq = rng.choice(seqs)
            pool.books.free(seq)
            del pool.want[seq]
        elif op == "compact":
            pool.copy(pool.books.compact())
            held = {p for s in pool.want for p in pool.books.pages_of(s)}
            assert held == set(range(len(held)))
        pool.check()
    for seq in list(pool.want):
        pool.books.free(seq)
    assert pool.books.free_pages == 40


def test_forks_share_until_a_write() -> None:
    books = PageBooks(8, 4)
    a = books.add()
    assert books.grow([a], [6]) == []
    b = books.fork(a)
    assert books.free_pages == 6 and books.pages_of(a) == books.pages_of(b)
    copies = books.grow([a, b], [1, 1])  # the first writer gets the copy, the second keeps the page
    assert len(copies) == 1 and copies[0][0] == books.pages_of(b)[1] and copies[0][1] == books.pages_of(a)[1]
    assert books.pages_of(a)[0] == books.pages_of(b)[0]
    assert books.grow([a, b], [1, 1]) == []


def test_full_pages_need_no_copy() -> None:
    books = PageBooks(8, 4)
    a = books.add()
    books.grow([a], [8])
    b = books.fork(a)
    assert books.grow([b], [1]) == []
    assert books.pages_of(b)[:2] == books.pages_of(a)


@pytest.mark.parametrize("call", [
    lambda b: b.grow([0, 0], [1, 1]),
    lambda b: b.grow([0], [0]),
    lambda b: b.grow([0], [1, 1]),
    lambda b: b.truncate(0, 3),
    lambda b: b.truncate(0, -1),
    lambda b: PageBooks(0, 16),
])
def test_refusals(call) -> None:
    books = PageBooks(4, 4)
    books.grow([books.add()], [2])
    with pytest.raises(ValueError):
        call(books)


def test_unknown_sequence_and_full_pool() -> None:
    books = PageBooks(2, 4)
    with pytest.raises(KeyError):
        books.free(7)
    a = books.add()
    books.grow([a], [8])
    b = books.add()
    with pytest.raises(RuntimeError, match="full"):
        books.grow([b], [1])
    with pytest.raises(KeyError):
        books.grow([99], [1])
    assert books.length(b) == 0 and books.free_pages == 0
