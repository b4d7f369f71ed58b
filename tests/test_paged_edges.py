"""The paged KV cache's host side at its edges, on the CPU: pools that hold exactly what a call needs, calls that are refused
and change nothing."""

import random

import pytest
import torch

import collaborative_edge_system_b200 as cea
from collaborative_edge_system_b200 import _lib, paged

CPU = torch.device("cpu")


class HostCache(paged.PagedKVCache):
    """The cache with small buffers on the CPU."""

    def __init__(self, pages, page_size):
        super().__init__(1, pages, page_size, 1, 1, dtype=torch.float32, device=torch.device("cuda"))

    def _make_buffers(self, shape, dtype, device):
        self.k, self.v = torch.zeros(shape), torch.zeros(shape)
        self.device = CPU

    def _copy(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        self.k[:, dst], self.v[:, dst] = self.k[:, src], self.v[:, src]

    def state(self):
        return self.num_free_pages, list(self.pool.refs), {s: (self.pages(s), self.length(s)) for s in sorted(self._lengths)}


def _pages_needed(cache, seqs, counts):
    """Pages that an extension cannot do without: those behind the last, and one for each sequence that writes a page
    which some other sequence still has (the last of the writers keeps the page if nobody else has it)."""
    ps, need, writers = cache.page_size, 0, {}
    for s, c in zip(seqs, counts):
        n = cache.length(s)
        need += (n + c + ps - 1) // ps - (n + ps - 1) // ps
        if c and n % ps:
            writers.setdefault(cache.pages(s)[-1], []).append(s)
    for page, who in writers.items():
        others = [s for s in cache._lengths if page in cache.pages(s) and s not in who]
        need += len(who) if others else len(who) - 1
    return need


def test_two_owners_of_a_page_split_with_one_free_page():
    cache = HostCache(2, 4)
    a = cache.add()
    cache.extend([a], [4])
    b, = cache.fork(a)
    cache.truncate(a, 3)
    cache.truncate(b, 2)
    assert cache.pool.refs == [2, 0]
    cache.extend([a, b], [1, 2])
    assert sorted(cache.pages(a) + cache.pages(b)) == [0, 1] and cache.num_free_pages == 0
    assert (cache.length(a), cache.length(b)) == (4, 4)


@pytest.mark.parametrize("seed", range(12))
def test_extension_is_refused_only_where_the_pages_are_missing(seed):
    rnd = random.Random(seed)
    cache = HostCache(rnd.choice([4, 5, 7, 14]), rnd.choice([2, 3, 4]))
    refused = 0
    for _ in range(400):
        ids = sorted(cache._lengths)
        move = rnd.choice(["add", "extend", "extend", "extend", "fork", "twins", "truncate", "free"])
        if move == "add" or not ids:
            cache.add()
        elif move == "extend":
            some = rnd.sample(ids, rnd.choice([len(ids), rnd.randint(1, len(ids))]))
            counts = [rnd.randint(0, rnd.choice([1, 3])) for _ in some]
            need, free, before = _pages_needed(cache, some, counts), cache.num_free_pages, cache.state()
            if need > free:
                with pytest.raises(cea.OutOfPages):
                    cache.extend(some, counts)
                assert cache.state() == before
                refused += 1
            else:
                cache.extend(some, counts)
                assert cache.num_free_pages == free - need
        elif move == "fork":
            s = rnd.choice(ids)
            try:
                cache.fork(s, rnd.randint(0, cache.length(s)), rnd.randint(1, 2))
            except cea.OutOfPages:
                pass
        elif move == "twins":  # owners of full pages that all step back into the last one
            s = rnd.choice(ids)
            n = cache.length(s) // cache.page_size * cache.page_size
            if n:
                for t in [s] + cache.fork(s, n, rnd.randint(1, 2)):
                    cache.truncate(t, n - 1)
        elif move == "truncate":
            s = rnd.choice(ids)
            cache.truncate(s, rnd.randint(0, cache.length(s)))
        elif len(ids) > 2:
            cache.free(rnd.choice(ids))
        counted = [0] * len(cache.pool.refs)
        for s in cache._lengths:
            for p in cache.pages(s):
                counted[p] += 1
        assert counted == cache.pool.refs and cache.num_free_pages == counted.count(0)
    assert refused


@pytest.fixture
def anywhere(monkeypatch):
    """Checks that come before the kernels, on CPU tensors: what they let pass ends in ``reached``."""
    reached = []
    monkeypatch.setattr(_lib, "device_number", lambda *t: 0)
    for name in ("paged_attn", "paged_append", "copy_pages"):
        monkeypatch.setattr(_lib, name, lambda p, dev: reached.append(p))
    return reached


def test_cache_refuses_rows_that_are_not_the_batchs(anywhere):
    cache = HostCache(4, 4)
    batch = cache.extend([cache.add(), cache.add()], [3, 2])
    good = torch.zeros(5, 1, 1)
    cache.append(0, good, good, batch)
    cache.attend(0, good, batch)
    assert [p.T for p in anywhere] == [5, 5]
    anywhere.clear()
    for rows in (0, 4, 6):
        x = torch.zeros(rows, 1, 1)
        for call in (lambda: cache.append(0, x, x, batch), lambda: cache.append(0, good, x, batch),
                     lambda: cache.attend(0, x, batch)):
            with pytest.raises(ValueError):
                call()
    assert not anywhere


def test_allocator_refusals_change_nothing():
    a = cea.PageAllocator(4)
    a.alloc(3)
    a.share([1])
    before = list(a.refs), a.num_free
    for call in (lambda: a.release([0, 0]), lambda: a.release([0, 3]), lambda: a.release([1, 1, 1]), lambda: a.release([-1]),
                 lambda: a.release([0, 4]), lambda: a.share([0, 3]), lambda: a.share([-2]), lambda: a.share([0, 4]),
                 lambda: a.alloc(-1), lambda: a.move([0], [3, 3]), lambda: a.move([0], [1]), lambda: a.move([3], [0]),
                 lambda: a.move([0, 1], [3, 3]), lambda: a.move([0, 0], [3, 2])):
        with pytest.raises(ValueError):
            call()
        assert (list(a.refs), a.num_free) == before
    a.release([0, 1, 1])
    assert a.num_free == 3 and a.alloc(3) == [0, 1, 3]


def _call(**kw):
    x = {"q": torch.zeros(3, 4, 8), "k_pages": torch.zeros(5, 2, 4, 8), "v_pages": torch.zeros(5, 2, 4, 8),
         "page_table": torch.zeros(2, 3, dtype=torch.int32), "seq_lens": torch.ones(2, dtype=torch.int32),
         "q_offsets": torch.tensor([0, 1, 3], dtype=torch.int32)}
    return cea.paged_attention(**{**x, **kw})


@pytest.mark.parametrize("kw", [{"min_q_len": 2**31}, {"max_q_len": 2**40}, {"min_q_len": -(2**33)}, {"max_q_len": 1.5},
                                {"min_q_len": 1.0}, {"min_q_len": "1"}, {"scale": "1"}, {"scale": None, "max_q_len": 3.0}])
def test_numbers_that_are_no_count_or_scale_are_refused(anywhere, kw):
    with pytest.raises((ValueError, TypeError)):
        _call(**kw)
    assert not anywhere


def test_heads_without_columns_are_refused(monkeypatch):
    monkeypatch.setattr(_lib, "device_number", lambda *t: 0)
    codes = []
    monkeypatch.setattr(_lib, "paged_attn", lambda p, like: codes.append(_lib.paged_attn_kernels(p)))
    _call(q=torch.zeros(3, 4, 0), k_pages=torch.zeros(5, 2, 4, 0), v_pages=torch.zeros(5, 2, 4, 0))
    assert codes == [-1]  # the library's own refusal, not a division by zero
