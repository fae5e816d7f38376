"""Bookkeeping of the 4-bit cache's pages: every sequence keeps its positions whatever is forked, written, freed and compacted."""
import random

import pytest
import torch

from shiftaddllm_b200 import decode_ops
from shiftaddllm_b200.kv4 import PAGE, Kv4Cache


@pytest.fixture()
def on_cpu(monkeypatch):
    def copy(pool, src, dst):
        assert len(src) == len(dst) == len(set(dst)) and not set(src) & set(dst)
        pool[:, list(dst)] = pool[:, list(src)]

    monkeypatch.setattr(decode_ops, "copy_kv4_pages", copy)


def check(cache, content):
    seen = {}
    for slot, values in enumerate(content):
        pages = cache.pages_of(slot)
        assert cache.table[slot].tolist() == pages + [-1] * (cache.table.shape[1] - len(pages))
        assert len(set(pages)) == len(pages) >= -(-len(values) // PAGE)
        for p in pages:
            seen[p] = seen.get(p, 0) + 1
        for pos, v in enumerate(values):
            assert cache.pool[0, pages[pos // PAGE], 0, pos % PAGE] == v
    assert all(cache._users[p] == seen.get(p, 0) for p in range(cache.pages))
    assert sorted(cache._free) == [p for p in range(cache.pages) if p not in seen]


@pytest.mark.parametrize("seed", range(6))
def test_sequences_keep_what_was_written(on_cpu, seed):
    rng = random.Random(seed)
    slots, max_len = 5, 300
    cache = Kv4Cache(2, 1, 64, slots, max_len, pages=14, device="cpu")
    content = [[] for _ in range(slots)]
    for _ in range(300):
        what, s = rng.choice(("write", "write", "write", "fork", "free", "cut", "compact")), rng.randrange(slots)
        if what == "write":
            n = min(rng.choice((1, 1, 5, 70, 130)), max_len - len(content[s]))
            first, before = len(content[s]), (cache.free_pages, cache.pages_of(s))
            try:
                cache.reserve(s, first, first + n)
            except RuntimeError:
                assert (cache.free_pages, cache.pages_of(s)) == before
                continue
            for pos in range(first, first + n):
                page = cache.pages_of(s)[pos // PAGE]
                assert cache._users[page] == 1
                v = rng.randrange(256)
                cache.pool[:, page, 0, pos % PAGE] = v
                content[s].append(v)
        elif what == "fork":
            d = rng.randrange(slots)
            cache.fork(s, d)
            content[d] = list(content[s])
        elif what == "free":
            cache.free(s)
            content[s] = []
        elif what == "cut":
            content[s] = content[s][:rng.randrange(len(content[s]) + 1)]
            cache.truncate(s, len(content[s]))
        else:
            used = cache.compact()
            assert used == cache.pages - cache.free_pages and all(p < used for t in range(slots) for p in cache.pages_of(t))
        check(cache, content)


def test_refusals(on_cpu):
    cache = Kv4Cache(1, 2, 128, 2, 200, pages=3, device="cpu")
    assert cache.table.shape == (2, 4) and cache.free_pages == 3
    for args in ((0, -1, 5), (0, 5, 4), (0, 0, 201), (0, 65, 66)):
        with pytest.raises(ValueError):
            cache.reserve(*args)
    cache.reserve(0, 0, 130)
    with pytest.raises(RuntimeError):
        cache.reserve(1, 0, 1)
    cache.fork(0, 1)
    with pytest.raises(RuntimeError):      # the shared page cannot be copied
        cache.reserve(1, 130, 131)
    assert cache.pages_of(0) == cache.pages_of(1) == [0, 1, 2]
    cache.free(0)
    cache.reserve(1, 130, 131)
    with pytest.raises(ValueError):
        cache.truncate(1, -1)
    for bad in (dict(layers=0), dict(slots=0), dict(max_len=0), dict(pages=0)):
        with pytest.raises(ValueError):
            Kv4Cache(**{**dict(layers=1, kv_heads=1, hd=64, slots=1, max_len=1, device="cpu"), **bad})
