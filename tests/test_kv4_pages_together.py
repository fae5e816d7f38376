"""Pages of several sequences taken at once: what was written stays, whatever is forked, freed and refused in between."""
import random

import pytest
import torch

from shiftaddllm_b200 import decode_ops
from shiftaddllm_b200.kv4 import PAGE, Kv4Cache


@pytest.mark.parametrize("seed", range(4))
def test_sequences_written_together(monkeypatch, seed):
    def copy(pool, src, dst):
        assert len(src) == len(dst) == len(set(dst)) and not set(src) & set(dst)
        pool[:, list(dst)] = pool[:, list(src)]

    monkeypatch.setattr(decode_ops, "copy_kv4_pages", copy)
    rng, slots = random.Random(seed), 6
    cache = Kv4Cache(2, 1, 64, slots, 300, pages=16, device="cpu")
    content, refused = [[] for _ in range(slots)], 0
    for _ in range(150):
        what, s = rng.choice(("write", "write", "write", "fork", "free", "cut", "compact")), rng.randrange(slots)
        if what == "write":
            ranges = [(b, len(content[b]), min(300, len(content[b]) + rng.choice((0, 1, 7, 64, 100)))) for b in rng.sample(range(slots), rng.randint(1, slots))]
            before = cache.free_pages, [cache.pages_of(b) for b in range(slots)], list(cache._users), cache.table.clone()
            try:
                cache.reserve_all(ranges)
            except RuntimeError:
                refused += 1
                assert (cache.free_pages, [cache.pages_of(b) for b in range(slots)], list(cache._users)) == before[:3] and torch.equal(cache.table, before[3])
                continue
            for b, first, last in ranges:
                for pos in range(first, last):
                    page = cache.pages_of(b)[pos // PAGE]
                    assert cache._users[page] == 1
                    content[b].append(rng.randrange(256))
                    cache.pool[:, page, 0, pos % PAGE] = content[b][-1]
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
            cache.compact()
        uses = [p for b in range(slots) for p in cache.pages_of(b)]
        assert all(cache._users[p] == uses.count(p) for p in range(cache.pages)) and sorted(cache._free) == sorted(set(range(cache.pages)) - set(uses))
        for b in range(slots):
            pages = cache.pages_of(b)
            assert cache.table[b].tolist() == pages + [-1] * (cache.table.shape[1] - len(pages))
            assert [int(cache.pool[1, pages[p // PAGE], 0, p % PAGE]) for p in range(0, len(content[b]), 5)] == content[b][::5]
    assert refused
