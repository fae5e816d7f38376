"""What the batch decoder keeps of its sequences on the host, with a model without blocks on the CPU: no kernel of the framework runs."""
from types import SimpleNamespace

import pytest
import torch
import torch.nn.functional as F

from shiftaddllm_b200 import decode_ops
from shiftaddllm_b200.decoder import BcqLlamaBatchDecoder, LlamaShape

BATCH, VOCAB = 3, 50


@pytest.fixture()
def make(lib, monkeypatch):
    """make(**kw) -> a decoder whose logits follow from the token alone."""

    def norm(x, delta, weight, out, x_out, eps):
        out.copy_(F.rms_norm(x, x.shape[1:], weight, eps))

    def copy(pool, src, dst):
        assert len(src) == len(dst) == len(set(dst)) and not set(src) & set(dst)
        pool[:, list(dst)] = pool[:, list(src)]

    def sample(logits, u, token, *settings):
        token.copy_((u * logits.shape[1]).long())      # the number alone decides

    monkeypatch.setattr(decode_ops, "residual_rmsnorm_rows", norm)
    monkeypatch.setattr(decode_ops, "copy_kv4_pages", copy)
    monkeypatch.setattr(decode_ops, "sample_token", sample)
    monkeypatch.setattr(decode_ops, "attention_kv4_check", lambda workspace: None, raising=False)
    shape = LlamaShape(64, 1, 1, 1, 64, vocab=VOCAB)
    gen = torch.Generator().manual_seed(0)
    weight = lambda *size: torch.randn(*size, generator=gen).half()
    like = SimpleNamespace(embed=weight(VOCAB, 64), lm_head=weight(VOCAB, 64), final_norm=weight(64), blocks=[])
    return lambda **kw: BcqLlamaBatchDecoder(shape, **{**dict(max_len=300, batch=BATCH, like=like, device="cpu", cache_bits=4), **kw})


def state(model):
    return (model.lengths, model.pos.tolist(), model.token.tolist(), model.cache.free_pages, [model.cache.pages_of(b) for b in range(BATCH)])


def test_a_device_side_wait_that_ran_out_is_an_error(make, monkeypatch):
    looked = []

    def ran_out(workspace):
        looked.append(workspace)
        raise RuntimeError("ran out")

    model = make()
    model.prefill([[1, 2], [3], []])
    before = state(model)[:3]
    monkeypatch.setattr(decode_ops, "attention_kv4_check", ran_out)
    with pytest.raises(RuntimeError, match="ran out"):
        model.prefill([[1], [2], [3]])
    assert state(model)[:3] == before and looked[0] is not model._attn_ws
    for call in (lambda: model.generate(2), lambda: model.feed([[1, 2, 3]])):
        with pytest.raises(RuntimeError, match="ran out"):
            call()
    assert looked[1] is looked[2] is model._attn_ws


def test_the_check_reads_the_workspace_s_status(lib, monkeypatch):
    from shiftaddllm_b200 import _lib

    codes = [_lib.SAL_E_TIMEOUT, 0]
    ws = torch.zeros(16, dtype=torch.uint8)
    monkeypatch.setattr(_lib, "load", lambda: SimpleNamespace(sal_workspace_status=lambda p, s: codes.pop(0) if p == ws.data_ptr() else -1,
                                                              sal_status_string=lib.sal_status_string))
    monkeypatch.setattr(decode_ops, "_on", lambda device: decode_ops._HERE)
    monkeypatch.setattr(decode_ops, "_stream", lambda t: 0)
    with pytest.raises(RuntimeError, match="status"):
        decode_ops.attention_kv4_check(ws)
    decode_ops.attention_kv4_check(ws)


def test_a_refused_prompt_takes_no_pages(make):
    model = make(pages=4)
    before = state(model)
    with pytest.raises(RuntimeError):
        model.prefill([[1] * 200, [2] * 100, []])      # six pages
    assert state(model) == before
    model.prefill([[], [2] * 100, []])
    assert model.lengths == [0, 100, 0] and model.cache.free_pages == 2
    model.prefill([[1] * 64, [], []])
    for call in (lambda: model.generate(1), lambda: model.feed([[1, 2, 3]]), model.capture):      # two sequences need a page, one is left
        before = state(model)
        with pytest.raises(RuntimeError):
            call()
        assert state(model) == before


def test_a_full_sequence_takes_no_pages_of_the_others(make):
    model = make(max_len=130)
    model.prefill([[1] * 10, [2] * 64, [3] * 130])
    before = state(model)
    for call in (lambda: model.generate(1), lambda: model.prefill([[], [1], [1]])):
        with pytest.raises(ValueError):
            call()
        assert state(model) == before


def test_pages_for_several_sequences_or_for_none(make):
    cache = make(pages=6).cache
    cache.reserve(0, 0, 130)
    cache.fork(0, 1), cache.fork(0, 2)
    used = lambda: (cache.free_pages, [cache.pages_of(b) for b in range(BATCH)], list(cache._users))
    before = used()
    for bad in ([(0, 130, 140), (1, 130, 140), (2, 100, 193)],      # three copies and a page
                [(0, 130, 131), (0, 131, 132)], [(0, 130, 131), (1, 193, 194)], [(0, 130, 131), (1, 5, 301)]):
        with pytest.raises((RuntimeError, ValueError)):
            cache.reserve_all(bad)
        assert used() == before
    cache.pool[0, :, 0, 0] = torch.arange(6, dtype=torch.uint8)
    cache.reserve_all([(0, 130, 140), (1, 100, 140), (2, 130, 140)])      # the last of them keeps the third page; 1 has a second one of its own
    assert cache.pages_of(2) == before[1][2] and cache.free_pages == 0 and [cache._users[p] for p in before[1][0]] == [3, 2, 1]
    for b in range(BATCH):
        assert [int(cache.pool[0, p, 0, 0]) for p in cache.pages_of(b)] == [0, 1, 2]
        assert cache.table[b].tolist() == cache.pages_of(b) + [-1, -1]


def test_pages_are_given_back_if_they_cannot_be_copied(make, monkeypatch):
    def fails(pool, src, dst):
        raise RuntimeError("no copy")

    cache = make(pages=5).cache
    cache.reserve(0, 0, 130)
    cache.fork(0, 1)
    monkeypatch.setattr(decode_ops, "copy_kv4_pages", fails)
    with pytest.raises(RuntimeError, match="no copy"):
        cache.reserve(1, 130, 131)
    assert cache.free_pages == 2 and cache.pages_of(1) == cache.pages_of(0) and [cache._users[p] for p in cache.pages_of(0)] == [2, 2, 2]


@pytest.mark.parametrize("bits", [4, 16])
def test_fed_prompts_draw_with_their_own_numbers(make, bits):
    rows, u = [[1, 2, 3], [4, 5, 6]], torch.rand(6, BATCH, generator=torch.Generator().manual_seed(1))

    def drawn(before):
        model = make(cache_bits=bits)
        model.set_sampling(0.9)
        if before:
            model.feed([[7, 8, 9]], u=u[4])
            model.generate(1, u=u[5:])
        model.feed(rows, u=u[0])
        return torch.cat((model.token[None].clone(), model.generate(3, u=u[1:4])))

    first = drawn(False)
    assert torch.equal(first, drawn(True)) and torch.equal(first[0], (u[0] * VOCAB).long())
    model = make(cache_bits=bits)
    model.set_sampling(0.9)
    for bad in (None, u, u[0, :2]):
        with pytest.raises(ValueError):
            model.feed(rows, u=bad)
    model.feed([])
    model.set_sampling(None)
    model.feed(rows)


def test_numbers_are_looked_at_before_a_prompt_takes_pages(make):
    model = make()
    model.set_sampling(0.9)
    before = state(model)
    for bad in (None, torch.rand(2), torch.rand(1, BATCH)):
        with pytest.raises(ValueError):
            model.prefill([[1], [2], [3]], u=bad)
    assert state(model) == before


@pytest.mark.parametrize("name", ["step", "generate_step"])
def test_single_steps_make_room_and_count(make, name):
    model = make(pages=7)
    model.prefill([[1] * 63, [2] * 130, [3] * 20])      # 1 + 3 + 1 pages
    model.fork(0, 2)
    for i in range(2):
        getattr(model, name)()
        assert model.lengths == model.pos.tolist() == [64 + i, 131 + i, 64 + i]
        pages = [model.cache.pages_of(b) for b in range(BATCH)]
        assert not set(pages[0]) & set(pages[2]) and [len(p) for p in pages] == [1 + i, 3, 1 + i]      # position 63, then 64
    assert model.cache.free_pages == 0
    model.lengths = [64, 192, 64]      # the fourth page of the second one
    model.pos.copy_(torch.tensor(model.lengths))
    before = state(model)
    with pytest.raises(RuntimeError):
        getattr(model, name)()
    assert state(model) == before


def test_a_graph_s_replays_count_too(make, monkeypatch):
    model = make()
    model.prefill([[1], [2, 3], []])
    model.graph = SimpleNamespace(replay=model._step)
    model.generate(2), model.feed([[1, 2, 3]])
    assert model.lengths == model.pos.tolist() == [4, 5, 3]


def test_ids_outside_the_vocabulary_are_refused(make):
    model = make()
    before = state(model)
    for bad in (-1, VOCAB, 1 << 40):
        for call in (lambda: model.prefill([[1], [2, bad], [3]]), lambda: model.feed([[1, 2, 3], [1, 2, bad]]), lambda: model.feed(torch.tensor([[1, bad, 3]]))):
            with pytest.raises(ValueError, match="49"):
                call()
            assert state(model) == before
    model.prefill([[0], torch.tensor([VOCAB - 1]), torch.tensor([], dtype=torch.int64)])
    model.feed(torch.tensor([[1, 2, 3]]))
    assert model.lengths == [2, 2, 1]


@pytest.mark.parametrize("slot", [-1, -BATCH, BATCH, 1 << 20])
def test_there_is_one_name_for_a_sequence(make, slot):
    model = make(pages=6)
    model.prefill([[1] * 100, [2], [3] * 70])
    before = state(model), list(model.cache._users)
    c = model.cache
    for call in (lambda: c.fork(0, slot), lambda: c.fork(slot, 0), lambda: c.fork(slot, slot), lambda: c.free(slot), lambda: c.truncate(slot, 1), lambda: c.pages_of(slot),
                 lambda: c.reserve(slot, 0, 1), lambda: c.reserve_all([(0, 100, 101), (slot, 0, 1)]), lambda: model.fork(0, slot), lambda: model.fork(slot, 0)):
        with pytest.raises(ValueError):
            call()
        assert (state(model), list(c._users)) == before
    model.fork(1, 1)
    assert (state(model), list(c._users)) == before


def test_settings_of_another_size_change_nothing(make):
    model = make()
    model.graph = graph = object()
    for bad in (dict(temperature=[1.0, 2.0]), dict(temperature=0.5, top_k=[1] * 4), dict(temperature=0.5, min_p="x")):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            model.set_sampling(**bad)
        assert model.sampling is None and model.graph is graph
    model.set_sampling(0.7, top_k=[3, 4, 5], top_p=0.9, min_p=torch.tensor([0.1, 0.0, 0.2]))
    assert model.graph is None
    model.graph, before = graph, [t.clone() for t in model.sampling]
    with pytest.raises(RuntimeError):
        model.set_sampling(0.1, top_k=2, top_p=[0.5, 0.5])
    assert all(map(torch.equal, model.sampling, before)) and model.graph is graph and model.sampling[1].tolist() == [3, 4, 5]
