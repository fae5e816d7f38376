"""The state of the batch decoder's sequences between its calls: tokens, positions, pages and lengths stay in step, whatever is called next."""
import pytest
import torch

from shiftaddllm_b200 import _lib, decode_ops
from shiftaddllm_b200.decoder import SHAPES, BcqLlamaBatchDecoder, BcqLlamaDecoder, benchmark_batch

pytestmark = pytest.mark.gpu
BATCH = 3


@pytest.fixture(scope="module")
def like():
    return BcqLlamaDecoder(SHAPES["tiny"], max_len=8, seed=3, fused=False)


def make(like, bits=4, **kw):
    return BcqLlamaBatchDecoder(SHAPES["tiny"], max_len=300, batch=BATCH, like=like, cache_bits=bits, **kw)


def prompts(lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (n,), generator=g).tolist() for n in lengths]


@pytest.mark.parametrize("bits", [4, 16])
def test_capture_behind_work_that_is_still_in_flight(like, bits):
    """The caller's stream is a tenth of a second behind when the step is captured."""
    rows = torch.tensor(prompts([9] * BATCH, seed=1)).t()
    forced = torch.tensor([11, 500, 999], device="cuda")
    eager, captured = make(like, bits), make(like, bits)
    for m in (eager, captured):
        if bits == 4:
            m.prefill(prompts([5, 130, 70]))
        m.token.zero_()
        torch.cuda.synchronize()
        if m is captured:
            torch.cuda._sleep(200_000_000)
        m.feed(rows)
        m.token.copy_(forced)
        if m is captured:
            m.capture()
    assert torch.equal(captured.generate(8), eager.generate(8)) and torch.equal(captured.logits, eager.logits)
    assert torch.equal(captured.pos, eager.pos)


def test_a_wait_that_ran_out_is_reported_once(like):
    """The device's word, written here as a kernel writes it."""
    model = make(like)
    model.prefill(prompts([5, 130, 70]))
    for call in (lambda: model.generate(2), lambda: model.feed([[1, 2, 3]])):
        model._attn_ws[:4].view(torch.int32).fill_(_lib.SAL_E_TIMEOUT)
        with pytest.raises(RuntimeError, match="wait"):
            call()
        call()
    decode_ops.attention_kv4_check(model._attn_ws)


def test_single_steps_are_what_generate_does(like):
    """Over a page's end and on forked sequences, whose common page neither may write to."""
    stepped, at_once = make(like), make(like)
    for m in (stepped, at_once):
        m.prefill(prompts([60, 125, 3]))
        m.fork(0, 2)
        m.token[2] = 77
    want = at_once.generate(12)
    got = []
    for _ in range(12):
        stepped.step()
        got.append(stepped.token.clone())
    assert torch.equal(torch.stack(got), want) and torch.equal(stepped.logits, at_once.logits) and stepped.lengths == stepped.pos.tolist()


def test_generating_behind_the_benchmark(like):
    model, fresh = make(like), make(like)
    benchmark_batch(model, 60, 8)
    assert model.lengths == model.pos.tolist() == [68] * BATCH
    ids = torch.randint(0, 1000, (60, BATCH), generator=torch.Generator().manual_seed(0))      # its prompts
    fresh.prefill(ids.t().tolist())
    fresh.generate(8)
    assert torch.equal(model.generate(6), fresh.generate(6)) and torch.equal(model.logits, fresh.logits)


@pytest.mark.parametrize("bits", [4, 16])
def test_a_capture_leaves_the_state_as_it_was(like, bits):
    """Behind a prompt, not forked and of no whole number of pages, with no wait of the host in between."""
    model = make(like, bits)
    if bits == 4:
        model.prefill(prompts([5, 130, 70]))
    else:
        model.feed(torch.tensor(prompts([7] * BATCH)).t())
    before = [t.clone() for t in (model.token, model.pos, model.logits)]
    model.capture()
    assert all(map(torch.equal, before, (model.token, model.pos, model.logits)))
