"""The batch decoder on a 4-bit cache, with sampled tokens: cache, attention, pages and sampler in one run, as they are used together."""

import pytest
import torch

from shiftaddllm_b200 import decode_ops, decoder
from shiftaddllm_b200.decoder import SHAPES, BcqLlamaBatchDecoder, BcqLlamaDecoder

pytestmark = pytest.mark.gpu
BATCH = 3


@pytest.fixture(scope="module")
def like():
    return BcqLlamaDecoder(SHAPES["tiny"], max_len=8, seed=3, fused=False)


def make(like, **kw):
    return BcqLlamaBatchDecoder(SHAPES["tiny"], max_len=300, batch=BATCH, like=like, cache_bits=4, **kw)


def prompts(lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (n,), generator=g).tolist() for n in lengths]


def plain_attention(q, pool, table, pos, out, heads, kv_heads, hd, scale, workspace, rows=None):
    """The same call in 64 bits on the values read back."""
    batch = pos.numel()
    m, t = q.numel() // (batch * heads * hd), table.shape[1] * 64
    k, v = (torch.empty(batch, t, kv_heads, hd, device="cuda") for _ in range(2))
    decode_ops.read_kv4(pool, table, torch.zeros_like(pos), k, v, kv_heads, hd)
    k, v = (x.double().repeat_interleave(heads // kv_heads, 2).transpose(1, 2) for x in (k, v))
    s = q.view(batch, m, heads, hd).transpose(1, 2).double() @ k.transpose(2, 3) * scale
    last = pos[:, None] + torch.arange(m, device="cuda")
    s.masked_fill_(torch.arange(t, device="cuda") > last[:, None, :, None], float("-inf"))
    o = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(batch, m, -1).half()
    valid = (torch.arange(m, device="cuda") < (rows[:, None] if rows is not None else m)).expand(batch, m)
    out.view(batch, m, -1)[valid] = o[valid]


def test_logits_against_plain_attention(like, monkeypatch):
    model = make(like)
    model.prefill(prompts([5, 130, 64]))
    first = model.logits.clone()
    tokens = model.generate(6)
    logits = model.logits.clone()
    monkeypatch.setattr(decode_ops, "attention_kv4", plain_attention)
    other = make(like)
    other.prefill(prompts([5, 130, 64]))
    assert (other.logits - first).norm() <= 5e-3 * first.norm()
    other.token.copy_(first.argmax(-1))
    other.cache.reserve(0, 5, 11), other.cache.reserve(1, 130, 136), other.cache.reserve(2, 64, 70)
    for i in range(6):
        other.step()
        other.token.copy_(tokens[i])      # the same tokens, whatever a tie gave
    assert (other.logits - logits).norm() <= 5e-3 * logits.norm()


def test_prompts_of_different_lengths_as_token_by_token(like):
    """The rows of a prompt come from the tensor-core products, single steps from the tables: a key or value then differs in its last 16-bit digits,
    and where it lies near the middle between two codes, in its code.  In the first layer, where the inputs are the same, that is one step of its
    group at most (two neighbouring codes), plus what the digits themselves move: the products are exact to 4.3e-4 and 2.1e-4 of a row's largest
    number, and a turned number is the sum of two, so 2e-3 of the largest covers the lowest value's and the scale's shift too.  Behind the
    first layer the steps have no such bound, so the logits are compared with plain arithmetic on the same cache (above) instead."""
    model, ps = make(like), prompts([1, 70, 200])
    model.prefill(ps)
    for b, p in enumerate(ps):
        one = make(like)
        one.feed([[t] * BATCH for t in p])
        assert one.lengths == [len(p)] * BATCH and one.pos.tolist() == one.lengths
        zero = torch.zeros(BATCH, dtype=torch.int64, device="cuda")
        got = []
        for m in (model, one):
            kv = [torch.empty(BATCH, len(p), 2, 64, device="cuda") for _ in range(2)]
            decode_ops.read_kv4(m.cache.pool[0], m.cache.table, zero, *kv, 2, 64)
            got.append(torch.stack(kv)[:, b])
        x, y = got
        step = (torch.maximum(x.amax(-1), y.amax(-1)) - torch.minimum(x.amin(-1), y.amin(-1))) / 15
        largest = y.abs().amax((-1, -2))      # of a position's row
        assert ((x - y).abs() <= step[..., None] + 2e-3 * largest[..., None, None]).all()
    assert model.lengths == [1, 70, 200] and model.pos.tolist() == model.lengths
    before = model.logits.clone()
    model.prefill([[], [7, 8], []])
    assert torch.equal(model.logits[0], before[0]) and torch.equal(model.logits[2], before[2]) and model.lengths == [1, 72, 200]


def test_a_captured_step_and_forked_sequences(like):
    """One prompt, forked, drawn with numbers of their own; the graph gives what single steps give, and so does a compacted cache."""
    torch.manual_seed(5)
    u = torch.rand(80, BATCH, device="cuda")

    def start(model):
        model.set_sampling([0.8, 1.0, 0.0], top_k=[40, 0, 0], top_p=0.9, min_p=0.01)
        model.prefill(prompts([100, 0, 0]), u=u[0])
        free = model.cache.free_pages
        model.fork(0, 1)
        model.fork(0, 2)
        assert model.cache.free_pages == free and model.lengths == [100] * 3

    eager, captured, moved = make(like), make(like), make(like)
    for m in (eager, captured, moved):
        start(m)
    want = eager.generate(60, u=u[1:61])
    assert len(set(map(tuple, want.t().tolist()))) > 1
    captured.capture()
    assert torch.equal(captured.generate(60, u=u[1:61]), want) and torch.equal(captured.logits, eager.logits)
    got = moved.generate(30, u=u[1:31])
    moved.cache.free(1)
    moved.lengths[1], moved.pos[1] = 0, 0
    used = moved.cache.compact()
    assert all(p < used for b in (0, 2) for p in moved.cache.pages_of(b))
    rest = moved.generate(30, u=u[31:61])
    assert torch.equal(got, want[:30]) and torch.equal(rest[:, [0, 2]], want[30:][:, [0, 2]])


def test_the_sampler_s_first_token_is_the_greedy_one(like):
    greedy, drawn = make(like), make(like)
    drawn.set_sampling(0.7, top_k=1)
    for m in (greedy, drawn):
        m.prefill(prompts([20, 30, 40]), u=torch.rand(BATCH, device="cuda"))
    assert torch.equal(greedy.generate(10), drawn.generate(10, u=torch.rand(10, BATCH, device="cuda")))


def test_refusals(like):
    model = make(like, pages=4)
    with pytest.raises(RuntimeError):
        model.prefill(prompts([200, 100, 0]))      # five pages
    for bad in (lambda: model.prefill(prompts([1, 2])), lambda: model.prefill(prompts([301, 0, 0])), lambda: make(like, fused=False),
                lambda: BcqLlamaBatchDecoder(SHAPES["tiny"], batch=2, like=like, cache_bits=8)):
        with pytest.raises(ValueError):
            bad()
    model.set_sampling(1.0)
    for bad in (lambda: model.generate(2), lambda: model.generate(2, u=torch.rand(2, 2, device="cuda")), lambda: model.prefill(prompts([1, 1, 1]))):
        with pytest.raises(ValueError):
            bad()
    full = BcqLlamaBatchDecoder(SHAPES["tiny"], max_len=64, batch=2, like=like)
    with pytest.raises(RuntimeError):
        full.fork(0, 1)
    with pytest.raises(RuntimeError):
        full.prefill([[1], [2]])


def test_the_command(capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["decoder", "--model", "tiny", "--batch", "4", "--cache-bits", "4", "--prompt", "70", "--new", "8", "--temperature", "0.8", "--top-p", "0.9"])
    decoder.main()
    assert '"cache_bits": 4' in capsys.readouterr().out
