"""The next token from logits, against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from shiftaddllm_b200 import decode_ops

pytestmark = pytest.mark.gpu


def chosen(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Token of one row, and how near a border it was: the running sum's distance from u * total, and the prefix's from top_p, both relative."""
    x = x.astype(np.float64)
    ok = x > -np.inf          # NaN: False
    if not ok.any():
        return 0, 1.0
    best = np.flatnonzero(ok)
    best = best[np.lexsort((best, -x[best]))]
    if not temperature > 0:
        return int(best[0]), 1.0
    top = x[best[0]]
    with np.errstate(all="ignore"):
        w = np.where(x[best] == top, 1.0, np.exp((x[best] - top) / temperature))
    if top_k > 0:
        best, w = best[:top_k], w[:top_k]
    near = 1.0
    if top_p < 1:
        before = np.cumsum(w) - w
        near = np.abs(before[1:] - top_p * w.sum()).min(initial=1.0) / w.sum()
        n = max(1, int((before < top_p * w.sum()).sum()))
        best, w = best[:n], w[:n]
    keep = w >= min(min_p, 1.0)
    near = min(near, np.abs(w / max(min_p, 1e-300) - 1).min(initial=1.0)) if min_p > 0 else near
    best, w = best[keep], w[keep]
    order = np.argsort(best)
    run = np.cumsum(w[order])
    goal = np.float64(u) * run[-1]
    near = min(near, np.abs(run[:-1] - goal).min(initial=1.0) / run[-1])
    return int(best[order][min(int((run <= goal).sum()), len(best) - 1)]), near


# Weights carry a relative error below 2**-21 (a 32-bit power function of two steps, its exponent exact to 2**-40, one more rounding): a token
# can differ where the running sum comes that near to a border, and nowhere else.
NEAR = 2.0 ** -20


def check(x, u, **filters):
    token = torch.full((x.shape[0],), -7, dtype=torch.int64, device="cuda")
    decode_ops.sample_token(x, u, token, **filters)
    again = torch.full_like(token, -7)
    decode_ops.sample_token(x, u, again, **filters)
    assert torch.equal(token, again)
    one = {k: v.tolist() if isinstance(v, torch.Tensor) else [v] * x.shape[0] for k, v in filters.items()}
    for r, (row, got) in enumerate(zip(x.cpu().numpy(), token.tolist())):
        want, near = chosen(row, u[r].item(), **{k: v[r] for k, v in one.items()})
        assert got == want or near < NEAR, (r, got, want, near, {k: v[r] for k, v in one.items()})
    return token


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 1000), (70, 1001), (4, 32000), (1, 50257), (2, 131071), (1, 262144)])
def test_filters_one_by_one_and_together(dtype, rows, vocab):
    torch.manual_seed(vocab)
    x = (3 * torch.randn(rows, vocab, device="cuda")).to(dtype)
    for f in (dict(), dict(temperature=0.3), dict(temperature=0.0), dict(top_k=1), dict(top_k=40), dict(top_k=vocab), dict(top_p=0.9), dict(top_p=1e-6),
              dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0), dict(temperature=1.7, top_k=200, top_p=0.7, min_p=0.01), dict(top_p=0.9999999)):
        check(x, torch.rand(rows, device="cuda"), **f)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_every_row_asks_for_something_else(dtype):
    torch.manual_seed(1)
    rows, vocab = 97, 5003
    x = (2.5 * torch.randn(rows, vocab, device="cuda")).to(dtype)
    t = torch.rand(rows, device="cuda") * 2
    t[::9] = 0
    t[::11] = -1
    check(x, torch.rand(rows, device="cuda"), temperature=t, top_k=torch.randint(-1, 300, (rows,), device="cuda", dtype=torch.int32),
          top_p=torch.rand(rows, device="cuda") * 1.2, min_p=torch.rand(rows, device="cuda") * 0.2 - 0.05)


@pytest.mark.parametrize("vocab", [1, 5, 999, 4096, 40001])
def test_equal_logits_go_by_index(vocab):
    x = torch.full((4, vocab), 1.25, dtype=torch.float16, device="cuda")
    u = torch.tensor([0.0, 0.3, 0.77, 0.9999999], device="cuda")
    for f in (dict(), dict(top_k=3), dict(top_p=0.31), dict(top_k=max(2, vocab // 2), top_p=0.5), dict(min_p=1.0), dict(temperature=0.0)):
        got = check(x, u, **f)
        assert got[0] == 0
    x[:, ::2] = 2.0                                # two values, each many times
    for f in (dict(), dict(top_k=vocab // 2 + 2), dict(top_p=0.31), dict(top_p=0.9)):
        check(x, u, **f)


def test_what_can_never_be_chosen():
    inf, nan = math.inf, math.nan
    rows = [[nan, nan, nan, nan], [-inf, -inf, -inf, -inf], [nan, -inf, 1.0, nan], [inf, 0.0, inf, 5.0], [nan, 2.0, -inf, 2.0], [-0.0, 0.0, -0.0, 0.0],
            [-65504.0, 65504.0, 0.0, nan]]
    for dtype in (torch.float16, torch.float32):
        x = torch.tensor(rows, device="cuda").to(dtype)
        for u in (0.0, 0.4, 0.6, 0.9999999):
            for f in (dict(), dict(top_k=2), dict(top_p=0.7), dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=1e30), dict(min_p=0.5)):
                check(x, torch.full((len(rows),), u, device="cuda"), **f)
    x = torch.full((2, 3), -inf, device="cuda")
    x[1, 2] = -3.0e38
    assert check(x, torch.full((2,), 0.99, device="cuda")).tolist() == [0, 2]


def test_random_numbers_at_and_outside_their_range():
    x = torch.tensor([[0.0, 1.0, 2.0, -math.inf]], device="cuda").repeat(5, 1)
    u = torch.tensor([0.0, 1.0, 7.0, -2.0, math.nan], device="cuda")
    token = torch.empty(5, dtype=torch.int64, device="cuda")
    decode_ops.sample_token(x, u, token)
    assert token.tolist() == [0, 2, 2, 0, 0]       # at 1 and above the last token that can be chosen, below 0 and NaN the first


def test_draws_follow_the_weights():
    """Evenly spread random numbers give every token its share, to one draw."""
    torch.manual_seed(2)
    vocab, n = 50, 4096
    x = torch.randn(1, vocab, device="cuda").repeat(n, 1)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    token = torch.empty(n, dtype=torch.int64, device="cuda")
    decode_ops.sample_token(x, u, token, temperature=0.8)
    share = torch.softmax(x[0].double() / 0.8, 0)
    assert ((torch.bincount(token, minlength=vocab).double() - n * share).abs() <= 1.0 + n * NEAR).all()
    assert (token[1:] >= token[:-1]).all()


def test_captured_and_replayed_with_new_numbers():
    torch.manual_seed(3)
    x, u, token = torch.randn(6, 32000, device="cuda").half(), torch.rand(6, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    t, p = torch.full((6,), 0.8, device="cuda"), torch.full((6,), 0.9, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        decode_ops.sample_token(x, u, token, temperature=t, top_k=50, top_p=p)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            decode_ops.sample_token(x, u, token, temperature=t, top_k=50, top_p=p)
    for _ in range(3):
        x.copy_(torch.randn(6, 32000, device="cuda"))
        u.copy_(torch.rand(6, device="cuda"))
        p.copy_(torch.rand(6, device="cuda"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        again = torch.empty_like(token)
        decode_ops.sample_token(x, u, again, temperature=t, top_k=50, top_p=p)
        assert torch.equal(token, again)


def test_refusals():
    x, u, token = torch.zeros(3, 100, device="cuda"), torch.zeros(3, device="cuda"), torch.full((3,), -7, dtype=torch.int64, device="cuda")
    for kw in (dict(logits=x.cpu()), dict(logits=x.double()), dict(logits=x.bfloat16()), dict(logits=x.t()), dict(logits=x[:, :0]), dict(u=u.double()),
               dict(u=u[:2]), dict(token=token.int()), dict(token=token[:1]), dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:1]),
               dict(min_p=u.cpu()), dict(logits=torch.zeros(1, 262145, device="cuda"), u=u[:1], token=token[:1])):
        with pytest.raises(RuntimeError):
            decode_ops.sample_token(**{**dict(logits=x, u=u, token=token), **kw})
    torch.cuda.synchronize()
    assert token.tolist() == [-7] * 3


@pytest.mark.parametrize("dtype,off", [(torch.float16, 1), (torch.float16, 7), (torch.float32, 3)])
def test_rows_that_begin_anywhere(dtype, off):
    """Rows and slices at any alignment, and nothing read in front of them or behind."""
    torch.manual_seed(off)
    for rows, vocab in ((3, 4097), (2, 33001), (1, 130003)):
        whole = torch.full((off + rows * vocab + 9,), 60000.0, dtype=dtype, device="cuda")      # larger than any logit
        x = whole[off:off + rows * vocab].view(rows, vocab)
        x.copy_(2.5 * torch.randn(rows, vocab, device="cuda"))
        for f in (dict(), dict(top_k=30, top_p=0.8), dict(top_p=0.95), dict(temperature=0.0)):
            check(x, torch.rand(rows, device="cuda"), **f)


@pytest.mark.parametrize("rows,vocab", [(300, 2048), (40, 60000), (1, 8192)])
def test_few_values_many_times(rows, vocab):
    """Logits on a coarse grid: windows full of equal logits, in one bin and in many."""
    torch.manual_seed(rows)
    for levels in (2, 5, 60):
        x = (torch.randint(0, levels, (rows, vocab), device="cuda").float() / levels * 4).half()
        for f in (dict(top_k=vocab // 3), dict(top_p=0.6), dict(top_k=vocab // 2, top_p=0.5, min_p=0.2)):
            check(x[:4].contiguous(), torch.rand(min(rows, 4), device="cuda"), **f)
        token = torch.empty(rows, dtype=torch.int64, device="cuda")
        decode_ops.sample_token(x, torch.rand(rows, device="cuda"), token, top_p=0.6)
        assert ((token >= 0) & (token < vocab)).all()
