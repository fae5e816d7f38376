"""A top_p near to 1 that parts tokens whose weights are some hundreds of the units of 2**-44 in which weights are summed, rounded down."""
import numpy as np
import pytest
import torch

from shiftaddllm_b200 import decode_ops

pytestmark = pytest.mark.gpu
ROWS = 6


@pytest.mark.parametrize("k_of", [0, 5])
@pytest.mark.parametrize("vocab,units,spread,share", [(262144, 1700, 0.05, 0.5), (262144, 1700, 0.3, 0.5), (262144, 1700, 0.8, 0.5), (262144, 3400, 0.6, 0.6), (262144, 2000, 0.2, 0.8), (262144, 9000, 1.0, 0.3), (200000, 3000, 0.4, 0.7),
                                                      (131071, 5000, 0.1, 0.6), (50000, 20000, 0.05, 0.5)])
def test_the_border_lies_among_small_weights(vocab, units, spread, share, k_of):
    """One likely token and many with weights of `units`, of whose sum `share` is kept.  A token is expected where whole numbers of units put it; the
    kernel's weights are exact to 3e-7, so that the sums are off by less than a token's weight."""
    rng = np.random.default_rng(vocab + units)
    x = (np.log(units * 2.0 ** -44) + spread * (rng.random((ROWS, vocab)) - 0.5)).astype(np.float32)
    x[:, 0] = 0.0
    k = vocab - vocab // k_of if k_of else 0
    top_p = np.empty(ROWS, dtype=np.float32)
    kept, runs = [], []
    for r in range(ROWS):
        w = np.floor(np.exp(x[r].astype(np.float64)) * 2.0 ** 44).astype(np.int64)
        order = np.argsort(-x[r], kind="stable")[: k if k else vocab]
        total = float(w[order].sum())
        top_p[r] = (2.0 ** 44 + (share + 0.01 * r) * (total - 2.0 ** 44)) / total
        before = np.cumsum(w[order]) - w[order]
        kept.append(np.sort(order[before < float(top_p[r]) * total]))
        assert 2 < len(kept[r]) < len(order) - 2
        runs.append(np.cumsum(w[kept[r]]))
    x = torch.from_numpy(x).cuda()
    for number in (0.25, 1.0 - 30 * 2.0 ** -24, float(np.nextafter(np.float32(1), np.float32(0)))):
        token = torch.full((ROWS,), -1, dtype=torch.int64, device="cuda")
        u = torch.full((ROWS,), number, device="cuda")
        decode_ops.sample_token(x, u, token, top_k=k, top_p=torch.from_numpy(top_p).cuda())
        for got, tokens, run in zip(token.tolist(), kept, runs):
            want = int(np.searchsorted(run, np.floor(number * float(run[-1])), side="right"))
            assert got in tokens[max(0, want - 1): want + 2], (got, want, tokens[want])


@pytest.mark.parametrize("min_p", [1.0, 1.5, float("inf")])
def test_min_p_of_one_and_above_keeps_the_largest(min_p):
    x = torch.randn(4, 9000, generator=torch.Generator().manual_seed(0)).cuda()
    x[:, [17, 5000]] = 9.0      # two of them
    u, token = torch.tensor([0.0, 0.49, 0.51, 1.0], device="cuda"), torch.full((4,), -1, dtype=torch.int64, device="cuda")
    for kw in (dict(), dict(top_k=50), dict(top_p=0.99)):
        decode_ops.sample_token(x, u, token.fill_(-1), min_p=min_p, **kw)
        assert token.tolist() == [17, 17, 5000, 5000]
