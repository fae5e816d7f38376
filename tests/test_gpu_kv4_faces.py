"""The same refusals from the compiled module and from its Python steps."""
import pytest
import torch

from shiftaddllm_b200 import decode_ops

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "python"])
def face(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(decode_ops, "_compiled", False)
    else:
        assert decode_ops._native()


def test_numbers_that_do_not_fit(face):
    logits, u, token = torch.zeros(1, 10, device="cuda"), torch.full((1,), 0.55, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    for bad in ((1 << 32) + 1, float("inf"), float("nan"), -(1 << 33)):
        with pytest.raises(RuntimeError):
            decode_ops.sample_token(logits, u, token, top_k=bad)
    for k, want in ((0, 5), (5, 2), (-1, 5), ((1 << 31) - 1, 5)):      # floor(u * kept), equal weights
        decode_ops.sample_token(logits, u, token, top_k=k)
        assert token.item() == want
    pool = torch.zeros(1, 4, 1, 16, dtype=torch.uint8, device="cuda")
    for src, dst in (([1 << 32], [1]), ([0], [(1 << 32) + 1]), ([-1], [1]), ([0], [4])):
        with pytest.raises(RuntimeError):
            decode_ops.copy_kv4_pages(pool, src, dst)
    pool[0, 0] = 7
    decode_ops.copy_kv4_pages(pool, [0], [3])
    assert (pool[0, :, 0, 0] == torch.tensor([7, 0, 0, 7], device="cuda")).all()
