"""Numbers that do not fit the C entries' types, in the calls' Python steps: refused, not wrapped around."""
from types import SimpleNamespace

import pytest
import torch

from shiftaddllm_b200 import _lib, decode_ops


class OnGpu(torch.Tensor):
    is_cuda = True


@pytest.fixture()
def reached(monkeypatch):
    """The calls that reach the library, of tensors that only say that they are on a GPU."""
    seen = []
    monkeypatch.setattr(decode_ops, "_compiled", False)
    monkeypatch.setattr(decode_ops, "_on", lambda device: decode_ops._HERE)
    monkeypatch.setattr(decode_ops, "_stream", lambda t: 0)
    monkeypatch.setattr(_lib, "load", lambda: SimpleNamespace(sal_copy_kv4_pages=lambda *a: seen.append(a) or 0, sal_sample_token=lambda *a: seen.append(a) or 0))
    return seen


def test_pages(reached):
    pool = torch.zeros(2, 4, 1, 16, dtype=torch.uint8).as_subclass(OnGpu)
    for src, dst in (([1 << 32], [1]), ([0], [(1 << 32) + 1]), ([-1], [1]), ([0], [4])):
        with pytest.raises(RuntimeError):
            decode_ops.copy_kv4_pages(pool, src, dst)
    assert not reached
    decode_ops.copy_kv4_pages(pool, [0, 1], (2, 3))
    assert len(reached) == 1


def test_top_k(reached):
    logits, u, token = (torch.zeros(1, 10).as_subclass(OnGpu), torch.zeros(1), torch.zeros(1, dtype=torch.int64))
    for bad in ((1 << 32) + 1, float("inf"), float("nan"), -(1 << 33)):
        with pytest.raises(RuntimeError):
            decode_ops.sample_token(logits, u, token, top_k=bad)
    assert not reached
    for k in (0, 5, -1, (1 << 31) - 1):
        decode_ops.sample_token(logits, u, token, top_k=k)
        assert reached.pop()[10] == k


def test_angles_of_any_shape(reached, monkeypatch):
    """As in the compiled module: rows of hd / 2 numbers, whatever the dimensions in front of them are."""
    monkeypatch.setattr(_lib, "load", lambda: SimpleNamespace(sal_rope_kv4_write_f16=lambda *a: reached.append(a) or 0))
    half, pos, table = torch.zeros(1, 1, 128, dtype=torch.float16), torch.zeros(1, dtype=torch.int64), torch.zeros(1, 1, dtype=torch.int32)
    pool = torch.zeros(2, 2, 64 * 72, dtype=torch.uint8).as_subclass(OnGpu)
    for shape in ((10, 32), (1, 10, 32), (2, 5, 32)):
        decode_ops.rope_kv4_write(half, half, half, torch.zeros(shape), torch.zeros(shape), pos, table, pool, half, 2, 2, 64)
        assert reached.pop()[15] == 10
    for cos, sin in (((10, 32), (9, 32)), ((10, 64), (10, 64)), ((0, 32), (10, 32))):
        with pytest.raises(RuntimeError):
            decode_ops.rope_kv4_write(half, half, half, torch.zeros(cos), torch.zeros(sin), pos, table, pool, half, 2, 2, 64)
    for heads in (0, -1):
        with pytest.raises(RuntimeError):
            decode_ops.rope_kv4_write(half, half, half, torch.zeros(10, 32), torch.zeros(10, 32), pos, table, pool, half, heads, 2, 64)
    assert not reached
