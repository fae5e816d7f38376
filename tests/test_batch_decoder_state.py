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
