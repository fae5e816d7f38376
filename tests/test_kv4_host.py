"""The 4-bit cache's and the sampler's C entries and Python faces refuse bad arguments before any GPU work."""
import ctypes

import pytest
import torch

from shiftaddllm_b200 import _lib, decode_ops


@pytest.fixture()
def ptr():
    buf = ctypes.create_string_buffer(8192)
    yield (ctypes.addressof(buf) + 15) & ~15
    del buf


def test_write_entry(lib, ptr):
    def call(null=None, off=None, batch=1, m=1, heads=4, kvh=2, hd=128, max_len=8, max_pages=1, pages=1):
        p = [ptr] * 10
        p[6] = None                                            # rows may be missing
        if null is not None:
            p[null] = None
        if off is not None:
            p[off] += 2
        return lib.sal_rope_kv4_write_f16(*p, batch, m, heads, kvh, hd, max_len, max_pages, pages, None)

    for i in (0, 1, 2, 3, 4, 5, 7, 8, 9):
        assert call(null=i) == _lib.SAL_E_NULL
    for i in (0, 1, 2, 3, 4, 8, 9):
        assert call(off=i) == _lib.SAL_E_ALIGN
    for hd in (0, 32, 96, 192, 512):
        assert call(hd=hd) == _lib.SAL_E_UNSUPPORTED
    for bad in (dict(batch=0), dict(m=0), dict(heads=0), dict(kvh=0), dict(max_len=0), dict(max_pages=0), dict(pages=0), dict(batch=65536), dict(m=70000),
                dict(batch=300, m=300), dict(max_pages=1 << 25)):
        assert call(**bad) == _lib.SAL_E_SHAPE


def test_read_and_attention_entries(lib, ptr):
    for i in range(5):
        p = [ptr] * 5
        p[i] = None
        assert lib.sal_read_kv4(*p, 1, 1, 1, 2, 128, 1, 1, None) == _lib.SAL_E_NULL
    assert lib.sal_read_kv4(ptr, ptr, ptr, ptr, ptr, 1, 1, 1, 2, 80, 1, 1, None) == _lib.SAL_E_UNSUPPORTED
    assert lib.sal_read_kv4(ptr, ptr, ptr, ptr, ptr + 4, 1, 1, 1, 2, 128, 1, 1, None) == _lib.SAL_E_ALIGN
    need = lib.sal_attention_kv4_workspace_bytes(1, 1, 4, 2, 128)
    assert need > 0 and lib.sal_attention_kv4_workspace_bytes(1, 1, 5, 2, 128) == 0 and lib.sal_attention_kv4_workspace_bytes(0, 1, 4, 2, 128) == 0

    def call(null=None, off=None, batch=1, m=1, heads=4, kvh=2, hd=128, ws=need):
        p = [ptr, ptr, ptr, ptr, None, ptr]
        if null is not None:
            p[null] = None
        if off is not None:
            p[off] += 8
        return lib.sal_attention_kv4_f16(*p, batch, m, heads, kvh, hd, 1, 1, 1.0, ptr, ws, None)

    for i in (0, 1, 2, 3, 5):
        assert call(null=i) == _lib.SAL_E_NULL
    for i in (0, 1, 5):
        assert call(off=i) == _lib.SAL_E_ALIGN
    assert call(heads=5) == _lib.SAL_E_SHAPE and call(batch=70000) == _lib.SAL_E_SHAPE and call(hd=64 + 16) == _lib.SAL_E_UNSUPPORTED
    assert call(ws=need - 1) == _lib.SAL_E_WORKSPACE


def test_copy_entry(lib, ptr):
    def call(src, dst, pages=8, layers=2, size=160, pool=ptr):
        a, b = (ctypes.c_int32 * len(src))(*src), (ctypes.c_int32 * len(dst))(*dst)
        return lib.sal_copy_kv4_pages(pool, ctypes.addressof(a), ctypes.addressof(b), len(src), layers, pages, size, None)

    assert lib.sal_copy_kv4_pages(None, None, None, 0, 1, 1, 16, None) == _lib.SAL_OK       # nothing to copy
    assert lib.sal_copy_kv4_pages(ptr, None, None, 1, 1, 1, 16, None) == _lib.SAL_E_NULL
    for src, dst in (([0], [8]), ([8], [0]), ([-1], [0]), ([0], [-1]), ([1, 2], [3, 3]), ([1, 2], [2, 3]), ([4], [4])):
        assert call(src, dst) == _lib.SAL_E_SHAPE
    assert call([0], [1], size=150) == _lib.SAL_E_SHAPE and call([0], [1], layers=0) == _lib.SAL_E_SHAPE
    assert call([0], [1], pool=ptr + 8) == _lib.SAL_E_ALIGN


def test_sample_entry(lib, ptr):
    def call(logits=ptr, rows=1, vocab=10, u=ptr, token=ptr):
        return lib.sal_sample_token(logits, 1, rows, vocab, u, None, None, None, None, 1.0, 0, 1.0, 0.0, token, None)

    for kw in (dict(logits=None), dict(u=None), dict(token=None)):
        assert call(**kw) == _lib.SAL_E_NULL
    for kw in (dict(rows=0), dict(rows=65536), dict(vocab=0), dict(vocab=262145)):
        assert call(**kw) == _lib.SAL_E_SHAPE


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(1, 1, 256, dtype=torch.float16)
    pos, table = torch.zeros(1, dtype=torch.int64), torch.zeros(1, 1, dtype=torch.int32)
    pool = decode_ops.kv4_pool(1, 2, 2, 128, "cpu")
    assert pool.shape == (1, 2, 2, 64 * 144)
    with pytest.raises(RuntimeError):
        decode_ops.attention_kv4(x, pool[0], table, pos, x, 2, 2, 128, 1.0, torch.zeros(1024, dtype=torch.uint8))
    with pytest.raises(RuntimeError):
        decode_ops.rope_kv4_write(x, x, x, x, x, pos, table, pool[0], x, 2, 2, 128)
    with pytest.raises(RuntimeError):
        decode_ops.copy_kv4_pages(pool, [0], [1])
    with pytest.raises(RuntimeError):
        decode_ops.sample_token(torch.zeros(1, 10), torch.zeros(1), torch.zeros(1, dtype=torch.int64))
    for hd in (32, 96, 192):
        with pytest.raises(RuntimeError):
            decode_ops.kv4_pool(1, 1, 1, hd, "cpu")


def test_a_refusal_with_a_number_in_it_is_an_exception(lib):
    """Numbers in the compiled module's messages: with a second C++ runtime inside the module they ended the process."""
    import subprocess
    import sys

    code = """
import torch
from shiftaddllm_b200 import _lib, build, lutgemm
build.build_extension()
_lib.load()
m = lutgemm.compiled_module()
try:
    m.lut_linear(torch.zeros(1, 30), torch.zeros(1), torch.zeros(1), None, 32, 32, 3, True)
except RuntimeError as e:
    print("refused", "32, got 30" in str(e))
"""
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=build_dir())
    assert got.returncode == 0 and "refused True" in got.stdout, got.stdout + got.stderr


def build_dir():
    from shiftaddllm_b200 import build

    return build.REPO_DIR
