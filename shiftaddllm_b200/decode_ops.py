"""Python face of include/sal_decode_ops.h: the fused steps between the LUT-GEMV calls of a
batch-1 decode step.  Tensors must be contiguous CUDA tensors; launches go to torch's current
stream and are CUDA-graph capturable (the position is read from a device tensor)."""
from __future__ import annotations

import contextlib
import ctypes
import math
import warnings

import torch

from . import _lib


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


_HERE = contextlib.nullcontext()


def _on(device):
    """Makes `device` the current one for a launch, where it is not."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def residual_rmsnorm(x, delta, weight, out, x_out, eps: float):
    """t = x (+ delta); x_out = t (if given, may be x itself); out = rmsnorm(t) * weight."""
    lib = _lib.load()
    _lib.check(lib.sal_residual_rmsnorm_f16(x.data_ptr(), None if delta is None else delta.data_ptr(), weight.data_ptr(),
                                            out.data_ptr(), None if x_out is None else x_out.data_ptr(), x.numel(),
                                            float(eps), _stream(x)), "sal_residual_rmsnorm_f16")


def rope_kv_write(q, k, v, cos, sin, pos, k_cache, v_cache, heads, kv_heads, hd):
    lib = _lib.load()
    _lib.check(lib.sal_rope_kv_write_f16(q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                         pos.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), heads, kv_heads, hd,
                                         k_cache.shape[0], _stream(q)), "sal_rope_kv_write_f16")


def residual_rmsnorm_fixedacc(x, delta32, weight, out, x_out, eps: float, zero_a=None, zero_b=None):
    """As residual_rmsnorm with an int64 fixed-point accumulator as delta (consumed and zeroed); zero_a / zero_b:
    further accumulators to clear."""
    lib = _lib.load()
    _lib.check(lib.sal_residual_rmsnorm_fixedacc(x.data_ptr(), None if delta32 is None else delta32.data_ptr(), weight.data_ptr(),
                                               out.data_ptr(), None if x_out is None else x_out.data_ptr(), x.numel(), float(eps),
                                               None if zero_a is None else zero_a.data_ptr(), 0 if zero_a is None else zero_a.numel(),
                                               None if zero_b is None else zero_b.data_ptr(), 0 if zero_b is None else zero_b.numel(),
                                               _stream(x)), "sal_residual_rmsnorm_fixedacc")


def rope_kv_write_fixedacc(q32, k32, v32, q_out, cos, sin, pos, k_cache, v_cache, heads, kv_heads, hd):
    lib = _lib.load()
    _lib.check(lib.sal_rope_kv_write_fixedacc(q32.data_ptr(), k32.data_ptr(), v32.data_ptr(), q_out.data_ptr(), cos.data_ptr(),
                                            sin.data_ptr(), pos.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), heads,
                                            kv_heads, hd, k_cache.shape[0], _stream(q_out)), "sal_rope_kv_write_fixedacc")


def attention_workspace(heads: int, hd: int, device) -> torch.Tensor:
    """Zero-filled scratch for the split form of attention_decode (one per stream that uses it)."""
    lib = _lib.load()
    return torch.zeros(lib.sal_attention_workspace_bytes(int(heads), int(hd)), dtype=torch.uint8, device=device)


def attention_decode(q, k_cache, v_cache, pos, out, heads, kv_heads, hd, scale: float, workspace=None):
    """Single-query attention over cache positions 0..pos.  With a `workspace` (attention_workspace) the
    positions are split over many CTAs and merged; shapes that form does not take fall back to one CTA
    per head."""
    lib = _lib.load()
    if workspace is not None:
        rc = lib.sal_attention_decode_split_f16(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), pos.data_ptr(),
                                                out.data_ptr(), heads, kv_heads, hd, k_cache.shape[0], float(scale),
                                                workspace.data_ptr(), workspace.numel(), _stream(q))
        if rc != _lib.SAL_E_UNSUPPORTED:
            _lib.check(rc, "sal_attention_decode_split_f16")
            return
    _lib.check(lib.sal_attention_decode_f16(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), pos.data_ptr(),
                                            out.data_ptr(), heads, kv_heads, hd, k_cache.shape[0], float(scale),
                                            _stream(q)), "sal_attention_decode_f16")


def rope_attention_decode(q, k_new, v_new, cos, sin, pos, k_cache, v_cache, out, heads, kv_heads, hd, scale: float, workspace):
    """Rotary step of the new token, cache write and split attention in one kernel.  q / k_new / v_new: fp16
    projections (left untouched) or int64 fixed-point accumulators (consumed and cleared).  Returns False — having done
    nothing — for shapes the split kernel does not take."""
    lib = _lib.load()
    f32 = q.dtype == torch.int64          # fixed-point accumulators (consumed and cleared)
    if k_new.dtype != q.dtype or v_new.dtype != q.dtype or q.dtype not in (torch.float16, torch.int64):
        raise RuntimeError("q, k_new and v_new must all be float16 or all int64 fixed-point accumulators")
    rc = lib.sal_rope_attention_decode(q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), 1 if f32 else 0, cos.data_ptr(),
                                       sin.data_ptr(), pos.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                                       heads, kv_heads, hd, k_cache.shape[0], float(scale), workspace.data_ptr(),
                                       workspace.numel(), _stream(out))
    if rc == _lib.SAL_E_UNSUPPORTED:
        return False
    _lib.check(rc, "sal_rope_attention_decode")
    return True


def residual_rmsnorm_rows(x, delta, weight, out, x_out, eps: float):
    """residual_rmsnorm for every row of [rows, n] tensors (one weight vector)."""
    lib = _lib.load()
    rows, n = x.shape[0], x.shape[1]
    _lib.check(lib.sal_residual_rmsnorm_rows_f16(x.data_ptr(), None if delta is None else delta.data_ptr(), weight.data_ptr(),
                                                 out.data_ptr(), None if x_out is None else x_out.data_ptr(), rows, n, float(eps),
                                                 _stream(x)), "sal_residual_rmsnorm_rows_f16")


def attention_workspace_batch(batch: int, heads: int, hd: int, device) -> torch.Tensor:
    lib = _lib.load()
    return torch.zeros(int(batch) * lib.sal_attention_workspace_bytes(int(heads), int(hd)), dtype=torch.uint8, device=device)


def rope_attention_decode_batch(q, k_new, v_new, cos, sin, pos, k_cache, v_cache, out, heads, kv_heads, hd, scale: float, workspace):
    """rope_attention_decode for `batch` sequences in lock step: q [batch, heads*hd], k_new / v_new [batch, kv_heads*hd] (fp16),
    caches [batch, max_len, kv_heads, hd], out [batch, heads*hd].  Returns False — having done nothing — for shapes
    the split kernel does not take."""
    lib = _lib.load()
    rc = lib.sal_rope_attention_decode_batch(q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                                             pos.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), q.shape[0], heads,
                                             kv_heads, hd, k_cache.shape[1], float(scale), workspace.data_ptr(), workspace.numel(),
                                             _stream(out))
    if rc == _lib.SAL_E_UNSUPPORTED:
        return False
    _lib.check(rc, "sal_rope_attention_decode_batch")
    return True


def greedy_token(logits_f16, logits_f32, token, pos):
    """End of a greedy step in one launch: fp32 copy of the fp16 logits (``logits_f32`` may be None), ``token[0]`` =
    argmax (first of equal maxima), ``pos[0] += 1``.  False if the vocabulary size is not a multiple of 8."""
    vocab = logits_f16.numel()
    if vocab % 8 != 0 or logits_f16.dtype != torch.float16 or not logits_f16.is_contiguous():
        return False
    lib = _lib.load()
    _lib.check(lib.sal_greedy_token_f16(logits_f16.data_ptr(), logits_f32.data_ptr() if logits_f32 is not None else None, vocab,
                                        token.data_ptr(), pos.data_ptr(), _stream(logits_f16)), "sal_greedy_token_f16")
    return True


def silu_mul(gate, up, out):
    lib = _lib.load()
    _lib.check(lib.sal_silu_mul_f16(gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.numel(), _stream(gate)),
               "sal_silu_mul_f16")


def rope_rows(q, k, v, cos, sin, pos0: int, k_cache, v_cache, heads, kv_heads, hd) -> bool:
    """Rotary step of a prompt's rows at positions pos0, pos0 + 1, ..: q [m, heads * hd] in place, keys and values into the cache rows.
    False where the helper does not take the shape (nothing is launched then)."""
    lib = _lib.load()
    rc = lib.sal_rope_rows_f16(q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(), int(pos0), q.shape[0],
                               k_cache.data_ptr(), v_cache.data_ptr(), heads, kv_heads, hd, k_cache.shape[0], _stream(q))
    if rc in (_lib.SAL_E_SHAPE, _lib.SAL_E_ALIGN):
        return False
    _lib.check(rc, "sal_rope_rows_f16")
    return True


def causal_softmax(scores, first: int, scale: float):
    """scores fp16 [heads, m, T] -> probabilities, in place; row i sees positions 0 .. first + i."""
    lib = _lib.load()
    _lib.check(lib.sal_causal_softmax_f16(scores.data_ptr(), scores.shape[0], scores.shape[1], scores.shape[2], int(first), float(scale),
                                          _stream(scores)), "sal_causal_softmax_f16")


# ---- a cache in 4 bits, in pages, for sequences of different lengths ----------------------------------------------------

KV4_PAGE = _lib.SAL_KV4_PAGE


_compiled = None   # the compiled module with these calls; False where it has not been built or cannot be imported


def _native():
    """The compiled module (csrc/decode_ext.cpp), whose calls make the checks below in a few microseconds less, or False."""
    global _compiled
    if _compiled is None:
        from . import lutgemm

        _lib.load()   # the module links to the library by name: the one loaded here is the one it finds
        try:
            module = lutgemm.compiled_module()
            _compiled = module if hasattr(module, "attention_kv4") else False
        except (RuntimeError, ImportError, OSError) as e:   # not built, or for another interpreter or torch
            warnings.warn(f"the compiled module cannot be imported, the 4-bit cache's calls take their steps in Python: {e}")
            _compiled = False
    return _compiled


def _want(what, name, t, dtype, shape, device):
    """`t` is a contiguous tensor of this dtype on this device; `shape`: so many numbers in all, so many in its last dimension."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{what}: {name} must be a torch.Tensor")
    if t.device != device or t.dtype != dtype or not t.is_contiguous() or t.numel() != math.prod(shape) or (t.dim() > 0 and t.shape[-1] != shape[-1]):
        raise RuntimeError(f"{what}: {name} must be a contiguous {dtype} tensor {list(shape)} on {device}, got {list(t.shape)} {t.dtype} on {t.device}")


def _kv4_pool_check(what, pool, table, pos, rows, kv_heads, hd):
    """Checks what every call on a layer's pool takes; returns (device, batch, max_pages, pages)."""
    if not isinstance(pool, torch.Tensor) or not pool.is_cuda:
        raise RuntimeError(f"{what}: pool must be a CUDA tensor (there is no CPU path)")
    record = kv4_record_bytes(hd)
    if pool.dim() != 3 or pool.shape[1] != kv_heads or pool.shape[2] != record or pool.dtype != torch.uint8 or not pool.is_contiguous():
        raise RuntimeError(f"{what}: pool must be a contiguous uint8 tensor [pages, {kv_heads}, {record}], got {tuple(pool.shape)} {pool.dtype}")
    device, batch = pool.device, pos.numel()
    _want(what, "pos", pos, torch.int64, (batch,), device)
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.shape[0] != batch or table.shape[1] < 1:
        raise RuntimeError(f"{what}: table must be an int32 tensor [{batch}, pages of a sequence]")
    _want(what, "table", table, torch.int32, table.shape, device)
    if rows is not None:
        _want(what, "rows", rows, torch.int32, (batch,), device)
    return device, batch, table.shape[1], pool.shape[0]


def _rows_per_sequence(what, name, t, batch, width):
    """m of a tensor [batch, m, width] (or [batch * m, width])."""
    if not isinstance(t, torch.Tensor) or batch < 1 or width < 1 or t.numel() == 0 or t.numel() % (batch * width):
        raise RuntimeError(f"{what}: {name} must hold the same number of rows of {width} numbers for each of {batch} sequences")
    return t.numel() // (batch * width)


def kv4_record_bytes(hd: int) -> int:
    """Bytes of a page and kv head: 64 positions of codes and parameters, keys and values."""
    if hd not in (64, 128, 256):
        raise RuntimeError(f"the 4-bit cache takes heads of 64, 128 or 256 numbers, got {hd}")
    return KV4_PAGE * (hd + hd // 8)


def kv4_pool(layers: int, pages: int, kv_heads: int, hd: int, device) -> torch.Tensor:
    """Zero-filled pages for `layers` layers: uint8 [layers, pages, kv_heads, record]; a layer's pool is `pool[layer]`."""
    return torch.zeros(layers, pages, kv_heads, kv4_record_bytes(hd), dtype=torch.uint8, device=device)


def rope_kv4_write(q, k, v, cos, sin, pos, table, pool, q_out, heads, kv_heads, hd, rows=None):
    """Rotary step of m new rows of each of `batch` sequences, and their keys and values into a 4-bit cache (the format, and what is left
    unwritten, stand in include/sal_decode_ops.h).  q, q_out fp16 [batch, m, heads * hd] (q_out may be q), k, v fp16 [batch, m, kv_heads * hd],
    cos, sin fp32 [max_len, hd / 2], pos int64 [batch]: position of each sequence's first new row, table int32 [batch, pages of a sequence],
    pool: one layer's uint8 [pages, kv_heads, record].  rows int32 [batch]: how many of the m rows there are (None: all)."""
    native = _compiled if _compiled is not None else _native()
    if native:
        return native.rope_kv4_write(q, k, v, cos, sin, pos, table, pool, q_out, heads, kv_heads, hd, rows)
    device, batch, max_pages, pages = _kv4_pool_check("rope_kv4_write", pool, table, pos, rows, kv_heads, hd)
    m = _rows_per_sequence("rope_kv4_write", "q", q, batch, heads * hd)
    for name, t, width in (("q", q, heads), ("q_out", q_out, heads), ("k", k, kv_heads), ("v", v, kv_heads)):
        _want("rope_kv4_write", name, t, torch.float16, (batch, m, width * hd), device)
    angles = cos.numel() // (hd // 2)
    for name, t in (("cos", cos), ("sin", sin)):
        _want("rope_kv4_write", name, t, torch.float32, (angles, hd // 2), device)
    lib = _lib.load()
    with _on(device):
        _lib.check(lib.sal_rope_kv4_write_f16(q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(), pos.data_ptr(),
                                              None if rows is None else rows.data_ptr(), table.data_ptr(), pool.data_ptr(), q_out.data_ptr(),
                                              batch, m, heads, kv_heads, hd, angles, max_pages, pages, _stream(q)), "sal_rope_kv4_write_f16")


def read_kv4(pool, table, pos, k_out, v_out, kv_heads, hd):
    """The values of m positions of each sequence, from pos[b] on: k_out and v_out [batch, m, kv_heads, hd] in float32 (as they are) or
    float16 (rounded); zeros where a sequence has no page."""
    native = _compiled if _compiled is not None else _native()
    if native:
        return native.read_kv4(pool, table, pos, k_out, v_out, kv_heads, hd)
    device, batch, max_pages, pages = _kv4_pool_check("read_kv4", pool, table, pos, None, kv_heads, hd)
    m = _rows_per_sequence("read_kv4", "k_out", k_out, batch, kv_heads * hd)
    if k_out.dtype not in (torch.float32, torch.float16):
        raise RuntimeError(f"read_kv4: k_out must be float32 or float16, got {k_out.dtype}")
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        _want("read_kv4", name, t, k_out.dtype, (batch, m, kv_heads, hd), device)
    lib = _lib.load()
    with _on(device):
        _lib.check(lib.sal_read_kv4(pool.data_ptr(), table.data_ptr(), pos.data_ptr(), k_out.data_ptr(), v_out.data_ptr(),
                                    1 if k_out.dtype == torch.float32 else 0, batch, m, kv_heads, hd, max_pages, pages, _stream(pool)), "sal_read_kv4")


def attention_kv4_workspace(batch: int, m: int, heads: int, kv_heads: int, hd: int, device) -> torch.Tensor:
    """Zero-filled scratch for attention_kv4 calls of up to this size (one per stream that uses it)."""
    lib = _lib.load()
    need = lib.sal_attention_kv4_workspace_bytes(int(batch), int(m), int(heads), int(kv_heads), int(hd))
    if need == 0:
        raise RuntimeError(f"attention_kv4_workspace: no such shape: batch {batch}, {m} rows, {heads} heads over {kv_heads}, {hd} numbers")
    return torch.zeros(need, dtype=torch.uint8, device=device)


def attention_kv4(q, pool, table, pos, out, heads, kv_heads, hd, scale: float, workspace, rows=None):
    """Attention of m rows of each of `batch` sequences over a 4-bit cache: row i of sequence b sees the positions 0 .. pos[b] + i as far as
    their pages exist (none: zeros).  q (rotated) and out fp16 [batch, m, heads * hd]; the other arguments as rope_kv4_write takes them."""
    native = _compiled if _compiled is not None else _native()
    if native:
        return native.attention_kv4(q, pool, table, pos, out, heads, kv_heads, hd, scale, workspace, rows)
    device, batch, max_pages, pages = _kv4_pool_check("attention_kv4", pool, table, pos, rows, kv_heads, hd)
    m = _rows_per_sequence("attention_kv4", "q", q, batch, heads * hd)
    for name, t in (("q", q), ("out", out)):
        _want("attention_kv4", name, t, torch.float16, (batch, m, heads * hd), device)
    _want("attention_kv4", "workspace", workspace, torch.uint8, workspace.shape, device)
    lib = _lib.load()
    with _on(device):
        _lib.check(lib.sal_attention_kv4_f16(q.data_ptr(), pool.data_ptr(), table.data_ptr(), pos.data_ptr(),
                                             None if rows is None else rows.data_ptr(), out.data_ptr(), batch, m, heads, kv_heads, hd, max_pages,
                                             pages, float(scale), workspace.data_ptr(), workspace.numel(), _stream(q)), "sal_attention_kv4_f16")


def attention_kv4_check(workspace):
    """Waits for the current stream; RuntimeError if a wait of an attention_kv4 call with this workspace ran out since the last look.  That call went
    on without the pages that it waited for, so its outputs, and all that was made of them, are wrong."""
    lib = _lib.load()
    with _on(workspace.device):
        _lib.check(lib.sal_workspace_status(workspace.data_ptr(), _stream(workspace)), "attention_kv4 on the device")


def copy_kv4_pages(pool, src, dst):
    """Page dst[i] of `pool` (uint8 [layers, pages, ..]) becomes a copy of page src[i], in every layer.  src and dst are sequences of whole
    numbers on the host; no page may be written twice, or written and read in the same call."""
    native = _compiled if _compiled is not None else _native()
    if native:
        return native.copy_kv4_pages(pool, src, dst)
    if not isinstance(pool, torch.Tensor) or not pool.is_cuda or pool.dtype != torch.uint8 or pool.dim() < 3 or not pool.is_contiguous():
        raise RuntimeError("copy_kv4_pages: pool must be a contiguous uint8 CUDA tensor [layers, pages, ..]")
    n = len(src)
    if len(dst) != n:
        raise RuntimeError(f"copy_kv4_pages: {n} pages to copy, {len(dst)} places")
    if n == 0:
        return
    if not all(0 <= p < pool.shape[1] for p in (*src, *dst)):      # a 32-bit number of them would wrap around
        raise RuntimeError(f"copy_kv4_pages: pages must be 0 .. {pool.shape[1] - 1}")
    lib = _lib.load()
    pages = (ctypes.c_int32 * (2 * n))(*src, *dst)
    with _on(pool.device):
        _lib.check(lib.sal_copy_kv4_pages(pool.data_ptr(), ctypes.addressof(pages), ctypes.addressof(pages) + 4 * n, n, pool.shape[0], pool.shape[1],
                                          pool[0, 0].numel(), _stream(pool)), "sal_copy_kv4_pages (no page twice, none both read and written)")


# ---- the next token ---------------------------------------------------------------------------------------------------


def sample_token(logits, u, token, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """token[r] (int64) = the next token of row r of logits (fp16 or fp32 [rows, vocab]), drawn with the random number u[r] (fp32, in [0, 1)).
    temperature, top_k, top_p and min_p are one number for all rows or a tensor of one per row (float32; top_k int32).  What each filter keeps,
    and in which order they apply, stands in include/sal_decode_ops.h."""
    native = _compiled if _compiled is not None else _native()
    if native:
        return native.sample_token(logits, u, token, temperature, top_k, top_p, min_p)
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in (torch.float16, torch.float32) or not logits.is_contiguous() \
            or logits.numel() == 0:
        raise RuntimeError("sample_token: logits must be a contiguous float16 or float32 CUDA tensor [rows, vocab]")
    vocab = logits.shape[-1]
    rows, device = logits.numel() // vocab, logits.device
    _want("sample_token", "u", u, torch.float32, (rows,), device)
    _want("sample_token", "token", token, torch.int64, (rows,), device)
    ptr, one = [], []
    for name, v, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32)):
        if isinstance(v, torch.Tensor):
            _want("sample_token", name, v, dtype, (rows,), device)
            ptr.append(v.data_ptr())
            one.append(0)
        else:
            if name == "top_k" and not abs(v) <= 0x7fffffff:
                raise RuntimeError(f"sample_token: top_k must be a 32-bit number, got {v}")
            ptr.append(None)
            one.append(v)
    lib = _lib.load()
    with _on(device):
        _lib.check(lib.sal_sample_token(logits.data_ptr(), 1 if logits.dtype == torch.float32 else 0, rows, vocab, u.data_ptr(), *ptr, float(one[0]),
                                        int(one[1]), float(one[2]), float(one[3]), token.data_ptr(), _stream(logits)), "sal_sample_token")
