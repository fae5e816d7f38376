"""The 4-bit cache on the GPU: rows written and read back, attended to, pages copied, against plain 64-bit arithmetic."""
import math

import numpy as np
import pytest
import torch

from shiftaddllm_b200 import decode_ops

pytestmark = pytest.mark.gpu
PAGE = 64


# ---- the format, from its definition -------------------------------------------------------------------


def place(g, p, groups):
    s = (p & 3) ^ ((p >> 1) & 2)
    return g ^ (s if groups == 4 else s >> 1 if groups == 2 else 0)


def quantise(x):
    """x fp16 [.., hd] -> (codes [.., G, 64], scale, low fp16 [.., G])."""
    g = x.astype(np.float32).reshape(*x.shape[:-1], -1, 64)
    low, high = g.min(-1), g.max(-1)
    with np.errstate(all="ignore"):
        scale = ((high - low) / np.float32(15)).astype(np.float16)
        inv = np.where(scale > 0, np.float32(1) / scale.astype(np.float32), np.float32(0))
        code = np.minimum(np.rint((g - low[..., None]) * inv[..., None]), 15)
    bad = ~np.isfinite(g).all(-1)
    code[bad] = 0
    scale[bad] = low[bad] = np.nan
    return code.astype(np.uint8), scale, low.astype(np.float16)


def put(pool, page, h, p, hd, k, v):
    """Writes the row of position p (within its page) into a numpy pool."""
    groups, size = hd // 64, 32 * hd
    for i, x in enumerate((k, v)):
        code, scale, low = quantise(x)
        for g in range(groups):
            at = i * size + p * hd // 2 + place(g, p, groups) * 32
            pool[page, h, at:at + 32] = code[g, 0::2] | code[g, 1::2] << 4
            par = np.array([scale[g], low[g]], np.float16).view(np.uint8)
            if np.isnan(scale[g]):
                par = np.array([0x7fff, 0x7fff], np.uint16).view(np.uint8)
            at = 2 * size + i * size // 8 + (p * groups + g) * 4
            pool[page, h, at:at + 4] = par


def values(pool, hd):
    """numpy pool [pages, kv_heads, record] -> K, V float64 [pages, kv_heads, 64, hd]."""
    groups, size = hd // 64, 32 * hd
    got = []
    for i in range(2):
        codes = pool[..., i * size:(i + 1) * size].reshape(*pool.shape[:2], PAGE, groups, 32)
        par = np.ascontiguousarray(pool[..., 2 * size + i * size // 8: 2 * size + (i + 1) * size // 8]).view(np.float16)
        par = par.reshape(*pool.shape[:2], PAGE, groups, 2).astype(np.float64)
        out = np.empty((*pool.shape[:2], PAGE, groups, 64))
        for p in range(PAGE):
            for g in range(groups):
                b = codes[:, :, p, place(g, p, groups)]
                out[:, :, p, g, 0::2], out[:, :, p, g, 1::2] = b & 15, b >> 4
        with np.errstate(all="ignore"):
            got.append((out * par[..., :1] + par[..., 1:]).reshape(*pool.shape[:2], PAGE, hd))
    return got


def rotated(x, cos, sin):
    """x fp16 [heads, hd]; cos, sin fp32 [hd / 2]: exact, rounded to 32 and then to 16 bits."""
    a, b = np.split(x.astype(np.float64), 2, -1)
    c, s = cos.astype(np.float64), sin.astype(np.float64)
    with np.errstate(all="ignore"):
        return np.concatenate((a * c - b * s, b * c + a * s), -1).astype(np.float32).astype(np.float16)


def angles(n, hd):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def random_pool(rng, pages, kvh, hd):
    return rng.integers(0, 256, (pages, kvh, PAGE * (hd + hd // 8)), dtype=np.uint8)


# ---- writing and reading -------------------------------------------------------------------------------------


@pytest.mark.parametrize("hd,heads,kvh,m,pos,rows,in_place", [
    (128, 4, 2, 1, [0, 63, 64, 200], None, False),
    (64, 3, 1, 1, [5, 127], None, True),
    (256, 2, 2, 3, [61, 0, 130], [3, 0, 2], False),
    (128, 8, 8, 70, [60, 1], [70, 33], True),
    (64, 16, 1, 5, [-2, 252, 10 ** 15, -(10 ** 15)], None, False),       # rows in front of the text and behind the table
])
def test_rows_are_written_bit_for_bit(hd, heads, kvh, m, pos, rows, in_place):
    rng = np.random.default_rng(hd + m)
    batch, width = len(pos), 4
    pages = batch * width + 2
    table = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32)
    table[0, 1], table[-1, 2] = -1, pages                                # pages that do not exist
    q, k, v = (rng.standard_normal((batch, m, n * hd)).astype(np.float16) for n in (heads, kvh, kvh))
    k[..., ::17] *= 8
    k[0, 0, :64] = 0.25                                                     # a group without a range
    v[-1, 0, 3], v[0, -1, 5] = np.inf, np.nan
    max_len = 250
    cos, sin = angles(max_len, hd)
    pool = random_pool(rng, pages, kvh, hd)
    q_out = q.copy() if in_place else np.full_like(q, 7)
    want_pool, want_q = pool.copy(), q_out.copy()
    for b in range(batch):
        for i in range(m if rows is None else rows[b]):
            p = pos[b] + i
            if not 0 <= p < min(max_len, width * PAGE):
                continue
            want_q[b, i] = rotated(q[b, i].reshape(heads, hd), cos[p], sin[p]).reshape(-1)
            kr = rotated(k[b, i].reshape(kvh, hd), cos[p], sin[p])
            page = table[b, p // PAGE]
            if 0 <= page < pages:
                for h in range(kvh):
                    put(want_pool, page, h, p % PAGE, hd, kr[h], v[b, i].reshape(kvh, hd)[h])
    g_pool, g_table, g_pos, g_q = cuda(pool), cuda(table), torch.tensor(pos).cuda(), cuda(q)
    g_out = g_q if in_place else cuda(q_out)
    g_rows = None if rows is None else torch.tensor(rows, dtype=torch.int32).cuda()
    decode_ops.rope_kv4_write(g_q, cuda(k), cuda(v), cuda(cos), cuda(sin), g_pos, g_table, g_pool, g_out, heads, kvh, hd, rows=g_rows)
    assert np.array_equal(g_out.cpu().numpy(), want_q)
    assert np.array_equal(g_pool.cpu().numpy(), want_pool)
    # and read back: the values in 32 bits are low + scale * code rounded once
    n = 6
    k_out, v_out = (torch.full((batch, n, kvh, hd), 9.0, device="cuda") for _ in range(2))
    decode_ops.read_kv4(g_pool, g_table, g_pos, k_out, v_out, kvh, hd)
    k_half, v_half = torch.empty_like(k_out, dtype=torch.float16), torch.empty_like(k_out, dtype=torch.float16)
    decode_ops.read_kv4(g_pool, g_table, g_pos, k_half, v_half, kvh, hd)
    kv = values(want_pool, hd)
    for x, got, half in ((kv[0], k_out, k_half), (kv[1], v_out, v_half)):
        want = np.zeros((batch, n, kvh, hd))
        for b in range(batch):
            for i in range(n):
                p = pos[b] + i
                page = table[b, p // PAGE] if 0 <= p < width * PAGE else -1
                if 0 <= page < pages:
                    want[b, i] = x[page, :, p % PAGE]
        with np.errstate(all="ignore"):
            assert np.array_equal(got.cpu().numpy(), want.astype(np.float32), equal_nan=True)
            assert np.array_equal(half.cpu().numpy(), want.astype(np.float32).astype(np.float16), equal_nan=True)


def test_a_value_is_half_a_step_off_at_most():
    """|value - x| <= scale / 2 plus what the roundings add: the scale's own (2**-11 of it, times 15 codes) and the clamp."""
    rng = np.random.default_rng(0)
    hd, kvh, n = 128, 4, 200
    x = (rng.standard_normal((1, n, kvh * hd)) * np.exp(rng.uniform(-6, 6, (1, n, kvh * hd)))).astype(np.float16)
    pool, table = decode_ops.kv4_pool(1, 4, kvh, hd, "cuda")[0], torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    cos, sin = torch.ones(256, hd // 2, device="cuda"), torch.zeros(256, hd // 2, device="cuda")
    pos, g = torch.zeros(1, dtype=torch.int64, device="cuda"), cuda(x)
    decode_ops.rope_kv4_write(g, g, g, cos, sin, pos, table, pool, torch.empty_like(g), kvh, kvh, hd)
    k, v = torch.empty(1, n, kvh, hd, device="cuda"), torch.empty(1, n, kvh, hd, device="cuda")
    decode_ops.read_kv4(pool, table, pos, k, v, kvh, hd)
    groups = x.astype(np.float64).reshape(n, -1, 64)
    step = (groups.max(-1) - groups.min(-1)) / 15
    bound = (step * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -10) + 16 * 2.0 ** -24)[..., None]   # a step below 2**-14 is a multiple of 2**-24
    for got in (k, v):
        assert (np.abs(got.cpu().numpy().astype(np.float64).reshape(n, -1, 64) - groups) <= bound).all()


# ---- attention --------------------------------------------------------------------------------------------------


def attention(q, pool, table, pos, rows, heads, kvh, hd, scale):
    """float64 result and the bound on a kernel's error, [batch, m, heads, hd]; rows that are not there: NaN."""
    batch, m = q.shape[:2]
    k, v = values(pool, hd)
    out = np.full((batch, m, heads, hd), np.nan)
    bound = np.zeros_like(out)
    for b in range(batch):
        for i in range(m if rows is None else rows[b]):
            n = min(pos[b] + i + 1, table.shape[1] * PAGE)
            at = [t for t in range(max(n, 0)) if 0 <= table[b, t // PAGE] < pool.shape[0]]
            for h in range(heads):
                if not at:
                    out[b, i, h] = 0
                    continue
                x = q[b, i].reshape(heads, hd)[h].astype(np.float64)
                kk = k[table[b, np.array(at) // PAGE], h // (heads // kvh), np.array(at) % PAGE]
                vv = v[table[b, np.array(at) // PAGE], h // (heads // kvh), np.array(at) % PAGE]
                s = kk @ x * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[b, i, h] = w @ vv
                # scores are sums of hd products in 32 bits (and of the groups' parts), so off by (hd + 8) 2**-24 of the sum of magnitudes; a
                # weight by twice that relative and 2**-20 for the exponential, the division and its two 16-bit parts; the output's
                # rounding is half a step of 16 bits; sums of n weights and products in 32 bits
                ds = (hd + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                spread = w @ (np.abs(vv) + np.abs(vv).max(0) * 2.0 ** -3)
                bound[b, i, h] = 2.0 ** -11 * np.abs(out[b, i, h]) + 2.0 ** -25 + (2 * ds + 2.0 ** -20 + 2.0 ** -24 * math.sqrt(n)) * spread
    return out, bound


def filled(rng, batch, width, kvh, hd, extra=2, spread=1.0):
    pages = batch * width + extra
    pool = random_pool(rng, pages, kvh, hd)
    x = rng.standard_normal((2, pages, kvh, PAGE, hd)) * spread
    x[..., :: hd // 4] *= 4
    x = x.astype(np.float16)
    groups, size = hd // 64, 32 * hd
    for i in range(2):
        code, scale, low = quantise(x[i])
        c = code[..., 0::2] | code[..., 1::2] << 4
        order = np.array([[place(g, p, groups) for g in range(groups)] for p in range(PAGE)])
        c = np.take_along_axis(c, order[None, None, :, :, None], 3)
        pool[..., i * size:(i + 1) * size] = c.reshape(pages, kvh, -1)
        par = np.stack((scale, low), -1)
        pool[..., 2 * size + i * size // 8:2 * size + (i + 1) * size // 8] = par.reshape(pages, kvh, -1).view(np.uint8).reshape(pages, kvh, -1)
    return pool, rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32)


def poison(pool, table, b, first, hd):
    """Everything of sequence b from position `first` on becomes NaN and infinities: scales, lowest values and codes."""
    size, groups = 32 * hd, hd // 64
    for p in range(first, table.shape[1] * PAGE):
        page = table[b, p // PAGE]
        if not 0 <= page < pool.shape[0]:
            continue
        for i in range(2):
            at = 2 * size + i * size // 8 + (p % PAGE) * groups * 4
            bits = np.array([0x7e00, 0xfc00] if p % 2 else [0x7c00, 0x7e00], np.uint16).view(np.uint8)
            pool[page, :, at:at + groups * 4] = np.tile(bits, groups)
            pool[page, :, i * size + (p % PAGE) * hd // 2: i * size + (p % PAGE + 1) * hd // 2] = 0xff


def check_attention(q, pool, table, pos, rows, heads, kvh, hd, scale=None):
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    batch, m = q.shape[:2]
    want, bound = attention(q, pool, table, pos, rows, heads, kvh, hd, scale)
    out = torch.full((batch, m, heads * hd), 5.0, dtype=torch.float16, device="cuda")
    ws = decode_ops.attention_kv4_workspace(batch, m, heads, kvh, hd, "cuda")
    args = (cuda(q), cuda(pool), cuda(table), torch.tensor(pos).cuda())
    g_rows = None if rows is None else torch.tensor(rows, dtype=torch.int32).cuda()
    decode_ops.attention_kv4(*args, out, heads, kvh, hd, scale, ws, rows=g_rows)
    first = out.clone()
    decode_ops.attention_kv4(*args, out, heads, kvh, hd, scale, ws, rows=g_rows)
    assert torch.equal(out, first) or torch.isnan(first).any()      # the same bits again, on scratch that was used before
    got = out.view(batch, m, heads, hd).double().cpu().numpy()
    absent = np.isnan(want).all((2, 3))
    assert (got[absent] == 5.0).all()                               # rows that are not there keep what they hold
    off = np.abs(got - want)[~absent]
    assert (off <= bound[~absent]).all(), (off / bound[~absent]).max()
    return got


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (4, 2), (8, 1), (16, 1), (6, 2), (7, 7), (20, 2)])
def test_one_row_of_every_head_layout(hd, heads, kvh):
    rng = np.random.default_rng(hd + heads)
    pos = [0, 62, 63, 64, 200, 255]
    pool, table = filled(rng, len(pos), 4, kvh, hd)
    for b, p in enumerate(pos):
        poison(pool, table, b, p + 1, hd)
    check_attention(rng.standard_normal((len(pos), 1, heads * hd)).astype(np.float16), pool, table, pos, None, heads, kvh, hd)


@pytest.mark.parametrize("heads,kvh,hd,m", [(4, 2, 64, 2), (8, 1, 128, 5), (4, 4, 128, 17), (8, 2, 128, 33), (2, 1, 256, 9), (3, 1, 64, 130), (4, 4, 128, 300),
                                            (10, 2, 256, 40), (16, 1, 128, 100)])
def test_several_rows(heads, kvh, hd, m):
    rng = np.random.default_rng(m)
    pos, rows = [0, 70, -1, 129], [m, max(1, m // 2), m, 0]
    width = (129 + m) // PAGE + 1
    pool, table = filled(rng, 4, width, kvh, hd)
    for b, p in enumerate(pos):
        poison(pool, table, b, max(0, p + rows[b]), hd)      # row m - 1's last position is the last that anybody sees
    check_attention(rng.standard_normal((4, m, heads * hd)).astype(np.float16), pool, table, pos, rows, heads, kvh, hd)


def test_a_later_rows_nan_is_not_an_earlier_rows():
    """Rows of one tile see different positions: what is NaN for the last row must not reach the first."""
    rng = np.random.default_rng(3)
    heads, kvh, hd, m = 4, 1, 128, 4
    pool, table = filled(rng, 1, 2, kvh, hd)
    q = rng.standard_normal((1, m, heads * hd)).astype(np.float16)
    clean = check_attention(q, pool, table, [60], None, heads, kvh, hd)
    poison(pool, table, 0, 62, hd)                          # rows 2 and 3 (positions 62, 63) see it, rows 0 and 1 do not
    out = torch.empty(1, m, heads * hd, dtype=torch.float16, device="cuda")
    ws = decode_ops.attention_kv4_workspace(1, m, heads, kvh, hd, "cuda")
    decode_ops.attention_kv4(cuda(q), cuda(pool), cuda(table), torch.tensor([60]).cuda(), out, heads, kvh, hd, 1 / math.sqrt(hd), ws)
    got = out.view(1, m, heads, hd).double().cpu().numpy()
    assert np.isnan(got[:, 2:]).all()
    assert np.array_equal(got[:, :2], clean[:, :2])


@pytest.mark.parametrize("m", [1, 40])
def test_pages_that_do_not_exist_are_not_seen(m):
    rng = np.random.default_rng(5)
    heads, kvh, hd = 4, 2, 128
    pool, table = filled(rng, 4, 3, kvh, hd)
    table[0, 0], table[1, 1], table[2] = -1, 2 ** 31 - 1, pool.shape[0]
    pos = [130, 185, 150, 10 ** 12]                          # the third sees nothing at all, the fourth all there is
    check_attention(rng.standard_normal((4, m, heads * hd)).astype(np.float16), pool, table, pos, None, heads, kvh, hd)


def test_rows_with_nothing_to_see_get_zeros():
    rng = np.random.default_rng(6)
    pool, table = filled(rng, 2, 1, 2, 64)
    got = check_attention(rng.standard_normal((2, 3, 4 * 64)).astype(np.float16), pool, table, [-3, -2], None, 4, 2, 64)
    assert (got[0] == 0).all() and (got[1, 0] == 0).all() and (got[1, 2] != 0).any()


@pytest.mark.parametrize("spread", [1e-4, 1.0, 300.0])
def test_small_and_large_numbers(spread):
    """Values below what 16-bit weights resolve, and scores far apart."""
    rng = np.random.default_rng(7)
    pool, table = filled(rng, 2, 5, 2, 128, spread=spread)
    check_attention(rng.standard_normal((2, 1, 8 * 128)).astype(np.float16), pool, table, [300, 17], None, 8, 2, 128)


def test_pages_shared_by_sequences():
    rng = np.random.default_rng(8)
    pool, table = filled(rng, 3, 4, 2, 128)
    table[1, :3] = table[0, :3]
    table[2] = table[0, 0]                                    # even the same page several times in one sequence
    check_attention(rng.standard_normal((3, 2, 4 * 128)).astype(np.float16), pool, table, [250, 251, 200], None, 4, 2, 128)


def long_reference(q, k, v, scale):
    s = torch.einsum("hd,thd->ht", q.double(), k.double()) * scale
    return torch.einsum("ht,thd->hd", torch.softmax(s, -1), v.double())


def test_long_texts_of_different_lengths():
    """Many pages, work that is split within sequences: against 64-bit arithmetic on the values read back."""
    torch.manual_seed(0)
    heads, kvh, hd = 16, 4, 128
    pos = torch.tensor([30011, 5, 777, 12345], device="cuda")
    width = 30011 // PAGE + 1
    pages = 4 * width
    pool = decode_ops.kv4_pool(1, pages, kvh, hd, "cuda")[0]
    table = torch.randperm(pages, device="cuda").view(4, width).int()
    n = width * PAGE
    cos, sin = torch.ones(n, hd // 2, device="cuda"), torch.zeros(n, hd // 2, device="cuda")
    for b in range(4):
        for c0 in range(0, n, 8192):
            r = min(8192, n - c0)
            k, v = (torch.randn(1, r, kvh * hd, device="cuda").half() for _ in range(2))
            dummy = k.clone()
            decode_ops.rope_kv4_write(dummy, k, v, cos, sin, torch.tensor([c0], device="cuda"), table[b:b + 1].contiguous(), pool, dummy, kvh, kvh, hd)
    q = torch.randn(4, 1, heads * hd, device="cuda").half()
    out = torch.empty_like(q)
    ws = decode_ops.attention_kv4_workspace(4, 1, heads, kvh, hd, "cuda")
    decode_ops.attention_kv4(q, pool, table, pos, out, heads, kvh, hd, 0.2, ws)
    for b in range(4):
        t = int(pos[b]) + 1
        k, v = torch.empty(1, t, kvh, hd, device="cuda"), torch.empty(1, t, kvh, hd, device="cuda")
        decode_ops.read_kv4(pool, table[b:b + 1].contiguous(), torch.zeros(1, dtype=torch.int64, device="cuda"), k, v, kvh, hd)
        k, v = (x[0].repeat_interleave(heads // kvh, 1) for x in (k, v))
        want = long_reference(q[b, 0].view(heads, hd), k, v, 0.2)
        # half a step of 16 bits, and 2**-16 of the values' size (about 1, a few of them per text are 4) for sums and weights in 32 bits
        assert ((out[b, 0].view(heads, hd).double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -16).all()


def test_a_pool_beyond_32_bit_offsets():
    hd, kvh = 128, 8
    record = decode_ops.kv4_record_bytes(hd)
    pages = (1 << 32) // (kvh * record) + 64
    pool = torch.empty(pages, kvh, record, dtype=torch.uint8, device="cuda")
    small = decode_ops.kv4_pool(1, 4, kvh, hd, "cuda")[0]
    high = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda").view(1, 4)
    low = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    torch.manual_seed(1)
    m = 200
    q, k, v = (torch.randn(1, m, kvh * hd, device="cuda").half() for _ in range(3))
    cos, sin = (cuda(x) for x in angles(256, hd))
    pos, outs = torch.zeros(1, dtype=torch.int64, device="cuda"), []
    for p, t in ((pool, high), (small, low)):
        q_out, out, one = torch.empty_like(q), torch.empty_like(q), torch.empty(1, 1, kvh * hd, dtype=torch.float16, device="cuda")
        decode_ops.rope_kv4_write(q, k, v, cos, sin, pos, t, p, q_out, kvh, kvh, hd)
        ws = decode_ops.attention_kv4_workspace(1, m, kvh, kvh, hd, "cuda")
        decode_ops.attention_kv4(q_out, p, t, pos, out, kvh, kvh, hd, 0.1, ws)
        decode_ops.attention_kv4(q_out[:, -1:].contiguous(), p, t, pos + m - 1, one, kvh, kvh, hd, 0.1, ws)
        outs += [q_out, out, one, p[t[0].long()]]
    for a, b in zip(outs[:4], outs[4:]):
        assert torch.equal(a, b)
    two = pool.view(1, pages, kvh, record)
    decode_ops.copy_kv4_pages(two, [pages - 2], [pages - 9])
    assert torch.equal(pool[pages - 9], small[2])


def test_captured_and_replayed_beside_another_graph():
    """Positions, pages and rows are read when the launch runs; two graphs with scratch of their own run side by side."""
    rng = np.random.default_rng(9)
    heads, kvh, hd = 8, 2, 128
    pool, table = filled(rng, 2, 20, kvh, hd)
    g_pool, g_table, pos = cuda(pool), cuda(table), torch.tensor([5, 100]).cuda()
    q = cuda(rng.standard_normal((2, 1, heads * hd)).astype(np.float16))
    graphs = []
    for _ in range(2):
        out, ws, stream = torch.empty_like(q), decode_ops.attention_kv4_workspace(2, 1, heads, kvh, hd, "cuda"), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            decode_ops.attention_kv4(q, g_pool, g_table, pos, out, heads, kvh, hd, 0.1, ws)
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                decode_ops.attention_kv4(q, g_pool, g_table, pos, out, heads, kvh, hd, 0.1, ws)
        graphs.append((g, out, stream, ws))
    for step in ([70, 1], [1200, 1279], [0, 640]):
        pos.copy_(torch.tensor(step))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, _out, stream, _ws in graphs:
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(q)
        decode_ops.attention_kv4(q, g_pool, g_table, pos, eager, heads, kvh, hd, 0.1, decode_ops.attention_kv4_workspace(2, 1, heads, kvh, hd, "cuda"))
        assert torch.equal(graphs[0][1], eager) and torch.equal(graphs[1][1], eager)


# ---- pages ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("layers,pages,kvh,hd,n", [(1, 2, 1, 64, 1), (3, 40, 2, 128, 20), (2, 1200, 1, 64, 600), (5, 9, 3, 256, 4)])
def test_pages_are_copied_in_every_layer(layers, pages, kvh, hd, n):
    rng = np.random.default_rng(n)
    pool = torch.randint(0, 256, (layers, pages, kvh, decode_ops.kv4_record_bytes(hd)), dtype=torch.uint8, device="cuda")
    order = rng.permutation(pages).tolist()
    src, dst = order[:n], order[n:2 * n]
    src = [src[0]] * n if n == 4 else src                # one page copied several times
    want = pool.clone()
    want[:, dst] = pool[:, src]
    decode_ops.copy_kv4_pages(pool, src, dst)
    assert torch.equal(pool, want)
    decode_ops.copy_kv4_pages(pool, [], [])
    assert torch.equal(pool, want)


def test_refusals_leave_everything_as_it_was():
    hd, kvh, heads = 128, 2, 4
    pool = decode_ops.kv4_pool(2, 8, kvh, hd, "cuda")
    before = pool.clone()
    for src, dst in (([0], [8]), ([-1], [1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]), ([0], [1, 2])):
        with pytest.raises(RuntimeError):
            decode_ops.copy_kv4_pages(pool, src, dst)
    f16 = dict(dtype=torch.float16, device="cuda")
    q, k = torch.zeros(2, 1, heads * hd, **f16), torch.zeros(2, 1, kvh * hd, **f16)
    cos = torch.ones(64, hd // 2, device="cuda")
    pos, table = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    ws = decode_ops.attention_kv4_workspace(2, 1, heads, kvh, hd, "cuda")
    layer = pool[0]

    def attend(**kw):
        a = dict(q=q, pool=layer, table=table, pos=pos, out=torch.empty_like(q), heads=heads, kv_heads=kvh, hd=hd, scale=1.0, workspace=ws)
        decode_ops.attention_kv4(**{**a, **kw})

    def write(**kw):
        a = dict(q=q, k=k, v=k, cos=cos, sin=cos, pos=pos, table=table, pool=layer, q_out=torch.empty_like(q), heads=heads, kv_heads=kvh, hd=hd)
        decode_ops.rope_kv4_write(**{**a, **kw})

    attend(), write()
    bad = [dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:1]), dict(q=q.transpose(0, 1).expand(2, 2, -1)), dict(table=table.long()), dict(table=table[0]),
           dict(table=table.t()), dict(pos=pos.int()), dict(pos=pos[:1]), dict(pool=pool), dict(pool=layer[..., :-16]), dict(pool=layer.cpu()),
           dict(rows=pos), dict(rows=pos.int()[:1]), dict(hd=96), dict(heads=3)]
    for kw in bad:
        with pytest.raises(RuntimeError):
            attend(**kw)
        with pytest.raises(RuntimeError):
            write(**kw)
    for kw in (dict(workspace=ws[:64]), dict(out=torch.empty_like(q, dtype=torch.float32)), dict(workspace=ws.float())):
        with pytest.raises(RuntimeError):
            attend(**kw)
    for kw in (dict(k=q), dict(cos=cos[:, :8]), dict(sin=cos[:8]), dict(cos=cos.half()), dict(q_out=k)):
        with pytest.raises(RuntimeError):
            write(**kw)
    with pytest.raises(RuntimeError):
        decode_ops.read_kv4(layer, table, pos, torch.empty(2, 1, kvh, hd, device="cuda"), torch.empty(2, 1, kvh, hd, **f16), kvh, hd)
    torch.cuda.synchronize()
    assert torch.equal(pool[1], before[1]) and torch.equal(pool[0, 1:], before[0, 1:])


def test_the_same_without_the_compiled_module(monkeypatch):
    """The Python steps make the same checks and the same calls."""
    monkeypatch.setattr(decode_ops, "_compiled", False)
    rng = np.random.default_rng(11)
    pool, table = filled(rng, 2, 2, 2, 128)
    check_attention(rng.standard_normal((2, 2, 4 * 128)).astype(np.float16), pool, table, [100, 3], [2, 1], 4, 2, 128)
    test_rows_are_written_bit_for_bit(128, 4, 2, 1, [0, 63, 64, 200], None, False)
    test_pages_are_copied_in_every_layer(3, 40, 2, 128, 20)
    test_refusals_leave_everything_as_it_was()
    logits, u, token = torch.randn(3, 100, device="cuda"), torch.rand(3, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    decode_ops.sample_token(logits, u, token, 0.7, 20, torch.full((3,), 0.9, device="cuda"), 0.01)
    monkeypatch.setattr(decode_ops, "_compiled", None)
    again = torch.zeros_like(token)
    decode_ops.sample_token(logits, u, again, 0.7, 20, torch.full((3,), 0.9, device="cuda"), 0.01)
    assert decode_ops._compiled and torch.equal(token, again)


@pytest.mark.parametrize("heads,kvh,m", [(8, 1, 1), (2, 2, 1), (2, 1, 40)])
def test_the_mean_of_many_values_keeps_its_digits(heads, kvh, m):
    """The output of a long text is small beside the values it is the mean of.  Its rounding to 16 bits is off by at most 2**-11 of each number,
    so by that of the norm too; on average it is 0.4 of that, which leaves the sums 0.9 of it."""
    torch.manual_seed(4)
    hd, n = 128, 100001
    pages = (n + PAGE - 1) // PAGE
    pool, table = decode_ops.kv4_pool(1, pages, kvh, hd, "cuda")[0], torch.randperm(pages, device="cuda").view(1, -1).int()
    cos, sin = torch.ones(pages * PAGE, hd // 2, device="cuda"), torch.zeros(pages * PAGE, hd // 2, device="cuda")
    for c0 in range(0, n, 50000):
        k, v = (torch.randn(1, min(50000, n - c0), kvh * hd, device="cuda").half() for _ in range(2))
        dummy = torch.empty_like(k)
        decode_ops.rope_kv4_write(k, k, v, cos, sin, torch.tensor([c0], device="cuda"), table, pool, dummy, kvh, kvh, hd)
    q = torch.randn(1, m, heads * hd, device="cuda").half()
    out, pos = torch.empty_like(q), torch.tensor([n - m], device="cuda")
    decode_ops.attention_kv4(q, pool, table, pos, out, heads, kvh, hd, hd ** -0.5, decode_ops.attention_kv4_workspace(1, m, heads, kvh, hd, "cuda"))
    got = []
    for c0 in range(0, n, 50000):
        k, v = (torch.empty(1, min(50000, n - c0), kvh, hd, device="cuda") for _ in range(2))
        decode_ops.read_kv4(pool, table, torch.tensor([c0], device="cuda"), k, v, kvh, hd)
        got.append((k, v))
    k, v = (torch.cat(x, 1)[0].repeat_interleave(heads // kvh, 1).transpose(0, 1).double() for x in zip(*got))            # [heads, n, hd]
    s = (q.view(m, heads, hd).transpose(0, 1).double() @ k.transpose(1, 2)) * hd ** -0.5
    s.masked_fill_(torch.arange(n, device="cuda") > (n - m + torch.arange(m, device="cuda"))[:, None], float("-inf"))
    want = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(1, m, -1)
    assert (out.double() - want).norm() <= 2.0 ** -11 * want.norm()


def test_one_workspace_for_calls_of_every_size():
    """Scratch of the largest call serves the smaller ones in any order: what one leaves there does not disturb the next."""
    rng = np.random.default_rng(12)
    heads, kvh, hd, width = 8, 2, 128, 40
    pool, table = filled(rng, 4, width, kvh, hd)
    g_pool, g_table = cuda(pool), cuda(table)
    ws = decode_ops.attention_kv4_workspace(4, 300, heads, kvh, hd, "cuda")
    calls = []
    for batch, m, pos in ((1, 1, [2500]), (4, 300, [2200, 0, 77, 1500]), (2, 5, [2000, 900]), (3, 1, [1, 2, 2555]), (4, 16, [2000] * 4), (1, 200, [2300])):
        q = cuda(rng.standard_normal((batch, m, heads * hd)).astype(np.float16))
        args = (q, g_pool, g_table[:batch].contiguous(), torch.tensor(pos, device="cuda"))
        alone = torch.empty_like(q)
        decode_ops.attention_kv4(*args, alone, heads, kvh, hd, 0.09, decode_ops.attention_kv4_workspace(batch, m, heads, kvh, hd, "cuda"))
        calls.append((args, alone))
    for i in rng.permutation(np.repeat(np.arange(len(calls)), 6)):
        args, alone = calls[i]
        out = torch.empty_like(alone)
        decode_ops.attention_kv4(*args, out, heads, kvh, hd, 0.09, ws)
        assert torch.equal(out, alone)


def written(kvh, hd, lengths, width):
    """A pool with random rows, its table, and a function that reads a sequence back as K, V [kvh, n, hd] in 64 bits."""
    batch = len(lengths)
    pages = sum(-(-n // PAGE) for n in lengths)
    pool = decode_ops.kv4_pool(1, pages, kvh, hd, "cuda")[0]
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    order, at = torch.randperm(pages, device="cuda").int(), 0
    cos, sin = torch.ones(width * PAGE, hd // 2, device="cuda"), torch.zeros(width * PAGE, hd // 2, device="cuda")
    for b, n in enumerate(lengths):
        k = -(-n // PAGE)
        table[b, :k] = order[at:at + k]
        at += k
        for c0 in range(0, n, 50000):
            x, y = (torch.randn(1, min(50000, n - c0), kvh * hd, device="cuda").half() for _ in range(2))
            decode_ops.rope_kv4_write(x, x, y, cos, sin, torch.tensor([c0], device="cuda"), table[b:b + 1].contiguous(), pool, torch.empty_like(x), kvh, kvh, hd)

    def back(b, heads):
        got = []
        for c0 in range(0, lengths[b], 50000):
            k, v = (torch.empty(1, min(50000, lengths[b] - c0), kvh, hd, device="cuda") for _ in range(2))
            decode_ops.read_kv4(pool, table[b:b + 1].contiguous(), torch.tensor([c0], device="cuda"), k, v, kvh, hd)
            got.append((k[0, :, heads].double(), v[0, :, heads].double()))
        return (torch.cat(x).transpose(0, 1) for x in zip(*got))

    return pool, table, back


def against_64_bits(q, out, back, b, pos, kv_head, heads, kvh, hd, scale):
    """Rows of the query heads of one kv head; the bound as in test_the_mean_of_many_values_keeps_its_digits."""
    rep, m = heads // kvh, q.shape[1]
    k, v = back(b, [kv_head])
    x = q[b].view(m, heads, hd)[:, kv_head * rep:(kv_head + 1) * rep].transpose(0, 1).double()      # [rep, m, hd]
    s = x @ k[0].T * scale
    s.masked_fill_(torch.arange(s.shape[-1], device="cuda") > pos + torch.arange(m, device="cuda")[:, None], float("-inf"))
    want = torch.softmax(s, -1) @ v[0]
    got = out[b].view(m, heads, hd)[:, kv_head * rep:(kv_head + 1) * rep].transpose(0, 1).double()
    assert (got - want).norm() <= 2.0 ** -11 * want.norm(), (b, kv_head)


def test_runs_of_many_pages():
    """So much work that a thread block's run has several hundred pages."""
    torch.manual_seed(6)
    heads, kvh, hd, lengths = 32, 32, 64, [150001, 70, 90017]
    pool, table, back = written(kvh, hd, lengths, -(-150001 // PAGE))
    q = torch.randn(3, 1, heads * hd, device="cuda").half()
    out, pos = torch.empty_like(q), torch.tensor([n - 1 for n in lengths], device="cuda")
    decode_ops.attention_kv4(q, pool, table, pos, out, heads, kvh, hd, 0.125, decode_ops.attention_kv4_workspace(3, 1, heads, kvh, hd, "cuda"))
    for b, h in ((0, 0), (0, 31), (1, 7), (2, 0), (2, 30)):
        against_64_bits(q, out, back, b, lengths[b] - 1, h, heads, kvh, hd, 0.125)


@pytest.mark.parametrize("batch,m,heads,kvh,hd", [(300, 1, 4, 2, 64), (40, 70, 8, 1, 128), (300, 3, 2, 2, 256)])
def test_more_sequences_than_the_list_takes(batch, m, heads, kvh, hd):
    """A thread block takes an item then, long texts among them."""
    torch.manual_seed(7)
    lengths = [1 + (b * 37) % 200 + m for b in range(batch)]
    lengths[3], lengths[-1] = 20011, 9000
    pool, table, back = written(kvh, hd, lengths, -(-20011 // PAGE))
    q = torch.randn(batch, m, heads * hd, device="cuda").half()
    out, pos = torch.empty_like(q), torch.tensor([n - m for n in lengths], device="cuda")
    decode_ops.attention_kv4(q, pool, table, pos, out, heads, kvh, hd, 0.1, decode_ops.attention_kv4_workspace(batch, m, heads, kvh, hd, "cuda"))
    for b in (0, 3, 17, batch - 2, batch - 1):
        against_64_bits(q, out, back, b, lengths[b] - m, kvh - 1, heads, kvh, hd, 0.1)


def test_queries_may_be_overwritten_by_the_outputs():
    rng = np.random.default_rng(13)
    pool, table = filled(rng, 2, 60, 2, 128)
    q = cuda(rng.standard_normal((2, 3, 8 * 128)).astype(np.float16))
    args = (cuda(pool), cuda(table), torch.tensor([3700, 40], device="cuda"))
    out, ws = torch.empty_like(q), decode_ops.attention_kv4_workspace(2, 3, 8, 2, 128, "cuda")
    decode_ops.attention_kv4(q, *args, out, 8, 2, 128, 0.1, ws)
    decode_ops.attention_kv4(q, *args, q, 8, 2, 128, 0.1, ws)
    assert torch.equal(q, out)


@pytest.mark.parametrize("heads,kvh,hd,m", [(1, 1, 128, 65), (1, 1, 64, 128), (3, 1, 128, 43), (5, 1, 64, 77), (8, 2, 128, 17), (64, 1, 64, 2), (2, 2, 128, 257)])
@pytest.mark.parametrize("far", [0, 1500])
def test_tiles_of_many_columns(heads, kvh, hd, m, far):
    """Up to, at and behind the end of a tile of 128 columns; with `far` an item's pages are split."""
    rng = np.random.default_rng(m + far)
    pos, rows = [far, 63, -2, far + 65], [m, max(1, m // 3), m, 0]
    width = (far + 65 + m) // PAGE + 1
    pool, table = filled(rng, 4, width, kvh, hd)
    for b, p in enumerate(pos):
        poison(pool, table, b, max(0, p + rows[b]), hd)
    check_attention(rng.standard_normal((4, m, heads * hd)).astype(np.float16), pool, table, pos, rows, heads, kvh, hd)


@pytest.mark.parametrize("spread", [1e-4, 1.0, 300.0])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_columns_of_small_and_large_numbers(hd, spread):
    rng = np.random.default_rng(17)
    pool, table = filled(rng, 1, 5, 2, hd, spread=spread)
    q = (rng.standard_normal((1, 70, 2 * hd)) * 3).astype(np.float16)
    check_attention(q, pool, table, [240], None, 2, 2, hd, scale=0.5 if spread < 1 else None)


def test_a_later_rows_nan_in_a_tile_of_many_columns():
    rng = np.random.default_rng(18)
    heads, kvh, hd, m = 4, 1, 128, 40
    pool, table = filled(rng, 1, 2, kvh, hd)
    q = rng.standard_normal((1, m, heads * hd)).astype(np.float16)
    clean = check_attention(q, pool, table, [50], None, heads, kvh, hd)
    poison(pool, table, 0, 60, hd)                          # rows from 10 on see it
    out = torch.empty(1, m, heads * hd, dtype=torch.float16, device="cuda")
    ws = decode_ops.attention_kv4_workspace(1, m, heads, kvh, hd, "cuda")
    decode_ops.attention_kv4(cuda(q), cuda(pool), cuda(table), torch.tensor([50]).cuda(), out, heads, kvh, hd, 1 / math.sqrt(hd), ws)
    got = out.view(1, m, heads, hd).double().cpu().numpy()
    assert np.isnan(got[:, 10:]).all()
    want, bound = attention(q, filled(np.random.default_rng(18), 1, 2, kvh, hd)[0], table, [50], None, heads, kvh, hd, 1 / math.sqrt(hd))
    assert (np.abs(got - want)[:, :10] <= bound[:, :10]).all() and np.isfinite(clean).all()


def test_many_columns_without_some_pages():
    rng = np.random.default_rng(19)
    heads, kvh, hd, m = 4, 2, 128, 70
    pool, table = filled(rng, 4, 9, kvh, hd)
    table[0, 0], table[0, 4:6], table[1, 8], table[2] = -1, -7, 2 ** 31 - 1, pool.shape[0]
    pos = [430, 9 * PAGE - 71, 300, 10 ** 12]                # the third sees nothing at all, the fourth all there is
    check_attention(rng.standard_normal((4, m, heads * hd)).astype(np.float16), pool, table, pos, None, heads, kvh, hd)


@pytest.mark.parametrize("heads,kvh,m", [(2, 1, 70), (1, 1, 65)])
def test_the_mean_of_many_values_in_a_tile_of_many_columns(heads, kvh, m):
    test_the_mean_of_many_values_keeps_its_digits(heads, kvh, m)


def test_many_queries_may_be_overwritten_by_the_outputs():
    rng = np.random.default_rng(20)
    pool, table = filled(rng, 2, 60, 2, 128)
    q = cuda(rng.standard_normal((2, 40, 8 * 128)).astype(np.float16))
    args = (cuda(pool), cuda(table), torch.tensor([3700, 40], device="cuda"))
    out, ws = torch.empty_like(q), decode_ops.attention_kv4_workspace(2, 40, 8, 2, 128, "cuda")
    decode_ops.attention_kv4(q, *args, out, 8, 2, 128, 0.1, ws)
    decode_ops.attention_kv4(q, *args, q, 8, 2, 128, 0.1, ws)
    assert torch.equal(q, out)
