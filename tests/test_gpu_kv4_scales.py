"""One position whose values are far larger than all others and which nobody attends to: the others' weights keep their digits."""
import math

import pytest
import torch

from shiftaddllm_b200 import decode_ops

pytestmark = pytest.mark.gpu

SEEN = 4000           # positions in front of the first row
TAIL = 16             # all but the first have a weight of 2**-TAIL of its


def cache(kvh, hd, at):
    """Keys that are one number a position, so that the weights are known; values of a few groups' largest numbers and many near the lowest, so that a
    lost weight shows (their codes are all far below the middle)."""
    n = SEEN + 300
    g = torch.Generator(device="cuda").manual_seed(hd + kvh)
    scale = 1 / math.sqrt(hd)
    score = torch.full((n,), -TAIL * math.log(2) / (scale * hd), device="cuda")
    score[0] = 0.0
    v = 0.01 * torch.rand(n, kvh, hd, device="cuda", generator=g)
    v[..., 7::64] = 1.0 + torch.rand(n, kvh, hd // 64, device="cuda", generator=g)
    for p in at:
        score[p] = -40.0                              # a weight of nothing
        v[p] = 60000 * (2 * torch.rand(kvh, hd, device="cuda", generator=g) - 1)
    pages = -(-n // 64)
    pool = decode_ops.kv4_pool(1, pages, kvh, hd, "cuda")[0]
    table, pos = torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int64, device="cuda")
    one = torch.ones(n, hd // 2, device="cuda")
    k = score[:, None].expand(n, kvh * hd).half().contiguous()
    decode_ops.rope_kv4_write(k.clone(), k, v.half().view(n, -1), one, torch.zeros_like(one), pos, table, pool, torch.empty_like(k), kvh, kvh, hd)
    back = [torch.empty(1, n, kvh, hd, device="cuda") for _ in range(2)]
    decode_ops.read_kv4(pool, table, pos, *back, kvh, hd)
    return pool, table, scale, back[0][0, :, :, 0].double() * hd * scale, back[1][0].double()


@pytest.mark.parametrize("at", [3, 130, 1000])
@pytest.mark.parametrize("heads,kvh,hd,m,batch", [(32, 32, 128, 1, 30), (64, 8, 128, 1, 120), (64, 8, 128, 5, 120), (32, 32, 128, 150, 4), (32, 32, 64, 150, 4),
                                                  (32, 32, 64, 1, 30), (16, 16, 256, 1, 30), (16, 2, 256, 1, 120), (16, 16, 256, 70, 10)])
def test_a_position_of_far_larger_values(heads, kvh, hd, m, batch, at):
    pool, table, scale, score, v = cache(kvh, hd, [at])
    q, pos = torch.ones(batch, m, heads * hd, dtype=torch.float16, device="cuda"), torch.full((batch,), SEEN, dtype=torch.int64, device="cuda")
    out, ws = torch.empty_like(q), decode_ops.attention_kv4_workspace(batch, m, heads, kvh, hd, "cuda")
    decode_ops.attention_kv4(q, pool, table.expand(batch, -1).contiguous(), pos, out, heads, kvh, hd, scale, ws)
    # Beside the output's rounding (half a step of 16 bits): the positions of the step (32 keys) or page (64) that holds the large one lose up to all of
    # their weight times 8 scales, a scale being (2 - 0) / 15 at most; a weight times a scale elsewhere keeps 2**-31 of a scale of 2**-2, times 8; and 32-bit
    # arithmetic, of exponents up to 20, 2**-19 of the largest value.
    own, total = 64 if m * heads // kvh > 64 and hd < 256 else 32, 1.0 + SEEN * 2.0 ** -TAIL
    slack = (own * 2.0 ** -TAIL * 8 * 2 / 15 + SEEN * 2.0 ** -33 * 8) / total + 2 * 2.0 ** -19
    for row in {0, m - 1}:
        n = SEEN + row + 1
        want = torch.einsum("ph,phd->hd", torch.softmax(score[:n], 0), v[:n]).repeat_interleave(heads // kvh, 0)
        got = out.view(batch, m, heads, hd)[:, row].double()
        assert ((got - want).abs() <= want.abs() * 2.0 ** -11 + slack).all(), float((got - want).abs().max())
