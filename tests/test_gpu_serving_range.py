"""The serving operators at the ends of their types' ranges, against plain 64-bit forms."""
import math

import numpy as np
import pytest
import torch

from test_gpu_serving import HALF, TYPES, gen, ints, pool

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------- attention --
def softmax_rows(c, q, length, most, scale):
    """out of the last `most` of `length` positions in 64 bits, pages 0, 1, ... in order."""
    n = -(-length // c.page_tokens)
    k, v = ((codes[:n].double() * scales[:n].double()[..., None, None]).transpose(1, 2).reshape(-1, c.kv_heads, c.head_dim)[:length]
            for codes, scales in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)))
    group = q.shape[1] // c.kv_heads
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    x = torch.einsum("ihd,jhd->hij", q.double(), k) * scale
    hidden = torch.arange(length, device="cuda") > torch.arange(length - most, length, device="cuda")[:, None]
    return torch.einsum("hij,jhd->ihd", torch.softmax(x.masked_fill(hidden, -math.inf), 2), v)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("most,heads,kv_heads,many", [(1, 4, 2, False), (3, 8, 2, False), (64, 40, 40, True), (130, 48, 24, True)])
@pytest.mark.parametrize("gap", [14.0, 26.0])
@pytest.mark.parametrize("first", [True, False])
def test_attention_keeps_small_weights_beside_a_large_one(dtype, dim, most, heads, kv_heads, many, gap, first):
    # One key 2^gap above several thousand others has no value: the others are the result.
    length = 4000
    c = pool(-(-length // 64), 64, kv_heads, dim, fill=False)
    g = gen(dim + most)
    near = torch.randint(-3, 4, c.k_codes.shape[:3], device="cuda", generator=g).to(torch.int8)
    c.k_codes[..., 0] = near
    c.v_codes.copy_(torch.randint(32, 128, c.v_codes.shape, device="cuda", generator=g))
    at = 0 if first else length - most
    c.k_codes[at // 64, :, at % 64, 0] = 100
    c.v_codes[at // 64, :, at % 64] = 0
    c.k_scales.fill_(1.0)
    c.v_scales.fill_(2.0 ** -5)
    q = torch.zeros(most, heads, dim, device="cuda", dtype=TYPES[dtype])
    q[..., 0] = 1
    scale = float(np.float32(gap * math.log(2) / 100))
    want = softmax_rows(c, q, length, most, scale)
    got = c.attention(q, ints([0, most]), ints([length]), torch.arange(len(c.k_codes), dtype=torch.int32, device="cuda")[None], most,
                      scale=scale)
    c.check()
    # All terms are positive, so that the bound is relative to the output.  Scores of at most 27
    # powers of two round four times at 2^-24, the power itself and the other roundings of a
    # weight are under 2^-20, the sum rounds once for each 16 keys.
    bound = 0.7 * 27 * 4 * 2.0 ** -24 + 2.0 ** -20 + (length / 16 + 8) * 2.0 ** -23
    # 16-bit results take a weight as one fp16 number (half a step, and twice that for its own
    # rounding's place), f32 ones two.  In the kernel of many queries fp16's smallest step,
    # 2^-24, counts where the row's largest weight is 2^14 at least.
    bound += 2.0 ** -21 if dtype == "f32" else 2.0 ** -11
    if many:
        bound += 2.0 ** -25 / 2.0 ** (14 - gap * 1.03)
    err = (got.double() - want).abs()
    assert (err <= (bound + HALF[q.dtype]) * want).all(), (err / want).max().item()
