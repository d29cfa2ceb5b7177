"""The serving operators at the ends of their types' ranges, against plain 64-bit forms."""
import math

import numpy as np
import pytest
import torch

import serving_cases as ref
from emufpga_b200 import kv8, sampling
from emufpga_b200._lib import SpmError
from test_gpu_serving import HALF, TICKS, TYPES, Serving, check_append, check_sample, gen, ints, pool

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- plan --
@pytest.mark.parametrize("R", [3, 700])
@pytest.mark.parametrize("cached,new", [(16, 0), (1, 1), (20, 30)])
def test_plan_refuses_a_row_that_gives_back_what_it_keeps(R, cached, new):
    cached, new, ended = np.where(np.arange(R) == R - 1, cached, 0), np.where(np.arange(R) == R - 1, new, 1), np.zeros(R, int)
    ended[R - 1] = 1
    table = np.full((R, 4), -1)
    table[R - 1, :2] = 0, 1
    free = np.concatenate([np.arange(2, 2 * R), np.full(2, -1)])
    t, f, c, status = ints(table), ints(free), ints([2 * R - 2]), ints([0])
    got = kv8.plan(ints(cached), ints(new), t, f, c, 16, 800, ended=ints(ended), status=status)
    assert status.item() == 18
    with pytest.raises(SpmError):
        kv8.check(status)
    assert not got.starts.any() and not got.lens.any() and (got.slots == -1).all() and (got.positions == -1).all()
    assert t.tolist() == table.tolist() and f.tolist() == free.tolist() and c.item() == 2 * R - 2
    cached[R - 1] = 0  # the same without tokens kept
    kv8.plan(ints(cached), ints(new), t, f, c, 16, 800, ended=ints(ended), status=status)
    kv8.check(status)


# -------------------------------------------------------------- attention --
def softmax_rows(c, q, length, most, scale, sizes=False):
    """out of the last `most` of `length` positions in 64 bits, pages 0, 1, ... in order; with `sizes`
    the sums of |weight * value| and the largest weight * 127 scales (a page's largest value at most) too."""
    n = -(-length // c.page_tokens)
    k, v = ((codes[:n].double() * scales[:n].double()[..., None, None]).transpose(1, 2).reshape(-1, c.kv_heads, c.head_dim)[:length]
            for codes, scales in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)))
    group = q.shape[1] // c.kv_heads
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    x = torch.einsum("ihd,jhd->hij", q.double(), k) * scale
    hidden = torch.arange(length, device="cuda") > torch.arange(length - most, length, device="cuda")[:, None]
    w = torch.softmax(x.masked_fill(hidden, -math.inf), 2)
    out = torch.einsum("hij,jhd->ihd", w, v)
    if not sizes:
        return out
    most_of = (c.v_scales[:n].double() * 127).repeat_interleave(c.page_tokens, 0)[:length].repeat_interleave(group, 1)
    return out, torch.einsum("hij,jhd->ihd", w, v.abs()), (w * most_of.t()[:, None]).amax(2).t()[:, :, None]


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


def weight_error(q, c, length, scale):
    """How far a weight may be off, relative: its score's sums and products, its power, the sum over keys (serving_cases.attention)."""
    k = (c.k_codes.double() * c.k_scales.double()[..., None, None]).abs().amax((0, 2))
    bits = (q.double().abs() * k.repeat_interleave(q.shape[1] // c.kv_heads, 0)).sum(2).max().item() * abs(scale) * 1.4427
    return 2 * (0.6932 * bits * 2.0 ** -23 * (c.head_dim / 8 + 4) + 2.0 ** -20 + (length / 16 + 8) * 2.0 ** -23)


def table_of(c):
    return torch.arange(c.pages, dtype=torch.int32, device="cuda")[None]


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("most,heads,kv_heads", [(1, 4, 2), (1, 32, 2), (3, 8, 2), (64, 40, 40), (130, 48, 24)])
def test_f16_attention_is_off_by_its_own_rounding(dim, most, heads, kv_heads):
    length = 300
    c = pool(-(-length // 32), 32, kv_heads, dim, seed=dim)
    q = torch.randn(most, heads, dim, device="cuda", generator=gen(most)).half()
    scale = float(np.float32(dim ** -0.5))
    want, size, _ = softmax_rows(c, q, length, most, scale, sizes=True)
    got = c.attention(q, ints([0, most]), ints([length]), table_of(c), most, scale=scale)
    c.check()
    # two parts of a weight: 2^-22 of it; then half a step of the result
    bound = (weight_error(q, c, length, scale) + 2.0 ** -21) * size + HALF[q.dtype] * want.abs() + 2.0 ** -25
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max().item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most,kv_heads", [(1, 2), (30, 2), (30, 40)])  # the last: the kernel of many queries
@pytest.mark.parametrize("lo,hi", [(-60, 60), (-30, 8), (-24, -10)])
def test_attention_where_pages_differ_widely_in_every_type(dtype, most, kv_heads, lo, hi):
    c = pool(13, 16, kv_heads, 128)
    g = gen(7 + hi)
    c.v_scales.copy_(2.0 ** torch.randint(lo, hi + 1, c.v_scales.shape, device="cuda", generator=g))
    c.k_codes[4], c.v_codes[4], c.k_scales[4], c.v_scales[4] = 0, 0, 0, 0
    q = torch.randn(most, 2 * kv_heads, 128, device="cuda", generator=g).to(TYPES[dtype])
    for length in (200, 16, 17):  # (the second: every other page is masked)
        n = min(most, length)
        scale = float(np.float32(0.02))
        want, size, large = softmax_rows(c, q[:n], length, n, scale, sizes=True)
        got = c.attention(q[:n], ints([0, n]), ints([length]), table_of(c), n, scale=scale).double()
        c.check()
        # a weight's parts; and fp16's smallest step where the largest weighted scale's is 2^14 at least
        bound = (weight_error(q, c, length, scale) + (2.0 ** -11 if dtype == "bf16" else 2.0 ** -21)) * size
        bound = bound + length * 2.0 ** -39 * large + HALF[q.dtype] * want.abs() + (2.0 ** -25 if dtype == "f16" else 0)
        top = torch.finfo(q.dtype).max * (1 + HALF[q.dtype] / 2)
        over, under = want.abs() - bound >= top, want.abs() + bound < top
        assert got[over].isinf().all() and (got[over].sign() == want[over].sign()).all()
        assert ((got - want).abs() <= bound)[under].all(), ((got - want).abs() / bound)[under].max().item()
        assert (over | under).any()  # (f16: pages of 2^60 take every output past its range)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("most", [1, 3])
@pytest.mark.parametrize("large", [1.25, 1.99, 1.996])
def test_attention_queries_are_fixed_point_of_23_bits(dim, most, large):
    # A large element meets a key dimension of zeros: the others' bits are what is left of 23, or of 22
    # where the three digits do not hold the largest one's.  Two keys of values 127 and -127.
    rows = 256 * most
    c = pool(1, 16, 1, dim, fill=False)
    c.k_codes.copy_(torch.randint(-100, 101, c.k_codes.shape, device="cuda", generator=gen(dim)))
    c.k_codes[..., 0] = 0
    c.k_scales.fill_(1.0)
    c.v_codes[0, 0, 0], c.v_codes[0, 0, 1:most + 1], c.v_codes[0, 0, most + 1:] = 127, -127, 50
    c.k_codes[0, 0, 2:most + 1] = c.k_codes[0, 0, 1]
    c.v_scales.fill_(2.0 ** -7)
    q = torch.randn(rows, 2, dim, device="cuda", generator=gen(most))
    q[..., 0] = large * 1024
    scale = float(np.float32(1 / (60 * dim ** 0.5)))
    starts, lens = ints(range(0, rows + 1, most)), ints([most + 1] * 256)
    got = c.attention(q, starts, lens, ints([[0]] * 256), most, scale=scale)[::most].double()
    c.check()
    # the first row of each request sees two keys
    k = c.k_codes[0, 0, :2].double()
    p = torch.sigmoid(q[::most].double() @ (k[0] - k[1]) * scale)
    unit = 2.0 ** (10 - 22 + (large > 1.992))
    # d out / d score is 127 / 64 p (1 - p); an element is off by unit / sqrt(12) in the mean square
    want_rms = (scale * unit / 12 ** 0.5 * (k[0] - k[1]).square().sum().sqrt() * 127 / 64 * p * (1 - p)).square().mean().sqrt()
    off = (got - (127 / 128 * (2 * p - 1))[..., None]).square().mean().sqrt()
    assert off <= 1.2 * want_rms + 2.0 ** -22, (off / want_rms).item()


@pytest.mark.parametrize("dim,requests,most,heads,kv_heads", [
    (64, 64, 1, 8, 2), (128, 64, 1, 8, 2), (128, 32, 2, 16, 2), (192, 32, 1, 4, 2), (256, 32, 2, 8, 2)])
def test_attention_over_many_keys_has_no_bias(dim, requests, most, heads, kv_heads):
    # Values of one sign, each CTA with thousands of keys: a sum that truncates loses 2^-24 of itself
    # at every product.  What is rounded to nearest has no bias; a step's own products (four of 16 keys
    # each at most) truncate by 2^-24 each on average, the powers of two are within 2^-22.
    length = 16384
    c = pool(length // 64, 64, kv_heads, dim, seed=dim)
    c.v_codes.copy_(c.v_codes.abs().clamp(min=1))
    c.k_scales.fill_(2.0 ** -7)
    q = torch.randn(requests * most, heads, dim, device="cuda", generator=gen(dim))
    scale = float(np.float32(0.08))
    got = c.attention(q, ints([most * i for i in range(requests + 1)]), ints([length] * requests),
                      table_of(c).repeat(requests, 1), most, scale=scale)
    c.check()
    want = softmax_rows(c, q[:most], length, most, scale)
    assert abs(((got[:most] - want) / want).mean().item()) <= 4 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -22


@pytest.mark.parametrize("dtype,length,bound", [
    # f32: a tile's products truncate, eight of 16 keys each (the low parts' are too small to count) by
    # 2^-24 on average; the powers of two are within 2^-22
    ("f32", 4096, 2.0 ** -21 + 2.0 ** -22), ("f32", 16384, 2.0 ** -21 + 2.0 ** -22),
    # 16 bits: an eighth of their rounding where one accumulator is kept, else the mean of so many roundings
    ("f16", 8192, 2.0 ** -14), ("f16", 16384, 2.0 ** -16), ("f16", 65536, 2.0 ** -16),
    ("bf16", 16384, 2.0 ** -11), ("bf16", 163840, 2.0 ** -12)])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
def test_prompt_attention_over_many_keys_has_no_bias(dtype, length, bound, dim):
    # values of one sign, of a size of its own in each dimension
    most, heads, kv_heads, last = 600, 16, 4, 24
    c = pool(length // 64, 64, kv_heads, dim, seed=dim)
    size = torch.rand(kv_heads, 1, dim, device="cuda", generator=gen(3)) * 0.8 + 0.2
    c.v_codes.copy_((c.v_codes.abs().clamp(min=1) * size).ceil())
    c.k_scales.fill_(2.0 ** -7)
    c.v_scales.fill_(2.0 ** -5)
    q = torch.randn(most, heads, dim, device="cuda", generator=gen(dim)).to(TYPES[dtype])
    scale = float(np.float32(0.08))
    got = c.attention(q, ints([0, most]), ints([length]), table_of(c), most, scale=scale)[-last:]
    c.check()
    want = softmax_rows(c, q[-last:], length, last, scale)
    off = ((got.double() - want) / want)
    assert abs(off.mean().item()) <= bound and off.abs().max().item() <= HALF[q.dtype] * 1.25 + 2.0 ** -18


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("news,lens,width", [([1, 1, 1], [900, 3, 0], 64), ([700, 33, 300], [3000, 40, 300], 64), ([700], [900], 8300)])
def test_attention_in_place(dtype, dim, news, lens, width):
    # the queries' memory receives the result, whatever shares a row's keys or dimensions out; the last: a long table
    c = pool(60, 64, 4, dim, seed=dim)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    for r, n in enumerate(lens):
        table[r, :-(-n // 64)] = torch.arange(-(-n // 64), device="cuda") + r
    starts, ln = ints(np.concatenate([[0], np.cumsum(news)])), ints(lens)
    q = torch.randn(sum(news) + 2, 16, dim, device="cuda", generator=gen(dim)).to(TYPES[dtype])
    want = c.attention(q, starts, ln, table, max(news))
    for _ in range(20):
        same = q.clone()
        assert c.attention(same, starts, ln, table, max(news), out=same) is same
        assert torch.equal(same[:-2], want[:-2]) and torch.equal(same[-2:], q[-2:])
    c.check()


# ----------------------------------------------------------------- append --
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("old,new", [(-126, 22), (-126, 23), (-126, 24), (-126, 31), (-126, 120), (-80, 100), (-40, 110), (-30, 119)])
def test_append_where_the_scale_grows_by_more_than_a_float_holds(dtype, old, new):
    # rows stored at 2^old under a row at 2^new: from 2^150 on the ratio is none of f32's
    c = pool(2, 16, 2, 64, fill=False)
    x = torch.randn(2, 5, 2, 64, device="cuda", generator=gen(1)).clamp(-3, 3)
    x[:, :4] *= 2.0 ** (old + 5)
    x[:, 4] *= 2.0 ** (new + 5)
    x = x.to(TYPES[dtype])
    check_append(c, x[0, :4], x[1, :4], [16, 17, 18, 19])
    check_append(c, x[0, 4:], x[1, 4:], [20])
    assert not c.k_codes[1, :, :4].any() and c.k_codes[1, :, 4].any()


# --------------------------------------------------------------- sampling --
@pytest.mark.parametrize("vocab,every", [(5000, 3), (40000, 20), (70000, 40), (151936, 100)])
def test_sample_of_many_ties_over_all_slices(vocab, every):
    # 1500 and more equal tokens on the border of top-p, some in every CTA's slice
    n = 16
    x = torch.randn(n, vocab, device="cuda", generator=gen(9)) - 40
    x[:, ::every] = 3.0
    rng = np.random.default_rng(vocab)
    p, u = rng.uniform(0.05, 0.99, n), rng.random(n)
    first = check_sample(x, np.ones(n), [0] * n, p, [0.0] * n, u)
    f = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    pp, uu = f(p), f(u)
    for _ in range(100):
        again = sampling.sample(x, uu, top_p=pp)
        assert torch.equal(again.token, first.token) and torch.equal(again.kept, first.kept) and torch.equal(again.prob, first.prob)


# ---------------------------------------------------------------- streams --
def test_check_sees_calls_on_every_stream():
    c = pool(4, 16, 2, 64)
    x, bad, none, much = torch.zeros(1, 2, 64, device="cuda"), ints([77]), ints([0]), ints([17])
    pages = kv8.Pages(1, 1, 1, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)
            c.append(x, x, bad)
            pages.plan(none, much, 17)
        with pytest.raises(SpmError):
            c.check()
        with pytest.raises(SpmError):
            pages.check()
        c.check()
        pages.check()


# -------------------------------------------------------------- gradients --
def test_tensors_that_require_a_gradient_are_refused():
    c = pool(4, 16, 2, 64)
    x = torch.randn(2, 2, 64, device="cuda", generator=gen(2))
    starts, lens, table, u = ints([0, 1, 2]), ints([16, 5]), ints([[0], [1]]), torch.full((2,), 0.5, device="cuda")
    calls = {"q": lambda t: c.attention(t, starts, lens, table, 1), "out": lambda t: c.attention(x, starts, lens, table, 1, out=t),
             "k": lambda t: c.append(t, x, ints([0, 1])), "v": lambda t: c.append(x, t, ints([0, 1])),
             "logits": lambda t: sampling.sample(t.flatten(1), u).token}
    for f in calls.values():
        leaf = x.clone().requires_grad_()
        with pytest.raises(SpmError, match="gradient"):
            f(leaf * 1.0)
        with pytest.raises(SpmError, match="gradient"):
            f(leaf)
        with torch.no_grad():
            got = f(leaf)
        want = f(x.clone())
        assert want is None or torch.equal(got, want)


# --------------------------------------------------------------- together --
def test_ticks_attend_to_exactly_what_the_cache_holds():
    # every tick's slots, stored values, attention and picks against 64-bit forms over the cache's own values
    s = Serving()
    held = {}  # slot -> row of k, v
    for new, ended in TICKS:
        s.new.copy_(ints(new))
        s.ended.copy_(ints(ended))
        s.cached.masked_fill_(s.ended > 0, 0)
        slots, out, token = s.tick()
        s.pages.check()
        s.cache.check()
        starts, lens = np.concatenate([[0], np.cumsum(new)]).tolist(), s.cached.tolist()
        held.update({slot: i for i, slot in enumerate(slots.tolist()) if slot >= 0})
        for (codes, scales), rows in zip(((s.cache.k_codes, s.cache.k_scales), (s.cache.v_codes, s.cache.v_scales)), (s.k, s.v)):
            for r, n in enumerate(lens):
                for p in range(n):
                    slot = s.pages.table[r, p // 16].item() * 16 + p % 16
                    got = codes[slot // 16, :, slot % 16].double() * scales[slot // 16].double()[:, None]
                    # a value and its page's later growths: under one step of the scale
                    assert ((got - rows[held[slot]].double()).abs() <= scales[slot // 16].double()[:, None]).all()
        c = s.cache
        want, tol = ref.attention(s.q, starts, lens, s.pages.table, (c.k_codes, c.v_codes), (c.k_scales, c.v_scales), 0.125)
        assert ((out.double() - want).abs() <= tol).all() and not out[starts[-1]:].any()
        last = out[(ints(starts[1:]).long() - 1).clamp(min=0)].flatten(1)
        logits = (last @ s.head.t()).double().cpu().numpy()
        for r in range(4):
            assert token[r].item() == ref.pick(logits[r], 1.0, 7, float(np.float32(0.9)), 0.0, s.u[r].item())[0]
