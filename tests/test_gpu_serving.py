"""The serving operators on the device against plain 64-bit forms: page plan,
8-bit paged cache, attention over it, sampling, and a run of them together."""
import math

import numpy as np
import pytest
import torch

import serving_cases as ref
from emufpga_b200 import kv8, sampling
from emufpga_b200._lib import SpmError

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a step of a rounding to the type
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES.values()}


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------- plan --
def plan_case(rng, R, P, longest, prompt, readmit=False):
    cached = rng.integers(0, longest + 1, R)
    new = rng.integers(0, prompt + 1, R)
    ended = np.zeros(R, dtype=np.int64)
    gone = rng.random(R) < 0.3
    ended[gone] = cached[gone]
    cached[gone] = 0
    if not readmit:
        new[gone] = 0
    held = -(-(cached + ended) // P)
    width = max(1, int(np.max(-(-(np.maximum(cached + new, ended)) // P))))
    pages = int(held.sum()) + int((-(-(cached + new) // P)).sum()) + 3
    ids = rng.permutation(pages)
    table = np.full((R, width), -1)
    table[np.arange(width) < held[:, None]] = ids[:held.sum()]
    free = np.full(pages, -1)
    free[:pages - held.sum()] = ids[held.sum():]
    return cached, new, ended, table, free, pages - int(held.sum())


@pytest.mark.parametrize("R,P,longest,prompt,readmit", [
    (1, 16, 0, 1, False), (1, 256, 1000, 1, False), (3, 16, 40, 20, True), (64, 64, 500, 3, True), (65, 32, 100, 1, False),
    (513, 16, 64, 40, True), (8192, 16, 30, 2, True), (7, 128, 3000, 2000, False)])
@pytest.mark.parametrize("seed", range(2))
def test_plan(R, P, longest, prompt, readmit, seed):
    rng = np.random.default_rng(seed)
    cached, new, ended, table, free, count = plan_case(rng, R, P, longest, prompt, readmit)
    tokens = int(new.sum()) + seed * 37
    want_table, want_free = table.tolist(), free.tolist()
    starts, lens, positions, slots, left = ref.plan(cached.tolist(), new.tolist(), ended.tolist(), want_table, want_free,
                                                    count, P, tokens)
    t, f, c, status = ints(table), ints(free), ints([count]), ints([0])
    got = kv8.plan(ints(cached), ints(new), t, f, c, P, tokens, ended=ints(ended), status=status)
    kv8.check(status)
    assert got.starts.tolist() == starts and got.lens.tolist() == lens
    assert got.positions.tolist() == positions and got.slots.tolist() == slots
    assert t.tolist() == want_table and f.tolist() == want_free and c.item() == left


def test_plan_without_requests_or_tokens():
    e = ints([])
    got = kv8.plan(e, e, torch.empty((0, 4), dtype=torch.int32, device="cuda"), ints([0, 1]), ints([2]), 16, 3)
    assert got.starts.tolist() == [0] and got.slots.tolist() == [-1] * 3
    got = kv8.plan(ints([5]), ints([0]), ints([[1]]), ints([0, -1]), ints([1]), 16, 0)
    assert got.lens.tolist() == [5] and got.slots.numel() == 0


@pytest.mark.parametrize("what,code", [("negative", 11), ("long", 11), ("free", 12), ("tokens", 13), ("stack", 14), ("count", 14)])
@pytest.mark.parametrize("R", [3, 700])
def test_plan_that_fails_moves_nothing(what, code, R):
    cached, new, ended = np.full(R, 16), np.ones(R, int), np.zeros(R, int)
    table = np.full((R, 3), -1)
    table[:, 0] = np.arange(R)
    free = np.concatenate([np.arange(R, 2 * R), np.full(2, -1)])
    count, tokens = R, R
    if what == "negative":
        new[1] = -1
    elif what == "long":
        cached[2] = 48
    elif what == "free":
        count = R - 1
    elif what == "tokens":
        tokens = R - 1
    elif what == "stack":
        ended[:] = 48
    else:
        count = -1
    t, f, c, status = ints(table), ints(free), ints([count]), ints([0])
    got = kv8.plan(ints(cached), ints(new), t, f, c, 16, tokens, ended=ints(ended), status=status)
    assert status.item() == code
    with pytest.raises(SpmError):
        kv8.check(status)
    assert status.item() == 0
    assert not got.starts.any() and not got.lens.any() and (got.slots == -1).all() and (got.positions == -1).all()
    assert t.tolist() == table.tolist() and f.tolist() == free.tolist() and c.item() == count


def test_plan_marks_a_page_that_is_not_in_the_pool():
    status = ints([0])
    got = kv8.plan(ints([3]), ints([2]), ints([[9]]), ints([0]), ints([0]), 16, 2, status=status)
    assert got.slots.tolist() == [-1, -1] and got.positions.tolist() == [3, 4] and status.item() == 15


# ----------------------------------------------------------------- append --
def pool(pages, page, heads, dim, seed=0, fill=True):
    c = kv8.Cache(pages, page, heads, dim)
    if fill:
        g = gen(seed)
        for codes, scales in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)):
            codes.copy_(torch.randint(-127, 128, codes.shape, device="cuda", generator=g))
            scales.copy_(2.0 ** torch.randint(-9, -3, scales.shape, device="cuda", generator=g))
    return c


def as_numpy(c):
    return [(c.k_codes.double().cpu().numpy(), c.k_scales.double().cpu().numpy()),
            (c.v_codes.double().cpu().numpy(), c.v_scales.double().cpu().numpy())]


def check_append(c, k, v, slots):
    want = as_numpy(c)
    for (codes, scales), x in zip(want, (k, v)):
        ref.store(x.double().cpu().numpy(), slots, codes, scales)
    c.append(k, v, ints(slots))
    got = as_numpy(c)
    for (wc, ws), (gc, gs) in zip(want, got):
        np.testing.assert_array_equal(gs, ws)
        np.testing.assert_array_equal(gc, wc)


def slots_for(rng, page, runs, pages):
    """Runs (offset, count) on consecutive pages of a random permutation."""
    ids, out = list(rng.permutation(pages)), []
    for off, n in runs:
        pos = off
        page_id = ids.pop()
        for _ in range(n):
            if pos == page:
                page_id, pos = ids.pop(), 0
            out.append(page_id * page + pos)
            pos += 1
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_append(dtype, dim, page):
    rng = np.random.default_rng(dim + page)
    runs = [(0, 1), (page - 1, 1), (3, 2 * page), (0, page), (page - 2, 5), (5, 70)]
    slots = slots_for(rng, page, runs, 40)
    c = pool(40, page, 3, dim)
    x = torch.randn(2, len(slots), 3, dim, device="cuda", generator=gen(dim)) * 4.0
    x = x.to(TYPES[dtype])
    check_append(c, x[0], x[1], slots)
    c.check()


@pytest.mark.parametrize("page,tokens,heads", [(16, 1, 1), (32, 64, 1), (64, 65, 2), (128, 1000, 8), (256, 2049, 8), (16, 1500, 8)])
def test_append_window_edges(page, tokens, heads):
    rng = np.random.default_rng(tokens)
    slots = slots_for(rng, page, [(page // 2 + 1, tokens)], tokens // page + 3)
    c = pool(tokens // page + 3, page, heads, 64)
    x = torch.randn(2, tokens, heads, 64, device="cuda", generator=gen(1))
    check_append(c, x[0], x[1], slots)


def test_append_strided_and_unaligned():
    rng = np.random.default_rng(0)
    slots = slots_for(rng, 16, [(0, 40)], 5)
    for off, dtype in ((0, torch.bfloat16), (1, torch.bfloat16), (3, torch.float32)):
        flat = torch.randn(40 * 700 + 8, device="cuda", generator=gen(2)).to(dtype)
        # a fused projection's rows, heads apart, and a base off every vector's alignment
        k = flat[off:].as_strided((40, 2, 64), (700, 129, 1))
        v = flat[off:].as_strided((40, 2, 64), (700, 64, 1), 320 + off)
        check_append(pool(5, 16, 2, 64), k, v, slots)


def test_append_values_that_are_special():
    c = pool(8, 16, 1, 64)
    x = torch.zeros(12, 1, 64, device="cuda")
    x[1, 0, 5] = math.inf
    x[2, 0, 7] = math.nan
    x[4] = 2.0 ** -140                      # under the smallest scale's half step
    x[5, 0, 0] = 3.0e38
    x[6, 0, 0], x[6, 0, 1] = 127.0, -127.0
    x[7, 0, 0] = math.nextafter(127.0, 128.0) + 1e-5
    x[8, 0, 0] = -0.0
    x[9] = 0.5                               # ties of rows that are rounded again
    v = torch.randn(12, 1, 64, device="cuda", generator=gen(3))
    # pages 0..6 new with zeros, inf, NaN, zeros, tiny, huge, 127; then into pages that hold rows
    slots = [0, 16, 32, 48, 64, 80, 96, 112 + 3, 112 + 4, 112 + 5, -1, -1]
    check_append(c, x, v, slots)
    assert c.k_scales[0, 0] == 0 and c.k_scales[6, 0] == 1 and torch.isnan(c.k_scales[1:3, 0]).all()
    check_append(c, v, x, [1, 17, 33, 49, 65, 81, 97, 112 + 6, 112 + 7, 112 + 8, -1, -1])  # NaN stays, zeros are raised
    c.check()


def test_append_marks_slots_out_of_the_pool_and_stores_the_others():
    c = pool(4, 16, 2, 64)
    x = torch.randn(4, 2, 64, device="cuda", generator=gen(4))
    want = as_numpy(c)
    ref.store(x.double().cpu().numpy()[1:3], [0, 16], *want[0])
    c.append(x, x, ints([64, 0, 16, -7]))
    np.testing.assert_array_equal(as_numpy(c)[0][0], want[0][0])
    assert c.status.item() == 15
    with pytest.raises(SpmError):
        c.check()


def test_append_token_by_token_equals_the_plain_form():
    c = pool(2, 32, 2, 128, fill=False)
    x = torch.randn(32, 2, 128, device="cuda", generator=gen(5)) * torch.exp2(torch.arange(32, device="cuda") / 4)[:, None, None]
    want = as_numpy(c)
    for t in range(32):
        for codes, scales in want:
            ref.store(x[t:t + 1].double().cpu().numpy(), [32 + t], codes, scales)
        c.append(x[t:t + 1], x[t:t + 1], ints([32 + t]))
    for (wc, ws), (gc, gs) in zip(want, as_numpy(c)):
        np.testing.assert_array_equal(gc, wc)
        np.testing.assert_array_equal(gs, ws)
    # a step of the last scale at most (see the plain form's test)
    assert ((c.values()[0][1].transpose(0, 1) - x).abs() <= c.k_scales[1][:, None]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_values_of_chosen_pages(dtype):
    c = pool(9, 64, 3, 96)
    ids = ints([8, 0, 8, 11, 3])
    k, v = c.values(ids, dtype=TYPES[dtype])
    for got, codes, scales in ((k, c.k_codes, c.k_scales), (v, c.v_codes, c.v_scales)):
        want = codes.double() * scales.double()[:, :, None, None]
        for i, p in enumerate([8, 0, 8, None, 3]):
            assert torch.equal(got[i].double(), want[p] if p is not None else torch.zeros_like(want[0]))
    assert c.status.item() == 15


# -------------------------------------------------------------- attention --
def tables(rng, lens, page, spare=1):
    need = [-(-n // page) for n in lens]
    width = max(1, max(need)) + spare
    ids = rng.permutation(sum(need) + 1)
    table, at = np.full((len(lens), width), -1), 0
    for r, n in enumerate(need):
        table[r, :n] = ids[at:at + n]
        at += n
    return ints(table), sum(need) + 1


def check_attention(c, q, starts, lens, table, most, scale=None, out=None):
    want, tol = ref.attention(q, starts, lens, table, (c.k_codes, c.v_codes), (c.k_scales, c.v_scales),
                              q.shape[2] ** -0.5 if scale is None else scale)
    got = c.attention(q, ints(starts), ints(lens), table, most, scale=scale, out=out)
    c.check()
    n = starts[-1]
    if q.dtype != torch.float32:
        # weights in one fp16 part: half a step each, and the result's rounding
        big = max(c.v_codes.double().abs().max().item() * c.v_scales[~c.v_scales.isnan()].max().item(), 0)
        tol = tol + 2.0 ** -11 * big + HALF[q.dtype] * want.abs()
    err = (got[:n].double() - want[:n]).abs()
    assert torch.equal(got[:n].isnan(), want[:n].isnan())
    assert (err.nan_to_num(0.0) <= tol[:n]).all(), (err - tol[:n]).max().item()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (9, 3), (14, 2), (16, 1), (40, 2), (6, 6)])
def test_attention_of_one_token_each(dtype, dim, heads, kv_heads):
    rng = np.random.default_rng(dim)
    lens = [1, 0, 33, 700, 16, 129, 31]
    table, pages = tables(rng, lens, 32)
    c = pool(pages, 32, kv_heads, dim, seed=dim)
    q = torch.randn(len(lens), heads, dim, device="cuda", generator=gen(dim)).to(TYPES[dtype])
    got = check_attention(c, q, list(range(len(lens) + 1)), lens, table, 1)
    assert not got[1].any()  # no key: zero


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,dim,news,lens", [
    (4, 4, 64, [1, 2, 0, 5], [1, 200, 60, 5]),
    (8, 1, 128, [3, 1], [400, 3]),
    (12, 4, 128, [40, 1, 0, 17], [300, 129, 5, 17]),
    (32, 4, 128, [130], [1000]),
    (32, 8, 64, [257, 64], [257, 2100]),
    (10, 2, 256, [33, 20], [77, 20]),
    (8, 2, 96, [100], [163]),
    (4, 1, 192, [65], [65])])
def test_attention_of_several_tokens(dtype, page, heads, kv_heads, dim, news, lens):
    rng = np.random.default_rng(page)
    table, pages = tables(rng, lens, page)
    c = pool(pages, page, kv_heads, dim, seed=page)
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    q = torch.randn(starts[-1] + 2, heads, dim, device="cuda", generator=gen(page)).to(TYPES[dtype])
    got = check_attention(c, q, starts, lens, table, max(news))
    assert not got[starts[-1]:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page,heads,kv_heads,news,lens", [
    (16, 32, 16, [200], [777]), (64, 36, 12, [129, 0, 77], [129, 40, 1100]), (256, 24, 24, [300], [300]),
    (32, 64, 4, [33, 40], [64, 1500]), (128, 32, 32, [1, 250, 3], [129, 380, 3])])
def test_attention_of_many_tokens(dtype, dim, page, heads, kv_heads, news, lens):
    rng = np.random.default_rng(page + dim)
    table, pages = tables(rng, lens, page)
    c = pool(pages, page, kv_heads, dim, seed=dim)
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    q = torch.randn(starts[-1], heads, dim, device="cuda", generator=gen(page)).to(TYPES[dtype])
    out = torch.full_like(q, 7.0)
    check_attention(c, q, starts, lens, table, max(news), out=out)
    check_attention(c, q, starts, lens, table, max(news), scale=-0.05)


def test_attention_with_more_queries_than_keys_leaves_the_first_empty():
    table, pages = tables(np.random.default_rng(0), [3, 40], 16)
    c = pool(pages, 16, 2, 64)
    q = torch.randn(50, 4, 64, device="cuda", generator=gen(6))
    got = check_attention(c, q, [0, 8, 50], [3, 40], table, 42)
    assert not got[:5].any() and got[5:8].any() and not got[8:10].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most,kv_heads", [(1, 2), (30, 2), (30, 40)])  # the last: the kernel of many queries
def test_attention_where_pages_differ_widely(dtype, most, kv_heads):
    # scales from 2^-60 to 2^60, pages of zeros, and a page of NaN that no query sees
    table, pages = tables(np.random.default_rng(1), [300, 200], 16)
    c = pool(pages, 16, kv_heads, 128)
    heads = 2 * kv_heads
    g = gen(7)
    c.v_scales.copy_(2.0 ** torch.randint(-60, 61, c.v_scales.shape, device="cuda", generator=g))
    c.k_scales.copy_(2.0 ** torch.randint(-9, -3, c.k_scales.shape, device="cuda", generator=g))
    for row, n in ((0, 300), (1, 200)):
        p = table[row, 4].item()
        c.k_codes[p], c.v_codes[p], c.k_scales[p], c.v_scales[p] = 0, 0, 0, 0
    starts, lens = [0, most, 2 * most], [300, 200]
    q = torch.randn(2 * most, heads, 128, device="cuda", generator=g).to(TYPES[dtype])
    want, _ = ref.attention(q, starts, lens, table, (c.k_codes, c.v_codes), (c.k_scales, c.v_scales), 0.02)
    got = c.attention(q, ints(starts), ints(lens), table, most, scale=0.02)
    # outputs near 2^60 times a weight: an fp16 type overflows to infinity
    if dtype == "f16":
        want = want.to(torch.float16).double()
        assert torch.equal(got.isinf(), want.isinf()) or most
        return
    big = (c.v_codes.double().abs().amax((2, 3)) * c.v_scales).max()
    assert ((got.double() - want).abs() <= (2.0 ** -10 if dtype == "bf16" else 2.0 ** -17) * big).all()
    # a small page alone, with a huge one masked behind it, keeps its own precision
    c.v_scales[table[0, 0]] = 2.0 ** -60
    c.v_scales[table[0, 1]] = 2.0 ** 60
    one = torch.randn(1, heads, 128, device="cuda", generator=g).to(TYPES[dtype])
    check_attention(c, one, [0, 1], [16], table[:1].contiguous(), 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most,kv_heads", [(1, 2), (40, 2), (40, 40)])
def test_attention_masks_what_is_not_finite(dtype, most, kv_heads):
    # the page behind the last token is NaN, and so are the codes' scales of pages no table names
    lens = [40, 64]
    table, pages = tables(np.random.default_rng(2), lens, 16, spare=2)
    c = pool(pages, 16, kv_heads, 64)
    unused = [p for p in range(pages) if p not in table.flatten().tolist()]
    c.k_scales[unused[0]] = c.v_scales[unused[0]] = math.nan
    table[0, 3] = unused[0]
    q = torch.randn(2 * most, 2 * kv_heads, 64, device="cuda", generator=gen(8)).to(TYPES[dtype])
    got = check_attention(c, q, [0, most, 2 * most], lens, table, most)
    assert not got.isnan().any()
    # and a NaN page that queries do see makes theirs NaN, and no earlier query's
    if most > 1:
        p = table[1, 3].item()
        c.k_scales[p, 0::2] = c.v_scales[p, 1::2] = math.nan
        got = c.attention(q, ints([0, most, 2 * most]), ints(lens), table, most)
        seen = torch.arange(24, 64) >= 48
        assert torch.equal(got[most:].isnan().all(2).all(1).cpu(), seen) and not got[:most].isnan().any()
        assert not got[most:][~seen].isnan().any()


def test_attention_strides_scale_and_rows_behind_the_last():
    lens = [100, 50]
    table, pages = tables(np.random.default_rng(3), lens, 64)
    c = pool(pages, 64, 2, 128)
    wide = torch.randn(9, 8 * 128 + 77, device="cuda", generator=gen(9))
    q = wide[:, 3:].as_strided((9, 8, 128), (wide.stride(0), 128, 1), 3)
    out = torch.full((8, 9, 128), 7.0, device="cuda").transpose(0, 1)
    got = check_attention(c, q, [0, 3, 7], lens, table, 4, scale=-0.3, out=out)
    assert got is out and (out[7:] == 7.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news,rows,most,kv_heads", [
    ([1, 1, 0, 1], 4, 1, 2), ([1, 0, 0, 1], 9, 1, 2), ([0, 0], 3, 1, 2), ([], 5, 1, 2), ([0], 5, 0, 2),
    ([30, 0, 20], 60, 30, 2), ([30, 0, 20], 60, 30, 40)])
@pytest.mark.parametrize("before", [0, 2])
def test_attention_rows_of_no_request(dtype, news, rows, most, kv_heads, before):
    lens = [40 + 30 * i for i in range(len(news))]
    table, pages = tables(np.random.default_rng(6), lens or [1], 16)
    table = table[:len(lens)]
    c = pool(pages, 16, kv_heads, 64)
    q = torch.randn(before + rows, 2 * kv_heads, 64, device="cuda", generator=gen(20)).to(TYPES[dtype])
    starts = np.concatenate([[before], before + np.cumsum(news, dtype=np.int64)]).tolist()
    rest = torch.ones(before + rows, dtype=torch.bool, device="cuda")
    rest[before:starts[-1]] = False
    torch.full((4,) + q.shape, math.nan, dtype=q.dtype, device="cuda")  # what fresh memory may hold
    got = check_attention(c, q, starts, lens, table, most)
    assert (got[rest] == 0).all()
    out = torch.full_like(q, 7.0)
    c.attention(q, ints(starts), ints(lens), table, most, out=out)
    assert (out[rest] == 7).all() and torch.equal(out[~rest], got[~rest])
    same = q.clone()
    assert c.attention(same, ints(starts), ints(lens), table, most, out=same) is same  # in place
    assert torch.equal(same[~rest], got[~rest]) and torch.equal(same[rest], q[rest])


def test_attention_of_more_requests_than_a_grid_is_deep():
    R, lens = 65600, [20, 33]
    table, pages = tables(np.random.default_rng(7), lens, 16)
    c = pool(pages, 16, 1, 64)
    q = torch.randn(40, 4, 64, device="cuda", generator=gen(21))
    wide = torch.full((R, table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[0], wide[-1] = table[0], table[1]
    starts, all_lens = np.full(R + 1, 20), np.zeros(R, dtype=np.int64)
    starts[0], starts[-1], all_lens[0], all_lens[-1] = 0, 40, 20, 33
    got = c.attention(q, ints(starts), ints(all_lens), wide, 20)
    c.check()
    want, tol = ref.attention(q, [0, 20, 40], lens, table, (c.k_codes, c.v_codes), (c.k_scales, c.v_scales), 0.125)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("most,kv_heads", [(1, 2), (64, 2), (64, 40)])
def test_attention_marks_lengths_pages_and_rows_that_are_wrong(most, kv_heads):
    lens = [100, 50]
    table, pages = tables(np.random.default_rng(4), lens, 16, spare=0)
    c = pool(pages, 16, kv_heads, 64)
    q = torch.randn(2 * most, 2 * kv_heads, 64, device="cuda", generator=gen(10))
    s = [0, most, 2 * most]

    def code(starts, lens, table):
        c.attention(q, ints(starts), ints(lens), table, most)
        got = c.status.item()
        with pytest.raises(SpmError):
            c.check()
        return got

    assert code(s, [10 ** 6, 50], table) == 11
    assert code(s, [-5, 50], table) == 11
    bad = table.clone()
    bad[0, 1] = pages
    assert code(s, lens, bad) == 15
    bad[0, 1] = -1
    assert code(s, lens, bad) == 15
    assert code([0, most, 2 * most + 1], lens, table) == 16
    assert code([0, 2 * most, most], lens, table) == 16
    assert code([-1, 0, most], lens, table) == 16
    check_attention(c, q, s, lens, table, most)  # and the next call is whole


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_over_a_cache_past_32_bits(dtype):
    # 2^32 codes of keys alone; the last pages hold the request
    page, heads, dim = 256, 16, 256
    pages = (1 << 32) // (page * heads * dim) + 4
    c = kv8.Cache(pages, page, heads, dim)
    table = ints([[pages - 1, 0, pages - 2, pages - 4]])
    g = gen(11)
    k, v = (torch.randn(700, heads, dim, device="cuda", generator=g).to(TYPES[dtype]) for _ in range(2))
    p = kv8.plan(ints([0]), ints([700]), table, ints([pages - 4, pages - 2, 0, pages - 1]), ints([4]), page, 700)
    assert table[0, :3].tolist() == [pages - 1, 0, pages - 2]
    c.append(k, v, p.slots)
    keep = table[0, :3].long()
    q = torch.randn(1, heads, dim, device="cuda", generator=g).to(TYPES[dtype])
    got = c.attention(q, ints([0, 1]), ints([700]), table, 1)
    small = kv8.Cache.over(*(t[keep].contiguous() for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)))
    want = small.attention(q, ints([0, 1]), ints([700]), ints([[0, 1, 2]]), 1)
    assert torch.equal(got, want) and got.any()
    x, _ = c.values(ints([pages - 1]))
    assert torch.equal(x[0], small.values()[0][0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most,dim", [(1, 128), (20, 128), (200, 64), (200, 128), (200, 256)])
def test_attention_repeats_bit_for_bit(dtype, most, dim):
    lens = [5000, 300, 1200, 4000]
    table, pages = tables(np.random.default_rng(5), lens, 64)
    c = pool(pages, 64, 2, dim)
    q = torch.randn(4 * most, 16, dim, device="cuda", generator=gen(12)).to(TYPES[dtype])
    s = ints([most * i for i in range(5)])
    first = c.attention(q, s, ints(lens), table, most)
    for _ in range(30):
        assert torch.equal(c.attention(q, s, ints(lens), table, most), first)


# ---------------------------------------------------------------- sampling --
def check_sample(logits, temperature, k, p, m, u):
    n = logits.shape[0]
    f = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
    t, kk, pp, mm, uu = f(temperature), ints(k), f(p), f(m), f(u)
    got = sampling.sample(logits, uu, temperature=t, top_k=kk, top_p=pp, min_p=mm)
    rows = logits.double().cpu().numpy()
    for i in range(n):
        want = ref.pick(rows[i], t[i].item(), int(k[i]), pp[i].item(), mm[i].item(), uu[i].item())
        assert (got.token[i].item(), got.kept[i].item()) == want[:2], (i, want)
        # weights of 2^-44 of the largest, a 64-bit exponential and one rounding to f32
        assert abs(got.prob[i].item() - want[2]) <= want[2] * (2.0 ** -24 + 2.0 ** -30) + 2.0 ** -40
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 2048, 2049, 5000, 49152, 151936])
def test_sample(dtype, vocab):
    rng = np.random.default_rng(vocab)
    n = 12
    x = (torch.randn(n, vocab, device="cuda", generator=gen(vocab)) * 3).to(TYPES[dtype])
    on = lambda: rng.random(n) < 0.6  # noqa: E731
    check_sample(x, rng.uniform(0.3, 2.0, n), np.where(on(), rng.integers(1, min(vocab, 300) + 1, n), 0),
                 np.where(on(), rng.uniform(0.0, 1.0, n), 1.0), np.where(on(), rng.uniform(0, 0.3, n), 0.0), rng.random(n))


@pytest.mark.parametrize("vocab", [100, 40000])
@pytest.mark.parametrize("kind", ["equal", "few", "steps"])
def test_sample_ties_go_to_the_lowest_index(kind, vocab):
    n = 10
    if kind == "equal":
        x = torch.full((n, vocab), -1.5, device="cuda")
    elif kind == "few":
        x = torch.randint(0, 3, (n, vocab), device="cuda", generator=gen(1)).float()
    else:
        x = (torch.arange(vocab, device="cuda") % 7).float().expand(n, vocab).contiguous()
    rng = np.random.default_rng(0)
    check_sample(x, np.full(n, 0.7), [0, 1, 5, vocab // 2, vocab - 1, vocab, 0, 0, 9, 0],
                 [1, 1, 1, 1, 1, 1, 0.25, 0.5, 0.5, 0.999], [0, 0, 0, 0, 0, 0, 0, 0, 0, 1.0], rng.random(n))


def test_sample_rows_that_are_special():
    inf, nan = math.inf, math.nan
    x = torch.zeros(12, 4000, device="cuda")
    x[0] = -inf                       # nothing to pick
    x[1] = nan
    x[2] = -inf
    x[2, 77] = -3e38                  # one token
    x[3] = torch.randn(4000, device="cuda", generator=gen(2))
    x[3, ::2] = nan
    x[4, 5] = x[4, 900] = inf         # infinities share the mass
    x[5] = torch.finfo(torch.float32).min
    x[6, 3] = 3e38
    x[7] = -0.0
    x[7, 1::2] = 0.0
    x[8] = torch.randn(4000, device="cuda", generator=gen(3)) * 1e-38
    x[9] = -inf
    x[9, 1000:1003] = torch.tensor([1.0, 2.0, 1.0], device="cuda")
    got = check_sample(x, [1, 1, 1, 1, 1, 1, 1, 0, 0.5, 1, 0, 1e-30],
                       [0, 3, 5, 0, 0, 0, 2, 0, 0, 100, 0, 3], [1, 0.5, 0.9, 0.9, 0.9, 1, 1, 1, 0.3, 1, 1, 1],
                       [0, 0, 0, 0.1, 0, 0, 0, 0, 0, 0, 0, 0], [0.5, 0.1, 0.9, 0.7, 0.6, 0.99, 0.5, 0.4, 0.2, 0.99, 0.9, 0.4])
    assert got.token[0] == -1 and got.token[1] == -1 and got.token[7] == 0 and got.token[10] == 0


@pytest.mark.parametrize("vocab", [2000, 5000, 70000])
@pytest.mark.parametrize("spread", [3.0, 1e-3])
def test_sample_of_long_lists(vocab, spread):
    # borders with 1000 to 2000 tokens before or beside them, in one CTA's slice or several
    n = 8
    x = torch.randn(n, vocab, device="cuda", generator=gen(22)) * spread
    x[:, 300:] -= torch.tensor([0.0, 0.0, 0.0, 0.0, 30.0, 30.0, 30.0, 30.0], device="cuda")[:, None]
    x[4:, 300:1700] += 30.0 - spread
    rng = np.random.default_rng(9)
    for k, p in [(0, 0.5), (0, 0.97), (1100, 1.0), (1500, 0.8), (1999, 0.99), (600, 0.999)]:
        check_sample(x, np.linspace(0.5, 1.5, n), [k] * n, [p] * n, np.where(np.arange(n) % 3 == 0, 0.01, 0.0), rng.random(n))


def test_sample_at_the_smallest_temperatures():
    # gaps a little and far over the temperature, normal and subnormal
    t = [2.0 ** -100, 2.0 ** -110, 2.0 ** -126, 2.0 ** -140, 2.0 ** -149, 2.0 ** -60]
    x = torch.zeros(6, 300, device="cuda")
    for i, v in enumerate(t):
        x[i, 10:40] = torch.arange(30, device="cuda").double().mul(v).float()
        x[i, 50] = 25 * v
        x[i, 60] = -2.0 ** -90
    rng = np.random.default_rng(8)
    for k, p in [(0, 1.0), (0, 0.9), (20, 0.9), (45, 1.0)]:
        check_sample(x, t, [k] * 6, [p] * 6, [0.0] * 6, rng.random(6))


def test_sample_settings_at_their_edges():
    n = 9
    x = torch.randn(1, 3001, device="cuda", generator=gen(4)).repeat(n, 1)
    check_sample(x, np.ones(n), [0] * n, [1.0, 0.0, 1.5, 0.9, 1.0, 1.0, 1e-30, 1.0, 1.0], [0, 0, 0, 0, 0, -1.0, 0, 1.0, 0.5],
                 [0.0, 0.5, np.nextafter(np.float32(1), np.float32(0)), 0.0, 0.9999, 0.3, 0.7, 0.99, 0.0])
    # numbers out of [0, 1) take the first or the last kept token; NaN settings are off
    u = torch.tensor([-1.0, 1.0, 2.0, math.nan], device="cuda")
    got = sampling.sample(x[:4], u, top_k=ints([5] * 4))
    kept = torch.sort(x[0], descending=True)[1][:5].sort()[0].tolist()
    assert got.token.tolist() == [kept[0], kept[-1], kept[-1], kept[0]]
    off = torch.full((4,), math.nan, device="cuda")
    v = torch.tensor([0.2, 0.4, 0.6, 0.8], device="cuda")
    plain = sampling.sample(x[:4], v)
    with_nan = sampling.sample(x[:4], v, top_p=off, min_p=off)
    assert torch.equal(plain.token, with_nan.token) and torch.equal(plain.kept, with_nan.kept)


def test_sample_of_the_largest_vocabulary_and_strided_rows():
    wide = torch.randn(3, (1 << 19) + 5, device="cuda", generator=gen(5))
    x = wide[:, 3:3 + (1 << 19)]
    check_sample(x, [1.0, 0.8, 1.0], [0, 50, 0], [1.0, 0.9, 0.95], [0, 0, 0.01], [0.3, 0.6, 0.9])
    flat = torch.zeros(2, 1 << 19, device="cuda")  # the largest total mass
    got = check_sample(flat, [1.0, 1.0], [0, 0], [1.0, 0.5], [0, 0], [0.75, 0.75])
    assert got.token.tolist() == [(1 << 19) * 3 // 4, (1 << 18) * 3 // 4]


def test_sample_frequencies_follow_the_weights():
    logits = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5], device="cuda").repeat(4000, 1)
    u = (torch.arange(4000, device="cuda") + 0.5) / 4000
    got = sampling.sample(logits, u, top_k=ints([4] * 4000))
    w = torch.softmax(torch.tensor([0.0, 1.0, 2.0, -math.inf, 0.5], dtype=torch.float64), 0)
    # evenly spaced numbers: every count is within one of its share
    counts = torch.bincount(got.token, minlength=5).cpu()
    assert ((counts - 4000 * w).abs() <= 1).all()


# ---------------------------------------------------------------- together --
def test_refusals_of_the_python_calls():
    c = kv8.Cache(4, 16, 2, 64)
    x = torch.zeros(3, 2, 64, device="cuda")
    s = ints([0, 1, 2])
    for bad in (lambda: c.append(x, x[:2], s), lambda: c.append(x, x.half(), s), lambda: c.append(x, x, s.long()),
                lambda: c.append(x, x, s[:2]), lambda: c.append(x.cpu(), x, s), lambda: c.append(x.double(), x.double(), s),
                lambda: c.append(x.transpose(1, 2), x.transpose(1, 2), s), lambda: c.append(x[:, :1], x[:, :1], s),
                lambda: c.attention(x[:, :1], s[:2], s[:1], s[None], 1), lambda: c.attention(x, s, s[:1], s[None], 1),
                lambda: c.attention(x, s[:2], s[:1], s, 1), lambda: c.attention(x, s[:2], s[:1], s[None], -1),
                lambda: c.attention(x, s[:2], s[:1], s[None], 1, out=x[:2]), lambda: c.values(s.long()),
                lambda: c.values(dtype=torch.float64), lambda: kv8.Cache(4, 24, 2, 64), lambda: kv8.Cache(4, 16, 2, 72),
                lambda: kv8.Cache.over(c.k_codes, c.k_scales[:2], c.v_codes, c.v_scales),
                lambda: kv8.plan(s, s, s, s, s[:1], 16, 3), lambda: kv8.plan(s, s[:2], s[:, None].contiguous(), s, s[:1], 16, 3),
                lambda: kv8.plan(s, s, s[:, None].contiguous(), s, s[:1], 16, -1),
                lambda: sampling.sample(x[0, 0], x[0, 0]), lambda: sampling.sample(x[0], x[0, 0, :2].double()),
                lambda: sampling.sample(x[0], x[0, 0, :2], top_k=x[0, 0, :2]), lambda: sampling.sample(x[0].t(), x[0, 0]),
                lambda: sampling.sample(x[0], None), lambda: sampling.sample(x[0].cpu(), x[0, 0, :2])):
        with pytest.raises(SpmError):
            bad()


class Serving:
    """A small server's state: three ticks' worth of requests over one cache."""

    def __init__(self):
        self.pages = kv8.Pages(4, 8, 24, 16)
        self.cache = kv8.Cache(24, 16, 2, 64)
        self.cached, self.new, self.ended = ints([0] * 4), ints([0] * 4), ints([0] * 4)
        g = gen(20)
        self.k, self.v = (torch.randn(64, 2, 64, device="cuda", generator=g) for _ in range(2))
        self.q = torch.randn(64, 4, 64, device="cuda", generator=g)
        self.head = torch.randn(500, 4 * 64, device="cuda", generator=g)
        self.u = torch.rand(4, device="cuda", generator=g)

    def tick(self):
        p = self.pages.plan(self.cached, self.new, 64, ended=self.ended)
        self.cache.append(self.k, self.v, p.slots)
        o = self.cache.attention(self.q, p.starts, p.lens, self.pages.table, 60)
        last = o[(p.starts[1:].long() - 1).clamp(min=0)].flatten(1)
        r = sampling.sample(last @ self.head.t(), self.u, top_k=ints_like(self.u, 7), top_p=torch.full_like(self.u, 0.9))
        self.cached.copy_(p.lens)
        return p.slots, o, r.token


def ints_like(t, v):
    return torch.full(t.shape, v, dtype=torch.int32, device=t.device)


TICKS = [([30, 0, 12, 1], [0] * 4), ([1, 1, 1, 0], [0] * 4), ([1, 40, 1, 1], [0, 0, 0, 1]), ([0, 1, 20, 1], [32, 0, 0, 0])]


def test_ticks_run_together_and_in_a_graph():
    eager, captured = Serving(), Serving()
    captured.tick()  # loads the kernels; no request has tokens yet
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = captured.tick()
    keys, values = [{} for _ in range(4)], [{} for _ in range(4)]
    for new, ended in TICKS:
        for s in (eager, captured):
            s.new.copy_(ints(new))
            s.ended.copy_(ints(ended))
            s.cached.masked_fill_(s.ended > 0, 0)
        before = eager.cached.tolist()
        got = eager.tick()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, outs):
            assert torch.equal(a, b)
        assert torch.equal(eager.pages.table, captured.pages.table) and torch.equal(eager.pages.count, captured.pages.count)
        # against rows kept in full, 64 bits
        at = 0
        for r in range(4):
            if ended[r]:
                keys[r], values[r] = {}, {}
            for i in range(new[r]):
                keys[r][before[r] + i], values[r][before[r] + i] = eager.k[at + i].double(), eager.v[at + i].double()
            L = len(keys[r])
            for i in range(new[r]):
                n = before[r] + i + 1
                k, v = (torch.stack([d[j] for j in range(n)]) for d in (keys[r], values[r]))
                for h in range(4):
                    w = torch.softmax(k[:, h // 2] @ eager.q[at + i, h].double() / 8, 0)
                    # codes within one step of 2^-5 (|x| under 4): scores move by less than
                    # 0.031 * sum|q| / 8 < 0.25, values by 0.031
                    assert ((w @ v[:, h // 2] - got[1][at + i, h]).abs() <= 0.031 + 0.3 * v.abs().max()).all()
            assert L == before[r] + new[r]
            at += new[r]
        eager.pages.check()
        eager.cache.check()


def test_two_captured_calls_share_nothing():
    # two graphs of the attention on two streams at once, each with scratch of its own
    lens = [4000, 3000]
    table, pages = tables(np.random.default_rng(6), lens, 64)
    c = pool(pages, 64, 2, 128)
    qs = [torch.randn(2, 16, 128, device="cuda", generator=gen(30 + i)) for i in range(2)]
    starts, ln = ints([0, 1, 2]), ints(lens)
    want = [c.attention(q, starts, ln, table, 1) for q in qs]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for q, st in zip(qs, streams):
        st.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(c.attention(q, starts, ln, table, 1))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)


def test_calls_on_another_stream():
    c = pool(8, 16, 2, 64)
    x = torch.randn(2, 30, 2, 64, device="cuda", generator=gen(40))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    slots = ints(list(range(30)))
    torch.cuda.synchronize()
    c.append(x[0], x[1], slots, stream=side)
    k, _ = c.values(stream=side)
    table, q = ints([[0, 1]]), torch.randn(1, 4, 64, device="cuda", generator=gen(41))
    starts, lens = ints([0, 1]), ints([30])
    side.wait_stream(torch.cuda.current_stream())
    o = c.attention(q, starts, lens, table, 1, stream=side)
    r = sampling.sample(q[0], torch.full((4,), 0.5, device="cuda"), stream=side)
    side.synchronize()
    assert torch.equal(k, c.values()[0]) and torch.equal(o, c.attention(q, starts, lens, table, 1))
    assert torch.equal(r.token, sampling.sample(q[0], torch.full((4,), 0.5, device="cuda")).token)
