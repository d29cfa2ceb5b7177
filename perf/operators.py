"""Measured cases of the serving operators: block tables and slot maps, the
paged 8-bit KV cache (append and attention) and the sampler.

Every state is made on the GPU from a seed.  `run` computes an operator in
elementary torch operations where `own` is false and through the package's
entry points where it is true; `exact` computes it from its definition in
64 bits.

Definitions.
  plan    Row r of the table has cached[r] tokens in ceil(cached[r] / P) pages
          and takes new[r] more; the pages of ended[r] tokens of its former
          request go back to the stack of free pages first, in row order.  New
          pages come off the stack's top in row order.  Token t of the call
          (rows one after the other) gets its position in its request and its
          slot, page * P + offset.  Places past the last token get -1.
  append  A page holds P tokens of one request; codes are int8 with one scale
          for each page and kv head, a power of two: the smallest 2^e with
          |x| <= 127 * 2^e for every value written.  Rows already in the page
          raise e, and are rounded again to it (half to even) when it grows.
          A call that writes a page's first row starts the page anew.
  attention  Query i of request r's n stands at position len - n + i and sees
          the keys up to it; softmax of scale * q.k in 32 bits.
  sample  Tokens sorted by (logit descending, index ascending), weights
          exp((logit - max) / temperature).  Kept is the shortest of three
          prefixes: the top_k first; the smallest whose mass reaches top_p of
          the top_k's; those of weight >= min_p.  The pick is the first token
          by index at which the kept mass exceeds u times its total; with
          temperature 0 the largest logit is taken, the first by index.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one decode tick of the largest batch a session takes: every call is launch latency
        {"name": "plan decode 8", "op": "plan", "requests": 8, "prompts": 0, "prompt": 0, "longest": 1280, "page": 64},
        # a serving tick that admits a wave of prompts beside many decoding requests
        {"name": "plan mixed 1024", "op": "plan", "requests": 1024, "prompts": 96, "prompt": 700, "longest": 4096, "page": 16},
        # a decode tick of the Qwen3-8B shape, eight clients
        {"name": "append decode 8", "op": "append", "dtype": "f32", "requests": 8, "new": 1, "longest": 768,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # one chunk of a prompt, as a session runs it
        {"name": "append prompt 1024", "op": "append", "dtype": "f32", "requests": 1, "new": 1024, "longest": 1024,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # a wave of ragged prompts, small pages
        {"name": "append ragged bf16", "op": "append", "dtype": "bf16", "requests": 37, "new": 700, "longest": 500,
         "heads": 32, "kv_heads": 4, "dim": 128, "page": 16},
        # a single client of the SmolLM2 shape: latency
        {"name": "attention one client", "op": "attention", "dtype": "f32", "requests": 1, "new": 1, "shortest": 96, "longest": 96,
         "heads": 9, "kv_heads": 3, "dim": 64, "page": 32},
        # eight clients of the Qwen3-30B-A3B shape at the end of their run
        {"name": "attention decode 8", "op": "attention", "dtype": "f32", "requests": 8, "new": 1, "shortest": 1024,
         "longest": 1280, "heads": 32, "kv_heads": 4, "dim": 128, "page": 64},
        # many clients, ragged and long: the cache is what is read
        {"name": "attention decode 64 long", "op": "attention", "dtype": "bf16", "requests": 64, "new": 1, "shortest": 1000,
         "longest": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # a prompt chunk over what its client has in the cache
        {"name": "attention prompt 1024", "op": "attention", "dtype": "bf16", "requests": 1, "new": 1024, "shortest": 4096,
         "longest": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # one client of the SmolLM2 vocabulary, every filter on
        {"name": "sample one 49152", "op": "sample", "dtype": "f32", "rows": 1, "vocab": 49152, "filters": "all"},
        # the largest session batch over the Qwen3 vocabulary, nucleus only
        {"name": "sample 8 151936", "op": "sample", "dtype": "f32", "rows": 8, "vocab": 151936, "filters": "p"},
        # a larger batch, each row with its own settings
        {"name": "sample 128 mixed", "op": "sample", "dtype": "bf16", "rows": 128, "vocab": 151936, "filters": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attention", "attention", "attention", "sample", "sample"])
    if op == "plan":
        requests = _log(rng, 1, 2048)
        prompts = rng.choice([0, rng.randint(0, max(1, min(requests, 128)))])
        return {"op": op, "requests": requests, "prompts": min(prompts, requests), "prompt": _log(rng, 2, 600),
                "longest": _log(rng, 1, 4096), "page": rng.choice([16, 32, 64, 128])}
    heads, kv_heads = rng.choice([(9, 3), (32, 8), (16, 16), (32, 4), (8, 1), (14, 2), (64, 4), (5, 5)])
    shape = {"dtype": rng.choice(["f32", "bf16", "f16"]), "heads": heads, "kv_heads": kv_heads,
             "dim": rng.choice([64, 96, 128, 128, 192, 256]), "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        row = kv_heads * shape["dim"]
        requests = _log(rng, 1, max(1, min(64, 9_000_000 // (row * shape["page"]))))
        return {"op": op, **shape, "requests": requests, "new": _log(rng, 1, max(1, min(2000, 9_000_000 // (requests * row)))),
                "longest": _log(rng, 1, 1000)}
    if op == "attention":
        if rng.random() < 0.65:  # decode, with a few tokens at once at times
            requests = _log(rng, 1, 64)
            new = rng.choice([1, 1, 1, 2, 5])
            longest = _log(rng, 8, max(16, min(16384, (1 << 30) // (requests * kv_heads * shape["dim"] * 4))))
        else:
            requests = rng.randint(1, 3)
            new = _log(rng, 17, 700)
            longest = new + _log(rng, 1, max(2, min(4000, 12_000_000_000 // (requests * heads * shape["dim"] * new) - new)))
        return {"op": op, **shape, "requests": requests, "new": new, "shortest": _log(rng, 1, longest), "longest": longest}
    return {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "rows": _log(rng, 1, 100), "vocab": _log(rng, 2, 152000),
            "filters": rng.choice(["none", "k", "p", "min", "all", "mixed"])}


# ------------------------------------------------------------------ inputs --
def _ints(values):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).cuda()


def _tables(rng, lens, page, spare=0):
    """A table of random distinct pages that holds `lens` tokens, and the number of pages it takes."""
    need = -(-lens // page)
    width = max(1, int(need.max()) if len(need) else 1)
    ids = rng.permutation(int(need.sum()) + spare)
    table = np.full((len(lens), width), -1, dtype=np.int32)
    at = np.arange(width)[None, :] < need[:, None]
    table[at] = ids[: int(need.sum())]
    return table, ids


def _prepare_plan(case, rng):
    R, P = case["requests"], case["page"]
    cached = rng.integers(0, case["longest"] + 1, R)
    new = np.ones(R, dtype=np.int64)
    ended = np.zeros(R, dtype=np.int64)
    rows = rng.permutation(R)[: case["prompts"]]
    cached[rows] = 0
    new[rows] = rng.integers((case["prompt"] + 1) // 2, case["prompt"] + 1, len(rows))
    gone = rng.random(R) < 0.1  # rows whose request has just ended, and idle ones
    gone[rows] = False
    ended[gone] = cached[gone]
    cached[gone] = 0
    new[gone] = 0
    need = -(-(cached + ended) // P)
    # a pool that holds every row at its longest, and a batch padded to its most tokens
    width = -(-max(case["longest"] + 1, case["prompt"]) // P)
    ids = rng.permutation(R * width)
    table = np.full((R, width), -1, dtype=np.int32)
    table[np.arange(width)[None, :] < need[:, None]] = ids[: int(need.sum())]
    spare = len(ids) - int(need.sum())
    free = np.full(len(ids), -1, dtype=np.int32)
    free[:spare] = ids[int(need.sum()):]
    return {"cached": _ints(cached), "new": _ints(new), "ended": _ints(ended), "table": _ints(table), "free": _ints(free),
            "count": _ints([spare]), "tokens": R + case["prompts"] * case["prompt"], "page": P}


def _quantised(x):
    """x [pages, heads, P, dim] as int8 codes and power-of-two scales."""
    m, e = torch.frexp(x.abs().amax((2, 3)))
    scale = ((e - 7 + (m > 127 / 128) + 127) << 23).view(torch.float32)
    return (x / scale[:, :, None, None]).round().to(torch.int8), scale


def _cache(gen, pages, case):
    """Pages of keys and values as projections give them: channels of different size, and pages of different size."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    out = []
    for spread in (0.6, 0.4):
        channel = torch.exp(spread * torch.randn(case["kv_heads"], 1, case["dim"], device="cuda", generator=gen))
        level = torch.exp(0.5 * torch.randn(pages, case["kv_heads"], 1, 1, device="cuda", generator=gen))
        codes = torch.empty(shape, dtype=torch.int8, device="cuda")
        scales = torch.empty(shape[:2], dtype=torch.float32, device="cuda")
        some = max(1, (1 << 27) // max(1, shape[1] * shape[2] * shape[3]))
        for a in range(0, pages, some):
            x = torch.randn((min(some, pages - a),) + shape[1:], device="cuda", generator=gen)
            codes[a:a + some], scales[a:a + some] = _quantised(x.mul_(channel).mul_(level[a:a + some]))
        out += [codes, scales]
    return out


def _prepare_append(case, rng, gen):
    R, P = case["requests"], case["page"]
    of_case = np.random.default_rng([R, P, case["new"], case["longest"], case["dim"], case["kv_heads"]])  # shapes do not go by the seed
    cached = of_case.integers(0, case["longest"] + 1, R)
    new = np.full(R, case["new"]) if case["new"] == 1 else of_case.integers(max(1, case["new"] // 2), case["new"] + 1, R)
    # the pages that the call touches, and of each request no more
    first = cached // P
    span = -(-(cached + new) // P) - first
    ids = rng.permutation(int(span.sum()))
    base = np.concatenate([[0], np.cumsum(span)])
    slots = np.concatenate([ids[base[r] + np.arange(cached[r], cached[r] + new[r]) // P - first[r]] * P
                            + np.arange(cached[r], cached[r] + new[r]) % P for r in range(R)])
    T, qw, kvw = len(slots), case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    qkv = torch.randn(T, qw + 2 * kvw, device="cuda", generator=gen)
    qkv *= torch.exp(torch.randn(1, qw + 2 * kvw, device="cuda", generator=gen))
    qkv = qkv.to(DTYPES[case["dtype"]])
    # keys and values as they lie in the fused projection's rows
    k = qkv[:, qw:qw + kvw].unflatten(1, (case["kv_heads"], case["dim"]))
    v = qkv[:, qw + kvw:].unflatten(1, (case["kv_heads"], case["dim"]))
    kc, ks, vc, vs = _cache(gen, len(ids), case)
    return {"k": k, "v": v, "slots": _ints(slots), "k_codes": kc, "k_scales": ks, "v_codes": vc, "v_scales": vs}


def _prepare_attention(case, rng, gen):
    R, P = case["requests"], case["page"]
    new = np.full(R, case["new"])
    lens = np.maximum(rng.integers(case["shortest"], case["longest"] + 1, R), new)
    lens[-1] = max(case["longest"], case["new"])
    table, ids = _tables(rng, lens, P)
    kc, ks, vc, vs = _cache(gen, len(ids), case)
    q = torch.randn(int(new.sum()), case["heads"], case["dim"], device="cuda", generator=gen)
    q *= torch.exp(0.3 * torch.randn(1, case["heads"], 1, device="cuda", generator=gen))
    return {"q": q.to(DTYPES[case["dtype"]]), "starts": _ints(np.concatenate([[0], np.cumsum(new)])), "lens": _ints(lens),
            "table": _ints(table), "most": case["new"], "scale": 1 / math.sqrt(case["dim"]),
            "k_codes": kc, "k_scales": ks, "v_codes": vc, "v_scales": vs}


def _prepare_sample(case, rng, gen):
    n, V, f = case["rows"], case["vocab"], case["filters"]
    x = torch.randn(n, V, device="cuda", generator=gen)
    # a few strong candidates over a broad body, as a language model's head gives
    x += 9.0 * torch.rand(n, V, device="cuda", generator=gen).pow_(2000 if V > 2000 else 8)
    x *= 1.0 + 1.5 * torch.rand(n, 1, device="cuda", generator=gen)
    on = lambda names: (np.full(n, f in names) if f != "mixed" else rng.random(n) < 0.5)  # noqa: E731
    return {"logits": x.to(DTYPES[case["dtype"]]),
            "temperature": torch.from_numpy(rng.uniform(0.5, 1.5, n).astype(np.float32) * (rng.random(n) < 0.95)).cuda(),
            "top_k": _ints(np.where(on(("k", "all")), np.exp(rng.uniform(0, math.log(200), n)).astype(int), 0)),
            "top_p": torch.from_numpy(np.where(on(("p", "all")), rng.uniform(0.3, 0.99, n), 1.0).astype(np.float32)).cuda(),
            "min_p": torch.from_numpy(np.where(on(("min", "all")), rng.uniform(0.001, 0.2, n), 0.0).astype(np.float32)).cuda(),
            "u": torch.from_numpy(rng.random(n).astype(np.float32)).cuda()}


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "plan":
        s = _prepare_plan(case, rng)
    elif case["op"] == "append":
        s = _prepare_append(case, rng, gen)
    elif case["op"] == "attention":
        s = _prepare_attention(case, rng, gen)
    else:
        s = _prepare_sample(case, rng, gen)
    s["op"] = case["op"]
    if own and "k_codes" in s:  # the handle that a program keeps over its cache's memory
        from emufpga_b200 import kv8

        s["cache"] = kv8.Cache.over(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    return s


# ------------------------------------------------------------- plain forms --
def _plan(s):
    cached, new, ended, P = s["cached"].long(), s["new"].long(), s["ended"].long(), s["page"]
    table, free, count = s["table"], s["free"], s["count"].long()
    R, W = table.shape
    lens = cached + new
    old, need, back = (cached + P - 1) // P, (lens + P - 1) // P, (ended + P - 1) // P
    j = torch.arange(W, device="cuda")[None, :]
    # pages of ended requests onto the stack (a spare place takes what is not one)
    rank = (back.cumsum(0) - back)[:, None] + j
    room = torch.cat([free, free.new_zeros(1)])
    room[torch.where(j < back[:, None], count + rank, len(free)).flatten()] = table.flatten()
    free.copy_(room[:-1])
    top = count + back.sum()
    fresh = need - old
    rank = (fresh.cumsum(0) - fresh)[:, None] + j - old[:, None]
    takes = (j >= old[:, None]) & (j < need[:, None])
    table.copy_(torch.where(takes, free[(top - 1 - rank).clamp(0, len(free) - 1)], table))
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(s["tokens"], device="cuda")
    r = torch.searchsorted(starts[1:], t, right=True)
    real = r < R
    r = r.clamp(max=R - 1)
    pos = cached[r] + t - starts[r]
    slots = table[r, (pos // P).clamp(0, W - 1)].long() * P + pos % P
    left = top - fresh.sum()
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"starts": i32(starts), "lens": i32(lens), "positions": i32(torch.where(real, pos, -1)),
            "slots": i32(torch.where(real, slots, -1)), "table": table, "free": free, "left": i32(left)}


def _store(x, slots, codes, scales):
    pages, heads, P, dim = codes.shape
    x = x.float()
    slots = slots.long()
    page, off = slots // P, slots % P
    amax = torch.zeros(pages, heads, device="cuda").index_reduce_(0, page, x.abs().amax(2), "amax")
    first = torch.full((pages,), P, device="cuda").index_reduce_(0, page, off, "amin")
    touched = (first < P)[:, None]
    m, e = torch.frexp(amax)
    scale = torch.where(amax > 0, ((e - 7 + (m > 127 / 128)).clamp(min=-126) + 127 << 23).view(torch.float32), 0.0)
    scale = torch.where((first > 0)[:, None], torch.maximum(scale, scales), scale)
    shrink = torch.where(scale > 0, scales / scale, torch.ones_like(scale))
    older = touched[:, :, None] & (torch.arange(P, device="cuda") < first[:, None, None])
    again = (codes.float() * shrink[:, :, None, None]).round().to(torch.int8)
    codes.copy_(torch.where(older[..., None], again, codes))
    scales.copy_(torch.where(touched, scale, scales))
    s = scales[page][:, :, None]
    codes[page, :, off] = torch.where(s > 0, x / s, torch.zeros_like(x)).round().to(torch.int8)
    return codes.float() * scales[:, :, None, None]


def _attend(s):
    q, table, starts, lens = s["q"], s["table"].long(), s["starts"].long(), s["lens"].long()
    T, H, D = q.shape
    R, N = len(lens), s["most"]
    keys = (s["k_codes"][table.clamp(min=0)].float() * s["k_scales"][table.clamp(min=0)][..., None, None])
    values = (s["v_codes"][table.clamp(min=0)].float() * s["v_scales"][table.clamp(min=0)][..., None, None])
    G = keys.shape[2]
    keys = keys.transpose(1, 2).flatten(2, 3)  # [R, kv head, position, dim]
    values = values.transpose(1, 2).flatten(2, 3)
    L = keys.shape[2]
    at = (starts[:-1, None] + torch.arange(N, device="cuda")).clamp(max=T - 1)
    qs = q[at].float().view(R, N, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(R, G, H // G * N, D)
    x = (qs @ keys.transpose(2, 3)).mul_(s["scale"]).view(R, G, H // G, N, L)
    place = lens[:, None] - (starts[1:] - starts[:-1])[:, None] + torch.arange(N, device="cuda")
    seen = torch.arange(L, device="cuda") <= place[..., None]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    y = (x.view(R, G, H // G * N, L) @ values).view(R, G, H // G, N, D) / total
    y = y.permute(0, 3, 1, 2, 4).reshape(R, N, H, D)
    real = torch.arange(N, device="cuda") < (starts[1:] - starts[:-1])[:, None]
    out = torch.zeros(T + 1, H, D, device="cuda")
    out[torch.where(real, at, T).flatten()] = y.flatten(0, 1)
    return out[:T].to(q.dtype)


def _pick(s):
    x = s["logits"].double()
    n, V = x.shape
    T = s["temperature"].double()[:, None]
    greedy = T <= 0
    top, best = x.max(1, keepdim=True)
    w = ((x - top) / torch.where(greedy, torch.ones_like(T), T)).exp()
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    ws = w.gather(1, order)
    cum = ws.cumsum(1)
    k = s["top_k"].long()[:, None]
    k = torch.where((k <= 0) | (k > V), V, k)
    p = s["top_p"].double()[:, None]
    mass = cum.gather(1, k - 1)
    np_ = torch.where(p < 1, 1 + (cum < p * mass).sum(1, keepdim=True), V)
    low = s["min_p"].double()[:, None]
    nm = torch.where(low > 0, (ws >= low).sum(1, keepdim=True), V)
    kept = torch.minimum(torch.minimum(k, np_), nm).clamp(min=1)
    kept = torch.where(greedy, 1, kept)
    stays = torch.zeros_like(w).scatter(1, order, (torch.arange(V, device="cuda") < kept).double())
    cum = (w * stays).cumsum(1)
    Z = cum[:, -1:]
    token = (cum <= s["u"].double()[:, None] * Z).sum(1, keepdim=True).clamp(max=V - 1)
    return {"token": token[:, 0].to(torch.int32), "kept": kept[:, 0].to(torch.int32),
            "prob": (w.gather(1, token) / Z)[:, 0].float()}


def run(state):
    s = state
    if own:
        from emufpga_b200 import kv8, sampling

        if s["op"] == "plan":
            p = kv8.plan(s["cached"], s["new"], s["table"], s["free"], s["count"], s["page"], s["tokens"], ended=s["ended"],
                         left=s.setdefault("left", torch.empty_like(s["count"])))
            return {"starts": p.starts, "lens": p.lens, "positions": p.positions, "slots": p.slots, "table": s["table"],
                    "free": s["free"], "left": s["left"]}
        if s["op"] == "append":
            s["cache"].append(s["k"], s["v"], s["slots"])
            k, v = s["cache"].values()
            return {"k": k, "v": v}
        if s["op"] == "attention":
            return s["cache"].attention(s["q"], s["starts"], s["lens"], s["table"], s["most"], scale=s["scale"])
        got = sampling.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        return {"token": got.token, "kept": got.kept, "prob": got.prob}
    if s["op"] == "plan":
        return _plan(s)
    if s["op"] == "append":
        return {"k": _store(s["k"], s["slots"], s["k_codes"], s["k_scales"]),
                "v": _store(s["v"], s["slots"], s["v_codes"], s["v_scales"])}
    return _attend(s) if s["op"] == "attention" else _pick(s)


def work(case):
    """Bytes and operations of one pass, from the case's expected lengths."""
    if case["op"] == "plan":
        P, R = case["page"], case["requests"]
        tokens = (R - case["prompts"]) * 0.9 + 0.75 * case["prompts"] * case["prompt"]
        moved = 0.75 * case["prompts"] * case["prompt"] / P + R / P + 0.1 * R * case["longest"] / 2 / P
        return {"bytes": 4 * (5 * R + 2 * tokens + 2 * moved), "flops": 0}
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 32), "flops": 0}
    size = 4 if case["dtype"] == "f32" else 2
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        each = 1 if case["new"] == 1 else 0.75 * case["new"]
        tokens = case["requests"] * each
        held = case["requests"] * (math.ceil((each - 1) / case["page"]) + (1 if case["new"] == 1 else 0.99)) * case["page"]
        # rows in, codes out; then the touched pages' codes in and their values out
        return {"bytes": 2 * row * (tokens * (size + 1) + held * 5), "flops": 0}
    mean = (case["shortest"] + case["longest"]) / 2
    lens = max(case["new"], ((case["requests"] - 1) * mean + case["longest"]) / case["requests"])
    seen = case["new"] * lens - case["new"] * (case["new"] - 1) / 2
    return {"bytes": case["requests"] * (2 * lens * row + 2 * case["new"] * case["heads"] * case["dim"] * size),
            "flops": 4 * case["requests"] * case["heads"] * case["dim"] * seen}


# ------------------------------------------------------------ definitions --
def _exact_plan(case, s):
    P = case["page"]
    cached, new, ended = (s[k].tolist() for k in ("cached", "new", "ended"))
    table, free, count = s["table"].tolist(), s["free"].tolist(), int(s["count"])
    top = count
    for r, n in enumerate(ended):
        for j in range(-(-n // P)):
            free[top] = table[r][j]
            top += 1
    starts, positions, slots = [0], [], []
    for r in range(len(cached)):
        for j in range(-(-cached[r] // P), -(-(cached[r] + new[r]) // P)):
            top -= 1
            table[r][j] = free[top]
        for p in range(cached[r], cached[r] + new[r]):
            positions.append(p)
            slots.append(table[r][p // P] * P + p % P)
        starts.append(starts[-1] + new[r])
    pad = [-1] * (s["tokens"] - len(slots))
    return {"starts": np.array(starts, np.int32), "lens": np.array([a + b for a, b in zip(cached, new)], np.int32),
            "positions": np.array(positions + pad, np.int32), "slots": np.array(slots + pad, np.int32),
            "table": np.array(table, np.int32), "free": np.array(free, np.int32), "left": np.array([top], np.int32)}


def _exact_store(x, slots, codes, scales):
    """Page after page, in exact arithmetic (every product is by a power of two)."""
    x, codes, scales = x.double().cpu().numpy(), codes.cpu().numpy().astype(np.float64), scales.double().cpu().numpy()
    P = codes.shape[2]
    at = 0
    while at < len(slots):
        page, off = divmod(int(slots[at]), P)
        n = 1
        while at + n < len(slots) and off + n < P and slots[at + n] == slots[at] + n:
            n += 1
        rows = x[at:at + n].transpose(1, 0, 2)
        for h in range(codes.shape[1]):
            big = np.abs(rows[h]).max()
            e = -math.inf
            if big > 0:
                e = max(-126, math.ceil(math.log2(big)) - 9)
                while big > 127 * 2.0 ** e:
                    e += 1
            if off and scales[page, h] > 0:
                e = max(e, math.log2(scales[page, h]))
            scale = 2.0 ** e if e > -math.inf else 0.0
            if scale:
                codes[page, h, :off] = np.rint(codes[page, h, :off] * (scales[page, h] / scale))
                codes[page, h, off:off + n] = np.rint(rows[h] / scale)
            else:
                codes[page, h, off:off + n] = 0
            scales[page, h] = scale
        at += n
    return codes * scales[:, :, None, None]


def _exact_attend(case, s):
    """One request and kv head after the other, in 64 bits."""
    q, starts, lens = s["q"].double(), s["starts"].tolist(), s["lens"].tolist()
    H, P = case["heads"], case["page"]
    G = H // case["kv_heads"]
    out = torch.zeros_like(q)
    for r, L in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        ids = s["table"][r, : -(-L // P)].long()
        hidden = torch.arange(L, device="cuda")[None, :] > torch.arange(L - (b - a), L, device="cuda")[:, None]
        for g in range(case["kv_heads"]):
            k, v = ((s[c][ids, g].double() * s[z][ids, g].double()[:, None, None]).reshape(-1, case["dim"])[:L]
                    for c, z in (("k_codes", "k_scales"), ("v_codes", "v_scales")))
            for h in range(g * G, g * G + G):
                x = (q[a:b, h] @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
                out[a:b, h] = torch.softmax(x, 1) @ v
    return out


def _exact_pick(case, s):
    x = s["logits"].double().cpu().numpy()
    V = case["vocab"]
    temps, ks, ps, ms, us = (s[k].double().cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p", "u"))
    token, kept, prob = [], [], []
    for row, T, k, p, m, u in zip(x, temps, ks, ps, ms, us):
        if T <= 0:
            token.append(int(np.argmax(row)))
            kept.append(1)
            prob.append(1.0)
            continue
        order = np.argsort(-row, kind="stable")
        w = np.exp((row[order] - row[order[0]]) / T)
        n = V if not 0 < k <= V else int(k)
        if p < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(w), p * np.sum(w[:n]), side="left")))
        if m > 0:
            n = min(n, int((w >= m).sum()))
        n = max(n, 1)
        some = np.argsort(order[:n])
        mass = np.cumsum(w[some])
        i = min(int(np.searchsorted(mass, u * mass[-1], side="right")), n - 1)
        token.append(int(order[some[i]]))
        kept.append(n)
        prob.append(w[some[i]] / mass[-1])
    return {"token": np.array(token, np.int32), "kept": np.array(kept, np.int32), "prob": np.array(prob)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(case, s)
    if case["op"] == "append":
        slots = s["slots"].tolist()
        return {"k": _exact_store(s["k"], slots, s["k_codes"], s["k_scales"]),
                "v": _exact_store(s["v"], slots, s["v_codes"], s["v_scales"])}
    return _exact_attend(case, s) if case["op"] == "attention" else _exact_pick(case, s)
