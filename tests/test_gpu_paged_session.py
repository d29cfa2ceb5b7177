"""Sessions over the paged 8-bit cache, and sampled steps, against a 64-bit
forward pass whose keys and values are rounded as the cache rounds them.

The bar is the repository's: logits within 1e-3 of the largest, greedy picks
the same -- until one of the client's stored values lies so near a tie between
two codes that the fp32 products decide it either way.  Key and value rows are
within 2^-21 of their largest (fp32 against 64 bits), which is 127 steps at
most: a value within 2^-14 of a step of a tie may take the other code, one step,
at most 2^-6 of the page's largest.  From then on the client is held to 2^-6,
and a pick to being within that of the largest."""
import math

import numpy as np
import pytest

import emufpga_b200 as eb
import serving_cases as ref
from emufpga_b200 import configs
from emufpga_b200._lib import LLAMA, SpmError
from emufpga_b200.sampling import Sampling
from emufpga_b200.scheduler import Request, serve_continuous

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-3


class Plain:
    """One client of a dense model in 64 bits, its cache in pages of `page` tokens."""

    def __init__(self, recipe, page, context):
        self.sh, self.page = recipe.shape, page
        self.img = eb.synth_gguf(recipe)
        self.w = {}
        n = -(-context // page)
        shape = (n, self.sh.kv_heads, page, self.sh.head_dim)
        self.cache = [[(np.zeros(shape), np.zeros(shape[:2])) for _ in range(2)] for _ in range(self.sh.layers)]
        self.len = 0
        self.tied = False

    def tensor(self, name):
        if name not in self.w:
            t = eb.gguf_find(self.img, name)
            v = eb.decode_blocks(t["dtype"], self.img[t["offset"]:t["offset"] + t["nbytes"]]).astype(np.float64)
            dims = [d for d in t["dims"] if d > 1]
            self.w[name] = v.reshape(dims[::-1]) if len(dims) > 1 else v
        return self.w[name]

    def norm(self, x, gain):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.sh.eps) * self.tensor(gain)

    def rope(self, x, pos):
        half = x.shape[-1] // 2
        angle = pos[:, None, None] / self.sh.rope_base ** (np.arange(half) / half)
        c, s = np.cos(angle), np.sin(angle)
        a, b = x[..., :half], x[..., half:]
        return np.concatenate([a * c - b * s, a * s + b * c], -1)

    def feed(self, tokens):
        """Tokens at the next positions, their keys and values stored in one call; the last one's logits."""
        sh, T = self.sh, len(tokens)
        pos = np.arange(self.len, self.len + T, dtype=np.float64)
        slots = list(range(self.len, self.len + T))
        x = self.tensor("token_embd.weight")[np.array(tokens)]
        for l in range(sh.layers):
            p = f"blk.{l}."
            h = self.norm(x, p + "attn_norm.weight")
            q, k, v = ((h @ self.tensor(p + f"attn_{n}.weight").T).reshape(T, -1, sh.head_dim) for n in "qkv")
            if sh.family != LLAMA:
                q, k = self.norm(q, p + "attn_q_norm.weight"), self.norm(k, p + "attn_k_norm.weight")
            q, k = self.rope(q, pos), self.rope(k, pos)
            for part, rows in zip(self.cache[l], (k, v)):
                ref.store(rows, slots, *part)
                scale = part[1][np.array(slots) // self.page][:, :, None]
                steps = np.abs(np.divide(rows, scale, out=np.zeros_like(rows), where=scale > 0))
                self.tied |= bool((np.abs(steps % 1 - 0.5) < 2.0 ** -14).any())
            keys, values = (((c * s[:, :, None, None]).transpose(0, 2, 1, 3)).reshape(-1, sh.kv_heads, sh.head_dim)
                            for c, s in self.cache[l])
            out = np.empty_like(q)
            for t in range(T):
                n = self.len + t + 1
                for g in range(sh.heads):
                    kv = g // (sh.heads // sh.kv_heads)
                    e = keys[:n, kv] @ q[t, g] / math.sqrt(sh.head_dim)
                    e = np.exp(e - e.max())
                    out[t, g] = e / e.sum() @ values[:n, kv]
            x = x + out.reshape(T, -1) @ self.tensor(p + "attn_output.weight").T
            h = self.norm(x, p + "ffn_norm.weight")
            a, b = (h @ self.tensor(p + f"ffn_{n}.weight").T for n in ("gate", "up"))
            x = x + (a / (1 + np.exp(-a)) * b) @ self.tensor(p + "ffn_down.weight").T
        self.len += T
        head = "token_embd.weight" if sh.tied else "output.weight"
        return self.norm(x[-1:], "output_norm.weight")[0] @ self.tensor(head).T


def close(got, want, tied=False):
    return np.abs(got - want).max() <= (2.0 ** -6 if tied else LOGIT_TOL) * np.abs(want).max()


def picked(best, want, tied):
    return want[best] >= want.max() - 2.0 ** -5 * np.abs(want).max() if tied else best == int(np.argmax(want))


DENSE = ["llama-q6_k", "qwen3-q6_k", "qwen3-g4-q5_k", "qwen3-g8-q6_k"]


@pytest.mark.parametrize("name", DENSE)
@pytest.mark.parametrize("graphs", [True, False])
def test_steps_match_the_plain_form(name, graphs):
    r = configs.TINY[name]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    s = eb.Session(m, 2, 64, graphs=graphs, paged=(8, 16))
    plain = [Plain(r, 16, 64) for _ in range(2)]
    prompts = [configs.prompt_tokens(3, i, 20, r.shape.vocab) for i in range(2)]
    toks = [p[0] for p in prompts]
    strict = 0
    for t in range(40):
        best, got = s.decode_step(toks, want_logits=True)
        want = [p.feed([tok]) for p, tok in zip(plain, toks)]
        strict += not all(p.tied for p in plain)
        assert all(close(g, w, p.tied) for g, w, p in zip(got, want, plain)), t
        assert all(picked(b, w, p.tied) for b, w, p in zip(best, want, plain)), t
        toks = [p[t + 1] if t + 1 < len(p) else b for p, b in zip(prompts, best)]
    assert strict
    assert s.free_pages == 8 - 2 * 3 and [s.length(i) for i in range(2)] == [40, 40]
    s.close()
    m.close()


@pytest.mark.parametrize("name,length", [("qwen3-q6_k", 70), ("llama-q6_k", 33), ("qwen3-g8-q6_k", 300)])
def test_prompts_match_the_plain_form(name, length):
    r = configs.TINY[name]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    s = eb.Session(m, 2, 400, paged=(60, 16))
    plain = Plain(r, 16, 400)
    prompt = configs.prompt_tokens(4, 0, length, r.shape.vocab)
    s.decode_step([1, 2])            # the other client holds a page between
    s.reset(0)
    s.prefill(0, prompt[:20])
    s.prefill(0, prompt[20:-1])
    plain.feed(prompt[:20])
    plain.feed(prompt[20:-1])
    toks = [prompt[-1], 5]
    for _ in range(6):
        best, got = s.decode_step(toks, want_logits=True)
        want = plain.feed([toks[0]])
        assert close(got[0], want, plain.tied) and picked(best[0], want, plain.tied)
        toks = best
    s.close()
    m.close()


@pytest.mark.parametrize("name", ["olmoe-q6_k", "qwen3moe-q5_k"])
def test_routed_models_serve_from_pages(name):
    # the same products and routing as an fp32 session's, keys and values to 8 bits:
    # the first token attends to itself alone, with its value off by half a step of
    # at most 1/64 of its largest
    r = configs.TINY[name]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    a, b = eb.Session(m, 2, 40), eb.Session(m, 2, 40, paged=(6, 16))
    _, want = a.decode_step([3, 4], want_logits=True)
    _, got = b.decode_step([3, 4], want_logits=True)
    assert np.abs(got - want).max() <= np.abs(want).max() / 64
    for _ in range(20):
        b.decode_step([5, 6])
    assert np.isfinite(b.decode_step([7, 8], want_logits=True)[1]).all()
    for s in (a, b):
        s.close()
    m.close()


def test_pages_run_out_and_come_back():
    r = configs.TINY["qwen3-q6_k"]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    s = eb.Session(m, 3, 64, paged=(4, 16))
    s.prefill(0, list(range(33)))    # three pages
    assert s.free_pages == 1
    with pytest.raises(SpmError) as e:
        s.prefill(1, list(range(17)))
    assert e.value.name == "SPM_E_CONTEXT" and s.free_pages == 1 and s.length(1) == 0
    with pytest.raises(SpmError):
        s.decode_step([1, 2, 3])     # two new pages
    assert [s.length(i) for i in range(3)] == [33, 0, 0]
    s.decode_step([1, 2])
    assert s.free_pages == 0 and [s.length(i) for i in range(3)] == [34, 1, 0]
    with pytest.raises(SpmError):
        s.decode_step([1, 2, 3])
    first = s.decode_step([7, 8], want_logits=True)[1][1]
    s.reset(0)
    assert s.free_pages == 3 and s.length(0) == 0
    s.decode_step([1, 2, 3])         # pages that another client held
    plain = Plain(r, 16, 64)
    plain.feed([2])
    want = plain.feed([8])
    assert close(first, want, plain.tied)
    s.reset(1)
    s.reset(1)
    s.reset(2)
    assert s.free_pages == 3
    s.close()
    with pytest.raises(SpmError):
        eb.Session(m, 1, 64).free_pages
    m.close()


@pytest.mark.parametrize("pages,page", [(0, 16), (-1, 16), (4, 24), (4, 0), (4, 512), (1 << 27, 64)])
def test_paged_sessions_refused(pages, page):
    r = configs.TINY["qwen3-q6_k"]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    with pytest.raises(SpmError):
        eb.Session(m, 1, 64, paged=(pages, page))
    m.close()


def test_paged_session_refuses_a_head_dim_that_the_cache_does_not_take():
    r = configs.TINY["llama-q8_0"]   # head_dim 16
    m = eb.Model(eb.synth_gguf(r), r.shape)
    with pytest.raises(SpmError) as e:
        eb.Session(m, 1, 64, paged=(4, 16))
    assert e.value.name == "SPM_E_ARG"
    m.close()


# ------------------------------------------------------------- sampled steps --
HOW = [None, Sampling(0.0), Sampling(0.7, top_k=5, seed=2), Sampling(1.3, top_p=0.8, min_p=0.01, seed=3)]


def test_sampled_steps_draw_from_the_steps_logits():
    r = configs.TINY["llama-q6_k"]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    s, plain = eb.Session(m, 4, 40), eb.Session(m, 4, 40)
    rng = np.random.default_rng(0)
    toks = [1, 2, 3, 4]
    for _ in range(12):
        u = [float(v) for v in rng.random(4, dtype=np.float32)]
        nxt, arg, logits = s.decode_step_sampled(toks, HOW, u, want_logits=True)
        best, want = plain.decode_step(toks, want_logits=True)
        assert arg == best and np.array_equal(logits, want)
        for i, w in enumerate(HOW):
            if w is None:
                assert nxt[i] == arg[i]
            else:
                f = [float(np.float32(v)) for v in (w.temperature, w.top_p, w.min_p)]
                assert nxt[i] == ref.pick(logits[i].astype(np.float64), f[0], w.top_k, f[1], f[2], u[i])[0]
        toks = nxt
    for bad in (dict(u=[0.5, 0.5, 0.5, 1.0]), dict(u=[0.5, -0.1, 0.5, 0.5]), dict(u=[0.5]), dict(how=HOW[:2]),
                dict(tokens=[1, 2, 3, 10 ** 6]), dict(u=[math.nan] * 4)):
        with pytest.raises(SpmError):
            s.decode_step_sampled(bad.get("tokens", toks), bad.get("how", HOW), bad.get("u", [0.5] * 4))
    assert s.length(0) == 12
    for x in (s, plain):
        x.close()
    m.close()


@pytest.mark.parametrize("paged", [None, (40, 16)])
def test_serving_with_sampling_does_not_depend_on_the_batch(paged):
    r = configs.TINY["qwen3-q6_k"]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    prompts = [configs.prompt_tokens(5, i, n, r.shape.vocab) for i, n in enumerate((4, 9, 6))]
    how = [Sampling(0.9, top_k=20, seed=1), None, Sampling(1.0, top_p=0.9, seed=2)]
    both, _ = eb.serve(m, prompts, 8, sampling=how, paged=paged)
    alone = [eb.serve(m, [p], 8, sampling=[w], paged=paged)[0][0][:8] for p, w in zip(prompts, how)]
    assert [b[:8] for b in both] == alone
    assert alone[1] == eb.serve(m, [prompts[1]], 8, paged=paged)[0][0][:8]
    s = eb.Session(m, 2, 40, paged=paged)
    requests = [Request(p, 8, arrival=i, sampling=w) for i, (p, w) in enumerate(zip(prompts, how))]
    assert serve_continuous(s, requests) == alone
    s.close()
    with pytest.raises(ValueError):
        eb.serve(m, prompts, 8, sampling=how[:2])
    m.close()
