"""Continuous batching host logic on CPU with a toy session whose greedy
pick depends only on the client's own history since its last reset (as in
the real engine, where clients share weights but nothing else)."""
import hashlib

import pytest

from emufpga_b200.scheduler import Request, serve_continuous


class ToySession:
    def __init__(self, max_clients, context, vocab=50):
        self.max_clients, self.context, self.vocab = max_clients, context, vocab
        self.hist = [[] for _ in range(max_clients)]
        self.steps = []
        self.prefills = []

    def reset(self, client):
        self.hist[client] = []

    def length(self, client):
        return len(self.hist[client])

    def prefill(self, client, tokens):
        # the prompt path: the same history as feeding the tokens one per step
        self.prefills.append((client, len(tokens)))
        self.hist[client].extend(tokens)

    def decode_step(self, tokens, want_logits=False):
        self.steps.append(len(tokens))
        best = []
        for i, t in enumerate(tokens):
            if len(self.hist[i]) >= self.context:
                raise RuntimeError("context exhausted")
            self.hist[i].append(t)
            h = hashlib.sha256(repr(self.hist[i]).encode()).digest()
            best.append(h[0] % self.vocab)
        return best, None


def alone(req, context=64):
    return serve_continuous(ToySession(1, context), [Request(req.prompt, req.max_new)])[0]


def test_each_request_gets_what_it_gets_alone():
    reqs = [Request([1, 2, 3], 5), Request([7], 9, arrival=2), Request([4, 4, 4, 4], 3, arrival=2),
            Request([9, 8], 6, arrival=5), Request([3, 1, 4, 1, 5], 4, arrival=6), Request([2], 2, arrival=30)]
    sess = ToySession(3, 64)
    got = serve_continuous(sess, reqs)
    for r, g in zip(reqs, got):
        assert g == alone(r)
        assert len(g) == r.max_new
    # never more clients in a step than slots, and slots were reused
    assert max(sess.steps) <= 3
    assert len(sess.steps) < sum(len(r.prompt) + r.max_new - 1 for r in reqs)


def test_single_request_matches_the_lockstep_rule():
    # serve-demo: prompt of L tokens, S generated tokens -> L + S - 1 steps
    sess = ToySession(1, 64)
    out = serve_continuous(sess, [Request([5, 6, 7, 8], 6)])
    assert len(out[0]) == 6
    assert len(sess.steps) == 4 + 6 - 1


def test_idle_slots_below_busy_ones_never_exhaust_the_context():
    # slot 0 finishes quickly; slot 1 runs long; slot 0 idles under it
    reqs = [Request([1], 1), Request([2, 3], 14)]
    got = serve_continuous(ToySession(2, 16), reqs)
    assert got[1] == alone(reqs[1], 16)


def test_requests_that_cannot_fit_are_refused():
    with pytest.raises(ValueError):
        serve_continuous(ToySession(2, 8), [Request([1] * 5, 4)])
    with pytest.raises(ValueError):
        serve_continuous(ToySession(2, 8), [Request([], 2)])


def test_prefill_of_joining_requests_changes_no_token():
    reqs = [Request([1, 2, 3, 9, 9], 5), Request([7], 9, arrival=2), Request([4, 4, 4, 4], 3, arrival=2),
            Request([5, 6, 7, 8, 1, 2], 4, arrival=6)]
    plain = ToySession(2, 32)
    fast = ToySession(2, 32)
    assert serve_continuous(fast, reqs, prefill=True) == serve_continuous(plain, reqs)
    # every prompt longer than one token went through prefill, all but its last token
    assert sorted(n for _, n in fast.prefills) == sorted(len(r.prompt) - 1 for r in reqs if len(r.prompt) > 1)
    assert len(fast.steps) < len(plain.steps)


class SampledSession:
    """A fake whose sampled step returns a token made of what it was given."""

    max_clients, context = 2, 64

    def __init__(self):
        self.lens, self.calls = [0, 0], []

    def reset(self, client):
        self.lens[client] = 0

    def length(self, client):
        return self.lens[client]

    def decode_step(self, tokens, want_logits=False):
        self.calls.append(("greedy", list(tokens)))
        for i in range(len(tokens)):
            self.lens[i] += 1
        return [t + 1 for t in tokens], None

    def decode_step_sampled(self, tokens, how, u, want_logits=False):
        self.calls.append(("sampled", list(tokens), list(how), list(u)))
        for i in range(len(tokens)):
            self.lens[i] += 1
        return [t + 1 if w is None else int(1000 * x) for t, w, x in zip(tokens, how, u)], None, None


def test_sampled_requests_draw_their_own_numbers():
    from emufpga_b200.sampling import Sampling

    how = [Sampling(seed=5), Sampling(seed=6)]

    def want(w, n):
        g = w.numbers()
        return [int(1000 * float(g.random(dtype="float32"))) for _ in range(n)]

    s = SampledSession()
    got = serve_continuous(s, [Request([1, 2, 3], 4, sampling=how[0]), Request([7], 2), Request([9, 9], 3, sampling=how[1])])
    assert got == [want(how[0], 4), [8, 9], want(how[1], 3)]
    # a greedy client's place in a sampled step has no settings, and a prompt's steps draw no number
    first = next(c for c in s.calls if c[0] == "sampled")
    assert first[2][1] is None and first[3] == [0.0, 0.0]
    s = SampledSession()
    assert serve_continuous(s, [Request([1], 2)]) == [[2, 3]] and all(c[0] == "greedy" for c in s.calls)


class PagedToySession(ToySession):
    """A toy session over one pool of pages: what finds too few free pages raises."""

    def __init__(self, max_clients, context, pages, page_tokens):
        super().__init__(max_clients, context)
        self.pages, self.page_tokens, self.least = pages, page_tokens, pages

    def held(self, extra=0):
        return sum(-(-(len(h) + (i < extra)) // self.page_tokens) for i, h in enumerate(self.hist))

    @property
    def free_pages(self):
        return self.pages - self.held()

    def prefill(self, client, tokens):
        super().prefill(client, tokens)
        if self.held() > self.pages:
            raise RuntimeError("pages exhausted")

    def decode_step(self, tokens, want_logits=False):
        if self.held(len(tokens)) > self.pages:
            raise RuntimeError("pages exhausted")
        got = super().decode_step(tokens)
        self.least = min(self.least, self.free_pages)
        return got


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("slots,context,pages,page,sizes", [
    (2, 64, 5, 16, [(10, 10), (40, 20)]),                            # an idle slot under a long request
    (2, 250, 16, 16, [(2, 8), (2, 200)]),
    (3, 64, 4, 16, [(1, 60), (5, 5), (30, 30), (2, 2)]),             # one request takes all pages: one after the other
    (8, 40, 10, 8, [(i % 7 + 1, 3 * i % 11 + 1) for i in range(30)]),
    (4, 32, 4, 8, [(3, 25), (1, 1), (1, 30), (8, 8), (9, 8), (16, 1)])])
def test_a_pool_smaller_than_all_clients_serves_every_request(prefill, slots, context, pages, page, sizes):
    reqs = [Request([(7 * i + j) % 50 for j in range(n)], new, arrival=i // 3) for i, (n, new) in enumerate(sizes)]
    sess = PagedToySession(slots, context, pages, page)
    sess.hist[slots - 1] = [1] * min(context, page + 1)              # what an earlier run left
    got = serve_continuous(sess, reqs, prefill=prefill)
    assert got == [alone(r, context) for r in reqs]
    assert sess.least >= 0 and sess.free_pages == pages              # all pages are back


def test_requests_share_a_pool_as_far_as_it_goes():
    # two requests of two pages each fit four pages together, the third one waits
    sess = PagedToySession(3, 64, 4, 16)
    serve_continuous(sess, [Request([1] * 16, 10)] * 3)
    assert max(sess.steps) == 2 and len(sess.steps) == 2 * 25


def test_a_request_that_no_pool_of_pages_holds_is_refused():
    with pytest.raises(ValueError):
        serve_continuous(PagedToySession(2, 64, 3, 16), [Request([1], 2), Request([1] * 30, 20)])
    got = serve_continuous(PagedToySession(2, 64, 3, 16), [Request([1] * 30, 19)])
    assert len(got[0]) == 19
