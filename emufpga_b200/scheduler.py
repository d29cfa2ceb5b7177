"""Continuous batching over one decode session.

The reference serves a fixed batch in lockstep (spm-batch/examples/
serve-demo.rs:45-91): every client starts at tick 0 and the batch ends with
its longest client.  Here requests join free client slots while other
clients are decoding and leave as soon as they are done, so the weight sweep
of every step is shared by whichever requests are in flight.  Each request
follows serve-demo's per-client rule on its own clock: it feeds its prompt
one token per step, then feeds back its greedy pick, and produces `max_new`
tokens -- the same tokens it would produce served alone.

A step runs clients 0..n-1 where n-1 is the highest busy slot; a free slot
below that decodes a filler token and is reset before a request takes it
(or when its cache would otherwise fill).

With `prefill=True` a joining request's prompt, all but its last token, runs
at once through the session's `prefill` (the tensor-core prompt path) when
it takes its slot; it then feeds its last prompt token in the next step and
decodes from there -- the batched prefill for late joiners that the
reference's lockstep server lacks (docs/results.md:1189-1191).

A paged session's clients share one pool of pages.  There a request starts only
when the pool holds its last token's page beside those of all requests in
flight, a finished request's pages come back at once, and a free slot that
decodes filler tokens holds one page at most, so that no step runs out of pages.
"""
from __future__ import annotations

import dataclasses
from typing import Protocol, Sequence


@dataclasses.dataclass(frozen=True)
class Request:
    prompt: Sequence[int]
    max_new: int
    arrival: int = 0  # first step at which the request may start
    sampling: object = None  # a sampling.Sampling; None: greedy


class DecodeSession(Protocol):
    """What the scheduler needs from a session (engine.Session has it)."""

    max_clients: int
    context: int

    def reset(self, client: int) -> None: ...

    def length(self, client: int) -> int: ...

    def decode_step(self, tokens: Sequence[int], want_logits: bool = False): ...

    # only with a sampled request: (next ids, argmax ids, logits)
    def decode_step_sampled(self, tokens: Sequence[int], how: Sequence, u: Sequence[float], want_logits: bool = False): ...

    # only with prefill=True: run tokens for `client` at its next positions
    def prefill(self, client: int, tokens: Sequence[int]) -> None: ...

    # only of a paged session (page_tokens neither missing nor None): its pages' length, and how many are free
    # page_tokens: int
    # free_pages: int


def serve_continuous(session: DecodeSession, requests: Sequence[Request], filler: int = 0,
                     prefill: bool = False) -> list[list[int]]:
    """Serve `requests` on `session`; returns each request's produced tokens.

    Requests start in arrival order (ties in list order) as slots free up.
    With prefill, a starting request's prompt but its last token is run at
    once by session.prefill.  A request with `sampling` feeds back tokens drawn
    with it, from its own seed's numbers, one for each token it produces, so
    that its tokens do not depend on what else is served.  Raises ValueError when a request cannot fit the
    session's context, or a paged session's pages (all of which it takes: every client starts empty)."""
    for r in requests:
        if not r.prompt or r.max_new < 1:
            raise ValueError("a request needs a prompt and at least one new token")
        if len(r.prompt) + r.max_new > session.context:
            raise ValueError("a request does not fit the session's context")
    page = getattr(session, "page_tokens", None)
    need, pages = [0] * len(requests), 0
    if page:
        for s in range(session.max_clients):
            if session.length(s):
                session.reset(s)
        pages = session.free_pages
        # the last token produced is not fed back
        need = [-(-(len(r.prompt) + r.max_new - 1) // page) for r in requests]
        if max(need, default=0) > pages:
            raise ValueError("a request does not fit the session's pages")
    waiting = sorted(range(len(requests)), key=lambda i: (requests[i].arrival, i))
    out: list[list[int]] = [[] for _ in requests]
    active: dict[int, list[int]] = {}  # slot -> [request, local step, next token]
    numbers = [None if r.sampling is None else r.sampling.numbers() for r in requests]
    step = 0
    while waiting or active:
        for s in range(session.max_clients):
            if not waiting or requests[waiting[0]].arrival > step:
                break
            if s in active:
                continue
            if page:
                # every slot of a step: its request's pages, or a free slot's one
                slots = range(max([s, *active]) + 1)
                if sum(need[waiting[0]] if t == s else need[active[t][0]] if t in active else 1 for t in slots) > pages:
                    break
            r = waiting.pop(0)
            session.reset(s)
            prompt = requests[r].prompt
            if prefill and len(prompt) > 1:
                session.prefill(s, list(prompt[:-1]))
                active[s] = [r, len(prompt) - 1, prompt[-1]]
            else:
                active[s] = [r, 0, prompt[0]]
        if not active:
            step = requests[waiting[0]].arrival
            continue
        n = max(active) + 1
        for s in range(n):
            if s not in active and (session.length(s) + 1 >= session.context or page and session.length(s) >= page):
                session.reset(s)
        feed = [active[s][2] if s in active else filler for s in range(n)]
        how = [requests[active[s][0]].sampling if s in active else None for s in range(n)]
        if any(w is not None for w in how):
            # a number for every client that produces a token in this step
            u = [float(numbers[active[s][0]].random(dtype="float32"))
                 if how[s] is not None and active[s][1] + 1 >= len(requests[active[s][0]].prompt) else 0.0 for s in range(n)]
            best, _, _ = session.decode_step_sampled(feed, how, u)
        else:
            best, _ = session.decode_step(feed)
        for s in list(active):
            st = active[s]
            r, k = st[0], st[1]
            prompt = requests[r].prompt
            if k + 1 < len(prompt):
                st[2] = prompt[k + 1]
            else:
                out[r].append(best[s])
                st[2] = best[s]
            st[1] = k + 1
            if len(out[r]) >= requests[r].max_new:
                del active[s]
                if page:
                    session.reset(s)
        if page:
            for s in range(max(active, default=-1) + 1, n):
                if session.length(s):
                    session.reset(s)
        step += 1
    return out
