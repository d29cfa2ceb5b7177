"""The serving operators' refusals, which the host makes before any device work
(no GPU needed), and the plain forms' own invariants."""
import ctypes as C
import random

import numpy as np
import pytest

from emufpga_b200 import _lib
from emufpga_b200._lib import Kv8, SpmError, call
from emufpga_b200.sampling import Sampling
from serving_cases import plan, store

A = 1 << 20  # a 16-byte aligned address that no refused call follows


def cache(**kw):
    f = dict(device=0, pages=4, page_tokens=16, kv_heads=2, head_dim=64, k_codes=A, v_codes=A, k_scales=A, v_scales=A,
             status=None)
    f.update(kw)
    return C.byref(Kv8(f["device"], f["pages"], f["page_tokens"], f["kv_heads"], f["head_dim"], 0, f["k_codes"],
                       f["v_codes"], f["k_scales"], f["v_scales"], f["status"]))


def refused(name, *args, code="SPM_E_ARG"):
    with pytest.raises(SpmError) as e:
        call(name, *args)
    assert e.value.name == code, e.value
    assert str(e.value)


BAD_CACHES = [dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=512), dict(head_dim=80), dict(head_dim=0),
              dict(kv_heads=0), dict(pages=-1), dict(pages=1 << 27), dict(k_codes=None), dict(v_scales=None),
              dict(k_codes=A + 8)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_cache_shapes_refused(bad):
    bad = dict(bad)
    if bad.get("pages") == 1 << 27:
        bad["page_tokens"] = 256  # 2^35 slots
    refused("spm_kv8_append", cache(**bad), _lib.F32, A, 64, 64, A, 64, 64, 1, A, None)
    refused("spm_kv8_values", cache(**bad), _lib.F32, None, 1, A, A, None)
    n = C.c_uint64()
    refused("spm_kv8_attention_workspace", cache(**bad), 2, 1, 1, 1, C.byref(n))


def test_append_and_values_refused():
    refused("spm_kv8_append", None, _lib.F32, A, 64, 64, A, 64, 64, 1, A, None)
    refused("spm_kv8_append", cache(), _lib.Q8_0, A, 64, 64, A, 64, 64, 1, A, None, code="SPM_E_ENCODING")
    refused("spm_kv8_append", cache(), _lib.F32, A, 64, 64, A, 64, 64, -1, A, None)
    refused("spm_kv8_append", cache(), _lib.F32, None, 64, 64, A, 64, 64, 1, A, None)
    refused("spm_kv8_append", cache(), _lib.F32, A, 64, 64, A, 64, 64, 1, None, None)
    refused("spm_kv8_values", cache(), _lib.BF16, None, 1, A + 4, A, None)
    refused("spm_kv8_values", cache(), 7, None, 1, A, A, None, code="SPM_E_ENCODING")
    refused("spm_kv8_values", cache(), _lib.F32, None, -1, A, A, None)
    call("spm_kv8_append", cache(), _lib.F32, None, 64, 64, None, 64, 64, 0, None, None)  # nothing to do
    call("spm_kv8_values", cache(), _lib.F32, None, 0, A, A, None)


def attend(c=None, dtype=_lib.F32, q=A, heads=4, rows=2, starts=A, lens=A, requests=2, most=1, table=A, width=3, out=A,
           work=A, size=1 << 40, clear=0, code="SPM_E_ARG"):
    refused("spm_kv8_attention", c or cache(), dtype, q, 256, 64, heads, rows, starts, lens, requests, most, table, width,
            0.125, out, 256, 64, clear, work, size, None, code=code)


def test_attention_refused():
    attend(heads=3)
    attend(heads=0)
    attend(dtype=2, code="SPM_E_ENCODING")
    for name in ("q", "starts", "lens", "table", "out", "work"):
        attend(**{name: None})
    attend(rows=-1)
    attend(requests=-1)
    attend(most=-1)
    attend(width=1 << 28)
    attend(size=15)
    attend(work=A + 8)
    attend(requests=1 << 20, most=1 << 20)
    attend(most=(1 << 30) - 1)
    attend(heads=1 << 30, most=1)
    for name in ("q", "starts", "out", "work"):
        attend(requests=0, clear=1, **{name: None})
    n = C.c_uint64()
    call("spm_kv8_attention_workspace", cache(), 4, 2, 1, 3, C.byref(n))
    attend(size=n.value - 1)
    call("spm_kv8_attention", cache(), _lib.F32, None, 256, 64, 4, 0, None, None, 0, 1, None, 3, 0.125, None, 256, 64, 0,
         None, 0, None)  # no requests: nothing to do


def planned(requests=2, page=16, width=4, pages=8, tokens=8, code="SPM_E_ARG", **kw):
    f = dict(cached=A, fresh=A, ended=None, table=A, free=A, count=A, left=A, starts=A, lens=A, positions=A, slots=A)
    f.update(kw)
    refused("spm_page_plan", 0, f["cached"], f["fresh"], f["ended"], requests, page, f["table"], width, f["free"], pages,
            f["count"], f["left"], tokens, f["starts"], f["lens"], f["positions"], f["slots"], None, None, code=code)


def test_plan_refused():
    planned(requests=-1)
    planned(requests=8193)
    planned(page=17)
    planned(page=8)
    planned(tokens=-1)
    planned(pages=-1)
    planned(width=1 << 28)
    planned(pages=1 << 28)
    for name in ("cached", "fresh", "table", "free", "count", "left", "starts", "lens", "positions", "slots"):
        planned(**{name: None})


def drawn(rows=1, vocab=10, dtype=_lib.F32, code="SPM_E_ARG", **kw):
    f = dict(logits=A, u=A, token=A)
    f.update(kw)
    refused("spm_sample", 0, dtype, f["logits"], vocab, rows, vocab, None, None, None, None, f["u"], f["token"], None, None,
            None, code=code)


def test_sample_refused():
    drawn(rows=-1)
    drawn(vocab=0)
    drawn(vocab=(1 << 19) + 1)
    drawn(dtype=13, code="SPM_E_ENCODING")
    for name in ("logits", "u", "token"):
        drawn(**{name: None})
    call("spm_sample", 0, _lib.F32, None, 1, 0, 1, None, None, None, None, None, None, None, None, None)  # no rows


def test_sampling_settings_refused():
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-2), dict(top_p=-0.1), dict(min_p=1.5)):
        with pytest.raises(ValueError):
            Sampling(**bad)
    a, b = Sampling(seed=3).numbers(), Sampling(seed=3).numbers()
    assert a.random() == b.random()


def test_no_device_is_an_error():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    refused("spm_sample", 0, _lib.F32, A, 10, 1, 10, None, None, None, None, A, A, None, None, None, code="SPM_E_NO_DEVICE")


@pytest.mark.parametrize("seed", range(4))
def test_a_page_filled_token_by_token_stays_within_a_step(seed):
    # the scale may grow at every token; each rounding adds half a step of its
    # own scale, and scales double, so the total stays under one final step
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((16, 1, 8)) * 2.0 ** np.sort(rng.uniform(-8, 8, 16))[:, None, None]
    codes, scales = np.zeros((1, 1, 16, 8)), np.zeros((1, 1))
    for t in range(16):
        store(x[t:t + 1], [t], codes, scales)
    assert np.abs(codes).max() <= 127
    assert np.abs(codes[0, 0] * scales[0, 0] - x[:, 0]).max() <= scales[0, 0]


def test_plan_serves_many_ticks_without_losing_a_page():
    rng = random.Random(7)
    R, P, W, N = 5, 16, 6, 24
    table, free, top = [[-1] * W for _ in range(R)], list(range(N)), N
    held = [0] * R
    for _ in range(200):
        ended = [h if h and rng.random() < 0.2 else 0 for h in held]
        cached = [0 if e else h for h, e in zip(held, ended)]
        back = sum(-(-e // P) for e in ended)
        new = [rng.choice([0, 1, 1, 20]) for _ in range(R)]
        new = [min(n, W * P - c) for n, c in zip(new, cached)]
        if sum(-(-(c + n) // P) + -c // P for c, n in zip(cached, new)) > top + back:
            new = [0] * R
        *_, slots, top = plan(cached, new, ended, table, free, top, P, 200)
        held = [c + n for c, n in zip(cached, new)]
        used = [table[r][j] for r in range(R) for j in range(-(-held[r] // P))]
        assert sorted(used + free[:top]) == list(range(N))
        assert len({s for s in slots if s >= 0}) == sum(new)
