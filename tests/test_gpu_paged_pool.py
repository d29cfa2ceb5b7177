"""Requests that come and go over a pool of pages smaller than all clients' contexts."""
import ctypes as C

import pytest
import torch

import emufpga_b200 as eb
from emufpga_b200 import _lib, configs
from emufpga_b200._lib import LLAMA, QWEN3
from emufpga_b200.sampling import Sampling
from emufpga_b200.scheduler import Request, serve_continuous

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("clients,pages", [(2, 5), (3, 6), (3, 4)])
def test_requests_share_a_small_pool(prefill, clients, pages):
    r = configs.TINY["qwen3-q6_k"]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    sizes = [(10, 10), (40, 20), (3, 5), (17, 30), (2, 1), (33, 16)]
    requests = [Request(configs.prompt_tokens(6, i, n, r.shape.vocab), new, arrival=2 * i,
                        sampling=Sampling(0.9, top_k=30, seed=i) if i % 2 else None) for i, (n, new) in enumerate(sizes)]
    s = eb.Session(m, clients, 64, paged=(pages, 16))
    s.decode_step([1] * clients)
    got = serve_continuous(s, requests, prefill=prefill)
    assert s.free_pages == pages
    one = eb.Session(m, 1, 64, paged=(4, 16))
    assert got == [serve_continuous(one, [q], prefill=prefill)[0] for q in requests]
    with pytest.raises(ValueError):
        serve_continuous(eb.Session(m, clients, 64, paged=(2, 16)), requests)
    for x in (s, one):
        x.close()
    m.close()


def test_prompts_take_no_device_memory_of_their_own():
    # a prompt's scratch is there before its pages are taken: nothing can fail between the two
    r = configs.TINY["qwen3-q6_k"]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    s = eb.Session(m, 2, 8192, paged=(1024, 16))
    s.prefill(0, [1, 2])             # the layers' buffers
    s.decode_step([1, 2])
    before = torch.cuda.mem_get_info()[0]
    for n in (20, 64, 100, 300, 2500):
        s.reset(0)
        s.prefill(0, configs.prompt_tokens(7, 0, n, r.shape.vocab))
        assert s.length(0) == n and s.free_pages == 1024 - -(-n // 16) - 1
    assert torch.cuda.mem_get_info()[0] == before
    s.close()
    m.close()


@pytest.mark.parametrize("paged", [None, (40, 16)])
def test_prompts_do_not_depend_on_the_default_stream(paged):
    # the first prompt's buffers are cleared in order with what uses them, whatever else the device does
    r = configs.TINY["qwen3-q6_k"]
    m = eb.Model(eb.synth_gguf(r), r.shape)
    prompt = configs.prompt_tokens(8, 0, 200, r.shape.vocab)
    want = None
    for busy in (False, True):
        s = eb.Session(m, 2, 300, paged=paged)
        if busy:
            torch.cuda._sleep(200_000_000)  # a tenth of a second of the default stream
        for _ in range(20):
            s.reset(0)
            s.prefill(0, prompt)
            _, got = s.decode_step([3, 4], want_logits=True)
            s.reset(1)
            want = got if want is None else want
            assert (got == want).all()
        torch.cuda.synchronize()
        s.close()
    m.close()


class QkArgs(C.Structure):
    """csrc/prefill.h's."""
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "kcache", "vcache", "pos", "k_out", "kplanes", "vplanes", "rope",
                                          "q_norm", "k_norm")]
    _fields_ += [(n, C.c_int32) for n in ("client", "layer", "layers", "context", "pos0", "heads", "kv_heads", "head_dim",
                                          "family")]
    _fields_ += [("eps", C.c_float)]


@pytest.mark.parametrize("family", [LLAMA, QWEN3])
def test_rows_without_a_position_are_left_as_they_are(family):
    # a plan that fails on the device gives positions of -1, before the first angle
    launch = _lib.lib()["_ZN3spm21launch_qk_rope_appendERKNS_6QkArgsEiP11CUstream_st"]
    launch.argtypes, launch.restype = [C.POINTER(QkArgs), C.c_int, C.c_void_p], C.c_int
    T, heads, kv_heads, dim, context = 5, 4, 2, 64, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(T, h * dim, device="cuda", generator=g) for h in (heads, kv_heads, kv_heads))
    rope = torch.randn(context, dim, device="cuda", generator=g)
    gains = torch.ones(dim, device="cuda")
    pos = torch.tensor([3, -1, 0, -1, 7], dtype=torch.int32, device="cuda")
    had = q.clone(), k.clone()
    a = QkArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), pos=pos.data_ptr(), k_out=k.data_ptr(), rope=rope.data_ptr(),
               q_norm=gains.data_ptr(), k_norm=gains.data_ptr(), layers=1, context=context, heads=heads, kv_heads=kv_heads,
               head_dim=dim, family=family, eps=1e-5)
    torch.cuda.synchronize()
    assert launch(C.byref(a), T, None) == 0
    torch.cuda.synchronize()
    for now, then in zip((q, k), had):
        assert torch.equal(now[[1, 3]], then[[1, 3]])
        assert (now[[0, 2, 4]] != then[[0, 2, 4]]).any(1).all()
