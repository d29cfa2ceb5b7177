"""Requests that come and go over a pool of pages smaller than all clients' contexts."""
import pytest
import torch

import emufpga_b200 as eb
from emufpga_b200 import configs
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
