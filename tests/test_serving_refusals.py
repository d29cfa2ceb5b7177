"""Calls of the serving operators that the host refuses before any device work (no GPU needed)."""
import subprocess
import sys

import pytest

from emufpga_b200 import _lib, serve
from emufpga_b200.sampling import Sampling
from test_serving_host import A, cache, planned, refused


@pytest.mark.parametrize("tokens", [2 ** 31 - 1, 2 ** 31 - 65536])
def test_a_slot_map_whose_indexes_pass_32_bits_is_refused(tokens):
    planned(tokens=tokens)
    refused("spm_kv8_append", cache(), _lib.F32, A, 64, 64, A, 64, 64, tokens, A, None)


@pytest.mark.parametrize("top_k", [2 ** 31, 2 ** 32 + 1])
def test_a_top_k_past_32_bits_is_refused(top_k):
    # (a C int32 would hold -2^31, off, and 1, greedy)
    with pytest.raises(ValueError):
        Sampling(top_k=top_k)
    assert Sampling(top_k=2 ** 31 - 1).top_k == 2 ** 31 - 1


def test_the_package_does_not_load_torch_by_itself():
    code = ("from emufpga_b200 import *; import sys; assert 'torch' not in sys.modules; import emufpga_b200 as eb; "
            "eb.kv8.Cache, eb.sampling.Sampling; assert 'torch' in sys.modules")
    assert subprocess.run([sys.executable, "-c", code], capture_output=True, timeout=300).returncode == 0


@pytest.mark.parametrize("prompts,steps,ticks,pages", [([[1] * 5, [2]], 12, None, 1), ([[1] * 5, [2]], 13, None, 3),
                                                       ([[1], [2], [3]], 100, 33, 8)])
def test_serving_from_too_few_pages_is_refused_before_any_step(prompts, steps, ticks, pages):
    with pytest.raises(ValueError):
        serve(None, prompts, steps, max_ticks=ticks, paged=(pages, 16))
