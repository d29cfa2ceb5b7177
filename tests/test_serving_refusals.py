"""Calls of the serving operators that the host refuses before any device work (no GPU needed)."""
import pytest

from emufpga_b200 import _lib
from test_serving_host import A, cache, planned, refused


@pytest.mark.parametrize("tokens", [2 ** 31 - 1, 2 ** 31 - 65536])
def test_a_slot_map_whose_indexes_pass_32_bits_is_refused(tokens):
    planned(tokens=tokens)
    refused("spm_kv8_append", cache(), _lib.F32, A, 64, 64, A, 64, 64, tokens, A, None)
