"""Sampling from logits on the device: temperature, top-k, top-p and min-p from
given random numbers (spm_sample).

The reference picks greedily (spm-batch/examples/serve-demo.rs:74-79);
``engine.Session.decode_step_sampled``, ``engine.serve`` and
``scheduler.serve_continuous`` draw with ``Sampling``."""
from __future__ import annotations

import dataclasses
from typing import NamedTuple

import numpy as np
import torch

from ._lib import SpmError, call
from .kv8 import _cuda, _dtype, _forward_only, _on


@dataclasses.dataclass(frozen=True)
class Sampling:
    """How a request's tokens are drawn.  temperature 0 takes the largest logit;
    top_k 0, top_p 1 and min_p 0 are off; a request's numbers come from its seed."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self):
        if not self.temperature >= 0 or not 0 <= self.top_k < 2 ** 31 or not 0 <= self.top_p or not 0 <= self.min_p <= 1:
            raise ValueError("temperature, top_k and top_p are not negative, top_k is under 2^31, min_p lies in [0, 1]")

    def numbers(self) -> np.random.Generator:
        return np.random.default_rng(self.seed)


class Picks(NamedTuple):
    """Per row: the token (-1 where nothing can be picked), how many were kept, the pick's share of their mass."""
    token: torch.Tensor
    kept: torch.Tensor
    prob: torch.Tensor


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, stream=None) -> Picks:
    """A pick per row of logits [rows, vocab] with the uniform numbers u [rows].

    temperature, top_p, min_p (float32) and top_k (int32) are tensors of one
    value per row, or None for off; see spm_sample for what they do."""
    index = _cuda(logits, "logits")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise SpmError(-1, "logits must be rows x vocab, contiguous along vocab")
    _forward_only(logits, "logits")
    n, vocab = logits.shape

    def per_row(t, what, dtype=torch.float32):
        if t is None:
            return None
        if t.dtype is not dtype or t.get_device() != index or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
            raise SpmError(-1, f"{what} must be a contiguous {dtype} tensor of one value per row on cuda:{index}")
        return t.data_ptr()

    if u is None:
        raise SpmError(-1, "u: one uniform number per row")
    args = (per_row(temperature, "temperature"), per_row(top_k, "top_k", torch.int32), per_row(top_p, "top_p"),
            per_row(min_p, "min_p"), per_row(u, "u"))
    dt = _dtype(logits, "logits")
    raw, scratch = _on(index, stream)
    with scratch:
        token, kept, prob = u.new_empty(n, dtype=torch.int32), u.new_empty(n, dtype=torch.int32), u.new_empty(n)
    call("spm_sample", index, dt, logits.data_ptr(), logits.stride(0), n, vocab, *args, token.data_ptr(), kept.data_ptr(),
         prob.data_ptr(), raw)
    return Picks(token, kept, prob)
