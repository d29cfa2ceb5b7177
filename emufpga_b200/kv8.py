"""Page tables and a paged 8-bit KV cache on the device.

A serving tick: ``plan`` gives every request its pages and every token its
slot, from the requests' lengths; per layer ``Cache.append`` stores the tick's
keys and values and ``Cache.attention`` reads them.  Nothing synchronises or
leaves the device, and a tick can be captured into a CUDA graph.  What only the
device can see (a length past its table, a page that is not in the pool, an
empty stack of free pages) goes into a status word; ``check`` reads it and
raises.  The calls run on the current stream of the tensors' device, or on
``stream``, and have no backward pass (a tensor that requires a gradient is
refused).  The reference keeps f32 rows of one client (spm-kv/src/cache.rs:49-58);
see include/spmgpu.h for the definitions.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from typing import NamedTuple

import torch

from ._lib import BF16, F16, F32, Kv8, SpmError, call

DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
STATUS = {11: "a length is negative or past its table", 12: "more pages wanted than free",
          13: "more tokens than the slot map holds", 14: "more pages back than the pool has",
          15: "a page or slot is not in the pool", 16: "a request's rows are not what the call says",
          17: "a device wait gave up", 18: "a row gives back pages that its cached tokens keep"}


_I32 = torch.int32
_HERE = contextlib.nullcontext()
# the current stream's handle (torch.cuda.current_stream builds an object around it, 2 us)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _dtype(t: torch.Tensor, what: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise SpmError(-5, f"{what}: activations are float32, float16 or bfloat16, got {t.dtype}")
    return code


def _i32(t: torch.Tensor, what: str, index: int, n: int | None = None) -> int:
    """The address of a contiguous int32 tensor of n values on device `index`."""
    if t.dtype is not _I32 or t.get_device() != index or not t.is_contiguous():
        raise SpmError(-1, f"{what} must be a contiguous int32 tensor on cuda:{index}")
    if n is not None and t.numel() != n:
        raise SpmError(-1, f"{what} must have {n} values, got {t.numel()}")
    return t.data_ptr()


def _cuda(t: torch.Tensor, what: str) -> int:
    index = t.get_device()
    if index < 0:
        raise SpmError(-1, f"{what} must be a CUDA tensor")
    return index


def _forward_only(t: torch.Tensor, what: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise SpmError(-1, f"{what} requires a gradient, and the serving operators have none: call them under torch.no_grad()")


def _on(index: int, stream):
    """The raw stream to launch on, and a context in which scratch is allocated for it."""
    if stream is None:
        return _raw_stream(index), _HERE
    return stream.cuda_stream, torch.cuda.stream(stream)


def check(status: torch.Tensor) -> None:
    """Raise for a status word that a call has set, and clear it.  Waits for every stream of its device."""
    torch.cuda.synchronize(status.device)
    code = int(status.item())
    if code:
        status.zero_()
        torch.cuda.synchronize(status.device)  # before a call on any stream sets it again
        raise SpmError(-9 if code in (12, 13) else -8 if code == 17 else -1, STATUS.get(code, f"code {code}"))


class Plan(NamedTuple):
    """One tick's maps: per request ``starts`` (requests + 1) and ``lens``, per token ``positions`` and ``slots``."""
    starts: torch.Tensor
    lens: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


def plan(cached, new, table, free, count, page_tokens: int, tokens: int, ended=None, left=None, status=None,
         stream=None) -> Plan:
    """Block table and slot map of one tick (spm_page_plan).

    Row r of ``table`` (requests x width) holds ``cached[r]`` tokens and takes
    ``new[r]`` more; the pages of ``ended[r]`` tokens of its former request go
    back first (such a row has no cached tokens).  ``free`` is the stack of free pages, ``count`` its height (one
    int32), ``left`` (default: ``count``) receives the new height.  ``tokens``
    is the length of the slot map, -1 behind the last token."""
    index = _cuda(table, "table")
    if table.dim() != 2:
        raise SpmError(-1, "table must be requests x width")
    R, width = table.shape
    left = count if left is None else left
    if tokens < 0:
        raise SpmError(-1, "negative token count")
    args = (index, _i32(cached, "cached", index, R), _i32(new, "new", index, R),
            None if ended is None else _i32(ended, "ended", index, R), R, page_tokens, _i32(table, "table", index),
            width, _i32(free, "free", index), free.numel(), _i32(count, "count", index, 1),
            _i32(left, "left", index, 1), tokens)
    word = None if status is None else _i32(status, "status", index, 1)
    raw, scratch = _on(index, stream)
    with scratch:
        maps = table.new_empty(2 * R + 1 + 2 * tokens)
    starts, lens, positions, slots = maps.split_with_sizes((R + 1, R, tokens, tokens))
    at = maps.data_ptr()
    call("spm_page_plan", *args, at, at + 4 * (R + 1), at + 4 * (2 * R + 1), at + 4 * (2 * R + 1 + tokens), word, raw)
    return Plan(starts, lens, positions, slots)


class Pages:
    """The page tables of up to ``requests`` requests over a pool of ``pages`` pages, all free at first."""

    def __init__(self, requests: int, max_pages: int, pages: int, page_tokens: int, device: int = 0):
        dev = torch.device("cuda", device)
        self.page_tokens = page_tokens
        self.table = torch.full((requests, max_pages), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.count = torch.full((1,), pages, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)

    def plan(self, cached, new, tokens: int, ended=None, stream=None) -> Plan:
        return plan(cached, new, self.table, self.free, self.count, self.page_tokens, tokens, ended=ended,
                    status=self.status, stream=stream)

    def check(self) -> None:
        check(self.status)


class Cache:
    """One layer's keys and values: int8 codes [pages, kv_heads, page_tokens, head_dim] and a power-of-two
    scale for each (page, kv head)."""

    def __init__(self, pages: int, page_tokens: int, kv_heads: int, head_dim: int, device: int = 0):
        dev = torch.device("cuda", device)
        shape = (pages, kv_heads, page_tokens, head_dim)
        codes = [torch.zeros(shape, dtype=torch.int8, device=dev) for _ in range(2)]
        scales = [torch.zeros(shape[:2], dtype=torch.float32, device=dev) for _ in range(2)]
        self._take(codes[0], scales[0], codes[1], scales[1])

    @classmethod
    def over(cls, k_codes, k_scales, v_codes, v_scales) -> "Cache":
        """A cache over the caller's tensors."""
        self = cls.__new__(cls)
        self._take(k_codes, k_scales, v_codes, v_scales)
        return self

    def _take(self, k_codes, k_scales, v_codes, v_scales) -> None:
        self._index = _cuda(k_codes, "codes")
        dev = k_codes.device
        if k_codes.dim() != 4:
            raise SpmError(-1, "codes must be pages x kv_heads x page_tokens x head_dim")
        for c, s in ((k_codes, k_scales), (v_codes, v_scales)):
            if c.dtype is not torch.int8 or c.shape != k_codes.shape or c.device != dev or not c.is_contiguous():
                raise SpmError(-1, "codes must be contiguous int8 tensors of one shape and device")
            if s.dtype is not torch.float32 or s.shape != c.shape[:2] or s.device != dev or not s.is_contiguous():
                raise SpmError(-1, "scales must be contiguous float32 tensors of pages x kv_heads")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.pages, self.kv_heads, self.page_tokens, self.head_dim = k_codes.shape
        self.device = dev
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._c = Kv8(self._index, self.pages, self.page_tokens, self.kv_heads, self.head_dim, 0, k_codes.data_ptr(),
                      v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), self.status.data_ptr())
        self._ref = C.byref(self._c)
        self._work: dict = {}
        self._bytes(self.kv_heads, 0, 0, 0)  # refuses a shape that no call takes

    def _bytes(self, heads: int, requests: int, most: int, width: int) -> int:
        key = (heads, requests, most, width)
        n = self._work.get(key)
        if n is None:
            if len(self._work) >= 1024:  # (lengths of a long life)
                self._work.clear()
            v = C.c_uint64()
            call("spm_kv8_attention_workspace", self._ref, heads, requests, most, width, C.byref(v))
            n = self._work[key] = v.value
        return n

    def _rows(self, t, what: str) -> int:
        """Checks [tokens, heads, head_dim] rows (any strides over tokens and heads)."""
        if t.dim() != 3 or t.shape[2] != self.head_dim or t.get_device() != self._index:
            raise SpmError(-1, f"{what} must be tokens x heads x {self.head_dim} on {self.device}")
        if t.stride(2) != 1 and t.numel():
            raise SpmError(-1, f"{what} must be contiguous along head_dim")
        _forward_only(t, what)
        return t.data_ptr()

    def append(self, k, v, slots, stream=None) -> None:
        """Store rows k, v [tokens, kv_heads, head_dim] at ``slots`` (spm_kv8_append)."""
        kp, vp = self._rows(k, "k"), self._rows(v, "v")
        if k.shape != v.shape or k.dtype is not v.dtype or k.shape[1] != self.kv_heads:
            raise SpmError(-1, f"k and v must be of one type, tokens x {self.kv_heads} x {self.head_dim}")
        sp = _i32(slots, "slots", self._index, k.shape[0])
        raw = _raw_stream(self._index) if stream is None else stream.cuda_stream
        call("spm_kv8_append", self._ref, _dtype(k, "k"), kp, k.stride(0), k.stride(1), vp, v.stride(0), v.stride(1),
             k.shape[0], sp, raw)

    def values(self, pages=None, dtype=torch.float32, stream=None):
        """The values (k, v) that whole pages stand for: [n, kv_heads, page_tokens, head_dim] for the int32
        page numbers ``pages``, or for all (spm_kv8_values)."""
        n = self.pages if pages is None else pages.numel()
        ids = None if pages is None else _i32(pages, "pages", self._index)
        if dtype not in DTYPES:
            raise SpmError(-5, "values are float32, float16 or bfloat16")
        raw, scratch = _on(self._index, stream)
        with scratch:
            out = torch.empty((2, n, self.kv_heads, self.page_tokens, self.head_dim), dtype=dtype, device=self.device)
        k, v = out.unbind(0)
        call("spm_kv8_values", self._ref, DTYPES[dtype], ids, n, k.data_ptr(), v.data_ptr(), raw)
        return k, v

    def attention(self, q, starts, lens, table, most: int, scale: float | None = None, out=None, stream=None):
        """Causal attention of q [rows, heads, head_dim] over the cached tokens (spm_kv8_attention).

        Request r's rows starts[r] .. starts[r + 1] (at most ``most``) stand at
        the last of its lens[r] positions, whose pages are table[r].  ``scale``
        defaults to head_dim ** -0.5.  Rows of ``out`` that no request has are left
        as they were (zeros where ``out`` is not given); ``out`` may be ``q``."""
        qp, dt = self._rows(q, "q"), _dtype(q, "q")
        T, H, _ = q.shape
        if table.dim() != 2:
            raise SpmError(-1, "table must be requests x width")
        R, width = table.shape
        args = (_i32(starts, "starts", self._index, R + 1), _i32(lens, "lens", self._index, R), R, most,
                _i32(table, "table", self._index), width)
        raw, scratch = _on(self._index, stream)
        need = self._bytes(H, R, most, width)
        with scratch:
            clear = out is None
            if clear:
                out = q.new_empty(q.shape)
            elif out.shape != q.shape or out.dtype is not q.dtype:
                raise SpmError(-1, "out must have q's shape and type")
            work = table.new_empty(need // 4)
        op = out.data_ptr() if clear else self._rows(out, "out")
        call("spm_kv8_attention", self._ref, dt, qp, q.stride(0), q.stride(1), H, T, *args,
             head_scale(self.head_dim) if scale is None else scale, op, out.stride(0), out.stride(1), clear,
             work.data_ptr(), need, raw)
        return out

    def check(self) -> None:
        """Raise for what the device found wrong in the calls so far, on whichever stream (synchronises)."""
        check(self.status)


def head_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)
