"""A key/value cache in 8 bits: quantised as it is written, read back, or read
by ``prefix.prefix_attention`` in place.

``KVCache`` holds ``k`` and ``v`` of ``slots`` rows. Formats:

* ``"e4m3"``: float8_e4m3fn codes, and per (slot, head) a power-of-two scale held
  as the byte e + 127;
* ``"int8"``: the same with whole numbers of -127..127, finer where a head's
  values are of one size;
* ``"none"``: the 16-bit values.

Scales are powers of two, so a value is rounded once, and code * 2^e is exact in
float16 and bfloat16 (csrc/kv_cache.cu has the rule). Launches are the kernels of
csrc/kv_cache.cu through the C ABI. The reference keeps no cache.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .attention import HEAD_DIM, KV_HEADS, Context, EncodableRun, _need, _ptr, encode_run

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
FORMATS = {"none": _lib.KV_PLAIN, "e4m3": _lib.KV_E4M3, "int8": _lib.KV_INT8}
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class KVCache:
    """Keys and values of ``slots`` rows, [slots, heads, head_dim] each."""

    def __init__(self, slots: int, format: str = "e4m3", heads: int = KV_HEADS,
                 head_dim: int = HEAD_DIM, dtype: torch.dtype = torch.float16, device=None):
        _need(format in FORMATS, f"format must be one of {sorted(FORMATS)}")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None \
            else torch.device(device)
        shape = (slots, heads, head_dim)
        code = _CODES.get(format, dtype)
        scales = None
        if format != "none":
            scales = [torch.full((slots, heads), 127, dtype=torch.uint8, device=device)
                      for _ in range(2)]
        self._set(torch.zeros(shape, dtype=code, device=device),
                  torch.zeros(shape, dtype=code, device=device),
                  scales[0] if scales else None, scales[1] if scales else None, dtype)

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
             v_scale: Optional[torch.Tensor] = None,
             dtype: Optional[torch.dtype] = None) -> "KVCache":
        """A cache over tensors that exist already: codes (float8_e4m3fn or int8)
        with their scales (uint8 [slots, heads]), or 16-bit values without.
        ``dtype``: of the rows written and read (float16 unless k has one)."""
        self = cls.__new__(cls)
        if dtype is None:
            dtype = k.dtype if k.dtype in _DTYPES else torch.float16
        self._set(k, v, k_scale, v_scale, dtype)
        return self

    def _set(self, k, v, k_scale, v_scale, dtype) -> None:
        _need(dtype in _DTYPES, "dtype must be float16 or bfloat16")
        fmt = {torch.float8_e4m3fn: "e4m3", torch.int8: "int8", dtype: "none"}.get(k.dtype)
        _need(fmt is not None, "k must hold float8_e4m3fn, int8 or values of dtype")
        _need(k.is_cuda and k.dim() == 3 and k.is_contiguous() and v.is_contiguous()
              and v.shape == k.shape and v.dtype == k.dtype and v.device == k.device,
              "k and v must be contiguous CUDA tensors [slots, heads, head_dim] of one kind")
        if fmt == "none":
            _need(k_scale is None and v_scale is None, "16-bit values have no scales")
        else:
            for s in (k_scale, v_scale):
                _need(s is not None and s.dtype == torch.uint8 and s.is_contiguous()
                      and s.device == k.device and s.shape == k.shape[:2],
                      "scales must be contiguous uint8 tensors [slots, heads]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.format, self.dtype = fmt, dtype
        self.slots, self.heads, self.head_dim = k.shape
        self.device = k.device
        self.struct = _lib.KvCacheStruct(_DTYPES[dtype], FORMATS[fmt], self.heads, self.head_dim,
                                         self.slots, k.data_ptr(), v.data_ptr(),
                                         k_scale.data_ptr() if k_scale is not None else None,
                                         v_scale.data_ptr() if v_scale is not None else None)

    def nbytes(self) -> int:
        held = (self.k, self.v, self.k_scale, self.v_scale)
        return sum(t.numel() * t.element_size() for t in held if t is not None)


def _slots(slots: torch.Tensor, device) -> int:
    _need(isinstance(slots, torch.Tensor) and slots.device == device
          and slots.dtype == torch.int32 and slots.is_contiguous(),
          "slots must be a contiguous int32 tensor on the cache's device")
    return slots.numel()


def _rows(t: torch.Tensor, name: str, cache: KVCache, tokens: int) -> None:
    _need(isinstance(t, torch.Tensor) and t.dtype == cache.dtype and t.device == cache.device
          and tuple(t.shape) == (tokens, cache.heads, cache.head_dim)
          and t.stride(2) == 1 and (t.stride(1) == cache.head_dim or cache.heads == 1),
          f"{name} must be [tokens, heads, head_dim] of the cache's dtype and device, "
          "a token's heads contiguous")


class KVCacheKernel:
    """Writing rows into a cache's slots, and reading them back."""

    def __init__(self, device=None):
        self.ctx = Context.for_device(device)

    def create_write_run(self, cache: KVCache, k: torch.Tensor, v: torch.Tensor,
                         slots: torch.Tensor) -> EncodableRun:
        """Row t of k and v goes into slot ``slots[t]``, which must differ within
        a call; a slot outside the cache skips its row."""
        n = _slots(slots, cache.device)
        _rows(k, "k", cache, n)
        _rows(v, "v", cache, n)
        _need(cache.device.index == self.ctx.device, "the cache must be on the kernel's device")
        lib, h = self.ctx.lib, self.ctx.handle
        width = cache.heads * cache.head_dim
        # a single row has no stride of its own
        args = (ctypes.byref(cache.struct), _ptr(k), k.stride(0) if n > 1 else width, _ptr(v),
                v.stride(0) if n > 1 else width, _ptr(slots), n)
        return EncodableRun(lambda s: lib.qwa_kv_cache_write(h, *args, s), self.ctx,
                            "KV cache write")

    def create_read_run(self, cache: KVCache, slots: torch.Tensor, k_output: torch.Tensor,
                        v_output: torch.Tensor) -> EncodableRun:
        """k_output, v_output [tokens, heads, head_dim]; a slot outside the cache
        gives zeros."""
        n = _slots(slots, cache.device)
        for t, name in ((k_output, "k_output"), (v_output, "v_output")):
            _rows(t, name, cache, n)
            _need(t.is_contiguous(), f"{name} must be contiguous")
        _need(cache.device.index == self.ctx.device, "the cache must be on the kernel's device")
        lib, h = self.ctx.lib, self.ctx.handle
        args = (ctypes.byref(cache.struct), _ptr(slots), n, _ptr(k_output), _ptr(v_output))
        return EncodableRun(lambda s: lib.qwa_kv_cache_read(h, *args, s), self.ctx,
                            "KV cache read")


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                   stream=None) -> None:
    """Quantise rows k, v [tokens, heads, head_dim] into the cache's ``slots``
    (int32 [tokens])."""
    encode_run(stream, KVCacheKernel(cache.device.index).create_write_run(cache, k, v, slots))


def kv_cache_read(cache: KVCache, slots: torch.Tensor, k_out: Optional[torch.Tensor] = None,
                  v_out: Optional[torch.Tensor] = None, stream=None
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [tokens, heads, head_dim] of ``slots`` in the cache's dtype."""
    shape = (slots.numel(), cache.heads, cache.head_dim)
    if k_out is None:
        k_out = torch.empty(shape, dtype=cache.dtype, device=cache.device)
    if v_out is None:
        v_out = torch.empty(shape, dtype=cache.dtype, device=cache.device)
    encode_run(stream, KVCacheKernel(cache.device.index).create_read_run(cache, slots, k_out,
                                                                        v_out))
    return k_out, v_out
