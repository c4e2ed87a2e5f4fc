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

from typing import Optional, Tuple

import torch

from . import _lib
from .attention import HEAD_DIM, KV_HEADS, Context, EncodableRun, _as_stream, _launch, _need

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
FORMATS = {"none": _lib.KV_PLAIN, "e4m3": _lib.KV_E4M3, "int8": _lib.KV_INT8}
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_FORMAT_OF = {code: name for name, code in _CODES.items()}


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
        with their scales (uint8 [slots, heads]: e + 127, where 2^e is a number of
        ``dtype``), or 16-bit values without.
        ``dtype``: of the rows written and read (float16 unless k has one)."""
        self = cls.__new__(cls)
        if dtype is None:
            dtype = k.dtype if k.dtype in _DTYPES else torch.float16
        self._set(k, v, k_scale, v_scale, dtype)
        return self

    def _set(self, k, v, k_scale, v_scale, dtype) -> None:
        code = _DTYPES.get(dtype)
        _need(code is not None, "dtype must be float16 or bfloat16")
        kind, index, shape = k.dtype, k.get_device(), k.shape
        fmt = _FORMAT_OF.get(kind)
        if fmt is None and kind == dtype:
            fmt = "none"
        _need(fmt is not None, "k must hold float8_e4m3fn, int8 or values of dtype")
        _need(index >= 0 and len(shape) == 3 and v.shape == shape and v.dtype == kind
              and v.get_device() == index and k.is_contiguous() and v.is_contiguous(),
              "k and v must be contiguous CUDA tensors [slots, heads, head_dim] of one kind")
        slots, heads, dim = shape
        ks = vs = 0
        if fmt == "none":
            _need(k_scale is None and v_scale is None, "16-bit values have no scales")
        else:
            _need(k_scale is not None and v_scale is not None
                  and k_scale.shape == (slots, heads) and v_scale.shape == (slots, heads)
                  and k_scale.dtype == torch.uint8 and v_scale.dtype == torch.uint8
                  and k_scale.get_device() == index and v_scale.get_device() == index
                  and k_scale.is_contiguous() and v_scale.is_contiguous(),
                  "scales must be contiguous uint8 tensors [slots, heads]")
            ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.format, self.dtype, self.index = fmt, dtype, index
        self.slots, self.heads, self.head_dim = slots, heads, dim
        self.struct = _lib.kv_cache(code, FORMATS[fmt], heads, dim, slots, k.data_ptr(),
                                    v.data_ptr(), ks, vs)

    @property
    def device(self) -> torch.device:
        return self.k.device

    def nbytes(self) -> int:
        held = (self.k, self.v, self.k_scale, self.v_scale)
        return sum(t.numel() * t.element_size() for t in held if t is not None)


def _slots(slots: torch.Tensor, index: int) -> int:
    _need(slots.get_device() == index and slots.dtype == torch.int32 and slots.is_contiguous(),
          "slots must be a contiguous int32 tensor on the cache's device")
    return slots.numel()


def _rows(t: torch.Tensor, name: str, cache: KVCache, tokens: int, index: int) -> int:
    """Checks rows [tokens, heads, head_dim] of the cache; their token stride."""
    heads, dim = cache.heads, cache.head_dim
    if t.shape != (tokens, heads, dim) or t.dtype != cache.dtype or t.get_device() != index:
        raise ValueError(f"{name} must be [tokens, heads, head_dim] of the cache's dtype and "
                         "device")
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s1 != dim and heads != 1):
        raise ValueError(f"{name}: a token's heads must be contiguous")
    return s0 if tokens > 1 else heads * dim  # a single row has no stride of its own


def _write_args(ctx: Context, cache: KVCache, k, v, slots) -> tuple:
    index = ctx.device
    _need(cache.index == index, "the cache must be on the kernel's device")
    n = _slots(slots, index)
    return (cache.struct, k.data_ptr(), _rows(k, "k", cache, n, index),
            v.data_ptr(), _rows(v, "v", cache, n, index), slots.data_ptr(), n)


def _read_args(ctx: Context, cache: KVCache, slots, k_output, v_output):
    """(k's output, v's output, the C call's arguments); outputs of None are made"""
    index = ctx.device
    _need(cache.index == index, "the cache must be on the kernel's device")
    n = _slots(slots, index)
    width = cache.heads * cache.head_dim
    if k_output is None:
        k_output = cache.k.new_empty((n, cache.heads, cache.head_dim), dtype=cache.dtype)
    else:
        _need(_rows(k_output, "k_output", cache, n, index) == width, "k_output must be contiguous")
    if v_output is None:
        v_output = torch.empty_like(k_output)
    else:
        _need(_rows(v_output, "v_output", cache, n, index) == width, "v_output must be contiguous")
    return k_output, v_output, (cache.struct, slots.data_ptr(), n,
                                k_output.data_ptr(), v_output.data_ptr())


class KVCacheKernel:
    """Writing rows into a cache's slots, and reading them back."""

    def __init__(self, device=None):
        self.ctx = Context.for_device(device)

    def create_write_run(self, cache: KVCache, k: torch.Tensor, v: torch.Tensor,
                         slots: torch.Tensor) -> EncodableRun:
        """Row t of k and v goes into slot ``slots[t]``, which must differ within
        a call; a slot outside the cache skips its row."""
        args = _write_args(self.ctx, cache, k, v, slots)
        lib, h = self.ctx.lib, self.ctx.handle
        return EncodableRun(lambda s: lib.qwa_kv_cache_write(h, *args, s), self.ctx,
                            "KV cache write")

    def create_read_run(self, cache: KVCache, slots: torch.Tensor, k_output: torch.Tensor,
                        v_output: torch.Tensor) -> EncodableRun:
        """k_output, v_output [tokens, heads, head_dim]; a slot outside the cache
        gives zeros."""
        _need(k_output is not None and v_output is not None, "outputs are required")
        _, _, args = _read_args(self.ctx, cache, slots, k_output, v_output)
        lib, h = self.ctx.lib, self.ctx.handle
        return EncodableRun(lambda s: lib.qwa_kv_cache_read(h, *args, s), self.ctx,
                            "KV cache read")


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                   stream=None) -> None:
    """Quantise rows k, v [tokens, heads, head_dim] into the cache's ``slots``
    (int32 [tokens], all different)."""
    ctx = Context.for_device(cache.index)
    _launch(ctx, stream, ctx.lib.qwa_kv_cache_write, *_write_args(ctx, cache, k, v, slots))


def kv_cache_read(cache: KVCache, slots: torch.Tensor, k_out: Optional[torch.Tensor] = None,
                  v_out: Optional[torch.Tensor] = None, stream=None
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [tokens, heads, head_dim] of ``slots`` in the cache's dtype. Outputs that
    the call makes are of ``stream``."""
    ctx = Context.for_device(cache.index)
    if stream is not None:
        with torch.cuda.stream(_as_stream(stream, ctx.device)):
            return kv_cache_read(cache, slots, k_out, v_out)
    k_out, v_out, args = _read_args(ctx, cache, slots, k_out, v_out)
    _launch(ctx, stream, ctx.lib.qwa_kv_cache_read, *args)
    return k_out, v_out
