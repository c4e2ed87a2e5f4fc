"""Rotary positions on their own: the (cos, sin) table and its application.

``QKNormRopeKernel`` rotates behind the Q/K norm, whole heads in halves, from
position 0 (src/webgpu/ops.ts:104-166, table model.ts:76-83). This module has
the rotation alone, for q and k that are normed already or not at all: both pair
layouts, a part of the head, any positions, the way back (the gradient), and
tables for contexts longer than the model's (linear, ntk, yarn, llama3). A
table with ``rotary_dim`` 128 is also a ``rope_table`` for the fused kernels;
its rows from P on serve requests that begin at position P.

Launches are the kernels of csrc/rope.cu through the C ABI.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .attention import ROPE_THETA, Context, EncodableRun, _as_stream, _launch, _need

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_LAYOUTS = {"half": _lib.ROPE_HALF, "interleaved": _lib.ROPE_INTERLEAVED}


@dataclass(frozen=True)
class RopeScaling:
    """How frequencies change for longer contexts (include/qwa.h has the rules).
    ``attention_factor`` None: yarn's own, 0.1 ln(factor) + 1."""
    kind: str = "none"
    factor: float = 1.0
    original_positions: float = 0.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: Optional[float] = None
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0

    def struct(self) -> "_lib.RopeScalingStruct":
        _need(self.kind in _lib.ROPE_SCALING,
              f"scaling kind must be one of {sorted(_lib.ROPE_SCALING)}")
        _need(self.attention_factor is None
              or (self.attention_factor > 0 and math.isfinite(self.attention_factor)),
              "attention_factor must be a finite number above 0")
        return _lib.RopeScalingStruct(_lib.ROPE_SCALING[self.kind], self.factor,
                                      self.original_positions, self.beta_fast, self.beta_slow,
                                      self.attention_factor or 0.0, self.low_freq_factor,
                                      self.high_freq_factor)


def rope_table(positions: int, rotary_dim: int = 128, theta: float = ROPE_THETA,
               scaling: Optional[RopeScaling] = None, first: int = 0, device=None,
               out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """f32 [positions, rotary_dim / 2, 2]: (cos, sin) of positions ``first``,
    ``first`` + 1, ... with the angle in 64 bits. A table that the call makes is of
    ``stream``."""
    _need(0 <= positions < 2 ** 31 and rotary_dim >= 2,
          "positions must be in 0..2^31-1 and rotary_dim >= 2")
    _need(rotary_dim < 2 ** 31 and -2 ** 63 <= first < 2 ** 63,
          "rotary_dim must be a 32-bit number, first a 64-bit one")
    if out is not None:
        _need(out.is_cuda and out.dtype == torch.float32 and out.is_contiguous()
              and out.numel() >= positions * (rotary_dim // 2) * 2,
              "out must be a contiguous CUDA float32 tensor of [positions, rotary_dim / 2, 2]")
        device = out.device
    device = torch.device("cuda") if device is None else torch.device(device)
    ctx = Context.for_device(device.index)
    if stream is not None:
        with torch.cuda.stream(_as_stream(stream, ctx.device)):
            return rope_table(positions, rotary_dim, theta, scaling, first,
                              torch.device("cuda", ctx.device), out)
    if out is None:
        out = torch.empty(positions, rotary_dim // 2, 2, dtype=torch.float32,
                          device=torch.device("cuda", ctx.device))
    s = scaling.struct() if scaling is not None else None
    _launch(ctx, stream, ctx.lib.qwa_rope_table, out.data_ptr(), first, positions, rotary_dim,
            theta, ctypes.byref(s) if s is not None else None)
    return out


def _side(x: torch.Tensor, y: Optional[torch.Tensor], name: str, tokens: int, dim: int, dtype,
          index: int):
    """Checks one of q and k with its output (None: one is made); the output and
    their qwa_rope_tensor."""
    shape = x.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim or shape[1] >= 2 ** 31:
        raise ValueError(f"{name} must be [tokens, heads, head_dim] as the others")
    if x.dtype != dtype or x.get_device() != index:
        raise ValueError(f"{name} must agree with the others in dtype and device")
    x0, x1, x2 = x.stride()
    if y is None:
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        y0, y1, y2 = shape[1] * dim, dim, 1
    else:
        if y.shape != shape or y.dtype != dtype or y.get_device() != index:
            raise ValueError(f"{name}'s output must be of its shape, dtype and device")
        y0, y1, y2 = y.stride()
    if x2 != 1 or y2 != 1:
        raise ValueError(f"{name}: a head's values must be contiguous")
    return y, _lib.rope_tensor(x.data_ptr(), x0, x1, y.data_ptr(), y0, y1, shape[1])


def _rope_args(ctx: Context, q, k, table, positions, q_output, k_output, layout, inverse):
    """(q's output, k's output, the C call's arguments between context and stream)"""
    some = q if q is not None else k
    dtype, index, shape = some.dtype, ctx.device, some.shape
    code, order = _DTYPES.get(dtype), _LAYOUTS.get(layout)
    if code is None or len(shape) != 3:
        raise ValueError("q or k must be a CUDA float16 or bfloat16 tensor [tokens, heads, "
                         "head_dim]")
    if order is None:
        raise ValueError("layout must be 'half' or 'interleaved'")
    tokens, _, dim = shape
    if tokens >= 2 ** 31:
        raise ValueError("at most 2^31 - 1 tokens")
    rows, half, two = table.shape
    if two != 2 or table.dtype != torch.float32 or table.get_device() != index \
            or not table.is_contiguous():
        raise ValueError("table must be a contiguous float32 [rows, rotary_dim / 2, 2] on q's "
                         "device")
    if positions.dtype != torch.int32 or positions.get_device() != index \
            or positions.numel() < tokens or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32 tensor of one position a token")
    qs = ks = None
    if q is not None:
        q_output, qs = _side(q, q_output, "q", tokens, dim, dtype, index)
    if k is not None:
        k_output, ks = _side(k, k_output, "k", tokens, dim, dtype, index)
    return q_output, k_output, (code, qs, ks, tokens, dim, 2 * half, order, 1 if inverse else 0,
                                positions.data_ptr(), table.data_ptr(), rows)


class RopeKernel:
    """Rotation of q and k by a table (``rope_table``), beside QKNormRopeKernel."""

    def __init__(self, device=None):
        self.ctx = Context.for_device(device)

    def create_run(self, q: Optional[torch.Tensor], k: Optional[torch.Tensor],
                   table: torch.Tensor, positions: torch.Tensor,
                   q_output: Optional[torch.Tensor], k_output: Optional[torch.Tensor],
                   layout: str = "half", inverse: bool = False) -> EncodableRun:
        """q, k: [tokens, heads, head_dim], any strides with contiguous heads;
        either may be None. An output may be its input (in place). A token
        whose position is not a row of the table is left unwritten."""
        _need(q is not None or k is not None, "one of q and k is required")
        _need((q is None or q_output is not None) and (k is None or k_output is not None),
              "q and k need their outputs")
        _, _, args = _rope_args(self.ctx, q, k, table, positions, q_output, k_output, layout,
                                inverse)
        lib, h = self.ctx.lib, self.ctx.handle
        return EncodableRun(lambda s: lib.qwa_rope(h, *args, s), self.ctx, "rotary positions")


def rope(q: Optional[torch.Tensor], k: Optional[torch.Tensor], table: torch.Tensor,
         positions: torch.Tensor, layout: str = "half", inverse: bool = False,
         q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None, stream=None
         ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(q, k) rotated at each token's position (the way back with ``inverse``). Outputs
    that the call makes are of ``stream``."""
    some = q if q is not None else k
    _need(some is not None and some.is_cuda, "q or k must be a CUDA tensor")
    ctx = Context.for_device(some.get_device())
    if stream is not None:
        with torch.cuda.stream(_as_stream(stream, ctx.device)):
            return rope(q, k, table, positions, layout, inverse, q_out, k_out)
    q_out, k_out, args = _rope_args(ctx, q, k, table, positions, q_out, k_out, layout, inverse)
    _launch(ctx, stream, ctx.lib.qwa_rope, *args)
    return q_out, k_out
