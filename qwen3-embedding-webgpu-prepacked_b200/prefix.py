"""Attention of a batch of requests that share a cached prefix.

Requests of one service begin with the same text (an instruction, examples, a
document). Its keys and values are computed once, kept in a ``KVCache``, and
every request of a micro-batch attends to them and to its own keys:
``prefix_attention`` packs the query rows of all requests into the tensor cores'
tiles, so the prefix is read and multiplied once for the batch. It stands
beside ``attention.CausalAttentionKernel`` (src/webgpu/ops.ts:320-345): with a
prefix of length 0 both compute the same, and the sparse rule is the
reference's, on absolute positions.

Launches are the kernel of csrc/prefix_attention.cu through the C ABI. A
``PrefixPlan`` holds the work lists of given lengths; ``prefix_attention``
keeps the last few plans. Lengths that were not met before cost their plan: lists made on the
host, an allocation and a copy, and as it allocates it waits for what runs on the device
(16 ragged requests: 83 us of the host's time a call instead of 17; 16 of about 500 tokens
behind 2000: 219 instead of 22, in the shade of a kernel of 193). A model's layers share one.
"""
from __future__ import annotations

import ctypes
import threading
from typing import Optional, Sequence

import torch

from . import _lib
from .attention import (HEAD_DIM, MODE_AUTO, PREFIX, WINDOW, AttentionRun, Context, EncodableRun,
                        _as_stream, _launch, _need, encode_run)
from .kv_cache import _DTYPES, FORMATS, KVCache


_retired: list = []  # lists of plans that ended during a capture
_create_lock = threading.Lock()  # a context makes one plan at a time


def _lengths(cu) -> Optional[tuple]:
    """Host offsets as a tuple of Python ints (of a tensor: by value)."""
    if cu is None:
        return None
    return tuple(cu.tolist()) if isinstance(cu, torch.Tensor) else tuple(cu)


def _int32(**values) -> None:
    for name, value in values.items():
        _need(-2 ** 31 <= value < 2 ** 31, f"{name} must be a 32-bit number")


def _cu_arrays(cu_seqlens, cu_seqlens_k):
    cu_q, cu_k = _lengths(cu_seqlens), _lengths(cu_seqlens_k)
    _need(len(cu_q) >= 2, "cu_seqlens needs at least one request")
    _need(cu_k is None or len(cu_k) == len(cu_q),
          "cu_seqlens and cu_seqlens_k must be of the same requests")
    for cu in (cu_q, cu_k or cu_q):
        _int32(cu_seqlens=min(cu))
        _int32(cu_seqlens=max(cu))
    return _lib.cu_array(cu_q), _lib.cu_array(cu_k) if cu_k is not None else None


class PrefixPlan:
    """Work lists for requests of given lengths behind a prefix of ``prefix_len``
    keys. A request's queries are the last of its own keys; ``cu_seqlens_k`` None: as
    many keys as queries. A captured graph needs its plan for as long as it is
    replayed."""

    def __init__(self, cu_seqlens: Sequence[int], prefix_len: int, q_heads: int, kv_heads: int,
                 cu_seqlens_k: Optional[Sequence[int]] = None, mode: int = MODE_AUTO,
                 sparse_prefix: int = PREFIX, window: int = WINDOW, device=None,
                 ctx: Optional[Context] = None):
        self.ctx = ctx if ctx is not None else Context.for_device(device)
        self.handle = None
        cu_q, cu_k = _cu_arrays(cu_seqlens, cu_seqlens_k)
        _int32(prefix_len=prefix_len, q_heads=q_heads, kv_heads=kv_heads, mode=mode,
               sparse_prefix=sparse_prefix, window=window)
        _need(not _capturing(self.ctx.device),
              "a plan allocates memory: make it before the capture")
        while True:
            try:  # (threads that make plans at once share the list)
                lib, old = _retired.pop()
            except IndexError:
                break
            lib.qwa_prefix_plan_destroy(old)
        h = ctypes.c_void_p()
        with _create_lock:
            _lib.check(self.ctx.lib.qwa_prefix_plan_create(
                self.ctx.handle, cu_q, cu_k, len(cu_q) - 1, q_heads, kv_heads, prefix_len, mode,
                sparse_prefix, window, ctypes.byref(h)), self.ctx.handle)
        self.handle = h
        self.queries = cu_q[len(cu_q) - 1]
        self.keys = cu_k[len(cu_k) - 1] if cu_k is not None else self.queries
        self.prefix_len, self.q_heads, self.kv_heads = prefix_len, q_heads, kv_heads
        deal = ctypes.c_int(), ctypes.c_int()
        _lib.check(self.ctx.lib.qwa_prefix_plan_deal(h, ctypes.byref(deal[0]),
                                                     ctypes.byref(deal[1])))
        self.block_tokens, self.splits = deal[0].value, deal[1].value
        fn = self.ctx.lib.qwa_prefix_attention_workspace
        self.workspace = {name: fn(h, code) for name, code in FORMATS.items()}  # bytes

    def close(self) -> None:
        """Release the lists; waits for the device. During a stream capture
        (memory is not freed then) they are released by the next plan."""
        if self.handle:
            handle, self.handle = self.handle, None
            if _capturing(self.ctx.device):
                _retired.append((self.ctx.lib, handle))
            else:
                self.ctx.lib.qwa_prefix_plan_destroy(handle)

    def __del__(self):
        try:
            self.close()
        except Exception:  # at the interpreter's end
            pass


def _packed(t: torch.Tensor, name: str, tokens: int, heads: int, dtype, index: int) -> int:
    """Checks a packed [tokens, heads, 128] operand; its token stride."""
    if t.shape != (tokens, heads, HEAD_DIM) or t.dtype != dtype or t.get_device() != index:
        raise ValueError(f"{name} must be [{tokens}, {heads}, {HEAD_DIM}] of q's dtype and device")
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s1 != HEAD_DIM and heads != 1):
        raise ValueError(f"{name}: a token's heads must be contiguous")
    return s0 if tokens > 1 else heads * HEAD_DIM  # a single row has no stride of its own


def _attention_args(ctx: Context, plan: PrefixPlan, q, k, v, output, cache, first_slot):
    """(output, made if None; workspace or None; the C call's arguments between plan
    and stream)"""
    dtype, index = q.dtype, ctx.device
    code = _DTYPES.get(dtype)
    _need(code is not None, "q must be float16 or bfloat16")
    _need(plan.ctx.device == index, "the plan must be on the kernel's device")
    _need(plan.handle is not None, "the plan is closed")
    _need(-2 ** 63 <= first_slot < 2 ** 63, "first_slot must be a 64-bit number")
    n, hq, m, hk = plan.queries, plan.q_heads, plan.keys, plan.kv_heads
    if output is None:
        output = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _need(_packed(output, "output", n, hq, dtype, index) == hq * HEAD_DIM,
              "output must be contiguous")
    struct = workspace = None
    need = 0
    if cache is not None:
        _need(cache.index == index, "the cache must be on q's device")
        struct = cache.struct
        need = plan.workspace[cache.format]
        if need:
            workspace = q.new_empty(need, dtype=torch.uint8)
    else:
        _need(plan.prefix_len == 0, "a prefix needs its cache")
    return output, workspace, (
        code, q.data_ptr(), _packed(q, "q", n, hq, dtype, index), k.data_ptr(),
        _packed(k, "k", m, hk, dtype, index), v.data_ptr(), _packed(v, "v", m, hk, dtype, index),
        output.data_ptr(), struct, first_slot,
        workspace.data_ptr() if workspace is not None else None, need)


class PrefixAttentionKernel:
    """Shared-prefix attention, beside CausalAttentionKernel."""

    def __init__(self, device=None):
        self.ctx = Context.for_device(device)

    def create_run(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, output: torch.Tensor,
                   plan: PrefixPlan, cache: Optional[KVCache] = None,
                   first_slot: int = 0) -> AttentionRun:
        """q [queries, q_heads, 128], k, v [own keys, kv_heads, 128] packed
        request after request, output as q, contiguous; the prefix is in the
        cache's slots ``first_slot`` .. ``first_slot + plan.prefix_len - 1``. A run
        with ``owned_buffers`` is issued on one stream at a time (making it waits for
        the current stream), and a captured graph needs it for as long as it is replayed."""
        _need(output is not None, "an output is required")
        _, workspace, args = _attention_args(self.ctx, plan, q, k, v, output, cache, first_slot)
        lib, h, device = self.ctx.lib, self.ctx.handle, self.ctx.device
        if workspace is not None and not _capturing(device):
            # whatever stream the run is issued on, no work must be left that writes it
            torch.cuda.current_stream(device).synchronize()
        used = set()

        def launch(stream):
            _need(plan.handle is not None, "the plan is closed")
            if workspace is not None and stream not in used:
                # not handed out again, once the run is gone, before that stream is done
                workspace.record_stream(_as_stream(stream, device))
                used.add(stream)
            return lib.qwa_prefix_attention(h, plan.handle, *args, stream)

        return AttentionRun([EncodableRun(launch, self.ctx, "shared-prefix attention")],
                            [workspace] if workspace is not None else [])

    def encode(self, stream, run: AttentionRun) -> None:
        for command in run.commands:
            encode_run(stream, command)


MAX_PLANS = 64
# (device, lengths, ...) -> [plan, use, kept]: `use` counts up with every use, and
# plans that a graph was captured with are kept for good
_plans: dict = {}
_plans_lock = threading.Lock()
_uses = 0


def _capturing(device: int) -> bool:
    """Whether the device's current stream is being captured."""
    if torch._C._cuda_getDevice() == device:
        return torch._C._cuda_isCurrentStreamCapturing()
    with torch.cuda.device(device):
        return torch._C._cuda_isCurrentStreamCapturing()


def _plan_for(ctx: Context, *key) -> PrefixPlan:
    global _uses
    full = (ctx.device, *key)
    with _plans_lock:
        entry = _plans.get(full)
        if entry is not None:
            _uses = entry[1] = _uses + 1
            if not entry[2] and _capturing(ctx.device):
                entry[2] = True
            return entry[0]
    cu_q, cu_k, prefix_len, q_heads, kv_heads, mode, sparse_prefix, window = key
    plan = PrefixPlan(cu_q, prefix_len, q_heads, kv_heads, cu_k, mode, sparse_prefix, window,
                      ctx=ctx)
    old = None
    with _plans_lock:
        # another thread may have met the same lengths meanwhile, and captured a graph
        # with its plan: the first one stays
        entry = _plans.setdefault(full, [plan, 0, False])
        _uses = entry[1] = _uses + 1
        loose = [(e[1], k) for k, e in _plans.items() if not e[2]]
        if len(loose) > MAX_PLANS:
            old = _plans.pop(min(loose)[1])
    del old  # outside the lock: releasing its lists waits for the device
    return entry[0]


def prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     cu_seqlens: Sequence[int], cache: Optional[KVCache] = None,
                     prefix_len: int = 0, first_slot: int = 0,
                     cu_seqlens_k: Optional[Sequence[int]] = None, mode: int = MODE_AUTO,
                     sparse_prefix: int = PREFIX, window: int = WINDOW,
                     out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """softmax(q k / sqrt(128)) v of packed requests behind the ``prefix_len``
    keys in the cache's slots from ``first_slot`` on: q [queries, q_heads, 128], k, v
    [own keys, kv_heads, 128]. ``cu_seqlens`` (host) cuts q into requests, ``cu_seqlens_k``
    k and v (None: the same); a request's queries are the last of its keys.
    Lengths met before reuse their plan; inside a capture they must have been
    met before it, and a captured ``stream`` must be the current one. An output that the
    call makes is of ``stream``."""
    q_shape, k_shape = q.shape, k.shape
    _need(q.is_cuda and len(q_shape) == 3 and len(k_shape) == 3,
          "q and k must be CUDA tensors [tokens, heads, 128]")
    ctx = Context.for_device(q.get_device())
    if stream is not None:
        stream = _as_stream(stream, ctx.device)
        if not _capturing(ctx.device):
            # the graph would keep neither the plan nor a workspace
            with torch.cuda.stream(stream):
                _need(not torch._C._cuda_isCurrentStreamCapturing(),
                      "a captured stream must be the current one")
    plan = _plan_for(ctx, _lengths(cu_seqlens), _lengths(cu_seqlens_k), prefix_len,
                     q_shape[1], k_shape[1], mode, sparse_prefix, window)
    if stream is not None:
        with torch.cuda.stream(stream):
            return _attention(ctx, plan, q, k, v, out, cache, first_slot)
    return _attention(ctx, plan, q, k, v, out, cache, first_slot)


def _attention(ctx: Context, plan: PrefixPlan, q, k, v, out, cache, first_slot) -> torch.Tensor:
    """The call on the current stream, with an output and a workspace of that stream."""
    out, workspace, args = _attention_args(ctx, plan, q, k, v, out, cache, first_slot)
    _launch(ctx, None, ctx.lib.qwa_prefix_attention, plan.handle, *args)
    return out


def prefix_attention_work(cu_seqlens: Sequence[int], prefix_len: int, q_heads: int,
                          kv_heads: int, cu_seqlens_k: Optional[Sequence[int]] = None,
                          mode: int = MODE_AUTO, sparse_prefix: int = PREFIX,
                          window: int = WINDOW):
    """(kept pairs per query head, key tiles visited over all kv heads) of one call."""
    cu_q, cu_k = _cu_arrays(cu_seqlens, cu_seqlens_k)
    _int32(prefix_len=prefix_len, q_heads=q_heads, kv_heads=kv_heads, mode=mode,
           sparse_prefix=sparse_prefix, window=window)
    pairs, tiles = ctypes.c_int64(), ctypes.c_int64()
    _lib.check(_lib.load().qwa_prefix_attention_work(
        cu_q, cu_k, len(cu_q) - 1, q_heads, kv_heads, prefix_len, mode, sparse_prefix, window,
        ctypes.byref(pairs), ctypes.byref(tiles)))
    return pairs.value, tiles.value
