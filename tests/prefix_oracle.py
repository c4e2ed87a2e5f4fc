"""Plain 64-bit forms of the rotary, cache and shared-prefix operators, for the
tests: numpy and torch on the CPU, request by request."""
import math

import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def _e4m3_values():
    v = np.empty(256)
    for c in range(256):
        s, e, m = c >> 7, (c >> 3) & 15, c & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = np.nan if (c & 0x7f) == 0x7f else (-x if s else x)
    return v


E4M3 = _e4m3_values()
_POSITIVE = E4M3[:127]  # ascending codes 0..126


def to_e4m3(y):
    """Codes (uint8) of values y (f64, |y| <= 448 or NaN): nearest, ties to the even code."""
    a = np.abs(y)
    hi = np.clip(np.searchsorted(_POSITIVE, np.where(np.isnan(a), 0, a)), 0, 126)
    lo = np.maximum(hi - 1, 0)
    d_hi, d_lo = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(a), 127, code)
    return (code + 128 * np.signbit(y)).astype(np.uint8)


def quantise(x, fmt, dtype):
    """(codes, scale bytes) of x [..., dim] (CPU tensor of dtype) by the rule of include/qwa.h."""
    most, steps = (448.0, 8) if fmt == "e4m3" else (127.0, 6)
    low = {("e4m3", torch.float16): -15, ("int8", torch.float16): -24,
           ("e4m3", torch.bfloat16): -117, ("int8", torch.bfloat16): -126}[(fmt, dtype)]
    top = {("e4m3", torch.float16): 8, ("int8", torch.float16): 10,
           ("e4m3", torch.bfloat16): 120, ("int8", torch.bfloat16): 122}[(fmt, dtype)]
    finite = float(torch.finfo(dtype).max)
    v = x.double().numpy()
    amax = np.nanmax(np.where(np.isnan(v), 0, np.minimum(np.abs(v), finite)), axis=-1,
                     keepdims=True)
    e = np.zeros(amax.shape, int)
    for i in np.ndindex(amax.shape):  # the definition, word for word
        if amax[i] > 0:
            g = math.frexp(amax[i])[1] - steps - 2
            while amax[i] > most * 2.0 ** g:
                g += 1
            e[i] = max(g, low)
    limit = np.where(e == top, 240.0 if fmt == "e4m3" else 63.0, most)
    y = np.clip(v * np.exp2(-e.astype(float)), -limit, limit)
    if fmt == "e4m3":
        code = to_e4m3(y)
    else:
        code = np.where(np.isnan(y), 0, np.rint(y)).astype(np.int8)
    return code, (e[..., 0] + 127).astype(np.uint8)


def dequantise(code, scale, fmt):
    v = E4M3[code] if fmt == "e4m3" else code.astype(np.float64)
    return v * np.exp2(scale.astype(np.float64) - 127)[..., None]


def rope(x, table, positions, rotary, layout, inverse):
    """x [T, H, D] -> rotated in f64, with the f32 table given."""
    x = x.double().cpu()
    row = table.double().cpu()[positions.long().cpu()][:, None]
    c, s = row[..., 0], row[..., 1] * (-1 if inverse else 1)
    y, h = x.clone(), rotary // 2
    a, b = ((slice(0, h), slice(h, 2 * h)) if layout == "half"
            else (slice(0, 2 * h, 2), slice(1, 2 * h, 2)))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def rope_tolerance(x, y, table, positions, dtype):
    """Half a step of the result, and three roundings of f32 on products of at most
    |x|max * m in each head."""
    big = x.double().cpu().abs().amax(dim=-1, keepdim=True) * float(table.abs().max())
    return HALF_STEP[dtype] * y.abs() + SMALLEST[dtype] / 2 + 4 * 2.0 ** -24 * big


def prefix_attention(q, k, v, cu_q, cu_k, pk, pv, sparse, sparse_prefix, window):
    """(out, tolerance) in f64 for packed q [Tq, Hq, 128], k, v [Tk, Hk, 128] and
    the prefix's values pk, pv [P, Hk, 128] (f64).

    The tolerance counts, for a result o = sum p v / sum p of n keys with A =
    sum p |v| / sum p and u half a step of the 16-bit type: the rounding of o
    (u |o|); of every p (u A, and half of the type's smallest step against sum p >= 1); f32:
    scores of 128 products, twice for a sum that is not rounded to nearest,
    2 * 130 * 2^-24 * max sum |q k| / sqrt(128), doubled as both sums have them,
    exp2 (2^-21) and the sums over n keys (2 n 2^-24)."""
    dt = q.dtype
    u = HALF_STEP[dt]
    dev = q.device
    pk, pv = pk.to(dev).double(), pv.to(dev).double()
    P, group = pk.shape[0], q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    for b in range(len(cu_q) - 1):
        n, m = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if n == 0:
            continue
        keys = torch.arange(P + m, device=dev)
        pos = P + m - n + torch.arange(n, device=dev)
        keep = keys[None] <= pos[:, None]
        if sparse:
            keep &= (keys[None] < sparse_prefix) | (keys[None] > pos[:, None] - window)
        for h in range(q.shape[1]):
            kk = torch.cat([pk[:, h // group], k[cu_k[b]:cu_k[b + 1], h // group].double()])
            vv = torch.cat([pv[:, h // group], v[cu_k[b]:cu_k[b + 1], h // group].double()])
            qq = q[cu_q[b]:cu_q[b + 1], h].double()
            s = (qq @ kk.T / math.sqrt(128)).masked_fill(~keep, -math.inf)
            p = torch.softmax(s, dim=-1)
            # a dropped key adds nothing, whatever its value is
            o = torch.zeros(n, 128, dtype=torch.float64, device=dev)
            A = torch.zeros_like(o)
            fine = torch.isfinite(vv)
            clean = torch.where(fine, vv, torch.zeros_like(vv))
            o = p @ clean
            A = p @ clean.abs()
            kinds = [(~fine & torch.isnan(vv), math.nan), (vv == math.inf, math.inf),
                     (vv == -math.inf, -math.inf)]
            for where, what in kinds:
                hit = (keep.double() @ where.double()) > 0
                o = torch.where(hit, o + what, o)
            smax = float((qq.abs() @ kk.abs().T).max()) / math.sqrt(128) if kk.numel() else 0.0
            f32 = 4 * 130 * 2.0 ** -24 * smax + 2.0 ** -21 + 2 * (P + m) * 2.0 ** -24
            out[cu_q[b]:cu_q[b + 1], h] = o
            tol[cu_q[b]:cu_q[b + 1], h] = u * o.abs() + (u + f32) * A + \
                SMALLEST[dt] * (P + m) * clean.abs().max() + SMALLEST[dt]
    return out, tol
