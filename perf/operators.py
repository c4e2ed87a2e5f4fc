"""What is measured of the shared-prefix operators, and their plain forms.

Three operators serve a micro-batch of embedding requests that begin with the
same instruction: rotary positions, the key/value cache in 8 bits, and the
attention of requests that share a cached prefix. A case is a dict with the
operator under ``"op"``; ``run`` computes it from elementary torch operations
(``own`` false) or through the package's entry points (``own`` true).

Rotary positions
    y1 = x1 * c - x2 * s, y2 = x2 * c + x1 * s for the pairs of the first
    ``rotary`` values of each head (halves, or neighbours), (c, s) the row of
    a table at the token's position; the inverse takes -s. A table holds
    m * cos(p * f_i), m * sin(p * f_i).
Cache
    per (slot, head) one power of two 2^e and the values' codes, code =
    round(x / 2^e) to E4M3 or to a whole number of 8 bits; e is the least for
    which the largest value fits. The scale is held as the byte e + 127.
Attention
    query i of a request sits behind the P keys of the prefix and the
    request's own keys up to itself; in the sparse form a key is kept if its
    position is under 176 or within the last 432.
"""
import importlib
import math
import random

import torch

own = False

PACKAGE = "qwen3-embedding-webgpu-prepacked_b200"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
TOP_EXPONENT = {"f16": 15, "bf16": 127}  # of the largest finite value
SPARSE_PREFIX, SPARSE_WINDOW = 176, 432
HEAD = 128
THETA = 1e6


# ------------------------------------------------------------------- cases

def listed():
    return [
        # one new token for each of 16 requests: the latency of a launch
        {"name": "rope_16_tokens", "op": "rope", "tokens": 16, "q_heads": 16, "kv_heads": 8,
         "dim": 128, "rotary": 128, "layout": "half", "inverse": False, "dtype": "f16",
         "table": 8192, "scaling": "none", "row": 4096},
        # a micro-batch of 16 x 500 tokens, q and k rotated where the projection left them
        {"name": "rope_16x500_yarn", "op": "rope", "tokens": 8000, "q_heads": 16, "kv_heads": 8,
         "dim": 128, "rotary": 128, "layout": "half", "inverse": False, "dtype": "f16",
         "table": 32768, "scaling": "yarn", "row": 4096},
        # the way back (the gradient), neighbouring pairs in half of each head, an odd count
        {"name": "rope_back_pairs_20011", "op": "rope", "tokens": 20011, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "rotary": 64, "layout": "interleaved", "inverse": True,
         "dtype": "bf16", "table": 32768, "scaling": "linear", "row": 0},
        # the table of a context stretched to four times 32768
        {"name": "rope_table_131072_yarn", "op": "table", "positions": 131072, "rotary": 128,
         "first": 0, "scaling": "yarn"},
        # one token of each of 16 requests goes into the cache
        {"name": "cache_write_16_e4m3", "op": "write", "tokens": 16, "slots": 2048, "heads": 8,
         "dim": 128, "format": "e4m3", "dtype": "f16", "spread": True},
        # 16 x 5000 tokens at once
        {"name": "cache_write_80000_int8", "op": "write", "tokens": 80000, "slots": 81920,
         "heads": 8, "dim": 128, "format": "int8", "dtype": "f16", "spread": False},
        # a cached context of 8000 tokens, gathered back
        {"name": "cache_read_8000_e4m3", "op": "read", "tokens": 8000, "slots": 16384, "heads": 8,
         "dim": 128, "format": "e4m3", "dtype": "bf16", "spread": True},
        # one query a request, behind its own short text and an instruction of 1000 tokens
        {"name": "attn_16x1_e4m3", "op": "attention", "requests": 16, "least": 1, "most": 1,
         "before": 150, "prefix": 1000, "q_heads": 16, "kv_heads": 8, "format": "e4m3",
         "dtype": "f16", "sparse": False, "lens": 1},
        # the ragged micro-batch of 15 to 150 tokens behind a short instruction
        {"name": "attn_ragged_15_150", "op": "attention", "requests": 16, "least": 15,
         "most": 150, "before": 0, "prefix": 176, "q_heads": 16, "kv_heads": 8, "format": "none",
         "dtype": "f16", "sparse": False, "lens": 2},
        # 16 passages of 500 tokens behind a long instruction with examples
        {"name": "attn_16x500_e4m3", "op": "attention", "requests": 16, "least": 500, "most": 500,
         "before": 0, "prefix": 2000, "q_heads": 16, "kv_heads": 8, "format": "e4m3",
         "dtype": "f16", "sparse": False, "lens": 3},
        # 4 passages of 1500 tokens under the sparse rule
        {"name": "attn_4x1500_sparse_int8", "op": "attention", "requests": 4, "least": 1500,
         "most": 1500, "before": 0, "prefix": 1000, "q_heads": 16, "kv_heads": 8,
         "format": "int8", "dtype": "f16", "sparse": True, "lens": 4},
        # 4 documents of 5000 tokens behind a document of 5000
        {"name": "attn_4x5000_bf16", "op": "attention", "requests": 4, "least": 5000,
         "most": 5000, "before": 0, "prefix": 5000, "q_heads": 16, "kv_heads": 8,
         "format": "none", "dtype": "bf16", "sparse": False, "lens": 5},
    ]


def _log(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "table", "write", "read", "attention", "attention",
                     "attention", "attention"])
    dtype = rng.choice(["f16", "f16", "bf16"])
    if op == "rope":
        dim = rng.choice([64, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        q_heads = kv_heads * rng.choice([1, 2, 3, 4])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4 + 2])
        row = rng.choice([0, (q_heads + 2 * kv_heads) * dim])
        most = max(64, min(40000, 3 * 10 ** 7 // ((q_heads + kv_heads) * dim)))
        return {"op": "rope", "tokens": _log(rng, 1, most), "q_heads": q_heads,
                "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
                "layout": rng.choice(["half", "interleaved"]), "inverse": rng.random() < 0.3,
                "dtype": dtype, "table": rng.choice([8192, 32768]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "llama3"]), "row": row}
    if op == "table":
        return {"op": "table", "positions": _log(rng, 1, 131072),
                "rotary": rng.choice([20, 32, 64, 128]), "first": rng.choice([0, 0, 8191]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "llama3"])}
    if op in ("write", "read"):
        tokens = _log(rng, 1, 40000)
        return {"op": op, "tokens": tokens, "slots": tokens + rng.randrange(1, 2000),
                "heads": rng.choice([1, 2, 4, 8, 8]), "dim": rng.choice([64, 128, 128, 256]),
                "format": rng.choice(["e4m3", "int8", "none"]), "dtype": dtype,
                "spread": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 4, 8, 8, 8])
    q_heads = kv_heads * rng.choice([1, 2, 2, 4, 3])
    while True:
        requests = rng.randrange(1, 17)
        most = _log(rng, 1, 3000)
        prefix = _log(rng, 1, 8000)
        if requests * most * (prefix + most) * q_heads <= 4 * 5000 * 7500 * 16 // 2:
            break
    return {"op": "attention", "requests": requests, "least": rng.randrange(1, most + 1),
            "most": most, "before": rng.choice([0, 0, _log(rng, 1, 500)]), "prefix": prefix,
            "q_heads": q_heads, "kv_heads": kv_heads,
            "format": rng.choice(["none", "e4m3", "int8"]), "dtype": dtype,
            "sparse": rng.random() < 0.35, "lens": rng.randrange(10 ** 6)}


def _lengths(case):
    """(own queries, own keys) of each request."""
    r = random.Random(case["lens"])
    queries = [r.randint(case["least"], case["most"]) for _ in range(case["requests"])]
    before = [r.randint(0, case["before"]) for _ in range(case["requests"])]
    return queries, [n + m for n, m in zip(queries, before)]


def _offsets(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _kept_pairs(case):
    """Kept (query, key) pairs of one head."""
    queries, keys = _lengths(case)
    total = 0
    for n, m in zip(queries, keys):
        first, last = case["prefix"] + m - n, case["prefix"] + m - 1  # positions
        if not case["sparse"]:
            total += n * (first + last + 2) // 2
            continue
        for p in range(first, last + 1):
            seen = p + 1
            total += seen if seen <= SPARSE_PREFIX + SPARSE_WINDOW else \
                SPARSE_PREFIX + SPARSE_WINDOW
    return total


def work(case):
    op = case["op"]
    if op == "rope":
        values = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        rows = min(case["tokens"], case["table"])
        # what is not rotated is copied too, unless it stays where it is
        moved = case["dim"]
        return {"bytes": values * moved * 4 + rows * case["rotary"] * 4 + case["tokens"] * 4,
                "flops": 3 * values * case["rotary"]}
    if op == "table":
        n = case["positions"] * (case["rotary"] // 2)
        return {"bytes": 8 * n, "flops": 2 * n}
    if op in ("write", "read"):
        values = 2 * case["tokens"] * case["heads"] * case["dim"]
        code = 2 if case["format"] == "none" else 1
        scale = 0 if case["format"] == "none" else 2 * case["tokens"] * case["heads"]
        return {"bytes": values * (2 + code) + scale + 4 * case["tokens"], "flops": 2 * values}
    queries, keys = _lengths(case)
    code = 2 if case["format"] == "none" else 1
    scale = 0 if case["format"] == "none" else 2
    cached = case["prefix"] * case["kv_heads"] * (2 * HEAD * code + scale)
    if case["sparse"] and case["prefix"] > SPARSE_PREFIX + SPARSE_WINDOW:
        cached = cached * (SPARSE_PREFIX + SPARSE_WINDOW) // case["prefix"]
    return {"bytes": 2 * HEAD * (2 * sum(queries) * case["q_heads"]
                                 + 2 * sum(keys) * case["kv_heads"]) + cached,
            "flops": 4 * HEAD * case["q_heads"] * _kept_pairs(case)}


# -------------------------------------------------------------- definitions

def _scaling(name):
    """The parameters of a kind of scaling (the factor is 4, from 32768 or 8192 positions)."""
    return {"none": {"kind": "none"},
            "linear": {"kind": "linear", "factor": 4.0},
            "ntk": {"kind": "ntk", "factor": 4.0},
            "yarn": {"kind": "yarn", "factor": 4.0, "original_positions": 32768},
            "llama3": {"kind": "llama3", "factor": 4.0, "original_positions": 8192}}[name]


def _frequencies(rotary, scaling, device):
    """([rotary / 2] frequencies in 64 bits, the table's factor)."""
    half = rotary // 2
    s = _scaling(scaling)
    i = torch.arange(half, dtype=torch.float64, device=device)
    factor = s.get("factor", 1.0)
    plain = THETA ** (-i / half)
    if s["kind"] == "linear":
        return plain / factor, 1.0
    if s["kind"] == "ntk":
        return (THETA * factor ** (rotary / max(rotary - 2, 1))) ** (-i / half), 1.0
    if s["kind"] == "yarn":
        def at(turns):
            return half * math.log(s["original_positions"] / (turns * 2 * math.pi)) / \
                math.log(THETA)
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rotary - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return plain / factor * ramp + plain * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if s["kind"] == "llama3":
        turns = s["original_positions"] * plain / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - smooth) * plain / factor + smooth * plain, 1.0
    return plain, 1.0


def _table(positions, rotary, scaling, first, device):
    f, m = _frequencies(rotary, scaling, device)
    p = torch.arange(first, first + positions, dtype=torch.float64, device=device)
    angle = p[:, None] * f[None, :]
    return torch.stack([angle.cos() * m, angle.sin() * m], dim=-1).float()


def _encode(x, fmt, dtype):
    """(codes, scale bytes) of x [..., dim]: the cache's definition, in 32 bits (exact but for
    the one rounding to a code)."""
    if fmt == "none":
        return x.clone(), None
    most, bits = (448.0, 7) if fmt == "e4m3" else (127.0, 5)
    low = {("f16", "e4m3"): -15, ("f16", "int8"): -24, ("bf16", "e4m3"): -117,
           ("bf16", "int8"): -126}[(dtype, fmt)]
    v = x.float()
    top = v.abs().amax(dim=-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    limit = most / 512.0 if fmt == "e4m3" else most / 128.0
    e = exponent - (9 if fmt == "e4m3" else 7) + (mantissa > limit).int()
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(min=low)
    # a code that would stand for more than the type's largest value takes the one below it
    highest = torch.where(e == TOP_EXPONENT[dtype] - bits, 240.0 if fmt == "e4m3" else 63.0, most)
    r = torch.ldexp(torch.ldexp(v, -(e // 2)), -(e - e // 2))
    r = torch.minimum(torch.maximum(r, -highest), highest)
    code = r.to(torch.float8_e4m3fn) if fmt == "e4m3" else r.round().to(torch.int8)
    return code, (e.squeeze(-1) + 127).to(torch.uint8)


def _decode(code, scale):
    """The values, in 32 bits."""
    if scale is None:
        return code.float()
    e = scale.int() - 127
    return torch.ldexp(torch.ldexp(code.float(), (e // 2)[..., None]), (e - e // 2)[..., None])


# ------------------------------------------------------------------ prepare

def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    op = case["op"]
    if op == "table":
        return {"case": case, "device": device, "first": case["first"] + int(seed) % 7}
    dtype = DTYPES[case["dtype"]]
    if op == "rope":
        n, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
        if case["row"]:  # q, k and v of a token lie in one row, as the projection leaves them
            rows = normal(n, case["row"]).to(dtype)
            q = rows[:, :hq * d].view(n, hq, d)
            k = rows[:, hq * d:(hq + hk) * d].view(n, hk, d)
        else:
            q, k = normal(n, hq, d).to(dtype), normal(n, hk, d).to(dtype)
        start = torch.randint(0, max(1, case["table"] - n), (1,), generator=g, device=device)
        positions = (start + torch.arange(n, device=device)) % case["table"]
        return {"case": case, "q": q, "k": k, "positions": positions.to(torch.int32),
                "table": _table(case["table"], case["rotary"], case["scaling"], 0, device)}
    # keys after their norm: about one, some channels larger; values with rows of differing size
    def keys_values(n, heads, d):
        gain = 1 + 2 * (torch.rand(heads, d, generator=g, device=device) > 0.95).float()
        k = normal(n, heads, d) * gain
        v = normal(n, heads, d) * torch.exp(0.5 * normal(n, heads, 1))
        return k.to(dtype), v.to(dtype)

    if op in ("write", "read"):
        n, slots, h, d = case["tokens"], case["slots"], case["heads"], case["dim"]
        if case["spread"]:
            at = torch.randperm(slots, generator=g, device=device)[:n].to(torch.int32)
        else:
            at = torch.arange(n, device=device, dtype=torch.int32) + (slots - n) // 2
        if op == "write":
            k, v = keys_values(n, h, d)
            s = {"case": case, "slots": at, "k": k, "v": v}
            for name in ("k", "v"):
                code, scale = _encode(torch.zeros(slots, h, d, device=device, dtype=dtype),
                                      case["format"], case["dtype"])
                s[name + "_code"], s[name + "_scale"] = code, scale
            return s
        k, v = keys_values(slots, h, d)
        kc, ks = _encode(k, case["format"], case["dtype"])
        vc, vs = _encode(v, case["format"], case["dtype"])
        return {"case": case, "slots": at, "k_code": kc, "k_scale": ks, "v_code": vc,
                "v_scale": vs}
    queries, keys = _lengths(case)
    hk, p = case["kv_heads"], case["prefix"]
    q = normal(sum(queries), case["q_heads"], HEAD).to(dtype)
    k, v = keys_values(sum(keys), hk, HEAD)
    pk, pv = keys_values(p, hk, HEAD)
    kc, ks = _encode(pk, case["format"], case["dtype"])
    vc, vs = _encode(pv, case["format"], case["dtype"])
    return {"case": case, "q": q, "k": k, "v": v, "k_code": kc, "k_scale": ks, "v_code": vc,
            "v_scale": vs, "cu_q": _offsets(queries), "cu_k": _offsets(keys)}


# ---------------------------------------------------------------------- run

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    op = case["op"]
    if op == "rope":
        row = state["table"][state["positions"].long()]
        c, s = row[..., 0], row[..., 1]
        if case["inverse"]:
            s = -s
        return {"q": _plain_rope(state["q"], c, s, case), "k": _plain_rope(state["k"], c, s, case)}
    if op == "table":
        return _table(case["positions"], case["rotary"], case["scaling"], state["first"],
                      state["device"])
    at = state["slots"].long() if op != "attention" else None
    if op == "write":
        out = {}
        for name in ("k", "v"):
            code, scale = _encode(state[name], case["format"], case["dtype"])
            # (8-bit types have no indexed assignment of their own: moved as bytes)
            held = state[name + "_code"]
            if code.element_size() == 1:
                held.view(torch.uint8)[at] = code.view(torch.uint8)
            else:
                held[at] = code
            out[name] = held
            if scale is not None:
                state[name + "_scale"][at] = scale
                out[name + "_scale"] = state[name + "_scale"]
        return out
    if op == "read":
        out = {}
        for name in ("k", "v"):
            held, scale = state[name + "_code"], state[name + "_scale"]
            code = held.view(torch.uint8)[at].view(held.dtype) if scale is not None else held[at]
            out[name] = _decode(code, scale[at] if scale is not None else None).to(
                DTYPES[case["dtype"]])
        return out
    return _plain_attention(case, state)


def _plain_rope(x, c, s, case):
    half = case["rotary"] // 2
    v = x.float()
    turned, rest = v[..., :2 * half], v[..., 2 * half:]
    c, s = c[:, None, :], s[:, None, :]
    if case["layout"] == "half":
        x1, x2 = turned[..., :half], turned[..., half:]
        y = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s, rest], dim=-1)
    else:
        x1, x2 = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).flatten(-2)
        y = torch.cat([y, rest], dim=-1)
    return y.to(x.dtype)


def _plain_attention(case, state):
    """The prefix as one product for all rows, the own keys as a padded batch, one softmax."""
    q, hk, p = state["q"].float(), case["kv_heads"], case["prefix"]
    device, group = q.device, case["q_heads"] // case["kv_heads"]
    queries, keys = _lengths(case)
    n, m = torch.tensor(queries, device=device), torch.tensor(keys, device=device)
    cu_q = torch.tensor(state["cu_q"], device=device)
    cu_k = torch.tensor(state["cu_k"], device=device)
    total = q.shape[0]
    request = torch.repeat_interleave(torch.arange(len(queries), device=device), n,
                                      output_size=total)
    index = torch.arange(total, device=device) - cu_q[request]  # of a row in its request
    place = index + (m - n)[request]  # its place among the request's own keys
    position = p + place
    wide = max(keys)
    # own keys and values, padded to [requests, wide]
    at = (cu_k[:-1, None] + torch.arange(wide, device=device)[None, :]).clamp(
        max=max(state["k"].shape[0] - 1, 0))
    k, v = state["k"].float()[at], state["v"].float()[at]  # [requests, wide, hk, 128]
    rows = q.view(total, hk, group, HEAD) / math.sqrt(HEAD)
    pk = _decode(state["k_code"], state["k_scale"])
    pv = _decode(state["v_code"], state["v_scale"])
    shared = torch.matmul(rows.permute(1, 2, 0, 3).reshape(hk, group * total, HEAD),
                          pk.permute(1, 2, 0)).view(hk, group, total, p)
    # the rows, padded to [requests, tall]
    tall = max(queries)
    spread = torch.zeros(len(queries), tall, hk, group, HEAD, device=device)
    spread[request, index] = rows
    mine = torch.matmul(spread.permute(0, 2, 3, 1, 4).reshape(len(queries), hk, group * tall,
                                                              HEAD),
                        k.permute(0, 2, 3, 1)).view(len(queries), hk, group, tall, wide)
    mine = mine.permute(0, 3, 1, 2, 4)[request, index].permute(1, 2, 0, 3)  # [hk, g, total, wide]
    key = torch.arange(wide, device=device)[None, :]
    kept = key <= place[:, None]
    if case["sparse"]:
        at_key = p + key
        kept = kept & ((at_key < SPARSE_PREFIX) | (at_key + SPARSE_WINDOW > position[:, None]))
        first = torch.arange(p, device=device)[None, :]
        seen = (first < SPARSE_PREFIX) | (first + SPARSE_WINDOW > position[:, None])
        shared = shared.masked_fill(~seen, float("-inf"))
    mine = mine.masked_fill(~kept, float("-inf"))
    top = torch.maximum(shared.amax(dim=-1, keepdim=True), mine.amax(dim=-1, keepdim=True))
    shared, mine = torch.exp(shared - top), torch.exp(mine - top)
    below = shared.sum(dim=-1, keepdim=True) + mine.sum(dim=-1, keepdim=True)
    out = torch.matmul(shared.view(hk, group * total, p), pv.permute(1, 0, 2)).view(
        hk, group, total, HEAD)
    weights = torch.zeros(len(queries), tall, hk, group, wide, device=device)
    weights[request, index] = mine.permute(2, 0, 1, 3)
    part = torch.matmul(weights.permute(0, 2, 3, 1, 4).reshape(len(queries), hk, group * tall,
                                                               wide),
                        v.permute(0, 2, 1, 3)).view(len(queries), hk, group, tall, HEAD)
    out = out + part.permute(0, 3, 1, 2, 4)[request, index].permute(1, 2, 0, 3)
    return (out / below).permute(2, 0, 1, 3).reshape(total, case["q_heads"], HEAD).to(
        state["q"].dtype)


def _run_own(case, state):
    pkg = importlib.import_module(PACKAGE)
    op = case["op"]
    if op == "rope":
        q, k = pkg.rotary.rope(state["q"], state["k"], state["table"], state["positions"],
                               layout=case["layout"], inverse=case["inverse"])
        return {"q": q, "k": k}
    if op == "table":
        scaling = pkg.rotary.RopeScaling(**_scaling(case["scaling"]))
        return pkg.rotary.rope_table(case["positions"], case["rotary"], THETA, scaling,
                                     first=state["first"], device=state["device"])
    cache = pkg.kv_cache.KVCache.wrap(state["k_code"], state["v_code"], state["k_scale"],
                                      state["v_scale"], DTYPES[case["dtype"]])
    if op == "write":
        pkg.kv_cache.kv_cache_write(cache, state["k"], state["v"], state["slots"])
        out = {"k": cache.k, "v": cache.v}
        if cache.k_scale is not None:
            out["k_scale"], out["v_scale"] = cache.k_scale, cache.v_scale
        return out
    if op == "read":
        k, v = pkg.kv_cache.kv_cache_read(cache, state["slots"])
        return {"k": k, "v": v}
    return pkg.prefix.prefix_attention(
        state["q"], state["k"], state["v"], state["cu_q"], cache, case["prefix"],
        cu_seqlens_k=state["cu_k"],
        mode=pkg.attention.MODE_SPARSE if case["sparse"] else pkg.attention.MODE_FULL)


# -------------------------------------------------------------------- exact

def exact(case, seed):
    """The definitions in 64 bits, request by request and head by head."""
    if case["op"] == "write" and case["format"] == "int8":
        return None  # whole numbers only
    s = prepare(case, seed)
    op = case["op"]
    if op == "table":
        device, half = s["device"], case["rotary"] // 2
        f, m = _frequencies(case["rotary"], case["scaling"], device)
        out = torch.empty(case["positions"], half, 2, dtype=torch.float64, device=device)
        p = torch.arange(s["first"], s["first"] + case["positions"], dtype=torch.float64,
                         device=device)
        for i in range(half):
            out[:, i, 0] = m * torch.cos(p * f[i])
            out[:, i, 1] = m * torch.sin(p * f[i])
        return out
    if op == "rope":
        sign = -1.0 if case["inverse"] else 1.0
        row = s["table"].double()[s["positions"].long()]
        turn = torch.complex(row[..., 0], sign * row[..., 1])[:, None, :]
        out, half = {}, case["rotary"] // 2
        for name in ("q", "k"):
            x = s[name].double()
            y = x.clone()
            if case["layout"] == "half":
                z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
                y[..., :half], y[..., half:2 * half] = z.real, z.imag
            else:
                z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * turn
                y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
            out[name] = y
        return out
    if op == "write":
        out = {}
        for name in ("k", "v"):
            held = s[name + "_code"].double()
            if case["format"] == "none":
                held[s["slots"].long()] = s[name].double()
                out[name] = held
                continue
            x = s[name].double()
            top = x.abs().amax(dim=-1, keepdim=True).clamp(min=1e-300)
            low = -15 if case["dtype"] == "f16" else -117
            e = torch.ceil(torch.log2(top / 448.0))
            e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(min=low)
            y = x / torch.exp2(e)
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            held[s["slots"].long()] = torch.round(y / step) * step
            out[name], out[name + "_scale"] = held, None  # the scales are whole numbers
        return out
    if op == "read":
        out = {}
        for name in ("k", "v"):
            x = s[name + "_code"].double()
            if s[name + "_scale"] is not None:
                x = x * torch.exp2(s[name + "_scale"].double() - 127)[..., None]
            out[name] = x[s["slots"].long()]
        return out

    def values(code, scale):
        x = code.double()
        return x if scale is None else x * torch.exp2(scale.double() - 127)[..., None]

    pk, pv = values(s["k_code"], s["k_scale"]), values(s["v_code"], s["v_scale"])
    p, group = case["prefix"], case["q_heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(case["requests"]):
        q0, q1, k0, k1 = s["cu_q"][b], s["cu_q"][b + 1], s["cu_k"][b], s["cu_k"][b + 1]
        at_key = torch.arange(p + k1 - k0, device=out.device)
        at_query = p + (k1 - k0) - (q1 - q0) + torch.arange(q1 - q0, device=out.device)
        seen = at_key[None, :] <= at_query[:, None]
        if case["sparse"]:
            seen &= (at_key < SPARSE_PREFIX)[None, :] | \
                (at_key[None, :] > at_query[:, None] - SPARSE_WINDOW)
        for h in range(case["q_heads"]):
            k = torch.cat([pk[:, h // group], s["k"][k0:k1, h // group].double()])
            v = torch.cat([pv[:, h // group], s["v"][k0:k1, h // group].double()])
            x = s["q"][q0:q1, h].double() @ k.T * HEAD ** -0.5
            out[q0:q1, h] = torch.softmax(x.masked_fill(~seen, -math.inf), dim=-1) @ v
    return out
