"""Operators of a key/value cache held in 4 bits, timed beside their plain forms.

A key or value of one token under one kv head is a row of `d` codes between 0 and 15, two to a byte (the even element in the low half), and two bfloat16
numbers: an element stands for base + code * step in 32 bits.

  append     queries and keys normed by heads and rotated, keys and values put into 4 bits at their places in the cache; the pages that they went to read back
  attention  causal attention of a step's tokens over the cache: single tokens, a few tokens a request, prompt portions, all of them in one step

`run` computes them with elementary operations in 32 bits; with `own` it calls the engine's kernels.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
ITEM = {"bfloat16": 2, "float32": 4}
D = 128
EPS = 1e-6
POSITIONS = 40960
#          query heads, kv heads (head size 128): the 0.6B and 1.7B, the 4B and 8B, the 14B and the 32B models
HEADS = {"1.7b": (16, 8), "8b": (32, 8), "14b": (40, 8), "32b": (64, 8)}


def listed():
    a = {"op": "attention", "heads": "8b", "page": 16, "window": 0, "dtype": "bfloat16"}
    p = {"op": "append", "heads": "8b", "page": 16, "norm": True, "dtype": "bfloat16"}
    return [
        # one user's next token in a short conversation: launch and latency
        {"name": "attention_1x1_behind_1000", **a, "requests": 1, "tokens": 1, "cached": 1000, "mixed": False},
        # a small batch of like lengths
        {"name": "attention_16x1_behind_4096", **a, "requests": 16, "tokens": 1, "cached": 4096, "mixed": False},
        # a busy server, long conversations of all lengths
        {"name": "attention_64x1_behind_16000", **a, "requests": 64, "tokens": 1, "cached": 16000, "mixed": False},
        # the widest group of query heads, many short conversations, an odd number of them
        {"name": "attention_123x1_behind_777_32b", **a, "heads": "32b", "requests": 123, "tokens": 1, "cached": 777, "mixed": False},
        # tokens given several at a time behind long conversations, within a window, pages of 64
        {"name": "attention_12x5_window_2000", **a, "heads": "14b", "page": 64, "window": 2000, "requests": 12, "tokens": 5, "cached": 9001, "mixed": False},
        # a prompt portion behind the portions before it
        {"name": "attention_1x2048_behind_6144", **a, "requests": 1, "tokens": 2048, "cached": 6144, "mixed": False},
        # odd portions with single tokens among them, as a scheduler puts a step together
        {"name": "attention_9_mixed_behind_3001", **a, "requests": 9, "tokens": 801, "cached": 3001, "mixed": True},
        # the float32 path of the whole model, used to check others
        {"name": "attention_f32_4x1_behind_1500", **a, "heads": "1.7b", "requests": 4, "tokens": 1, "cached": 1500, "mixed": False, "dtype": "float32"},
        # one user's next token
        {"name": "append_1x1", **p, "requests": 1, "tokens": 1, "cached": 1000},
        # a full decode batch
        {"name": "append_128x1", **p, "requests": 128, "tokens": 1, "cached": 2000},
        # portions of an odd length, heads without a norm, pages of 64
        {"name": "append_3x637_plain", **p, "heads": "14b", "page": 64, "norm": False, "requests": 3, "tokens": 637, "cached": 123},
        # the largest portion that a step takes
        {"name": "append_1x8192", **p, "requests": 1, "tokens": 8192, "cached": 0},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op, heads, page = rng.choice(["attention", "attention", "append"]), rng.choice(sorted(HEADS)), rng.choice([16, 16, 16, 64, 1])
    if op == "append":
        requests = _log_int(rng, 1, 128)
        tokens = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, 6000 // requests))
        return {"op": op, "heads": heads, "page": page, "norm": rng.random() < 0.7, "dtype": "bfloat16", "requests": requests, "tokens": tokens, "cached": _log_int(rng, 1, 8192)}
    dtype = "float32" if rng.random() < 0.1 else "bfloat16"
    kind = rng.choice(["single", "single", "few", "portion", "mixed"]) if dtype == "bfloat16" else "single"
    case = {"op": op, "heads": heads, "page": page, "window": _log_int(rng, 16, 4096) if rng.random() < 0.2 else 0, "dtype": dtype, "mixed": kind == "mixed"}
    if kind == "single":
        requests = _log_int(rng, 1, 128 if dtype == "bfloat16" else 8)
        return {**case, "requests": requests, "tokens": 1, "cached": _log_int(rng, 1, min(16000, 800000 // requests) if dtype == "bfloat16" else 1500)}
    if kind == "few":
        requests = _log_int(rng, 1, 24)
        return {**case, "requests": requests, "tokens": rng.randint(2, 12), "cached": _log_int(rng, 1, 8192)}
    requests = rng.randint(1, 3) if kind == "portion" else rng.randint(2, 9)
    tokens = _log_int(rng, 13, 1600 // requests)
    return {**case, "requests": requests, "tokens": tokens, "cached": _log_int(rng, 1, 8000 // requests)}


# -- what a case has, apart from its values ------------------------------------------------------------

def _lengths(case):
    """(new tokens, cached tokens) of every request: the first has the most of both; where the step is mixed, half of the others bring one token."""
    rng = random.Random("%(op)s %(requests)d %(tokens)d %(cached)d" % case)
    B, n, C = case["requests"], case["tokens"], case["cached"]
    cached = [C] + [rng.randint(C // 2, C) for _ in range(B - 1)]
    if case["op"] == "append" or n == 1:
        return [n] * B, cached
    fewer = lambda: 1 if case.get("mixed") and rng.random() < 0.5 else rng.randint((n + 1) // 2, n)      # noqa: E731
    return [n] + [fewer() for _ in range(B - 1)], cached


def _seen_keys(case):
    """(keys that are read of every request, pairs of a token and a key that it sees)."""
    read, pairs, W = [], 0, case["window"]
    for n, c in zip(*_lengths(case)):
        read.append(min(n + c, n + W - 1) if W else n + c)
        pairs += sum(min(c + i + 1, W or c + i + 1) for i in range(n))
    return read, pairs


# -- inputs ----------------------------------------------------------------------------------------------

def _int32(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def _normal(seed, shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _angles():
    freq = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    at = torch.arange(POSITIONS, dtype=torch.float64)[:, None] * freq
    return torch.cat([at.cos(), at.sin()], dim=1).float().cuda()


def _cache(seed, pages, n_kv, page):
    """A cache of keys and values as they are met: keys with a few large elements (rotated pairs that carry position), values without."""
    out = []
    for i in range(2):
        x = _normal(seed + i, (pages, n_kv, page, D), torch.float32)
        if i == 0:
            x[..., 5::32] *= 4.0
        codes, step, base = _quantised(x)
        out += [_packed(codes), step, base]
    return out[0], out[3], torch.stack([out[1], out[2], out[4], out[5]], dim=-1)


def prepare(case, seed):
    n_q, n_kv = HEADS[case["heads"]]
    P, dtype = case["page"], DTYPES[case["dtype"]]
    tokens, cached = _lengths(case)
    T, B = sum(tokens), len(tokens)
    kv = [n + c for n, c in zip(tokens, cached)]
    width = -(-max(kv) // P)
    rng = np.random.RandomState(seed % (1 << 31))
    table = (rng.permutation(B * width) + 1).reshape(B, width).astype(np.int32)          # page 0 is where padding goes
    k, v, steps = _cache(seed, B * width + 1, n_kv, P)
    starts = np.concatenate([[0], np.cumsum(tokens)])
    state = {"case": case, "kv": [k, v], "steps": steps}
    if case["op"] == "attention":
        one = max(tokens) == 1
        state.update(q=_normal(seed + 5, (T, n_q, D), dtype), q_start=_int32(starts), kv_len=_int32(kv), table=torch.from_numpy(table).cuda(),
                     q_lens=None if one else tokens, kv_lens=None if one else kv)
        return state
    position = np.concatenate([np.arange(c, c + n) for n, c in zip(tokens, cached)])
    request = np.repeat(np.arange(B), tokens)
    page = table[request, position // P]
    state.update(qkv=_normal(seed + 5, (T, (n_q + 2 * n_kv) * D), dtype), positions=_int32(position), slots=_int32(page.astype(np.int64) * P + position % P),
                 touched=_int32(np.unique(page)), angles=_angles(), q_weight=1 + 0.05 * _normal(seed + 6, (D,), torch.float32) if case["norm"] else None,
                 k_weight=1 + 0.05 * _normal(seed + 7, (D,), torch.float32) if case["norm"] else None)
    return state


# -- the plain forms ------------------------------------------------------------------------------------------

def _quantised(x):
    """Rows of float32 -> codes (uint8), steps and bases (bfloat16)."""
    base = x.amin(-1).to(torch.bfloat16)
    step = ((x.amax(-1) - base.float()) * (1.0 / 15.0)).to(torch.bfloat16)
    codes = ((x - base.float()[..., None]) / step.float()[..., None]).round().clamp(0, 15).to(torch.uint8)
    return codes, step, base


def _packed(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _values(packed, step, base):
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2).float()
    return base.float()[..., None] + codes * step.float()[..., None]


def run(state):
    return _attention(state) if state["case"]["op"] == "attention" else _append(state)


_scratch = []          # the scratch tensors that a program keeps for all its steps


def _workspace():
    if not _scratch:
        from mini_sglang_b200.parts import Workspace
        _scratch.append(Workspace("cuda"))
    return _scratch[0]


def _normed(x, weight):
    if weight is None:
        return x
    mean = x.double().square().mean(-1, keepdim=True).float()          # in 64 bits: a code next to a border does not hang on the order of the sum
    return x * (1.0 / torch.sqrt(mean + EPS)) * weight


def _rotated(x, angles):
    cos, sin = angles[:, None, :D // 2], angles[:, None, D // 2:]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _append(s):
    case, qkv, T = s["case"], s["qkv"], s["qkv"].shape[0]
    n_q, n_kv = HEADS[case["heads"]]
    P, dtype = case["page"], DTYPES[case["dtype"]]
    if own:
        from mini_sglang_b200 import ops
        cache = ops.KV4Cache(*s["kv"], s["steps"])
        q = ops.qknorm_rope_kv4write(qkv, s["positions"], n_q, n_kv, D, q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, rope_table=s["angles"],
                                     out_loc=s["slots"], cache=cache)
        return [q, *ops.kv4_restore(cache, s["touched"], dtype)]
    x = qkv.float().view(T, n_q + 2 * n_kv, D)
    angles = s["angles"][s["positions"].long()]
    q = _rotated(_normed(x[:, :n_q], s["q_weight"]), angles)
    page, slot = s["slots"].long() // P, s["slots"].long() % P
    for i, rows in enumerate((_rotated(_normed(x[:, n_q:n_q + n_kv], s["k_weight"]), angles), x[:, n_q + n_kv:])):
        codes, step, base = _quantised(rows)
        s["kv"][i][page, :, slot] = _packed(codes)
        s["steps"][page, :, slot, 2 * i] = step
        s["steps"][page, :, slot, 2 * i + 1] = base
    at = s["touched"].long()
    return [q.to(dtype)] + [_values(s["kv"][i][at], s["steps"][at][..., 2 * i], s["steps"][at][..., 2 * i + 1]).to(dtype) for i in range(2)]


def _attention(s):
    case, q, table = s["case"], s["q"], s["table"].long()
    T, n_q, _ = q.shape
    n_kv, P, W, scale = HEADS[case["heads"]][1], case["page"], case["window"], D ** -0.5
    if own:
        from mini_sglang_b200 import ops
        out = torch.empty_like(q)
        ops.kv4_attention(q, out, ops.KV4Cache(*s["kv"], s["steps"]), q_start=s["q_start"], kv_len=s["kv_len"], block_table=s["table"], scale=scale, window=W,
                          q_lens=s["q_lens"], kv_lens=s["kv_lens"], workspace=_workspace())
        return out
    B, G, L, N = table.shape[0], n_q // n_kv, table.shape[1] * P, case["tokens"]
    keys, values = (_values(s["kv"][i][table], s["steps"][table][..., 2 * i], s["steps"][table][..., 2 * i + 1]).permute(0, 2, 1, 3, 4).reshape(B, n_kv, L, D) for i in range(2))
    first, kv = s["q_start"][:-1].long(), s["kv_len"].long()
    n = s["q_start"][1:].long() - first
    at = torch.arange(N, device=q.device)
    there = at < n[:, None]                                                                    # [B, N]
    row = torch.where(there, first[:, None] + at, 0)
    rows = q[row].float().reshape(B, N, n_kv, G, D).permute(0, 2, 1, 3, 4).reshape(B, n_kv, N * G, D)
    key, newest = torch.arange(L, device=q.device), (kv - n)[:, None] + at
    seen = key <= newest[..., None]
    if W:
        seen &= key > newest[..., None] - W
    seen = seen[:, None, :, None, :].expand(B, 1, N, G, L).reshape(B, 1, N * G, L)
    scores = (rows @ keys.transpose(2, 3) * scale).masked_fill_(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = p @ values / p.sum(-1, keepdim=True)
    return o.reshape(B, n_kv, N, G, D).permute(0, 2, 1, 3, 4).reshape(B, N, n_q, D)[there].to(q.dtype)


# -- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    n_q, n_kv = HEADS[case["heads"]]
    item, tokens = ITEM[case["dtype"]], _lengths(case)[0]
    T = sum(tokens)
    if case["op"] == "attention":
        read, pairs = _seen_keys(case)
        return {"bytes": sum(read) * n_kv * (D + 8) + 2 * T * n_q * D * item + 4 * (sum(read) // case["page"] + 2 * len(tokens)), "flops": 4 * pairs * n_q * D}
    pages = sum((c + n - 1) // case["page"] - c // case["page"] + 1 for n, c in zip(*_lengths(case)))
    restored = pages * case["page"] * n_kv
    return {"bytes": T * (2 * n_q + 2 * n_kv) * D * item + T * (4 * D + 8) + T * n_kv * (D + 8) + restored * (D + 8 + 2 * D * item), "flops": 20 * T * (n_q + 2 * n_kv) * D}


# -- the definitions in 64 bits --------------------------------------------------------------------------------

def _whole(s, i, pages):
    """Keys (i = 0) or values (i = 1) of some pages, [pages, kv heads, page, D] in 64 bits."""
    packed, st = s["kv"][i][pages], s["steps"][pages].double()
    codes = torch.empty(*packed.shape[:-1], D, dtype=torch.float64, device=packed.device)
    codes[..., 0::2] = (packed % 16).double()
    codes[..., 1::2] = (packed // 16).double()
    return st[..., 2 * i + 1, None] + codes * st[..., 2 * i, None]


def exact(case, seed):
    s = prepare(case, seed)
    n_q, n_kv = HEADS[case["heads"]]
    P, W = case["page"], case["window"] if case["op"] == "attention" else 0
    tokens, cached = _lengths(case)
    if case["op"] == "append":
        x = s["qkv"].double().view(-1, n_q + 2 * n_kv, D)
        turn = torch.complex(s["angles"][:, :D // 2].double(), s["angles"][:, D // 2:].double())[s["positions"].long()][:, None]

        def placed(y, weight):
            if weight is not None:
                y = y * torch.rsqrt((y * y).sum(-1, keepdim=True) / D + EPS) * weight.double()
            z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * turn
            return torch.cat([z.real, z.imag], dim=-1)

        out = [placed(x[:, :n_q], s["q_weight"])]
        where = torch.searchsorted(s["touched"].long(), s["slots"].long() // P)
        for i, rows in enumerate((placed(x[:, n_q:n_q + n_kv], s["k_weight"]), x[:, n_q + n_kv:])):
            low = rows.amin(-1, keepdim=True).to(torch.bfloat16).double()
            step = ((rows.amax(-1, keepdim=True) - low) / 15).to(torch.bfloat16).double()
            whole = _whole(s, i, s["touched"].long())
            whole[where, :, s["slots"].long() % P] = low + torch.clamp(torch.round((rows - low) / step), 0, 15) * step
            out.append(whole)
        return out
    out, t, G = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0, n_q // n_kv
    for b, (n, c) in enumerate(zip(tokens, cached)):
        pages = s["table"][b, :-(-(n + c) // P)].long()
        keys, values = (_whole(s, i, pages) for i in range(2))
        key, newest = torch.arange(n + c, device="cuda"), torch.arange(c, c + n, device="cuda")[:, None]
        hidden = (key > newest) | (key <= newest - W if W else torch.zeros_like(key > newest))
        for h in range(n_kv):
            k, v = (y[:, h].reshape(-1, D)[:n + c] for y in (keys, values))
            scores = torch.einsum("tgd,kd->gtk", s["q"][t:t + n, h * G:(h + 1) * G].double(), k) / math.sqrt(D)
            p = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=-1)
            out[t:t + n, h * G:(h + 1) * G] = torch.einsum("gtk,kd->tgd", p, v)
        t += n
    return out
