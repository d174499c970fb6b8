"""Operators timed beside their plain forms: what a serving step with drafted tokens needs around the model's layers.

A request hands the model a tree of drafted tokens behind its cached ones.  Draft 0 is the newest accepted token, the parent of any
other is an earlier draft; draft i lies in the cache at place `cached + i` and at position `cached + depth`.

  plan       draft lengths, cached lengths and parents -> offsets, lengths, positions, cache slots and ancestor masks of all drafts
  attention  every draft over all cached keys of its request and over its ancestors and itself
  accept     the longest path from draft 0 whose every token is the one that the model put after its parent; the keys and values
             of that path move to the places that follow the cached tokens
  logprobs   log probabilities of given tokens, the entropy of every row, and its most probable tokens

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
PAGE = 16
VOCAB = 151936
#          query heads, kv heads (head size 128): the 0.6B and 1.7B, the 4B and 8B, the 14B and the 32B models
HEADS = {"1.7b": (16, 8), "8b": (32, 8), "14b": (40, 8), "32b": (64, 8)}


def listed():
    return [
        # one user, a short draft behind a short conversation: launch and latency
        {"name": "attention_1x8_behind_1000", "op": "attention", "heads": "8b", "requests": 1, "drafts": 8, "cached": 1000, "tree": False, "dtype": "bfloat16"},
        # a batch that verifies chains of a small draft model
        {"name": "attention_16x5_behind_4096", "op": "attention", "heads": "8b", "requests": 16, "drafts": 5, "cached": 4096, "tree": False, "dtype": "bfloat16"},
        # a busy server with trees of an odd size behind long conversations
        {"name": "attention_48x49_behind_8192", "op": "attention", "heads": "8b", "requests": 48, "drafts": 49, "cached": 8192, "tree": True, "dtype": "bfloat16"},
        # the widest group of query heads, the largest tree, one long document
        {"name": "attention_2x128_behind_16000", "op": "attention", "heads": "32b", "requests": 2, "drafts": 128, "cached": 16000, "tree": True, "dtype": "bfloat16"},
        # the float32 path of the whole model, used to check others
        {"name": "attention_f32_4x26_behind_1500", "op": "attention", "heads": "1.7b", "requests": 4, "drafts": 26, "cached": 1500, "tree": True, "dtype": "float32"},
        # one user: the fields of a step of eight drafts
        {"name": "plan_1x8", "op": "plan", "requests": 1, "drafts": 8, "cached": 1000},
        # a full batch of large trees
        {"name": "plan_256x64", "op": "plan", "requests": 256, "drafts": 64, "cached": 8192},
        # one user, all layers of the smallest model
        {"name": "accept_1x8_28_layers", "op": "accept", "requests": 1, "drafts": 8, "cached": 100, "layers": 28, "dtype": "bfloat16"},
        # a batch of large trees, the layers of one cache group
        {"name": "accept_64x61_4_layers", "op": "accept", "requests": 64, "drafts": 61, "cached": 64, "layers": 4, "dtype": "bfloat16"},
        # one decoded token whose user asked for alternatives
        {"name": "logprobs_1_top_20", "op": "logprobs", "rows": 1, "vocab": VOCAB, "top": 20, "dtype": "float32"},
        # the tokens of a prompt portion scored, five alternatives each
        {"name": "logprobs_2048_top_5", "op": "logprobs", "rows": 2048, "vocab": VOCAB, "top": 5, "dtype": "float32"},
        # a batch over an odd vocabulary, bfloat16 logits
        {"name": "logprobs_100_odd_bf16", "op": "logprobs", "rows": 100, "vocab": 32003, "top": 8, "dtype": "bfloat16"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "plan", "accept", "logprobs", "logprobs"])
    if op == "attention":
        heads, dtype = rng.choice(sorted(HEADS)), "float32" if rng.random() < 0.15 else "bfloat16"
        requests, drafts = _log_int(rng, 1, 48), _log_int(rng, 1, 128)
        most = int(6e8 if dtype == "bfloat16" else 2e7) // (requests * drafts * HEADS[heads][0])      # pairs of a query and a key: no more than in the largest listed case
        return {"op": op, "heads": heads, "requests": requests, "drafts": drafts, "cached": _log_int(rng, 1, max(2, min(16000, most, 390000 // requests))),
                "tree": rng.random() < 0.6, "dtype": dtype}
    if op == "plan":
        return {"op": op, "requests": _log_int(rng, 1, 256), "drafts": _log_int(rng, 1, 64), "cached": _log_int(rng, 1, 8192)}
    if op == "accept":
        requests, dtype = _log_int(rng, 1, 64), rng.choice(["bfloat16", "bfloat16", "float32"])
        return {"op": op, "requests": requests, "drafts": _log_int(rng, 1, 61), "cached": _log_int(rng, 1, 64 if requests > 2 else 100),
                "layers": rng.randint(1, max(1, min(28, 512 // ITEM[dtype] // requests))), "dtype": dtype}
    vocab = _log_int(rng, 500, VOCAB)
    return {"op": op, "rows": _log_int(rng, 1, min(4096, 2048 * VOCAB // vocab)), "vocab": vocab, "top": rng.randint(0, 20), "dtype": rng.choice(["float32", "float32", "bfloat16"])}


# -- what a case has, apart from its values ------------------------------------------------------------

def _rng(case):
    """Random numbers that follow from a case's sizes alone."""
    return random.Random("%(op)s %(requests)d %(drafts)d %(cached)d" % case)


def _lengths(case):
    """(drafts, cached tokens) of every request: the first has the most of both, some of a larger batch bring no draft."""
    rng = _rng(case)
    B, D, C = case["requests"], case["drafts"], case["cached"]
    drafts = [D] + [0 if rng.random() < 0.04 else rng.randint((D + 1) // 2, D) for _ in range(B - 1)]
    cached = [C] + [rng.randint(C // 2, C) for _ in range(B - 1)]
    return drafts, cached


def _parents(case, n, rng):
    """A chain, or a tree whose drafts continue one of the nine before them."""
    return [-1] + [i - 1 if not case.get("tree", True) else rng.randint(max(0, i - 9), i - 1) for i in range(1, n)] if n else []


def _forest(case, rng):
    """Parents of every request's drafts (an index within the request, -1 for its first)."""
    return [_parents(case, n, rng) for n in _lengths(case)[0]]


def _agreed(case):
    """(parents, drafts that the model agrees with) of every request: a path from draft 0 of up to about a sixth of the tree."""
    rng, out = _rng(case), []
    for up in _forest(case, rng):
        path = [0] if up else []
        while path and len(path) < 1 + (len(up) + 5) // 6 and path[-1] in up:
            path.append(rng.choice([i for i, p in enumerate(up) if p == path[-1]]))
        out.append((up, path))
    return out


def _seen_pairs(case):
    """Pairs of a draft and a key that it sees: of the cached keys all, of the drafts about a path."""
    drafts, cached = _lengths(case)
    depth = (lambda n: n * (n + 1) // 2) if not case["tree"] else (lambda n: sum(1 + i // 5 for i in range(n)))
    return sum(n * c + depth(n) for n, c in zip(drafts, cached))


# -- inputs ----------------------------------------------------------------------------------------------

def _int32(values, device="cuda"):
    return torch.tensor(list(values), dtype=torch.int32, device=device)


def _tables(case, seed, per_request):
    """Block tables over pages in random order, page 0 left out (padding goes there) -> (table, number of pages)."""
    B = case["requests"]
    order = np.random.RandomState(seed % (1 << 31)).permutation(B * per_request) + 1
    return torch.from_numpy(order.reshape(B, per_request).astype(np.int32)).cuda(), B * per_request


def _ancestors(forest, width):
    """[B, width, width], 1 where the column is the row's draft or one of its ancestors, from the chain of parents, on the host."""
    out = np.zeros((len(forest), width, width), dtype=np.uint8)
    for b, up in enumerate(forest):
        for i, p in enumerate(up):
            if p >= 0:
                out[b, i] = out[b, p]
            out[b, i, i] = 1
    return out


def _values(seed, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def prepare(case, seed):
    op = case["op"]
    if op == "logprobs":
        N, V = case["rows"], case["vocab"]
        logits = _values(seed, (N, V), torch.float32, 2.5)
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        likely = torch.randint(0, V, (N, 4), generator=g, device="cuda")           # a few tokens stand out, as a model's do
        logits.scatter_add_(1, likely, torch.rand(N, 4, generator=g, device="cuda") * 12.0)
        logits = logits.to(DTYPES[case["dtype"]])
        return {"case": case, "logits": logits, "tokens": likely[:, 0].to(torch.int32).contiguous()}
    drafts, cached = _lengths(case)
    agreed = _agreed(case) if op == "accept" else None
    forest = [up for up, _ in agreed] if agreed else _forest(case, random.Random(seed))
    parents = [p for up in forest for p in up]
    D, B = case["drafts"], case["requests"]
    pages = -(-(case["cached"] + D) // PAGE)
    table, n_pages = _tables(case, seed, pages)
    state = {"case": case, "table": table, "drafts": _int32(drafts), "cached": _int32(cached), "parents": _int32(parents)}
    if op == "plan":
        return state
    starts = np.concatenate([[0], np.cumsum(drafts)])
    state.update(q_start=_int32(starts), kv_len=_int32(n + c for n, c in zip(drafts, cached)))
    dtype = DTYPES[case["dtype"]]
    if op == "attention":
        n_q, n_kv = HEADS[case["heads"]]
        words = -(-D // 32)
        bits = np.zeros((B, D, words * 32), dtype=np.uint8)
        bits[:, :, :D] = _ancestors(forest, D)
        packed = np.packbits(bits, axis=-1, bitorder="little").view(np.int32)
        state["mask"] = torch.from_numpy(np.concatenate([packed[b, :n] for b, n in enumerate(drafts)])).cuda()
        state["q"] = _values(seed, (len(parents), n_q, 128), dtype)
        state["k"] = _values(seed + 1, (n_pages + 1, n_kv, PAGE, 128), dtype)
        state["v"] = _values(seed + 2, (n_pages + 1, n_kv, PAGE, 128), dtype)
        return state
    # accept: the model agrees along one path of each tree and nowhere else but by chance
    rng = random.Random(seed)
    tokens = [rng.randrange(VOCAB) for _ in parents]
    following = [rng.randrange(VOCAB) for _ in parents]
    for first, (_, path) in zip(starts, agreed):
        for a, b in zip(path, path[1:]):
            following[first + a] = tokens[first + b]
    state.update(tokens=_int32(tokens), following=_int32(following))
    state["caches"] = [_values(seed + 10 + i, (n_pages + 1, 8, PAGE, 128), dtype) for i in range(2 * case["layers"])]
    return state


# -- the operators -----------------------------------------------------------------------------------------

def run(state):
    return {"attention": _attention, "plan": _plan, "accept": _accept, "logprobs": _logprobs}[state["case"]["op"]](state)


def _places(table, places):
    """Pages and rows of places [B, n] of every request."""
    return table.long().gather(1, places // PAGE), places % PAGE


def _attention(s):
    q, k, v, case = s["q"], s["k"], s["v"], s["case"]
    T, n_q, d = q.shape
    B, D, n_kv, scale = case["requests"], case["drafts"], k.shape[1], d ** -0.5
    if own:
        from mini_sglang_b200 import ops
        out = torch.empty_like(q)
        ops.tree_attention(q, out, k, v, q_start=s["q_start"], kv_len=s["kv_len"], block_table=s["table"], mask=s["mask"], n_kv=n_kv, page_size=PAGE,
                           scale=scale, max_draft=D)
        return out
    G, L = n_q // n_kv, s["table"].shape[1] * PAGE
    key = torch.arange(L, device=q.device)
    keys = k[s["table"].long()].float().permute(0, 2, 1, 3, 4).reshape(B, n_kv, L, d)
    values = v[s["table"].long()].float().permute(0, 2, 1, 3, 4).reshape(B, n_kv, L, d)
    first, n = s["q_start"][:-1].long(), s["drafts"].long()
    row = first[:, None] + torch.arange(D, device=q.device)
    there = torch.arange(D, device=q.device) < n[:, None]                                     # [B, D]
    row = torch.where(there, row, 0)
    rows = q[row].float().reshape(B, D, n_kv, G, d).permute(0, 2, 1, 3, 4).reshape(B, n_kv, D * G, d)
    bits = (s["mask"][row].long()[..., None] >> torch.arange(32, device=q.device)) & 1        # [B, D, words, 32]
    among = key[None, :] - s["cached"].long()[:, None]                                        # the key's number among the drafts
    drafted = bits.reshape(B, D, -1).gather(2, among.clamp(0, bits.shape[2] * 32 - 1)[:, None, :].expand(B, D, L)) > 0
    seen = torch.where((among < 0)[:, None, :], True, drafted & (among < n[:, None])[:, None, :])
    scores = rows @ keys.transpose(2, 3) * scale
    seen = seen[:, None, :, None, :].expand(B, n_kv, D, G, L).reshape(B, n_kv, D * G, L)
    scores = scores.masked_fill(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
    total = p.sum(-1, keepdim=True)
    values = values.masked_fill((key[None, :] >= s["kv_len"].long()[:, None])[:, None, :, None], 0.0)
    o = torch.where(total > 0, p @ values / total, 0.0)
    return o.reshape(B, n_kv, D, G, d).permute(0, 2, 1, 3, 4).reshape(B, D, n_q, d)[there].to(q.dtype)


def _closure(parents, first, there):
    """(ancestors [B, D, D] with the draft itself, parents [B, D]) of packed trees: the inverse of I - P, P a one where the column is the row's parent."""
    B, D = there.shape
    at = torch.arange(D, device=parents.device)
    up = torch.where(there, parents[torch.where(there, first[:, None] + at, 0)].long(), -1)
    eye = torch.eye(D, device=parents.device)
    step = (up[:, :, None] == at).float()
    return torch.linalg.solve_triangular(eye - step, eye.expand(B, D, D), upper=False, unitriangular=True), up


def _plan(s):
    if own:
        from mini_sglang_b200 import ops
        p = ops.draft_plan(s["parents"], s["drafts"], s["cached"], s["table"], page_size=PAGE, max_draft=s["case"]["drafts"])
        return [p.q_start, p.kv_len, p.positions, p.token_req, p.out_loc, p.mask]
    B, D = s["case"]["requests"], s["case"]["drafts"]
    at = torch.arange(D, device="cuda")
    n, cached = s["drafts"].long(), s["cached"].long()
    end = n.cumsum(0)
    there = at < n[:, None]
    above, _ = _closure(s["parents"], end - n, there)
    page, slot = _places(s["table"], cached[:, None] + at)
    words = torch.nn.functional.pad(above, (0, -D % 32)).long().reshape(B, D, -1, 32)
    words = (words << torch.arange(32, device="cuda")).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words)
    fields = [torch.cat([torch.zeros_like(end[:1]), end]), n + cached, (cached[:, None] + above.sum(-1).long() - 1)[there],
              torch.arange(B, device="cuda")[:, None].expand(B, D)[there], (page * PAGE + slot)[there], words[there]]
    return [f.to(torch.int32) for f in fields]


def _accept(s):
    if own:
        from mini_sglang_b200 import ops
        a = ops.draft_accept(s["tokens"], s["parents"], s["following"], s["q_start"], max_draft=s["case"]["drafts"], kv_len=s["kv_len"], block_table=s["table"],
                             caches=s["caches"])
        return [a.kept, a.path, a.tokens] + s["caches"]
    B, D = s["case"]["requests"], s["case"]["drafts"]
    at = torch.arange(D, device="cuda")
    n, cached, first = s["drafts"].long(), s["cached"].long(), s["q_start"][:-1].long()
    there = at < n[:, None]
    above, up = _closure(s["parents"], first, there)
    row = torch.where(there, first[:, None] + at, 0)
    token, after = s["tokens"][row], s["following"][row]
    wanted = (up >= 0) & (token == after.gather(1, up.clamp_min(0)))
    rival = (up[:, :, None] == up[:, None, :]) & wanted[:, None, :] & (at[None, :] < at[:, None])      # an earlier child of the same draft that fits as well
    fits = there & ((at == 0) | (wanted & ~rival.any(2)))
    whole = fits & ((above @ fits.float()[:, :, None])[:, :, 0] == above.sum(-1))
    kept = whole.sum(1)
    path = torch.where(whole, at, D).sort(1).values
    held = at < kept[:, None]
    moved = held & (path > at)
    source, target = (_places(s["table"], torch.where(moved, cached[:, None] + x, 0)) for x in (path, at))
    from_, to = ([torch.where(moved, x, 0).reshape(-1) for x in pair] for pair in (source, target))
    [c.__setitem__((to[0], slice(None), to[1]), c[from_[0], :, from_[1]]) for c in s["caches"]]        # what does not move: page 0, row 0 onto itself
    out = torch.where(held, after.gather(1, path.clamp_max(D - 1)), -1)
    return [kept.to(torch.int32), torch.where(held, path, -1).to(torch.int32), out.to(torch.int32)] + s["caches"]


def _logprobs(s):
    logits, tokens, top = s["logits"], s["tokens"], s["case"]["top"]
    if own:
        from mini_sglang_b200 import ops
        r = ops.token_logprobs(logits, tokens, top)
        return [r.logprobs, r.entropy, r.top_logprobs, r.top_tokens]
    parts = [_logprob_rows(x, t, top) for x, t in zip(logits.split(256), tokens.split(256))]
    return [torch.cat(x) for x in zip(*parts)]


def _logprob_rows(logits, tokens, top):
    given_as = logits.float()
    x = given_as - given_as.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    log_total = torch.log(total)
    given = x.gather(1, tokens.long()[:, None]).double() - log_total
    entropy = log_total - (e * x).sum(1, keepdim=True, dtype=torch.float64) / total
    # one whole number a token, higher for the more probable and among equals for the lower index
    order = (given_as + 0.0).view(torch.int32).long()
    order = torch.where(order < 0, -(order & 0x7FFFFFFF), order) * (1 << 20) - torch.arange(x.shape[1], device=x.device)
    best = order.topk(top, dim=1).values
    at = (-best) % (1 << 20)
    return [given[:, 0].float(), entropy[:, 0].float(), (x.gather(1, at).double() - log_total).float(), at.to(torch.int32)]


# -- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "logprobs":
        N, V = case["rows"], case["vocab"]
        return {"bytes": N * V * ITEM[case["dtype"]] + N * (12 + 8 * case["top"]), "flops": 6 * N * V}
    drafts, cached = _lengths(case)
    T, B = sum(drafts), case["requests"]
    if op == "plan":
        return {"bytes": 4 * (T * (4 + -(-case["drafts"] // 32)) + B * 5) + 8 * T // PAGE, "flops": T * case["drafts"]}
    if op == "accept":
        rows = sum(i != p for _, path in _agreed(case) for i, p in enumerate(path))
        return {"bytes": rows * 8 * 128 * ITEM[case["dtype"]] * 4 * case["layers"] + 4 * (3 * T + 2 * B * case["drafts"] + 3 * B), "flops": T * case["drafts"]}
    n_q, n_kv = HEADS[case["heads"]]
    read = sum(n + c for n, c in zip(drafts, cached) if n)
    return {"bytes": (2 * read * n_kv + 2 * T * n_q) * 128 * ITEM[case["dtype"]] + 4 * (T * -(-case["drafts"] // 32) + read // PAGE), "flops": 4 * _seen_pairs(case) * n_q * 128}


# -- the definitions in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        parts = []
        for x, t in zip(s["logits"].split(128), s["tokens"].split(128)):
            lp = torch.log_softmax(x.double(), 1)
            ids = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
            parts.append([lp.gather(1, t.long()[:, None])[:, 0], -(lp.exp() * lp).sum(1), lp.gather(1, ids), ids.to(torch.int32)])
        return [torch.cat(x) for x in zip(*parts)]
    if case["op"] == "plan":
        return None
    if case["op"] == "accept":
        for b, (_, path) in enumerate(_agreed(case)):
            base = int(s["cached"][b])
            for i, p in enumerate(path):
                to, at = base + i, base + p
                for c in s["caches"]:
                    c[s["table"][b, to // PAGE], :, to % PAGE] = c[s["table"][b, at // PAGE], :, at % PAGE]
        return [None, None, None] + [c.double() for c in s["caches"]]
    n_kv, drafts = s["k"].shape[1], _lengths(case)
    above, out, t = _ancestors(_forest(case, random.Random(seed)), case["drafts"]), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, c) in enumerate(zip(*drafts)):
        if n == 0:
            continue
        pages = s["table"][b].long()
        seen = torch.ones(n, n + c, dtype=torch.bool, device="cuda")
        seen[:, c:] = torch.from_numpy(above[b, :n, :n]).cuda() > 0
        for h in range(n_kv):
            keys, values = (x[pages, h].reshape(-1, 128)[:n + c].double() for x in (s["k"], s["v"]))
            group = slice(h * (s["q"].shape[1] // n_kv), (h + 1) * (s["q"].shape[1] // n_kv))
            scores = torch.einsum("tgd,kd->tgk", s["q"][t:t + n, group].double(), keys) / math.sqrt(128.0)
            p = torch.softmax(torch.where(seen[:, None, :], scores, -math.inf), dim=-1)
            out[t:t + n, group] = torch.einsum("tgk,kd->tgd", p, values)
        t += n
    return out
