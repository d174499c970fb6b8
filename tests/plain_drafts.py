"""Plain forms, on the host, of a step that verifies drafted tokens: trees, the fields of the step, attention, the accepted path."""
import random

import torch


def random_forest(lens, kind, seed):
    """Parents of every request's drafts: a chain, a bush (all children of draft 0) or a random tree."""
    rng = random.Random(seed)
    pick = {"chain": lambda i: i - 1, "bush": lambda i: 0, "tree": lambda i: rng.randrange(max(0, i - 7), i)}[kind]
    return [[-1] + [pick(i) for i in range(1, n)] if n else [] for n in lens]


def ancestors(up):
    """For every draft the set of its ancestors and itself; a parent that is no earlier draft is none."""
    out = []
    for i, p in enumerate(up):
        out.append((out[p] if 0 <= p < i else frozenset()) | {i})
    return out


def mask_rows(up, words):
    """The mask rows of one request as int32 words."""
    rows = []
    for anc in ancestors(up):
        bits = sum(1 << a for a in anc)
        rows.append([(w - (1 << 32) if w >= 1 << 31 else w) for w in ((bits >> (32 * k)) & 0xFFFFFFFF for k in range(words))])
    return rows


def random_tables(lens, cached, page_size, seed, spare=0):
    """(block table int32 [B, width], pages) over pages in random order; page 0 is for padding."""
    per = max((c + n + page_size - 1) // page_size for n, c in zip(lens, cached)) + spare
    per = max(per, 1)
    order = torch.randperm(per * len(lens), generator=torch.Generator().manual_seed(seed)) + 1
    return order.view(len(lens), per).to(torch.int32), per * len(lens)


def rows_of(cache, table_row, places):
    """Rows [n, kv heads, d] of a cache [pages, kv heads, page size, d]."""
    P = cache.shape[2]
    places = torch.as_tensor(places, device=cache.device, dtype=torch.long)
    return cache[table_row.to(cache.device).long()[places // P], :, places % P]


def tree_attention(q, k_cache, v_cache, table, lens, cached, masks, scale):
    """q [T, n_q, d]; masks: per request a bool [n, n] -> float64 [T, n_q, dv].  A key that a draft does not see counts for nothing, whatever it holds."""
    n_kv, d = k_cache.shape[1], q.shape[2]
    G, t, outs = q.shape[1] // n_kv, 0, []
    for r, (n, c) in enumerate(zip(lens, cached)):
        if n:
            kk, vv = (rows_of(x, table[r], torch.arange(c + n)).double() for x in (k_cache, v_cache))
            seen = torch.ones(n, c + n, dtype=torch.bool, device=q.device)
            seen[:, c:] = masks[r].to(q.device)
            for i in range(n):
                at = seen[i].nonzero()[:, 0]
                if len(at) == 0:
                    outs.append(torch.zeros(q.shape[1], v_cache.shape[3], dtype=torch.float64, device=q.device))
                    continue
                s = torch.einsum("hgd,khd->hgk", q[t + i].double().view(n_kv, G, d), kk[at]) * scale
                outs.append(torch.einsum("hgk,khd->hgd", s.softmax(-1), vv[at]).reshape(q.shape[1], -1))
        t += n
    return torch.stack(outs) if outs else torch.zeros(0, q.shape[1], v_cache.shape[3], dtype=torch.float64, device=q.device)


def accepted(up, tokens, following):
    """The path from draft 0 along the first children whose tokens are what the model put after their parents."""
    path, at = ([0] if up else []), 0
    while path:
        nxt = [i for i in range(at + 1, len(up)) if up[i] == at and tokens[i] == following[at]]
        if not nxt:
            return path
        at = nxt[0]
        path.append(at)
    return path
