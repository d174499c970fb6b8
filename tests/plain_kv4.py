"""A key/value cache in 4 bits, computed plainly: rows in separately rounded float32 operations (so that codes can be compared bit for bit), attention in 64 bits."""
import math

import torch


def quantised(x):
    """float32 rows [.., d] -> codes uint8 [.., d], step, base (bfloat16 [..])."""
    low, high = x.amin(-1), x.amax(-1)          # (both keep a NaN)
    base = low.to(torch.bfloat16)
    step = ((high - base.float()) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)).to(torch.bfloat16)
    bad = ~(base.float().isfinite() & step.float().isfinite())
    step = torch.where(bad | ~(step.float() >= 2.0 ** -100), torch.zeros_like(step), step)
    base = torch.where(bad, torch.full_like(base, math.nan), base)
    flat = step.float()[..., None] == 0
    codes = ((x - base.float()[..., None]) / torch.where(flat, 1.0, step.float()[..., None])).round().clamp(0, 15)
    return torch.where(flat, 0.0, codes).to(torch.uint8), step, base


def packed(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def values(cache, i):
    """Keys (i = 0) or values (i = 1) of a whole cache (k, v, steps), in 64 bits (what float32 holds: one rounding of base + code * step)."""
    p, steps = cache[i], cache[2].float()
    codes = torch.stack((p & 15, p >> 4), dim=-1).flatten(-2).float()
    return (steps[..., 2 * i + 1, None] + codes * steps[..., 2 * i, None]).double()


def append(qkv, positions, n_q, n_kv, d, q_weight, k_weight, eps, table, slots, cache, interleaved=False):
    """-> q [T, n_q, d] in float32 (not rounded to qkv's type); the cache (k, v, steps) is written in place."""
    x = qkv.float().view(-1, n_q + 2 * n_kv, d)
    T, P = x.shape[0], cache[0].shape[2]

    def placed(y, w):
        if w is not None:
            mean = (y.double().square().sum(-1, keepdim=True) / d).float()
            y = y * (1.0 / torch.sqrt(mean + torch.tensor(eps, dtype=torch.float32, device=y.device))) * w.float()
        if table is None:
            return y
        rot = table.shape[1]
        cs = table[positions.long().clamp(0, table.shape[0] - 1)][:, None]
        c, s, y, rest = cs[..., :rot // 2], cs[..., rot // 2:], y[..., :rot], y[..., rot:]
        a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:])
        turned = a * c - b * s, a * s + b * c
        return torch.cat([torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1), rest], -1)

    keep = (slots >= 0) & (slots < cache[0].shape[0] * P)
    at = slots[keep].long()
    for i, rows in enumerate((placed(x[:, n_q:n_q + n_kv], k_weight), x[:, n_q + n_kv:])):
        codes, step, base = quantised(rows[keep])
        cache[i][at // P, :, at % P] = packed(codes)
        cache[2][at // P, :, at % P, 2 * i] = step
        cache[2][at // P, :, at % P, 2 * i + 1] = base
    return placed(x[:, :n_q], q_weight)


def attention(q, cache, q_start, q_lens, kv_lens, block_table, scale, window=0):
    """-> (o [T, heads, d] in 64 bits, 0 where a token sees no key or no request brings it; per token and head: the largest sum |q_i k_i| * scale over its
    keys, the largest |v| and the largest step of a value among them, the largest |q| sum times key step * scale)."""
    T, n_q, d = q.shape
    pages, n_kv, P = cache[0].shape[:3]
    G = n_q // n_kv
    keys, vals = values(cache, 0), values(cache, 1)
    steps = cache[2].double()
    out, facts = torch.zeros(T, n_q, d, dtype=torch.float64, device=q.device), torch.zeros(T, n_q, 4, dtype=torch.float64, device=q.device)
    for r, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        t0 = int(q_start[r])
        for i in range(n):
            pos = kv - n + i
            lo = max(0, pos - window + 1) if window else 0
            if pos < lo:
                continue
            at = torch.arange(lo, pos + 1, device=q.device)
            page, slot = block_table[r].long()[at // P], at % P
            ok = (page >= 0) & (page < pages)
            pick = lambda x: torch.where(ok.view(-1, *[1] * (x.dim() - 2)), x[page.clamp(0, pages - 1), :, slot], 0.0)      # noqa: E731
            k, v, st = pick(keys), pick(vals), pick(steps)
            for h in range(n_kv):
                rows = q[t0 + i, h * G:(h + 1) * G].double()
                s = rows @ k[:, h].T * scale
                p = torch.softmax(s, dim=-1)
                out[t0 + i, h * G:(h + 1) * G] = p @ v[:, h]
                facts[t0 + i, h * G:(h + 1) * G, 0] = (rows.abs() @ k[:, h].abs().T).amax(-1) * scale
                facts[t0 + i, h * G:(h + 1) * G, 1] = v[:, h].abs().max()
                facts[t0 + i, h * G:(h + 1) * G, 2] = st[:, h, 2].max()
                facts[t0 + i, h * G:(h + 1) * G, 3] = rows.abs().sum(-1) * st[:, h, 0].max() * scale
    return out, facts
