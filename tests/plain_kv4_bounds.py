"""What attention over a cache in 4 bits may be off by, token by token and head by head, from the roundings of the path that computes it.

Every path: float32 sums of d products leave a score off by (d + 8) 2^-24 of its terms' sizes (Kahan's classic bound, a term a rounding); scores off by x leave normed weights off by
e^(2 x) - 1 of themselves; float32 sums of weights and values over n keys add 2 (n + 64) 2^-24 of the sum of p |v|.
  float32      nothing else.
  codes        (mma on float16) A score's sum of q c, cut off by 2^-22 of up to 16 sum |q| in each of d / 16 + 1 additions; queries kept to 2^-35 of the largest, 15 codes a product.
               A weight p step is rounded to float16, half a step being 2^-11 of it, or 2^-25 where that is more; the row's largest weight lies at 2^-6 or above, so that this is
               2^-19 of the largest weight; both count by codes up to 15.  Sums of weights times codes less the middles (128 at most, a byte at a time), cut off by 2^-22 in each addition of 16 keys.
  restored     keys rounded to bfloat16, half a step being 2^-8 of a key (2^-8 of the score's terms), values likewise, weights likewise.
The result's own rounding is apart."""
import torch

import plain_kv4 as plain

U = 2.0 ** -24


def attention(q, cache, starts, q_lens, kv_lens, block_table, scale, window, path):
    """(o [T, heads, d] in 64 bits, how far `path` ("float32", "codes" or "restored") may be off before the result is rounded); rows that no request brings: 0.  A row sees keys or
    its result is 0; pages that are none are no part of this."""
    T, n_q, d = q.shape
    n_kv, P = cache[0].shape[1:3]
    G = n_q // n_kv
    keys, vals, steps = plain.values(cache, 0), plain.values(cache, 1), cache[2].double()
    out, off = (torch.zeros(T, n_q, d, dtype=torch.float64, device=q.device) for _ in range(2))
    for r, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        if n == 0 or kv == 0:
            continue
        at = torch.arange(kv, device=q.device)
        page = block_table[r].long()[at // P]
        k, v, st = (x[page, :, at % P].transpose(0, 1) for x in (keys, vals, steps))          # [heads, keys, ..]
        rows = q[starts[r]:starts[r] + n].double().view(n, n_kv, G, d).permute(1, 2, 0, 3)       # [heads, group, tokens, d]
        pos = kv - n + torch.arange(n, device=q.device)[:, None]
        hidden = (at > pos) | (at <= pos - window if window else torch.zeros_like(at > pos))
        s = (rows @ k[:, None].transpose(2, 3) * scale).masked_fill(hidden, -torch.inf)
        p = torch.softmax(s, -1)
        S = (rows.abs() @ k[:, None].abs().transpose(2, 3) * scale).masked_fill(hidden, 0.0)
        ds = (d + 8) * U * S
        A = p @ v[:, None].abs()                                  # sum p |v|
        sizes = 2 * (kv + 64) * U * A
        if path == "codes":
            Q = (rows.abs().sum(-1, keepdim=True) * st[:, None, None, :, 0] * scale).masked_fill(hidden, 0.0)
            ds = ds + Q * (16 * (d / 16 + 1) * 2.0 ** -22 + 15 * d * 2.0 ** -35)
            w = p * st[:, None, None, :, 2]
            sizes = sizes + (15 * (2.0 ** -11 * w + torch.minimum(w, 2.0 ** -19 * w.amax(-1, keepdim=True))).sum(-1, keepdim=True)
                             + (kv / 16 + 8) * 2.0 ** -22 * 128 * w.sum(-1, keepdim=True))
        if path == "restored":
            ds = ds + 2.0 ** -8 * S
            sizes = sizes + 2 * 2.0 ** -8 * A
        x = sizes + torch.expm1(2 * ds.amax(-1, keepdim=True)) * A
        o = p @ v[:, None]
        for y, to in ((o, out), (x, off)):
            to[starts[r]:starts[r] + n] = y.permute(2, 0, 1, 3).reshape(n, n_q, d)
    return out, off
