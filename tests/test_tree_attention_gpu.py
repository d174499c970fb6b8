"""Attention for trees of drafted tokens against the plain softmax in 64 bits: trees of every shape, ragged lengths, any mask, cut and whole items,
pages of every size, values that hold no numbers where nobody looks."""
import math
import random

import plain_drafts as P
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def bools(up, n):
    m = torch.zeros(n, n, dtype=torch.bool)
    for i, anc in enumerate(P.ancestors(up)):
        m[i, list(anc)] = True
    return m


def words_of(masks, most):
    """bool [n, n] masks -> packed int32 rows, one request behind the other."""
    words, rows = -(-most // 32), []
    for m in masks:
        for row in m.tolist():
            bits = sum(1 << a for a, on in enumerate(row) if on)
            rows.append([(w - (1 << 32) if w >= 1 << 31 else w) for w in ((bits >> (32 * k)) & 0xFFFFFFFF for k in range(words))])
    return i32(rows).view(-1, words) if rows else torch.zeros((0, words), dtype=torch.int32, device=DEV)


def step(lens, cached, n_q, n_kv, d, page, dtype, masks, seed=0, most=None, spare=0):
    """(arguments of the call, the plain result) of a random step; what no key of a request lies in holds NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    table, pages = P.random_tables(lens, cached, page, seed + 1, spare)
    k, v = (torch.full((pages + 1, n_kv, page, d), math.nan, device=DEV, dtype=dtype) for _ in range(2))
    for r, (n, c) in enumerate(zip(lens, cached)):
        at = torch.arange(n + c, device=DEV)
        row = table[r].to(DEV).long()
        for x in (k, v):
            x[row[at // page], :, at % page] = torch.randn(n + c, n_kv, d, generator=g, device=DEV).to(dtype)
    q = (1.5 * torch.randn(sum(lens), n_q, d, generator=g, device=DEV)).to(dtype)
    most = most or max(max(lens), 1)
    kw = dict(q_start=i32([sum(lens[:r]) for r in range(len(lens) + 1)]), kv_len=i32([n + c for n, c in zip(lens, cached)]), block_table=table.to(DEV),
              mask=words_of(masks, most), n_kv=n_kv, page_size=page, scale=d ** -0.5, max_draft=most)
    return q, k, v, kw, table


def check(q, k, v, kw, table, lens, cached, masks):
    from mini_sglang_b200 import ops
    out = torch.full_like(q, 7.0)
    ops.tree_attention(q, out, k, v, **kw)
    want = P.tree_attention(q, k, v, table, lens, cached, masks, kw["scale"])
    err = (out.double() - want).abs()
    if q.dtype == torch.float32:
        # a score of size s is off by at most d half steps of its sum of products, which moves a weight by as much; the exponential by four, sums by
        # the number of keys a thread adds: with random signs far below 2^-24 x (d + keys / 32 + 64) of the largest value
        keys = max(n + c for n, c in zip(lens, cached))
        assert (err <= 2.0 ** -24 * (q.shape[2] + keys / 32 + 64) * 4 * max(1.0, float(want.abs().max()))).all()
    else:
        # every weight is rounded once to bfloat16 (half a step, 2^-9 of it, in the mean 0.29 of a step of 2^-8: 2^-9.8), with random signs over the
        # keys, so relative to a result of random signs its root mean square is no more than that; the result is rounded once likewise.
        # Largest: the sum of |p v| is at most sqrt(keys that weigh) times the result's size, below 8 here, each off by up to 2^-9; and half a step 2^-9 of |v| < 6
        assert err.pow(2).mean().sqrt() <= 2.0 ** -8 * want.pow(2).mean().sqrt() + 1e-9
        assert err.max() <= 2.0 ** -9 * (8 + 1) * max(1.0, float(want.abs().max()))
    return out


SHAPES = [
    # drafts, cached, n_q, n_kv, d, page, tree
    ([1], [0], 4, 1, 128, 16, "chain"), ([8], [1000], 32, 8, 128, 16, "tree"), ([1, 0, 3], [0, 7, 129], 8, 8, 128, 16, "tree"), ([33], [127], 16, 2, 128, 64, "tree"),
    ([5] * 16, [500 + 33 * i for i in range(16)], 32, 8, 128, 16, "chain"), ([64, 17, 1], [2000, 128, 383], 16, 8, 128, 16, "tree"), ([256], [300], 8, 1, 128, 16, "tree"),
    ([200, 90], [1, 0], 10, 5, 128, 32, "bush"), ([49] * 6, [700 + i for i in range(6)], 32, 8, 128, 8, "tree"), ([128], [9000], 64, 8, 128, 16, "tree"),
    ([3, 40], [5, 77], 6, 2, 128, 128, "tree"), ([12, 31], [256, 255], 7, 1, 128, 256, "tree"), ([2] * 70, [(13 * i) % 300 for i in range(70)], 4, 2, 128, 16, "chain"),
    ([8, 20], [333, 64], 8, 2, 64, 16, "tree"), ([129], [1500], 16, 4, 64, 16, "tree"),
    ([9], [100], 4, 2, 96, 16, "tree"), ([7, 3], [40, 90], 4, 4, 20, 16, "tree"), ([5], [70], 2, 1, 256, 16, "tree"), ([4], [50], 2, 2, 512, 16, "chain"),
    ([6, 6], [33, 200], 8, 2, 128, 1, "tree"), ([10], [90], 4, 1, 128, 48, "tree"), ([11], [75], 6, 3, 33, 5, "tree"), ([70], [600], 40, 8, 128, 16, "tree"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,cached,n_q,n_kv,d,page,kind", SHAPES)
def test_trees(lens, cached, n_q, n_kv, d, page, kind, dtype):
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, kind, 5), lens)]
    q, k, v, kw, table = step(lens, cached, n_q, n_kv, d, page, dtype, masks)
    out = check(q, k, v, kw, table, lens, cached, masks)
    again = torch.empty_like(out)
    from mini_sglang_b200 import ops
    ops.tree_attention(q, again, k, v, **kw)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype,d,page", [(torch.bfloat16, 128, 16), (torch.float32, 128, 16), (torch.bfloat16, 40, 16)])
def test_any_mask(dtype, d, page):
    """Masks that are no trees: random ones, none at all (with cached keys and without: then the row is 0), all; rows of q behind the last draft stay."""
    from mini_sglang_b200 import ops
    lens, cached = [40, 9, 33, 5], [100, 0, 0, 250]
    rng = torch.Generator().manual_seed(3)
    masks = [torch.rand(n, n, generator=rng) < 0.3 for n in lens]
    masks[1][:] = False
    masks[2][4:20] = False
    masks[3][:] = True
    q, k, v, kw, table = step(lens, cached, 8, 2, d, page, dtype, masks)
    out = check(q, k, v, kw, table, lens, cached, masks)
    assert not out[40:49].any() and not out[49 + 4:49 + 20].any()
    T = q.shape[0]
    more = dict(kw, mask=torch.cat([kw["mask"], torch.full((3, kw["mask"].shape[1]), -1, dtype=torch.int32, device=DEV)]))
    padded, held = torch.cat([q, q[:3]]), torch.full((T + 3, 8, d), 5.0, device=DEV, dtype=dtype)
    ops.tree_attention(padded, held, k, v, **more)
    assert torch.equal(held[:T], out) and (held[T:] == 5.0).all()


@pytest.mark.parametrize("dtype,d,page", [(torch.bfloat16, 128, 16), (torch.float32, 128, 16), (torch.bfloat16, 64, 16), (torch.bfloat16, 72, 3)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_may_be_anything(dtype, d, page, bad):
    """A draft whose key and value hold no numbers spoils the drafts that see it, and no other; and of those only the elements that it spoils."""
    from mini_sglang_b200 import ops
    lens, cached = [60, 20], [77, 128]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "tree", 8), lens)]
    q, k, v, kw, table = step(lens, cached, 8, 2, d, page, dtype, masks)
    clean = check(q, k, v, kw, table, lens, cached, masks)
    place = cached[0] + 3
    at = (int(table[0, place // page]), slice(None), place % page)
    v[at][..., 5] = bad
    spoiled = torch.empty_like(clean)
    ops.tree_attention(q, spoiled, k, v, **kw)
    sees = torch.zeros(80, dtype=torch.bool)
    sees[:60] = masks[0][:, 3]
    assert sees.sum() > 1 and torch.equal(spoiled[~sees.to(DEV)], clean[~sees.to(DEV)])
    assert not spoiled[sees.to(DEV)][..., 5].isfinite().any()
    rest = [c for c in range(d) if c != 5]
    assert torch.equal(spoiled[sees.to(DEV)][..., rest], clean[sees.to(DEV)][..., rest])
    k[at] = math.nan
    v[at] = bad
    ops.tree_attention(q, spoiled, k, v, **kw)
    assert torch.equal(spoiled[~sees.to(DEV)], clean[~sees.to(DEV)])


def test_large_scores_and_one_key():
    """Scores far from zero, where the reference of the exponentials has to move, and drafts that see a single key."""
    lens, cached = [30, 16], [1000, 0]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "tree", 2), lens)]
    masks[1] = torch.eye(16, dtype=torch.bool)
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, kw, table = step(lens, cached, 8, 2, 128, 16, dtype, masks)
        k[table[0].to(DEV).long()[40:]] *= 30            # later keys tower over the earlier ones
        if dtype == torch.float32:
            q.div_(8)
        out = check(q, k, v, kw, table, lens, cached, masks)
        one = P.rows_of(v, table[1], torch.arange(16)).repeat_interleave(4, 1)
        assert torch.equal(out[30:], one)


def test_random_steps():
    rng = random.Random(7)
    for i in range(25):
        B = rng.choice((1, 2, 5, 20))
        lens, cached = [rng.choice((0, 1, 2, 7, 30, 65, 128)) for _ in range(B)], [rng.choice((0, 1, 15, 100, 1023, 3000)) for _ in range(B)]
        if not sum(lens):
            continue
        n_kv = rng.choice((1, 2, 8))
        n_q = n_kv * rng.choice((1, 2, 4, 5, 8))
        d, page = rng.choice(((128, 16), (128, 32), (64, 16), (128, 7), (48, 16)))
        masks = [bools(up, n) for up, n in zip(P.random_forest(lens, rng.choice(("chain", "tree", "bush")), i), lens)]
        q, k, v, kw, table = step(lens, cached, n_q, n_kv, d, page, torch.bfloat16, masks, seed=i, spare=rng.choice((0, 3)))
        check(q, k, v, kw, table, lens, cached, masks)


def test_bad_fields_read_nothing_outside():
    """Pages outside the cache read as zeros, lengths beyond the table are cut, starts beyond the stream too."""
    from mini_sglang_b200 import ops
    masks = [bools([-1, 0, 0, 1], 4)]
    for dtype, d in ((torch.bfloat16, 128), (torch.float32, 32)):
        q, k, v, kw, table = step([4], [60], 4, 2, d, 16, dtype, masks)
        bad = table.clone()
        bad[0, 1], bad[0, 2] = 10 ** 6, -5
        out = torch.empty_like(q)
        ops.tree_attention(q, out, k, v, **dict(kw, block_table=bad.to(DEV)))
        k0, v0 = k.clone(), v.clone()
        for x in (k0, v0):
            x[table[0, 1:3].to(DEV).long()] = 0.0
        want = torch.empty_like(q)
        ops.tree_attention(q, want, k0, v0, **kw)
        assert torch.equal(out, want) and out.isfinite().all()
        ops.tree_attention(q, out, k, v, **dict(kw, kv_len=i32([10 ** 9])))
        ops.tree_attention(q, out, k, v, **dict(kw, q_start=i32([0, 10 ** 9])))
        ops.tree_attention(q, out, k, v, **dict(kw, kv_len=i32([-3])))
        assert not out.any()


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 128), (torch.float32, 40), (torch.bfloat16, 256)])
def test_drafts_beyond_the_bound_are_left_out(dtype, d):
    from mini_sglang_b200 import ops
    lens, cached = [40, 70], [200, 90]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "chain", 1), lens)]
    q, k, v, kw, table = step(lens, cached, 4, 2, d, 16, dtype, masks)
    out = check(q, k, v, kw, table, lens, cached, masks)
    part = torch.full_like(q, 3.0)
    ops.tree_attention(q, part, k, v, **dict(kw, max_draft=45))
    kept = torch.ones(110, dtype=torch.bool, device=DEV)
    kept[40 + 45:] = False
    assert (part[~kept] == 3.0).all()
    # (rows that another kernel or another cut of the work made: the same but for the order of the sums)
    torch.testing.assert_close(part[kept].float(), out[kept].float(), rtol=2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -14, atol=2.0 ** -7 if dtype == torch.bfloat16 else 1e-5)


def test_graph_other_lengths_and_streams():
    """Captured once, replayed on other lengths and masks; two streams at once; nothing is kept from call to call."""
    from mini_sglang_b200 import ops
    lens, cached = [20, 9, 1], [900, 40, 300]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "tree", 1), lens)]
    q, k, v, kw, table = step(lens, cached, 16, 4, 128, 16, torch.bfloat16, masks, spare=40)
    out, want = torch.empty_like(q), torch.empty_like(q)
    ops.tree_attention(q, want, k, v, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tree_attention(q, out, k, v, **kw)
    graph.replay()
    assert torch.equal(out, want)
    k.nan_to_num_(0.0), v.nan_to_num_(0.0)
    kw["q_start"].copy_(i32([0, 2, 30, 30]))
    kw["kv_len"].copy_(i32([500, 60, 10]))
    kw["mask"].copy_(kw["mask"].flip(0))
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = torch.empty_like(q)
        ops.tree_attention(q, other, k, v, **kw)
    graph.replay()
    torch.cuda.synchronize()
    # 28 drafts of the second request, 20 of them within the bound that the launch was made for: the rest keep what the first replay wrote
    assert torch.equal(out[:22], other[:22]) and torch.equal(out[22:], want[22:])
