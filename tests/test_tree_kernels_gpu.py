"""Each kernel of tree attention by itself, and that it is the one that ran: any mask, what is not seen, large scores, bad fields, drafts beyond the bound,
numbers that are none in items that are cut, more requests than a block has threads."""
import math

import plain_drafts as P
import pytest
import torch

from test_tree_attention_gpu import DEV, bools, check, i32, step

pytestmark = pytest.mark.gpu
SIMT, TILE, TC = 0, 1, 2
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def ran(monkeypatch):
    """The kernels that calls of tree_attention have launched."""
    from mini_sglang_b200 import ops
    lib, kinds = ops._draft_lib(), []

    class Library:
        def __getattr__(self, name):
            fn = getattr(lib, name)
            if name != "msgl_tree_attention":
                return fn

            def call(*a):
                kinds.append(a[-4])
                return fn(*a)
            return call

    monkeypatch.setattr(ops, "_drafts", Library())
    return kinds


# a table that is wide enough for three tiles of 64 keys an SM takes float32 steps, and the bfloat16 ones that are not for the tensor cores, to the 64-row kernel
FORMS = [(TC, BF16, 128, 16, 0), (TC, BF16, 64, 32, 0), (SIMT, F32, 128, 16, 0), (SIMT, BF16, 33, 5, 0), (SIMT, BF16, 256, 16, 0), (SIMT, F32, 300, 8, 0),
         (SIMT, F32, 512, 16, 0), (TILE, F32, 128, 16, 260), (TILE, F32, 33, 5, 800), (TILE, F32, 64, 7, 600),
         (TILE, BF16, 96, 16, 260), (TILE, BF16, 33, 5, 800)]
forms = pytest.mark.parametrize("kind,dtype,d,page,spare", FORMS)


@forms
def test_any_mask(ran, kind, dtype, d, page, spare):
    lens, cached = [40, 9, 33, 5], [100, 0, 0, 250]
    rng = torch.Generator().manual_seed(3)
    masks = [torch.rand(n, n, generator=rng) < 0.3 for n in lens]
    masks[1][:] = False
    masks[2][4:20] = False
    masks[3][:] = True
    q, k, v, kw, table = step(lens, cached, 8, 2, d, page, dtype, masks, spare=spare)
    out = check(q, k, v, kw, table, lens, cached, masks)
    assert not out[40:49].any() and not out[49 + 4:49 + 20].any() and set(ran) == {kind}


@forms
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_may_be_anything(ran, kind, dtype, d, page, spare, bad):
    from mini_sglang_b200 import ops
    lens, cached = [60, 20, 9], [77, 128, 3]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "tree", 8), lens)]
    q, k, v, kw, table = step(lens, cached, 8, 2, d, page, dtype, masks, spare=spare)
    clean = check(q, k, v, kw, table, lens, cached, masks)
    place = cached[0] + 3
    at = (int(table[0, place // page]), slice(None), place % page)
    v[at][..., 5] = bad
    spoiled = torch.empty_like(clean)
    ops.tree_attention(q, spoiled, k, v, **kw)
    sees = torch.zeros(sum(lens), dtype=torch.bool, device=DEV)
    sees[:60] = masks[0][:, 3].to(DEV)
    rest = [c for c in range(d) if c != 5]
    assert sees.sum() > 1 and torch.equal(spoiled[~sees], clean[~sees]) and torch.equal(spoiled[sees][..., rest], clean[sees][..., rest])
    assert not spoiled[sees][..., 5].isfinite().any()
    k[at] = math.nan
    v[at] = bad
    ops.tree_attention(q, spoiled, k, v, **kw)
    assert torch.equal(spoiled[~sees], clean[~sees]) and set(ran) == {kind}


@forms
def test_large_scores_and_one_key(ran, kind, dtype, d, page, spare):
    lens, cached = [30, 16], [1000, 0]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "tree", 2), lens)]
    masks[1] = torch.eye(16, dtype=torch.bool)
    q, k, v, kw, table = step(lens, cached, 8, 2, d, page, dtype, masks, spare=2 * spare)
    k[table[0].to(DEV).long()[640 // page:]] *= 30           # later keys tower over the earlier ones
    if dtype == F32:
        q.div_(8)
    out = check(q, k, v, kw, table, lens, cached, masks)
    one = P.rows_of(v, table[1], torch.arange(16)).repeat_interleave(4, 1)
    assert torch.equal(out[30:], one) and set(ran) == {kind}


@forms
def test_bad_fields(ran, kind, dtype, d, page, spare):
    from mini_sglang_b200 import ops
    lens, cached = [34, 4], [60, 9]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "tree", 3), lens)]
    q, k, v, kw, table = step(lens, cached, 8, 2, d, page, dtype, masks, spare=2 * spare)
    bad = table.clone()
    bad[0, 0], bad[0, 2] = 10 ** 6, -5
    out, want = torch.empty_like(q), torch.empty_like(q)
    ops.tree_attention(q, out, k, v, **dict(kw, block_table=bad.to(DEV)))
    k0, v0 = k.clone(), v.clone()
    for x in (k0, v0):
        x[table[0, [0, 2]].to(DEV).long()] = 0.0
    ops.tree_attention(q, want, k0, v0, **kw)
    assert torch.equal(out, want) and out.isfinite().all()
    k.nan_to_num_(0.0), v.nan_to_num_(0.0)
    ops.tree_attention(q, out, k, v, **dict(kw, kv_len=i32([10 ** 9, 2 ** 31 - 1])))
    assert out.isfinite().all()
    ops.tree_attention(q, out, k, v, **dict(kw, q_start=i32([0, 10 ** 9, -7])))
    ops.tree_attention(q, out, k, v, **dict(kw, kv_len=i32([-3, -2 ** 31])))
    assert not out.any() and set(ran) == {kind}


@forms
def test_drafts_beyond_the_bound(ran, kind, dtype, d, page, spare):
    from mini_sglang_b200 import ops
    lens, cached = [40, 70], [200, 90]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "chain", 1), lens)]
    q, k, v, kw, table = step(lens, cached, 8, 2, d, page, dtype, masks, spare=2 * spare)
    out = check(q, k, v, kw, table, lens, cached, masks)
    part = torch.full_like(q, 3.0)
    ops.tree_attention(q, part, k, v, **dict(kw, max_draft=45))
    kept = torch.ones(110, dtype=torch.bool, device=DEV)
    kept[40 + 45:] = False
    # the bound only leaves rows out; where the keys are cut may differ, so sums are taken in another order: in float32 the bound of `check` on either
    # result, in bfloat16 the same of 2^-8 a rounding of a weight or of the result
    steps = 2.0 ** -8 * 8 if dtype == BF16 else 2.0 ** -24 * (d + 10 + 64) * 8
    assert (part[~kept] == 3.0).all() and ((part[kept].double() - out[kept].double()).abs() <= steps * max(1.0, float(out.abs().max()))).all()
    assert set(ran) == {kind}


@forms
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_numbers_that_are_none_in_items_that_are_cut(ran, kind, dtype, d, page, spare, bad):
    """Drafts behind many keys: their items lie in several pieces, and the draft whose value is no number in the last. What sees it is spoiled in the one
    column as the formula has it, and cannot become a number where the piece weighs next to nothing beside the others."""
    from mini_sglang_b200 import ops
    lens, cached = [8 if kind == SIMT else 33, 8], [5000, 3100]         # (32 rows a kv head at most stay with the 32-row kernel)
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "tree", 8), lens)]
    q, k, v, kw, table = step(lens, cached, 8, 2, d, page, dtype, masks, spare=spare)
    clean = check(q, k, v, kw, table, lens, cached, masks)
    draft = 1 + int(masks[0][:, 1:].sum(0).argmax())                    # (the one with the most descendants, the root apart)
    at = (int(table[0, (cached[0] + draft) // page]), slice(None), (cached[0] + draft) % page)
    held = v[at].clone()
    v[at][..., 5] = bad
    sees = torch.zeros(sum(lens), dtype=torch.bool, device=DEV)
    sees[:lens[0]] = masks[0][:, draft].to(DEV)
    rest, out = [c for c in range(d) if c != 5], torch.empty_like(clean)
    ops.tree_attention(q, out, k, v, **kw)
    assert sees.sum() > 1 and torch.equal(out[~sees], clean[~sees]) and torch.equal(out[sees][..., rest], clean[sees][..., rest])
    assert torch.equal(out[sees][..., 5], torch.full_like(out[sees][..., 5], bad)) or (math.isnan(bad) and out[sees][..., 5].isnan().all())
    # one early key of every head has a score some thousands above all others
    place = 70
    first = (int(table[0, place // page]), slice(None), place % page)
    k[first] = 0.0
    q[..., 0], k[first][..., 0] = 8.0, 2048.0
    v[at] = held
    ops.tree_attention(q, clean, k, v, **kw)
    v[at][..., 5] = bad
    ops.tree_attention(q, out, k, v, **kw)
    assert torch.equal(out[~sees], clean[~sees]) and torch.equal(out[sees][..., rest], clean[sees][..., rest])
    assert not out[sees][..., 5].isfinite().any() and set(ran) == {kind}


@pytest.mark.parametrize("kind,dtype,d,page", [(TC, BF16, 128, 16), (TC, BF16, 64, 8), (SIMT, F32, 32, 4), (TILE, F32, 32, 8)])
@pytest.mark.parametrize("B", [300, 1300])
def test_more_requests_than_a_block_has_threads(ran, kind, dtype, d, page, B):
    """Several requests a thread where the work is cut, some of them without drafts, some without keys before them."""
    lens, cached = [(7 * r) % 4 if r % 50 > 20 else 0 for r in range(B)], [(13 * r) % 41 for r in range(B)]
    masks = [bools(up, n) for up, n in zip(P.random_forest(lens, "tree", 2), lens)]
    n_q = 32 if kind == TILE else 4
    q, k, v, kw, table = step(lens, cached, n_q, 2, d, page, dtype, masks)
    check(q, k, v, kw, table, lens, cached, masks)
    assert set(ran) == {kind}
