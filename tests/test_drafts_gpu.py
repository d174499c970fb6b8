"""The fields of a step of drafted tokens and the accepted path, exactly as the plain forms have them."""
import random

import plain_drafts as P
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


PLANS = [
    ([1], [0], "chain", 16, 1), ([8], [1000], "tree", 16, 8), ([0], [5], "tree", 16, 3), ([256], [77], "chain", 16, 256), ([256, 1, 0, 255], [0, 1, 2, 3], "tree", 1, 256),
    ([33, 32, 31, 64, 65], [15, 16, 17, 4095, 0], "tree", 16, 65), ([5, 5, 5], [10, 20, 30], "bush", 48, 7), ([0, 0, 3, 0], [4, 4, 4, 4], "chain", 8, 32),
    ([3] * 300, list(range(300)), "tree", 16, 33), ([64] * 256, [31 * i for i in range(256)], "tree", 16, 64),
]


@pytest.mark.parametrize("lens,cached,kind,page,most", PLANS)
@pytest.mark.parametrize("spare_rows", [0, 5])
def test_plan(lens, cached, kind, page, most, spare_rows):
    from mini_sglang_b200 import ops
    forest = P.random_forest(lens, kind, 3)
    table, _ = P.random_tables(lens, cached, page, 4)
    parents = i32([p for up in forest for p in up] + [7] * spare_rows)
    plan = ops.draft_plan(parents, i32(lens), i32(cached), table.to(DEV), page_size=page, max_draft=most)
    words, T = -(-most // 32), sum(lens)
    starts = [sum(lens[:r]) for r in range(len(lens) + 1)]
    assert plan.q_start.tolist() == starts and plan.kv_len.tolist() == [n + c for n, c in zip(lens, cached)]
    pad = [0] * spare_rows
    assert plan.positions.tolist() == [c + len(a) - 1 for up, c in zip(forest, cached) for a in P.ancestors(up)] + pad
    assert plan.token_req.tolist() == [r for r, n in enumerate(lens) for _ in range(n)] + pad
    assert plan.out_loc.tolist() == [int(table[r, (c + i) // page]) * page + (c + i) % page for r, (n, c) in enumerate(zip(lens, cached)) for i in range(n)] + pad
    assert plan.mask.shape == (T + spare_rows, words)
    assert plan.mask.tolist() == [row for up in forest for row in P.mask_rows(up, words)] + [[0] * words] * spare_rows


def test_plan_of_bad_fields():
    """Parents that are no earlier draft, lengths beyond the limits, places beyond the table: what the documentation says, and nothing read out of range."""
    from mini_sglang_b200 import ops
    up = [5, 1, 0, -7, 3, 2 ** 31 - 1, 6, -2 ** 31]                        # only drafts 2 and 4 have a parent
    table = i32([[3, 4], [5, 6]])
    plan = ops.draft_plan(i32(up + up), i32([8, 200]), i32([28, -4]), table, page_size=16, max_draft=20)
    assert plan.q_start.tolist() == [0, 8, 16] and plan.kv_len.tolist() == [36, 8]
    anc = P.ancestors(up)
    assert [len(a) for a in anc] == [1, 1, 2, 1, 2, 1, 1, 1]
    assert plan.mask.tolist() == P.mask_rows(up, 1) * 2
    assert plan.out_loc.tolist() == [4 * 16 + 12 + i for i in range(4)] + [0] * 4 + [5 * 16 + i for i in range(8)]
    far = ops.draft_plan(i32([-1]), i32([1]), i32([2 ** 31 - 1]), table[:1], page_size=16, max_draft=1)
    assert far.out_loc.tolist() == [0]
    none = ops.draft_plan(i32([]), i32([4, 4]), i32([1, 2]), table, page_size=16, max_draft=4)
    assert none.q_start.tolist() == [0, 0, 0] and none.kv_len.tolist() == [1, 2] and none.mask.shape == (0, 1)
    empty = ops.draft_plan(i32([1, 2]), i32([]), i32([]), table[:0], page_size=16, max_draft=4)
    assert empty.q_start.tolist() == [0] and not empty.mask.any() and empty.positions.tolist() == [0, 0]


def agreeing(forest, seed, share):
    """Tokens and the model's tokens after them from a small vocabulary, so that siblings share tokens; the model agrees often."""
    rng = random.Random(seed)
    tokens = [[rng.randrange(6) for _ in up] for up in forest]
    after = [[rng.randrange(6) for _ in up] for up in forest]
    for up, tok, nxt in zip(forest, tokens, after):
        for i in range(1, len(up)):
            if rng.random() < share and 0 <= up[i] < i:
                nxt[up[i]] = tok[i]
    return tokens, after


ACCEPTS = [
    ([1], "chain", 16, 128, torch.bfloat16), ([8], "tree", 16, 128, torch.bfloat16), ([256], "chain", 16, 64, torch.bfloat16), ([0, 5, 0], "chain", 8, 128, torch.float32),
    ([61] * 9, "tree", 16, 128, torch.bfloat16), ([33, 1, 64, 7], "tree", 1, 20, torch.bfloat16), ([12] * 40, "bush", 16, 33, torch.bfloat16),
    ([200, 199], "tree", 48, 7, torch.float32),
]


@pytest.mark.parametrize("lens,kind,page,d,dtype", ACCEPTS)
def test_accept(lens, kind, page, d, dtype):
    from mini_sglang_b200 import ops
    forest = P.random_forest(lens, kind, 11)
    tokens, after = agreeing(forest, 12, 0.9)
    cached = [(37 * r) % 50 for r in range(len(lens))]
    table, pages = P.random_tables(lens, cached, page, 13)
    starts = [sum(lens[:r]) for r in range(len(lens) + 1)]
    g = torch.Generator(device=DEV).manual_seed(1)
    shapes = [(pages + 1, 3, page, d)] * 3 + [(pages + 1, 1, page, 2 * d)]
    caches = [torch.randn(s, generator=g, device=DEV).to(dtype) for s in shapes]
    want, paths = [c.clone() for c in caches], [P.accepted(*x) for x in zip(forest, tokens, after)]
    for r, path in enumerate(paths):
        for w, c in zip(want, caches):
            if path:
                places = torch.arange(len(path), device=DEV) + cached[r]
                row = table[r].to(DEV).long()
                w[row[places // page], :, places % page] = P.rows_of(c, table[r], [cached[r] + i for i in path])
    flat = lambda x: i32([v for part in x for v in part])      # noqa: E731
    most = max(lens) + 2 if max(lens) < 255 else 256
    got = ops.draft_accept(flat(tokens), flat(forest), flat(after), i32(starts), max_draft=most, kv_len=i32([n + c for n, c in zip(lens, cached)]),
                           block_table=table.to(DEV), caches=caches + caches[:1])
    assert got.kept.tolist() == [len(p) for p in paths]
    assert got.path.tolist() == [p + [-1] * (most - len(p)) for p in paths]
    assert got.tokens.tolist() == [[after[r][i] for i in p] + [-1] * (most - len(p)) for r, p in enumerate(paths)]
    assert len(max(paths, key=len)) > 1 or lens == [1]
    for w, c in zip(want, caches):
        assert torch.equal(w, c)
    again = ops.draft_accept(flat(tokens), flat(forest), flat(after), i32(starts), max_draft=most)          # without caches
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_accept_leaves_out_what_is_not_there():
    """Places beyond the table and pages outside the cache are not touched; drafts beyond max_draft are not looked at."""
    from mini_sglang_b200 import ops
    chain = [-1, 0, 1, 1, 3]
    tokens, after = [9, 4, 8, 5, 6], [4, 5, 0, 6, 0]                       # path 0, 1, 3, 4: rows 3 and 4 move to 2 and 3
    cache = torch.arange(4 * 2, device=DEV, dtype=torch.float32).view(4, 1, 2, 1).repeat(1, 1, 1, 4).contiguous()
    before = cache.clone()
    args = (i32(tokens), i32(chain), i32(after), i32([0, 5]))
    got = ops.draft_accept(*args, max_draft=5, kv_len=i32([5]), block_table=i32([[1, 2]]), caches=[cache])      # places 0..3 have pages, place 4 has none
    assert got.path.tolist() == [[0, 1, 3, 4, -1]]
    want = before.clone()
    want[2, :, 0] = before[2, :, 1]
    assert torch.equal(cache, want)
    cache.copy_(before)
    ops.draft_accept(*args, max_draft=5, kv_len=i32([5]), block_table=i32([[1, 400, -3]]), caches=[cache])
    assert torch.equal(cache, before)
    assert ops.draft_accept(*args, max_draft=2).path.tolist() == [[0, 1]]
    two = ops.draft_accept(i32([9, 7, 4]), i32([-1, 0, 0]), i32([4, 0, 0]), i32([0, 3]), max_draft=3, kv_len=i32([5]), block_table=i32([[1, 2, 3]]), caches=[cache])
    assert two.path.tolist() == [[0, 2, -1]]                 # place 4 moves to place 3
    want = before.clone()
    want[2, :, 1] = before[3, :, 0]
    assert torch.equal(cache, want)
    cache.copy_(before)
    cut = ops.draft_accept(i32([9, 7, 4, 1]), i32([-1, 0, 0, 0]), i32([4, 0, 0, 0]), i32([0, 4]), max_draft=3, kv_len=i32([6]), block_table=i32([[1, 2, 3]]), caches=[cache])
    assert cut.path.tolist() == [[0, 2, -1]] and torch.equal(cache, want)          # a draft beyond the bound: the places are what they were


def test_plan_and_accept_in_a_graph():
    """Captured once and replayed on other lengths, trees and tables."""
    from mini_sglang_b200 import ops
    lens, cached = [6, 9, 4], [20, 3, 40]
    rows, most, page = 24, 12, 16
    static = {k: torch.zeros(s, dtype=torch.int32, device=DEV) for k, s in (("parents", rows), ("lens", 3), ("cached", 3), ("tokens", rows), ("after", rows))}
    table, pages = P.random_tables([12] * 3, [40] * 3, page, 1)
    table = table.to(DEV)
    cache = torch.randn(pages + 1, 2, page, 16, device=DEV)

    def step():
        plan = ops.draft_plan(static["parents"], static["lens"], static["cached"], table, page_size=page, max_draft=most)
        return plan, ops.draft_accept(static["tokens"], static["parents"], static["after"], plan.q_start, max_draft=most, kv_len=plan.kv_len, block_table=table, caches=[cache])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, got = step()
    for seed in (1, 2):
        forest = P.random_forest(lens, "tree", seed)
        tokens, after = agreeing(forest, seed, 0.8)
        for k, v in (("parents", forest), ("tokens", tokens), ("after", after)):
            flat = [x for part in v for x in part]
            static[k].copy_(i32(flat + [0] * (rows - len(flat))))
        static["lens"].copy_(i32(lens))
        static["cached"].copy_(i32(cached))
        start = cache.clone()
        graph.replay()
        paths = [P.accepted(*x) for x in zip(forest, tokens, after)]
        assert got.path.tolist() == [p + [-1] * (most - len(p)) for p in paths]
        assert plan.kv_len.tolist() == [n + c for n, c in zip(lens, cached)]
        for r, path in enumerate(paths):
            there = P.rows_of(cache, table[r], [cached[r] + i for i in range(len(path))])
            assert torch.equal(there, P.rows_of(start, table[r], [cached[r] + i for i in path]))
        lens, cached = [0, 12, 12], [1, 31, 0]
