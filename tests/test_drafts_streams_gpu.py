"""Plans and accepted paths of two steps at once, each on a stream of its own."""
import plain_drafts as P
import pytest
import torch

from test_drafts_gpu import DEV, agreeing, i32

pytestmark = pytest.mark.gpu


def one(seed, lens, page, d):
    """(arguments, caches, what the caches hold afterwards, paths) of a step."""
    forest = P.random_forest(lens, "tree", seed)
    tokens, after = agreeing(forest, seed + 1, 0.9)
    cached = [(37 * r + seed) % 50 for r in range(len(lens))]
    table, pages = P.random_tables(lens, cached, page, seed + 2)
    g = torch.Generator(device=DEV).manual_seed(seed)
    caches = [torch.randn(pages + 1, 3, page, d, generator=g, device=DEV) for _ in range(4)]
    want, paths = [c.clone() for c in caches], [P.accepted(*x) for x in zip(forest, tokens, after)]
    for r, path in enumerate(paths):
        places, row = torch.arange(len(path), device=DEV) + cached[r], table[r].to(DEV).long()
        for w, c in zip(want, caches):
            w[row[places // page], :, places % page] = P.rows_of(c, table[r], [cached[r] + i for i in path])
    flat = lambda x: i32([v for part in x for v in part])      # noqa: E731
    return dict(tokens=flat(tokens), parents=flat(forest), after=flat(after), lens=i32(lens), cached=i32(cached), table=table.to(DEV), caches=caches, want=want, paths=paths,
                page=page, most=max(lens))


def run(s):
    from mini_sglang_b200 import ops
    plan = ops.draft_plan(s["parents"], s["lens"], s["cached"], s["table"], page_size=s["page"], max_draft=s["most"])
    return ops.draft_accept(s["tokens"], s["parents"], s["after"], plan.q_start, max_draft=s["most"], kv_len=plan.kv_len, block_table=s["table"], caches=s["caches"])


def test_two_streams():
    for round_ in range(6):
        steps = [one(round_, [61] * 9, 16, 128), one(100 + round_, [20, 5, 33, 64] * 5, 8, 64)]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
        for stream, s in zip(streams, steps):
            with torch.cuda.stream(stream):
                got.append(run(s))
        torch.cuda.synchronize()
        for s, a in zip(steps, got):
            assert a.path.tolist() == [p + [-1] * (s["most"] - len(p)) for p in s["paths"]]
            assert all(torch.equal(c, w) for c, w in zip(s["caches"], s["want"]))
