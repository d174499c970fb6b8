"""Where attention over a cache in 4 bits can go wrong: rows that are no numbers, requests without keys, pages that are none, captures, streams, long sums, far pages."""
import math

import pytest
import torch

import plain_kv4 as plain
from mini_sglang_b200 import ops
from mini_sglang_b200.parts import Workspace
from test_kv4_gpu import BF, F32, bound, filled, i32, normal

pytestmark = pytest.mark.gpu
SHAPES = [(4, 2, 128, BF), (8, 1, 64, BF), (4, 4, 32, BF), (4, 2, 128, F32)]          # both kernels that read codes


def table_of(B, width, seed=0):
    return (torch.randperm(B * width, generator=torch.Generator().manual_seed(seed)) + 1).view(B, width).int().cuda()


def attend(q, c, kv, table, **kw):
    out = torch.full_like(q, 7.0)
    ops.kv4_attention(q, out, c, kv_len=i32(kv) if isinstance(kv, list) else kv, block_table=table, scale=q.shape[2] ** -0.5, **kw)
    return out


def near(out, q, c, lens, kv, table, window=0):
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    want, facts = plain.attention(q, c, starts, lens, kv, table, q.shape[2] ** -0.5, window)
    tol = torch.maximum(*(bound(facts, max(kv), q.shape[2], q.dtype, r) for r in (False, True)))
    nan = want.isnan()
    assert torch.equal(out.isnan(), nan)
    assert ((out.double() - want).abs() <= tol + torch.finfo(q.dtype).eps / 2 * (want.abs() + tol))[~nan].all()
    return want


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
def test_a_row_that_is_no_number_shows_only_where_it_is_seen(n_q, n_kv, d, dtype):
    lens, kv, page = [3, 1, 1], [70, 70, 40], 16
    table = table_of(3, 5)
    for which, window in ((1, 0), (3, 0), (1, 9), (3, 9)):          # a key's base, a value's
        c = filled(1, 16, n_kv, page, d)
        at = lambda r, key: (int(table[r, key // page]), slice(None), key % page, which)      # noqa: E731, B023
        c.steps[at(0, 69)] = math.nan          # seen by the last of three tokens
        c.steps[at(1, 5)] = math.nan           # outside the window of request 1, if there is one
        c.steps[at(2, 40)] = math.nan          # behind request 2's last key: in its last page, and in no one's sight
        c.steps[at(2, 47)] = math.inf
        c.steps[(*at(2, 44)[:3], 2)] = math.inf          # a step that is none, likewise
        q = normal(2, 5, n_q, d, dtype=dtype)
        out = attend(q, c, kv, table, window=window, q_start=i32([0, 3, 4, 5]), q_lens=lens, kv_lens=kv)
        assert out.isnan().flatten(1).all(1).tolist() == [False, False, True, window == 0, False] and torch.equal(out.isnan().flatten(1).any(1), out.isnan().flatten(1).all(1))
        clean = c._replace(steps=torch.where(c.steps.isfinite(), c.steps, 0.0))
        ok = torch.tensor([0, 1, 4], device="cuda")
        want, facts = plain.attention(q, clean, [0, 3, 4, 5], lens, kv, table, d ** -0.5, window)
        tol = bound(facts, 70, d, dtype, False)
        assert ((out.double() - want).abs() <= tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol))[ok].all()


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
def test_requests_without_keys_and_pages_that_are_none(n_q, n_kv, d, dtype):
    c, q = filled(4, 9, n_kv, 16, d), normal(5, 4, n_q, d, dtype=dtype)
    table = i32([1, 2, 3, 4, 9, -5, 6, 7, 2 ** 31 - 1, 8, 1, -2 ** 31]).view(4, 3)
    kv = [0, 40, 33, 48]          # request 1's first page is its fourth, its second is beyond the cache ...
    out = attend(q, c, kv, table)
    assert (out[0] == 0).all()
    near(out, q, c, [1] * 4, kv, table)
    negative = attend(q, c, [-3, 40, 33, 48], table)          # lengths below zero are none
    assert torch.equal(negative, out)
    long = attend(q, c, [10 ** 9, 48, 48, 48], table)          # and no more keys are seen than the table holds
    assert torch.isfinite(long).all()


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
def test_steps_and_bases_of_all_sizes(n_q, n_kv, d, dtype):
    """Values between 2^-60 and 2^60 times their neighbours', in falling and in rising order of the keys; keys whose scores leave one of them."""
    B, n = 3, 300
    c, table = filled(6, 3 * 19 + 1, n_kv, 16, d), table_of(B, 19)
    up = (2.0 ** torch.linspace(-60, 60, 19 * 16, device="cuda"))
    for r, order in enumerate((up, up.flip(0), up[torch.randperm(up.numel(), generator=torch.Generator().manual_seed(1)).cuda()])):
        c.steps[table[r].long(), :, :, 2:] *= order.view(19, 1, 16, 1).to(BF)
    q = normal(7, B, n_q, d, dtype=dtype) * torch.tensor([1.0, 30.0, 1e-3], device="cuda", dtype=dtype)[:, None, None]
    near(attend(q, c, [n] * B, table), q, c, [1] * B, [n] * B, table)


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
@pytest.mark.parametrize("power", [111, -90])
def test_values_of_either_end_of_the_range(n_q, n_kv, d, dtype, power):
    """All values times 2^111 (their steps are above 2^109; sums of 40 products with weights up to 2^8 stay below 2^128) or 2^-90 (their steps above 2^-100)."""
    B, n = 3, 40
    c, table = filled(10, 3 * 3 + 1, n_kv, 16, d), table_of(B, 3)
    c.steps[..., 2:] *= 2.0 ** power
    q = normal(11, B, n_q, d, dtype=dtype)
    assert torch.isfinite(near(attend(q, c, [n] * B, table), q, c, [1] * B, [n] * B, table)).all()


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
@pytest.mark.parametrize("kept", [True, False])
def test_a_captured_call_reads_what_is_there_when_it_is_replayed(n_q, n_kv, d, dtype, kept):
    B, width = 5, 40
    ws = Workspace("cuda") if kept else None
    c, q, kv, table = filled(8, B * width + 1, n_kv, 16, d), normal(9, B, n_q, d, dtype=dtype), i32([1] * B), table_of(B, width)
    out = torch.empty_like(q)
    run = lambda: ops.kv4_attention(q, out, c, kv_len=kv, block_table=table, scale=d ** -0.5, workspace=ws)      # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for k, lens in enumerate(([640, 3, 77, 500, 32], [1] * B, [100, 640, 640, 640, 639])):
        kv.copy_(i32(lens))
        table.copy_(table_of(B, width, k))
        q.copy_(normal(20 + k, B, n_q, d, dtype=dtype))
        for _ in range(2):          # the counters are clear again
            graph.replay()
            near(out, q, c, [1] * B, lens, table)
            out.fill_(7.0)
        run()
        near(out, q, c, [1] * B, lens, table)


def test_two_streams_with_scratch_of_their_own():
    n_q, n_kv, d, B, width = 32, 8, 128, 16, 128
    c, table = filled(10, B * width + 1, n_kv, 16, d), table_of(B, width)
    qs, kv = [normal(30 + i, B, n_q, d, dtype=BF) for i in range(2)], i32(range(width * 16 - B, width * 16))
    want = [attend(q, c, kv, table) for q in qs]
    streams, spaces, outs = [torch.cuda.Stream() for _ in range(2)], [Workspace("cuda") for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(attend(qs[i], c, kv, table, workspace=spaces[i]))
    torch.cuda.synchronize()
    for w, got in zip(want, outs):
        assert all(torch.equal(w, o) for o in got)


def test_the_same_call_gives_the_same_bits():
    n_q, n_kv, d, B = 40, 8, 128, 33
    c, table, ws = filled(11, B * 64 + 1, n_kv, 16, d), table_of(B, 64), Workspace("cuda")
    kv = [1 + (97 * i) % 1000 for i in range(B)]
    q, lens = normal(12, 3 * B, n_q, d, dtype=BF), [3] * B
    kv = [max(k, 3) for k in kv]
    kw = dict(q_start=i32(range(0, 3 * B + 1, 3)), q_lens=lens, kv_lens=kv, workspace=ws)
    first = attend(q, c, kv, table, **kw)
    for _ in range(10):
        assert torch.equal(first, attend(q, c, kv, table, **kw))


def test_a_mean_of_many_keys_keeps_its_digits():
    """64 requests of 16,000 keys give every warp a chain of a hundred units.  Rounded to bfloat16 the result is off by 2^-8 at most, weights rounded to 2^-11 add less than half of
    what that does on average: 2^-8 of its size in all."""
    B, n, n_q, n_kv, d = 64, 16000, 32, 8, 128
    c, ws = filled(13, 20001, n_kv, 16, d), Workspace("cuda")
    table = torch.randint(1, 20001, (B, n // 16), generator=torch.Generator().manual_seed(5)).int().cuda()
    q = normal(14, B, n_q, d, dtype=BF)
    out = attend(q, c, [n] * B, table, workspace=ws)
    keys, values = plain.values(c, 0).float(), plain.values(c, 1).float()
    for r in (0, 31, 63):
        k, v = (x[table[r].long()].permute(1, 0, 2, 3).reshape(n_kv, n, d).double() for x in (keys, values))
        s = torch.einsum("hgd,hkd->hgk", q[r].double().view(n_kv, n_q // n_kv, d), k) * d ** -0.5
        want = torch.einsum("hgk,hkd->hgd", torch.softmax(s, -1), v).reshape(n_q, d)
        assert (out[r].double() - want).norm() <= 2.0 ** -8 * want.norm()


@pytest.mark.parametrize("d,dtype", [(128, BF), (128, F32), (40, BF)])
def test_pages_past_32_bits_of_bytes(d, dtype):
    """Pages whose codes lie more than 2^32 bytes into the arrays: appended to, attended to (from codes and restored) and read back."""
    n_kv, page, n_q = 2, 64, 8
    pages = (1 << 32) // (n_kv * page * d // 2) + 20
    c = ops.kv4_cache(pages, n_kv, page, d)
    T, kv = 700, [500, 200]
    table = torch.stack([torch.arange(pages - 8, pages), torch.arange(pages - 16, pages - 8)]).int().cuda()
    qkv = normal(15, T, (n_q + 2 * n_kv) * d, dtype=dtype)
    slots = torch.cat([table[r].long().repeat_interleave(page)[:n] * page + torch.arange(n, device="cuda") % page for r, n in enumerate(kv)]).int()
    pos = i32(list(range(500)) + list(range(200)))
    q = ops.qknorm_rope_kv4write(qkv, pos, n_q, n_kv, d, q_weight=None, k_weight=None, eps=1e-6, rope_table=None, out_loc=slots, cache=c)
    small = ops.kv4_cache(17, n_kv, page, d)
    near_table = torch.stack([torch.arange(8) + 9, torch.arange(8) + 1]).int().cuda()
    near_slots = torch.cat([near_table[r].long().repeat_interleave(page)[:n] * page + torch.arange(n, device="cuda") % page for r, n in enumerate(kv)]).int()
    q2 = ops.qknorm_rope_kv4write(qkv, pos, n_q, n_kv, d, q_weight=None, k_weight=None, eps=1e-6, rope_table=None, out_loc=near_slots, cache=small)
    assert torch.equal(q, q2)
    for a, b in zip(ops.kv4_restore(c, table.flatten(), F32), ops.kv4_restore(small, near_table.flatten(), F32)):
        assert torch.equal(a, b)
    lens = dict(q_start=i32([0, 500, 700]), q_lens=kv, kv_lens=kv)
    assert torch.equal(attend(q, c, kv, table, **lens), attend(q, small, kv, near_table, **lens))
    one = q[[499, 699]].contiguous()
    assert torch.equal(attend(one, c, kv, table), attend(one, small, kv, near_table))


def test_tables_whose_rows_lie_apart_and_rows_of_q_behind_the_last_request():
    n_q, n_kv, d, B = 16, 2, 128, 4
    c, wide = filled(16, 81, n_kv, 16, d), table_of(B, 20)
    table, kv = wide[:, 3:15], [190, 17, 100, 64]
    assert table.stride(0) == 20
    q = normal(17, B, n_q, d, dtype=BF)
    assert torch.equal(attend(q, c, kv, table), attend(q, c, kv, table.contiguous()))
    lens, kvs = [70, 1, 2, 64], [190, 17, 100, 64]
    q = normal(18, 140, n_q, d, dtype=BF)
    kw = dict(q_start=i32([0, 70, 71, 73, 137]), q_lens=lens, kv_lens=kvs)
    a, b = attend(q, c, kvs, table, **kw), attend(q, c, kvs, table.contiguous(), **kw)
    assert torch.equal(a, b) and (a[137:] == 7.0).all()
    near(a[:137], q[:137], c, lens, kvs, table.contiguous())


def test_long_portions_restored_a_few_requests_at_a_time(monkeypatch):
    n_q, n_kv, d = 16, 2, 128
    lens, kv = [130, 1, 200, 300, 3, 129], [400, 90, 200, 777, 30, 129]
    c, table, ws = filled(19, 6 * 49 + 1, n_kv, 16, d), table_of(6, 49), Workspace("cuda")
    q = normal(20, sum(lens), n_q, d, dtype=BF)
    starts = [sum(lens[:i]) for i in range(7)]
    kw = dict(q_start=i32(starts), q_lens=lens, kv_lens=kv, workspace=ws)
    whole = attend(q, c, kv, table, **kw)
    near(whole, q, c, lens, kv, table)
    monkeypatch.setattr(ops, "KV4_RESTORE_BYTES", 4 * 2 * 128 * n_kv * d * 2)          # four pages of restored keys and values at a time, more where a request has more
    assert torch.equal(whole, attend(q, c, kv, table, **kw))


def test_steps_without_tokens():
    c, q = filled(21, 5, 2, 16, 128), normal(22, 3, 4, 128, dtype=BF)
    out = attend(q, c, [9, 20], i32([1, 2, 3, 4]).view(2, 2), q_start=i32([0, 0, 0]), q_lens=[0, 0], kv_lens=[9, 20])
    assert (out == 7.0).all()
    empty = q[:0]
    ops.kv4_attention(empty, empty, c, kv_len=i32([]), block_table=i32([]).view(0, 2), scale=1.0)
    ops.kv4_attention(empty, empty, c, kv_len=i32([]), block_table=i32([]).view(0, 2), scale=1.0, q_start=i32([0]), q_lens=[], kv_lens=[])
    assert ops.qknorm_rope_kv4write(normal(1, 0, 8 * 128), i32([]), 4, 2, 128, q_weight=None, k_weight=None, eps=1e-6, rope_table=None, out_loc=i32([]), cache=c).shape == (0, 4, 128)
