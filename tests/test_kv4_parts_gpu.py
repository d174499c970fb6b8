"""Portions over a cache in 4 bits whose restored keys are made in several parts, with key tiles cut in a part that is not the first: every row against 64 bits."""
import pytest
import torch

import plain_kv4 as plain
from mini_sglang_b200 import ops
from mini_sglang_b200.parts import Workspace
from test_kv4_edges_gpu import attend, table_of
from test_kv4_gpu import BF, bound, filled, i32, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_q,n_kv,lens,kv,pages", [
    (32, 8, [130, 1, 300, 200], [400, 90, 777, 8000], 12),              # the last request is a part by itself, and its tiles are cut
    (24, 8, [1, 250, 3, 180, 260, 1], [9, 5000, 40, 5100, 6000, 300], 88),      # two parts, both cut, short requests among them
    (40, 8, [140, 150, 160], [6000, 1500, 5200], 1)])                   # a part a request
def test_every_row_of_every_part(n_q, n_kv, lens, kv, pages, monkeypatch):
    d, ws = 128, Workspace("cuda")
    c, table = filled(31, len(kv) * 501 + 1, n_kv, 16, d), table_of(len(kv), 501)
    q = normal(32, sum(lens) + 2, n_q, d, dtype=BF)
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    kw = dict(q_start=i32(starts), q_lens=lens, kv_lens=kv, workspace=ws)
    plans, plan = [], ops.plan_tc_pieces
    monkeypatch.setattr(ops, "plan_tc_pieces", lambda a, *b, **k: plans.append((len(a), plan(a, *b, **k))) or plans[-1][1])
    monkeypatch.setattr(ops, "KV4_RESTORE_BYTES", pages * 2 * 128 * n_kv * d * 2)          # pages of restored keys and values at a time
    want, facts = plain.attention(q, c, starts, lens, kv, table, d ** -0.5)
    n = sum(lens)
    tol = torch.maximum(bound(facts[:n], max(kv), d, BF, True), bound(facts[:n], max(kv), d, BF, False))
    for _ in range(2):          # the second time over what the first left in the scratch memory
        plans.clear()
        out = attend(q, c, kv, table, **kw)
        ops.check_kernel_status()
        assert plans[-1][0] < len(lens) and plans[-1][1] is not None          # cut, and not the whole step
        err = (out[:n].double() - want[:n]).abs()
        assert (err <= tol + torch.finfo(BF).eps / 2 * (want[:n].abs() + tol)).all()
        # each request by itself: keys and values rounded to 2^-9 and the result once more make 2^-7 of its size at the very most
        for a, m in zip(starts, lens):
            assert err[a:a + m].norm() <= 2.0 ** -7 * want[a:a + m].norm()
        assert (out[n:] == 7.0).all()
