"""Portions over a cache in 4 bits whose restored keys are made in several parts, on the host: which tokens the launches of every part name (the libraries' entry points are recorded,
no GPU is needed)."""
import types

import pytest
import torch

from mini_sglang_b200 import ops
from mini_sglang_b200.parts import Workspace

META = torch.device("meta")


class Recorder:
    """A library whose entry points note their arguments."""

    def __init__(self, log):
        self.log = log

    def __getattr__(self, name):
        return lambda *a: self.log.append((name, a)) or 0


def launches(monkeypatch, q_lens, kv_lens, n_q=32, n_kv=8, d=128, workspace=True):
    log, plans, plan = [], [], ops.plan_tc_pieces
    for name, fake in dict(_need_cuda=lambda *t: None, _status_tensor=lambda dev: torch.zeros(1), _stream=lambda *a: 0, _attn_lib=lambda d: Recorder(log), _kv4_lib=lambda: Recorder(log),
                           sm_count=lambda *a: 148, poll_status=lambda *a: None,
                           plan_tc_pieces=lambda q, kv, **kw: plans.append((list(q), plan(q, kv, **kw), kw["bytes_per_piece"])) or plans[-1][1]).items():
        monkeypatch.setattr(ops, name, fake)
    T, B, width = sum(q_lens), len(q_lens), -(-max(kv_lens) // 16)
    q = torch.empty(T, n_q, d, dtype=torch.bfloat16, device=META)
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, device=META)      # noqa: E731
    ops._kv4_portions(q, torch.empty_like(q), ops.kv4_cache(4, n_kv, 16, d, device=META), i32(B), i32(B, width), d ** -0.5, 0, i32(B + 1), list(q_lens), list(kv_lens), 21,
                      Workspace("meta") if workspace else None, lambda beside: log.append(("others", beside)))
    tiles = [a for name, a in log if name == "msgl_attention_tc"]
    merges = [a for name, a in log if name == "msgl_attention_combine_range"]
    return types.SimpleNamespace(log=[name for name, _ in log], plans=plans, tiles=tiles, merges=merges)


#         the step's lengths, the requests of every part
STEPS = [([100] * 8, [40000] * 8, [6, 2]),                                         # eight long conversations that go on at once
         ([2000, 2000, 400], [131072, 131072, 60400], [2, 1]),
         ([200] * 9, [30200] * 9, [8, 1])]


@pytest.mark.parametrize("q_lens,kv_lens,parts", STEPS)
def test_every_part_merges_its_own_tokens(monkeypatch, q_lens, kv_lens, parts):
    got = launches(monkeypatch, q_lens, kv_lens)
    assert [len(q) for q, _, _ in got.plans] == parts and len(got.tiles) == len(parts)
    at, merged = 0, []
    for (lens, plan, per_piece), tile in zip(got.plans, got.tiles):
        first, n = sum(q_lens[:at]), sum(lens)
        at += len(lens)
        assert per_piece == n * 32 * 128 * 4          # what a cut costs counts the part's tokens only
        lo, plane = tile[35:37]
        if plan is not None:
            assert first <= lo < lo + plane <= first + n          # partial results are kept for the part's own tokens
            merged += [(lo, plane, first + a, m) for a, m in plan[2]]
    assert plan is not None          # (the last part, which is not the first, is cut)
    assert [m[5:9] for m in got.merges] == merged


def test_requests_left_out_ahead_of_a_part_count_too(monkeypatch):
    """Single tokens between the portions belong to no part's plan, but the tokens behind them are counted from the step's first."""
    q_lens, kv_lens = [1, 2000, 1, 1, 2000, 1, 400, 1], [50, 131072, 9, 9, 131072, 9, 60400, 7]
    got = launches(monkeypatch, q_lens, kv_lens)
    assert got.plans[1][1] is not None and got.merges[-1][5:9] == (4004, 400, 4004, 400) and got.log[-1] == "msgl_attention_combine_range"
    assert got.log.count("others") == 1


def test_a_step_in_one_part_counts_as_ever(monkeypatch):
    got = launches(monkeypatch, [100] * 3, [9000] * 3)
    (lens, plan, per_piece), = got.plans
    assert per_piece == 300 * 32 * 128 * 4 and [m[7:9] for m in got.merges] == [tuple(r) for r in plan[2]]
