"""Rows of a cache in 4 bits that are no numbers, in portions (keys and values restored for the prefill kernels): they show in the tokens that see them, and in no other."""
import math

import pytest
import torch

from mini_sglang_b200 import ops
from mini_sglang_b200.parts import Workspace
from test_kv4_edges_gpu import SHAPES as FEW, attend, table_of
from test_kv4_gpu import BF, F32, filled, i32, normal

pytestmark = pytest.mark.gpu
#         one of every prefill kernel: tcgen05, mma, scalar in bfloat16 and float32, tiles of float32
SHAPES = [(8, 2, 128, BF), (4, 2, 64, BF), (4, 4, 40, BF), (2, 1, 512, BF), (4, 2, 128, F32), (3, 1, 40, F32)]
LENS, KV = [150, 1, 60, 3], [200, 77, 300, 9]


def portions(monkeypatch, q, c, table, window):
    """The step's attention, its two long requests as portions."""
    taken, restored = [], ops._kv4_portions
    monkeypatch.setattr(ops, "_kv4_middle", lambda q_lens, kv_lens, direct, *a: direct)
    monkeypatch.setattr(ops, "_kv4_portions", lambda *a: taken.append(a[10]) or restored(*a))
    starts = [sum(LENS[:i]) for i in range(5)]
    out = attend(q, c, KV, table, window=window, q_start=i32(starts), q_lens=LENS, kv_lens=KV, workspace=Workspace("cuda"))
    ops.check_kernel_status()
    assert len(taken) == 1 and taken[0] <= 60
    return out


def check(monkeypatch, shape, which, window, keys):
    n_q, n_kv, d, dtype = shape
    table = table_of(4, 19)
    c, q = filled(71, 77, n_kv, 16, d), normal(72, sum(LENS) + 1, n_q, d, dtype=dtype)
    clean = portions(monkeypatch, q, c, table, window)
    assert torch.isfinite(clean).all()
    shown, t = [], 0
    for r, (n, kv) in enumerate(zip(LENS, KV)):
        for pos in range(kv - n, kv):
            shown.append(any(key <= pos and (not window or key > pos - window) for key in keys[r]))
        for key in keys[r]:
            c.steps[int(table[r, key // 16]), :, key % 16, which] = math.nan
    out = portions(monkeypatch, q, c, table, window)
    shown = torch.tensor(shown + [False], device="cuda")
    assert 0 < shown[:150].sum() < 150 and 0 < shown[151:211].sum() < 60          # some tokens of either portion
    assert torch.equal(out.isnan().flatten(1).all(1), shown) and torch.equal(out.isnan().flatten(1).any(1), shown)
    # the others are as without those rows, up to the order of a few sums
    torch.testing.assert_close(out[~shown].float(), clean[~shown].float(), rtol=2.0 ** -7 if dtype == BF else 1e-5, atol=2.0 ** -7 if dtype == BF else 1e-5)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window", [0, 40])
def test_keys(monkeypatch, shape, window):
    check(monkeypatch, shape, 1, window, [[120, 121], [], [250, 299], []])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window", [0, 40])
def test_values(monkeypatch, shape, window):
    """Earlier tokens of the same query tile have weights of 0 for such a row, and so have those whose window has passed it."""
    check(monkeypatch, shape, 3, window, [[120, 121], [], [250, 299], []])


def test_pages_read_back_as_they_are():
    c = filled(73, 3, 2, 16, 64)
    c.steps[1, :, 5, 3] = math.nan
    k, v = ops.kv4_restore(c, i32([1]), F32)
    assert torch.isfinite(k).all() and v[0, :, 5].isnan().all() and torch.isfinite(v[0, :, :5]).all()


@pytest.mark.parametrize("shape", SHAPES)
def test_a_key_alone_in_its_tile(monkeypatch, shape):
    """Position 192 starts a tile of 64 or 128 keys: the token there sees that key alone of it."""
    check(monkeypatch, shape, 1, 0, [[192], [], [256], []])


@pytest.mark.parametrize("n_q,n_kv,d,dtype", FEW)
@pytest.mark.parametrize("at", [3, 40, 99])
def test_rows_of_next_to_no_weight(n_q, n_kv, d, dtype, at):
    """A value row that is no number shows where it is seen, however small its weight (200 below the other scores): from codes and in portions."""
    c, table = filled(74, 2 * 7 + 1, n_kv, 16, d), table_of(2, 7)
    q = normal(75, 2, n_q, d, dtype=dtype) * 0.125 + 1
    page = int(table[0, at // 16])
    c.steps[page, :, at % 16, 0] = 0.0
    c.steps[page, :, at % 16, 1] = -200.0 / d ** 0.5
    c.steps[page, :, at % 16, 3] = math.nan
    out = attend(q, c, [100, 100], table)
    assert out[0].isnan().all() and torch.isfinite(out[1]).all()
    q = normal(76, 100, n_q, d, dtype=dtype) * 0.125 + 1
    out = attend(q, c, [100], table[:1], q_start=i32([0, 100]), q_lens=[100], kv_lens=[100])
    assert out[at:].isnan().all() and torch.isfinite(out[:at]).all()


@pytest.mark.parametrize("n_q,n_kv,d,dtype", FEW)
@pytest.mark.parametrize("which,value", [(2, math.inf), (2, math.nan), (3, math.inf), (3, -math.inf)])
def test_steps_and_bases_that_are_none_ahead_of_a_window(n_q, n_kv, d, dtype, which, value):
    """What no append writes: such rows count for nothing where they are not seen."""
    c, table = filled(77, 8, n_kv, 16, d), table_of(1, 7)
    for key in (60, 70, 90):
        c.steps[int(table[0, key // 16]), :, key % 16, which] = value
    q = normal(78, 3, n_q, d, dtype=dtype)
    out = attend(q, c, [100], table, window=8, q_start=i32([0, 3]), q_lens=[3], kv_lens=[100])          # positions 97 to 99: keys from 90, 91 and 92 on
    assert out[0].isfinite().flatten().tolist().count(True) == 0 and out[1:].isfinite().all()


def test_values_beyond_the_range_where_they_are_not_seen(monkeypatch):
    """Codes whose value passes the largest float32, ahead of windows and in later tokens: finite steps and bases, as append writes them for rows that reach the end of the range."""
    def place(c, table, r, keys):
        for key in keys:
            c.steps[int(table[r, key // 16]), :, key % 16, 2] = 1.5e37
            c.steps[int(table[r, key // 16]), :, key % 16, 3] = 1.5e38          # 15 steps above: 3.75e38

    for n_q, n_kv, d, dtype in FEW:
        c, table = filled(79, 8, n_kv, 16, d), table_of(1, 7)
        place(c, table, 0, (60, 70, 90, 99))
        out = attend(normal(80, 3, n_q, d, dtype=dtype), c, [100], table, window=8, q_start=i32([0, 3]), q_lens=[3], kv_lens=[100])
        assert out[1].isfinite().all() and (out[[0, 2]].abs().amax(-1) > 1e30).all(), (n_q, d, dtype)
    for n_q, n_kv, d, dtype in SHAPES:
        table = table_of(4, 19)
        c, q = filled(81, 77, n_kv, 16, d), normal(82, sum(LENS) + 1, n_q, d, dtype=dtype)
        place(c, table, 0, (120,))
        place(c, table, 2, (250, 299))
        for window in (0, 40):
            with monkeypatch.context() as m:
                out = portions(m, q, c, table, window)
            seen = torch.tensor([any(k <= pos and (not window or k > pos - window) for k in keys) for n, kv, keys in zip(LENS, KV, ((120,), (), (250, 299), ())) for pos in range(kv - n, kv)] + [False])
            assert torch.equal(out.isfinite().flatten(1).all(1).cpu(), ~seen), (n_q, d, dtype, window)
