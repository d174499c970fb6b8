"""Attention over a cache in 4 bits where value rows differ in size by more than a float16 holds: what a row does not see, or gives no weight, costs it no digits."""
import pytest
import torch

import plain_kv4_bounds as bounds
from test_kv4_edges_gpu import SHAPES, attend, table_of
from test_kv4_gpu import BF, filled, i32, normal

pytestmark = pytest.mark.gpu
LARGE = 2.0 ** 60


def check(q, c, lens, kv, table, window=0, **kw):
    d, dtype = q.shape[2], q.dtype
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    out = attend(q, c, kv, table, window=window, q_start=i32(starts), q_lens=lens, kv_lens=kv, **kw)
    want, off = bounds.attention(q, c, starts, lens, kv, table, d ** -0.5, window, "codes" if dtype == BF and d in (64, 128) else "float32")
    assert ((out.double() - want).abs() <= off + torch.finfo(dtype).eps / 2 * (want.abs() + off)).all()
    return want


def place(c, table, r, key, which, value):
    c.steps[int(table[r, key // 16]), :, key % 16, which] = value


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
def test_steps_of_keys_that_are_not_seen(n_q, n_kv, d, dtype):
    """Keys ahead of the window and keys of later tokens, in the unit of 32 of those that are seen: their values' steps are 2^60."""
    lens, kv, window = [1, 3, 2], [70, 70, 100], 9
    table = table_of(3, 7)
    c, q = filled(51, 22, n_kv, 16, d), normal(52, 6, n_q, d, dtype=dtype)
    for r, keys in enumerate(([33, 40, 59], [35, 69], [68, 99])):          # (69 and 99: the last tokens' own keys)
        for key in keys:
            place(c, table, r, key, 2, LARGE)
    want = check(q, c, lens, kv, table, window)
    assert want[[0, 1, 2, 4]].abs().max() < 10 and (want[[3, 5]].abs().amax(-1) > 2.0 ** 40).all()          # ordinary rows, and those that see the large ones


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
@pytest.mark.parametrize("at", [0, 40, 299])
def test_large_steps_with_next_to_no_weight(n_q, n_kv, d, dtype, at):
    """A key seen first, in the middle or last, whose score lies 68 below the others' (weight 2^-98) and whose value's step is 2^60: it counts for 2^-34 in all."""
    c, table = filled(53, 19 * 2 + 1, n_kv, 16, d), table_of(2, 19)
    q = normal(54, 2, n_q, d, dtype=dtype) * 0.125 + 1
    for r in range(2):
        place(c, table, r, at, 0, 0.0)
        place(c, table, r, at, 1, -68.0 / d ** 0.5)
        place(c, table, r, at, 2, LARGE)
    assert check(q, c, [1, 1], [300, 300], table).abs().max() < 10


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
def test_large_steps_that_others_outweigh_later(n_q, n_kv, d, dtype):
    """All keys of the first 64 have steps of 2^60 and scores 68 below those behind them, so that their weights, the largest at first, end as next to nothing."""
    c, table = filled(55, 13 * 2 + 1, n_kv, 16, d), table_of(2, 13)
    q = normal(56, 2, n_q, d, dtype=dtype) * 0.125 + 1
    for r in range(2):
        for key in range(64):
            place(c, table, r, key, 0, 0.0)
            place(c, table, r, key, 1, -68.0 / d ** 0.5)
            place(c, table, r, key, 2, LARGE)
    assert check(q, c, [1, 1], [200, 200], table).abs().max() < 10


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
def test_rows_of_one_request_with_weights_of_different_sizes(n_q, n_kv, d, dtype):
    """Queries of either sign: half the heads give all their weight to keys whose values have steps of 2^60, the others to ordinary ones."""
    c, table = filled(57, 8, n_kv, 16, d), table_of(1, 7)
    q = normal(58, 3, n_q, d, dtype=dtype) * 0.125 + 1
    q[:, ::2] *= -1
    for key in range(5, 100, 7):
        place(c, table, 0, key, 0, 0.0)
        place(c, table, 0, key, 1, -68.0 / d ** 0.5)
        place(c, table, 0, key, 2, LARGE)
    want = check(q, c, [3], [100], table)
    assert want[:, 1::2].abs().max() < 10 and (want[:, ::2].abs().amax(-1) > LARGE).all()


@pytest.mark.parametrize("n_q,n_kv,d,dtype", SHAPES)
@pytest.mark.parametrize("q_size", [1, 30])
def test_steps_of_all_sizes(n_q, n_kv, d, dtype, q_size):
    """Steps and bases between 2^-60 and 2^60 times what they were, in falling, rising and mixed order of the keys."""
    B, n = 3, 300
    c, table = filled(59, B * 19 + 1, n_kv, 16, d), table_of(B, 19)
    up = 2.0 ** torch.linspace(-60, 60, 19 * 16, device="cuda")
    for r, order in enumerate((up, up.flip(0), up[torch.randperm(up.numel(), generator=torch.Generator().manual_seed(1)).cuda()])):
        c.steps[table[r].long(), :, :, 2:] *= order.view(19, 1, 16, 1).to(BF)
    check(normal(60, B, n_q, d, dtype=dtype) * q_size, c, [1] * B, [n] * B, table)


@pytest.mark.parametrize("n_q,n_kv,d", [(4, 2, 128), (8, 1, 64)])
@pytest.mark.parametrize("low", [-68.0, -4.0])
def test_units_of_either_kind_in_one_warps_run(n_q, n_kv, d, low):
    """48 or 96 requests of the same 3,000 keys, so that a warp goes through several units: in every third unit of 32 the steps are 2^60 and the scores `low`, among them first and last ones."""
    B, n = 96 // n_kv, 3000
    c, pages = filled(61, 189, n_kv, 16, d), table_of(1, 188)
    q = normal(62, B, n_q, d, dtype=BF) * 0.125 + 1
    for page in range(188):
        if page // 2 % 3 == 0:
            c.steps[int(pages[0, page]), :, :, 0] = 0.0
            c.steps[int(pages[0, page]), :, :, 1] = low / d ** 0.5
            c.steps[int(pages[0, page]), :, :, 2] = LARGE
    kv = [n - 3 * i for i in range(B)]
    out = attend(q, c, kv, pages.repeat(B, 1))
    rows = [0, 1, 17, B - 1]
    want, off = bounds.attention(q[rows], c, [0, 1, 2, 3], [1] * 4, [kv[r] for r in rows], pages.repeat(4, 1), d ** -0.5, 0, "codes")
    assert ((out[rows].double() - want).abs() <= off + torch.finfo(BF).eps / 2 * (want.abs() + off)).all()
    assert want.abs().max() < 10 if low < -60 else (want.abs().amax(-1) > 2.0 ** 30).all()
