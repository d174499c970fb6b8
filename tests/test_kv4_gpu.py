"""A cache in 4 bits against plain forms: rows bit for bit, attention against 64 bits within bounds that follow from the kernels' roundings."""
import math

import pytest
import torch

import plain_kv4 as plain
from mini_sglang_b200 import ops
from mini_sglang_b200.parts import Workspace

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def normal(seed, *shape, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def i32(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def angles(rot, positions=4096):
    at = torch.arange(positions, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.cat((at.cos(), at.sin()), 1).float().cuda()


def filled(seed, pages, n_kv, page, d):
    """A cache whose rows are those of normal values, the keys with a few large elements."""
    c = ops.kv4_cache(pages, n_kv, page, d)
    for i in range(2):
        x = normal(seed + i, pages, n_kv, page, d)
        if i == 0:
            x[..., 3::16] *= 3.0
        codes, step, base = plain.quantised(x)
        c[i].copy_(plain.packed(codes))
        c.steps[..., 2 * i], c.steps[..., 2 * i + 1] = step, base
    return c


# -- appending and reading back --------------------------------------------------------------------------------

def same_rows(a, b):
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n_q,n_kv,d,rot,page,norm,interleaved", [
    (4, 2, 128, 128, 16, "f32", False), (8, 1, 64, 64, 16, "same", False), (3, 3, 32, 32, 8, None, False), (2, 2, 256, 256, 64, "f32", False),
    (4, 2, 128, 64, 16, "f32", False), (4, 2, 128, 128, 1, "same", True), (2, 1, 8, 4, 3, None, False), (5, 5, 40, 40, 16, "same", False), (2, 1, 512, 512, 16, "f32", False),
    (2, 2, 264, 0, 5, "f32", False), (6, 2, 128, 0, 16, None, False)])
@pytest.mark.parametrize("T", [1, 37])
def test_append_writes_the_rows_of_the_formula(dtype, n_q, n_kv, d, rot, page, norm, interleaved, T):
    seed = T + d + n_q
    wide = normal(seed, T, (n_q + 2 * n_kv) * d + 8, dtype=dtype)
    qkv = wide[:, :(n_q + 2 * n_kv) * d] if T > 1 else wide[:, :(n_q + 2 * n_kv) * d].contiguous()          # rows further apart than they are long
    wt = None if norm is None else dtype if norm == "same" else F32
    qw, kw = (None, None) if wt is None else ((1 + 0.1 * normal(seed + 1, d)).to(wt), (1 + 0.1 * normal(seed + 2, d)).to(wt))
    table = angles(rot, 100) if rot else None
    pages = T // page + 3
    slots = i32(torch.randperm(pages * page, generator=torch.Generator().manual_seed(seed))[:T].tolist())
    pos = i32((17 * i + 3) % 130 for i in range(T))          # some beyond the table: its last row
    got, want = filled(9, pages, n_kv, page, d), filled(9, pages, n_kv, page, d)
    q = ops.qknorm_rope_kv4write(qkv, pos, n_q, n_kv, d, q_weight=qw, k_weight=kw, eps=1e-6, rope_table=table, out_loc=slots, cache=got, interleaved=interleaved)
    q_plain = plain.append(qkv, pos, n_q, n_kv, d, qw, kw, 1e-6, table, slots, want, interleaved)
    same_rows(got, want)                       # rows that no token brings among them
    assert torch.equal(q, q_plain.to(dtype))


def test_append_leaves_out_slots_beyond_the_cache():
    c, before = filled(1, 3, 2, 16, 64), filled(1, 3, 2, 16, 64)
    qkv = normal(2, 4, 6 * 64, dtype=BF)
    ops.qknorm_rope_kv4write(qkv, i32([0, 1, 2, 3]), 2, 2, 64, q_weight=None, k_weight=None, eps=1e-6, rope_table=None, out_loc=i32([-1, 48, 2 ** 31 - 1, -2 ** 31]), cache=c)
    same_rows(c, before)


@pytest.mark.parametrize("d", [128, 40])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_without_width_and_rows_that_are_no_numbers(d, dtype):
    rows = torch.zeros(8, d, device="cuda")
    rows[1] = -3.25
    rows[2, 5] = math.inf
    rows[3, d - 1] = math.nan
    rows[4] = torch.where(torch.arange(d, device="cuda") % 2 == 0, 3e38, -3e38)          # wider than the type reaches
    rows[5, :] = 2.0 ** -110
    rows[5, 0] = 0.0
    rows[6] = torch.arange(d, device="cuda") * 1e-3
    rows[7] = -math.inf
    qkv = torch.cat([torch.zeros(8, d, device="cuda"), rows, rows.flip(0)], 1).to(dtype)
    got, want = ops.kv4_cache(1, 1, 8, d), ops.kv4_cache(1, 1, 8, d)
    args = (qkv, i32(range(8)), 1, 1, d)
    ops.qknorm_rope_kv4write(*args, q_weight=None, k_weight=None, eps=1e-6, rope_table=None, out_loc=i32(range(8)), cache=got)
    plain.append(*args, None, None, 1e-6, None, i32(range(8)), want)
    same_rows(got[:2], want[:2])
    assert torch.equal(got.steps.isnan(), want.steps.isnan()) and torch.equal(got.steps.nan_to_num(7.0), want.steps.nan_to_num(7.0))
    k, v = ops.kv4_restore(got, i32([0]), F32)
    nan = k[0, 0].isnan().all(-1)
    assert nan.tolist() == [False, False, True, True, True, False, False, True] and torch.equal(k[0, 0].isnan().any(-1), nan)
    assert torch.equal(v[0, 0].isnan().all(-1), nan.flip(0))
    assert torch.equal(k[0, 0, 0], rows[0]) and torch.equal(k[0, 0, 1], rows[1]) and (k[0, 0, 5] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n_kv,page,d", [(2, 16, 128), (3, 1, 40), (1, 48, 512), (8, 64, 8)])
def test_restore_reads_pages_back(dtype, n_kv, page, d):
    c = filled(3, 7, n_kv, page, d)
    numbers = [6, 0, 3, 3, 7, -1, 2 ** 31 - 1]
    k, v = ops.kv4_restore(c, i32(numbers), dtype)
    for i, got in enumerate((k, v)):
        whole = torch.cat([plain.values(c, i), torch.zeros(1, n_kv, page, d, dtype=torch.float64, device="cuda")])
        assert torch.equal(got, whole[[n if 0 <= n < 7 else 7 for n in numbers]].to(dtype))
    assert ops.kv4_restore(c, i32([]), dtype)[0].shape == (0, n_kv, page, d)


# -- attention -------------------------------------------------------------------------------------------------

def bound(facts, kv, d, dtype, restored):
    """How far an output may be off (the result's own rounding apart).  S: sum |q k| * scale, V: |v|, w: a value's step, Q: sum |q| * key step * scale.
    float32 arithmetic: a score is off by (d + 8) 2^-24 S, a weight by twice that relative to itself, sums of kv terms by 2 kv 2^-24 at most.
    bfloat16 from codes: sums of q (1 + c / 16), 16 key steps of them, kept to 2^-22 in each of d / 16 + 1 additions: 2 * 16 Q (d / 16 + 1) 2^-22; weights of
    codes up to 31 / 16 * 16 steps are rounded to 2^-9, but count by their codes alone (15 steps).
    bfloat16 from restored keys and values: keys off by 2^-9 S, values by 2^-9 V, weights rounded to 2^-9 and scores kept as above."""
    S, V, w, Q = facts.unbind(-1)
    ds = (d + 8) * 2.0 ** -24 * S
    rest = 2.0 * (kv + 64) * 2.0 ** -24 * V
    if dtype == BF and not restored:
        ds = ds + 2 * 16 * Q * (d / 16 + 1) * 2.0 ** -22
        rest = rest + 2.0 ** -9 * 15 * w + (kv + 64) * 2.0 ** -22 * 32 * w
    if dtype == BF and restored:
        ds = ds + 2.0 ** -9 * S
        rest = rest + 2 * 2.0 ** -9 * V
    return (2 * V * torch.expm1(ds) + rest)[..., None]


def check(q_lens, kv_lens, *, n_q, n_kv, d, dtype, page=16, window=0, seed=0, extra_rows=0, host=True, workspace=None, q_scale=1.0):
    B, T = len(q_lens), sum(q_lens) + extra_rows
    width = max(1, -(-max(kv_lens) // page))
    table = (torch.randperm(B * width, generator=torch.Generator().manual_seed(seed)) + 1).view(B, width).int().cuda()
    c = filled(seed + 3, B * width + 1, n_kv, page, d)
    q = normal(seed + 5, T, n_q, d, dtype=dtype) * q_scale
    starts = [0]
    for n in q_lens:
        starts.append(starts[-1] + n)
    out = torch.full_like(q, 7.0)
    lens = dict(q_lens=q_lens, kv_lens=kv_lens, q_start=i32(starts)) if host else {}
    ops.kv4_attention(q, out, c, kv_len=i32(kv_lens), block_table=table, scale=d ** -0.5, window=window, workspace=workspace, **lens)
    ops.check_kernel_status()
    want, facts = plain.attention(q, c, starts, q_lens, kv_lens, table, d ** -0.5, window)
    n = sum(q_lens)
    assert (out[n:] == 7.0).all()
    tol = torch.maximum(bound(facts[:n], max(kv_lens), d, dtype, True), bound(facts[:n], max(kv_lens), d, dtype, False))          # (from codes or from restored keys)
    err = (out[:n].double() - want[:n]).abs()
    tol = tol + torch.finfo(dtype).eps / 2 * (want[:n].abs() + tol)
    assert (err <= tol).all(), (err - tol).max()
    if dtype == BF and n:          # errors of many roundings cancel: well inside the bound of the worst case
        assert err.norm() <= 2.0 ** -7 * want[:n].norm() + 1e-30
    return out


GEOMETRIES = [(4, 2, 128, BF), (8, 1, 128, BF), (5, 1, 64, BF), (16, 1, 128, BF), (8, 4, 64, BF), (4, 4, 32, BF), (6, 2, 40, BF), (2, 1, 512, BF), (4, 2, 128, F32),
              (3, 1, 8, F32), (2, 1, 320, F32)]


@pytest.mark.parametrize("n_q,n_kv,d,dtype", GEOMETRIES)
@pytest.mark.parametrize("kv_lens", [[1], [5, 64, 1, 129], [700, 31, 32, 33], [2049]])
def test_single_tokens(n_q, n_kv, d, dtype, kv_lens):
    a = check([1] * len(kv_lens), kv_lens, n_q=n_q, n_kv=n_kv, d=d, dtype=dtype, host=False, workspace=Workspace("cuda"))
    b = check([1] * len(kv_lens), kv_lens, n_q=n_q, n_kv=n_kv, d=d, dtype=dtype, host=True, extra_rows=2)
    assert torch.equal(a, b[:len(kv_lens)])


@pytest.mark.parametrize("n_q,n_kv,d,dtype", GEOMETRIES)
def test_runs_of_all_lengths(n_q, n_kv, d, dtype):
    check([3, 1, 0, 70, 2, 9, 1], [3, 1, 17, 70, 300, 137, 512], n_q=n_q, n_kv=n_kv, d=d, dtype=dtype, extra_rows=3, workspace=Workspace("cuda"))


@pytest.mark.parametrize("page", [1, 3, 8, 16, 48, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 50, 1000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_pages_and_windows(page, window, dtype):
    check([1, 6, 1, 150], [333, 90, 12, 280], n_q=8, n_kv=2, d=128, dtype=dtype, page=page, window=window, seed=page)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_requests(dtype):
    kv = [1 + (37 * i) % 90 for i in range(300)]
    check([1] * 300, kv, n_q=4, n_kv=2, d=128, dtype=dtype, host=False, workspace=Workspace("cuda"))
    check([1 + i % 3 for i in range(300)], [k + 3 for k in kv], n_q=4, n_kv=2, d=64, dtype=dtype, workspace=Workspace("cuda"))
