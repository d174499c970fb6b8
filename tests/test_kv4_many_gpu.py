"""Appending many tokens to a cache in 4 bits, where lanes go through several heads of a token: the rows and queries of launches of few tokens, bit for bit."""
import pytest
import torch

import plain_kv4 as plain
from mini_sglang_b200 import ops
from test_kv4_gpu import BF, F32, angles, filled, i32, normal, same_rows

pytestmark = pytest.mark.gpu


def many(n_heads, d):
    """Tokens of more than four times as many heads as run at a time: 9 blocks of 128 threads an SM, 16 elements a lane."""
    return ops.sm_count("cuda") * 9 * 128 // (d // 16) * 4 // n_heads + 1


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n_q,n_kv,d,rope,page,norm", [(13, 3, 32, True, 16, "f32"), (2, 1, 64, True, 16, None), (12, 4, 128, True, 16, "same"), (40, 8, 128, False, 64, None), (7, 2, 128, False, 5, "f32"),
                                                       (16, 8, 256, True, 16, "same")])
@pytest.mark.parametrize("extra", [0, 777])
def test_many_tokens_leave_the_rows_of_few(dtype, n_q, n_kv, d, rope, page, norm, extra):
    n_heads = n_q + 2 * n_kv
    T = many(n_heads, d) + extra
    wide = normal(1, T, n_heads * d + 8, dtype=dtype)
    qkv = wide[:, :n_heads * d]          # rows further apart than they are long
    weights = [None if norm is None else (1 + 0.1 * normal(2 + i, d)).to(dtype if norm == "same" else F32) for i in range(2)]
    table = angles(d) if rope else None
    pages = T // page + 3
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[::97] = -1                     # some nowhere
    slots[5::101] = pages * page + 4
    slots, pos = slots.int().cuda(), torch.randint(-3, 5000, (T,), generator=g).int().cuda()          # some positions outside the table
    common = dict(q_weight=weights[0], k_weight=weights[1], eps=1e-6, rope_table=table)
    got, want = ops.kv4_cache(pages, n_kv, page, d), ops.kv4_cache(pages, n_kv, page, d)
    q = ops.qknorm_rope_kv4write(qkv, pos, n_q, n_kv, d, out_loc=slots, cache=got, **common)
    for a in range(0, T, T // 5):
        b = min(a + T // 5, T)
        part = ops.qknorm_rope_kv4write(qkv[a:b], pos[a:b], n_q, n_kv, d, out_loc=slots[a:b], cache=want, **common)
        assert torch.equal(q[a:b], part)
    same_rows(got, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(4, 2, 128, 16), (3, 1, 64, 7), (2, 2, 256, 16)])
def test_norm_without_rotation(dtype, n_q, n_kv, d, page):
    T = 300
    qkv, qw, kw, slots = normal(4, T, (n_q + 2 * n_kv) * d, dtype=dtype), 1 + 0.1 * normal(5, d), 1 + 0.1 * normal(6, d), i32(range(T))
    got, want = filled(7, T // page + 1, n_kv, page, d), filled(7, T // page + 1, n_kv, page, d)
    q = ops.qknorm_rope_kv4write(qkv, slots, n_q, n_kv, d, q_weight=qw, k_weight=kw, eps=1e-6, rope_table=None, out_loc=slots, cache=got)
    q_plain = plain.append(qkv, slots, n_q, n_kv, d, qw, kw, 1e-6, None, slots, want, False)
    same_rows(got, want)
    assert torch.equal(q, q_plain.to(dtype))
