"""Prefill on tcgen05 with query groups that do not divide a tile's 128 rows: tiles hold whole tokens, and the launch has blocks for all of them."""
import pytest
import torch

from mini_sglang_b200 import ops
from mini_sglang_b200.parts import Workspace

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [3, 5, 6, 7, 48])
@pytest.mark.parametrize("page", [16, 12])
def test_every_token_of_every_request_is_written(group, page):
    """151 tokens of group 5 are four tiles of 50 tokens, not three of 51; page sizes that TMA does not fetch go through the one-tile kernel."""
    lens, cached = [151, 130, 1, 204, 76], [43, 0, 9, 25, 37]
    kv = [n + c for n, c in zip(lens, cached)]
    n_kv, d, T, width = 2, 128, sum(lens), -(-max(kv) // page)
    g = torch.Generator(device="cuda").manual_seed(group)
    q, k, v = (torch.randn(s, generator=g, device="cuda").bfloat16() for s in ((T, n_kv * group, d), *[(5 * width + 1, n_kv, page, d)] * 2))
    table = (torch.arange(5 * width, device="cuda") + 1).view(5, width).int()
    starts = [sum(lens[:i]) for i in range(6)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")      # noqa: E731
    out = torch.full_like(q, 9.0)
    ops.attention_tc(q, out, k, v, q_start=i32(starts), kv_len=i32(kv), block_table=table, n_kv=n_kv, page_size=page, window=0, scale=d ** -0.5, qlen_min=2, qlen_max=1 << 30,
                     q_lens=lens, kv_lens=kv, workspace=Workspace("cuda"))
    ops.check_kernel_status()
    assert (out[starts[2]:starts[3]] == 9.0).all()          # a request shorter than qlen_min is left alone
    for r, (n, c) in enumerate(zip(lens, cached)):
        if n < 2:
            continue
        rows = q[starts[r]:starts[r + 1]].float().view(n, n_kv, group, d)
        keys, values = (x[table[r].long()].float().permute(1, 0, 2, 3).reshape(n_kv, -1, d)[:, :n + c] for x in (k, v))
        s = torch.einsum("thgd,hkd->thgk", rows, keys) * d ** -0.5
        seen = torch.arange(n + c, device="cuda") <= torch.arange(c, n + c, device="cuda")[:, None]
        want = torch.einsum("thgk,hkd->thgd", torch.softmax(s.masked_fill(~seen[:, None, None], float("-inf")), -1), values).reshape(n, n_kv * group, d)
        # weights and the result are rounded to 2^-9: at most 2^-9 of the largest value and of the result, with as much again for sums and exponentials
        assert ((out[starts[r]:starts[r + 1]].float() - want).abs() <= 2 * (2.0 ** -9 * values.abs().max() + 2.0 ** -9 * want.abs())).all(), r
