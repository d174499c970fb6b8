"""The cut of a step's keys over blocks (attention over a cache in 4 bits, from the codes): a long request among short ones, wherever it stands."""
import pytest
import torch

from test_kv4_edges_gpu import attend, near, table_of
from test_kv4_gpu import BF, filled, i32, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
def test_pieces_of_a_long_request_among_short_ones(d):
    """40 requests of 2 segments each, of which one has 94 units of keys in 5 pieces: whichever lane of the cutting warp it falls to, all pieces are added up."""
    n_kv, B, width = 2, 40, 188
    c, q = filled(41, 2 * width + 1, n_kv, 16, d), normal(42, B, 4, d, dtype=BF)
    table = table_of(2, width)[0].repeat(B, 1)
    for at in (0, 1, 2, 17, 31, 32, 38, 39):
        kv = [20 + (7 * i) % 60 for i in range(B)]
        kv[at] = 3000
        got = attend(q, c, kv, table)
        assert torch.equal(got, attend(q, c, kv, table, q_start=i32(range(B + 1)), q_lens=[1] * B, kv_lens=kv))
        rows = [at, (at + 1) % B, (at + 39) % B]
        near(got[rows], q[rows].contiguous(), c, [1] * 3, [kv[r] for r in rows], table[rows])
