"""Captured calls of attention over a cache in 4 bits that share a workspace with each other and with calls that outgrow it."""
import pytest
import torch

from mini_sglang_b200 import ops
from mini_sglang_b200.parts import Workspace
from test_kv4_edges_gpu import attend, table_of
from test_kv4_gpu import BF, filled, i32, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_q,n_kv,d", [(8, 2, 128), (16, 1, 64)])
def test_graphs_of_two_batch_sizes_and_a_step_between_them(n_q, n_kv, d):
    ws, width, graphs = Workspace("cuda"), 130, []
    c = filled(91, 40 * width + 1, n_kv, 16, d)
    for B in (3, 40):
        q, kv, table = normal(92 + B, B, n_q, d, dtype=BF), i32([1] * B), table_of(B, width, B)
        out = torch.empty_like(q)
        run = lambda q=q, out=out, kv=kv, table=table: ops.kv4_attention(q, out, c, kv_len=kv, block_table=table, scale=d ** -0.5, workspace=ws)      # noqa: E731
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
            run()
        graphs.append((graph, q, out, kv, table))
        # many rows a request, and portions: more counters, other scratch memory
        lens, kvs = [12, 300, 1], [2000, 400, 900]
        attend(normal(93, 313, n_q, d, dtype=BF), c, kvs, table_of(3, width), q_start=i32([0, 12, 312, 313]), q_lens=lens, kv_lens=kvs, workspace=ws)
    for k in range(4):
        for graph, q, out, kv, table in graphs[::-1] if k % 2 else graphs:
            lens = [1 + (977 * (i + k + 1) * (k + 1)) % (16 * width) for i in range(q.shape[0])]
            kv.copy_(i32(lens))
            q.copy_(normal(94 + k, *q.shape, dtype=BF))
            graph.replay()
            assert torch.equal(out, attend(q, c, lens, table))          # with scratch memory of its own
