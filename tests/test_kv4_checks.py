"""What the operators of a cache in 4 bits refuse, without a GPU: every argument is looked at before the device is."""
import pytest
import torch

from mini_sglang_b200 import ops

I = lambda *s: torch.zeros(s, dtype=torch.int32)      # noqa: E731, E741


def refused(match, call, *args, **kw):
    with pytest.raises(ops.KernelError, match=match):
        call(*args, **kw)


def cache(pages=4, n_kv=2, page=16, d=32):
    return ops.kv4_cache(pages, n_kv, page, d, device="cpu")


def test_cache_is_68_bytes_a_row_of_128():
    c = cache(3, 2, 16, 128)
    assert sum(t.numel() * t.element_size() for t in c) == 3 * 2 * 16 * ops.kv4_row_bytes(128) == 3 * 2 * 16 * 2 * 68
    for d in (0, 4, 12, 520):
        refused("head sizes", ops.kv4_cache, 3, 2, 16, d, device="cpu")


def test_append_refuses():
    f, c = ops.qknorm_rope_kv4write, cache()
    x = torch.zeros(3, 8 * 32)
    ok = dict(q_weight=None, k_weight=None, eps=1e-6, rope_table=None, out_loc=I(3), cache=c)
    call = lambda qkv=x, pos=I(3), sizes=(4, 2, 32), **kw: f(qkv, pos, *sizes, **{**ok, **kw})      # noqa: E731
    refused("qkv", call, qkv=x.half())
    refused("qkv", call, qkv=x[:, :-1])
    refused("qkv", call, qkv=x.t().contiguous().t())
    refused("qkv", call, sizes=(0, 4, 32))
    refused("kv heads", call, sizes=(2, 3, 32))
    refused("kv heads", call, sizes=(8, 4, 16), qkv=torch.zeros(3, 16 * 16))
    refused("positions", call, pos=I(3).long())
    refused("positions", call, pos=I(4))
    refused("out_loc", call, out_loc=I(2))
    refused("out_loc", call, out_loc=I(6)[::2])
    w = torch.ones(32)
    refused("norm weights", call, q_weight=w)
    refused("norm weights", call, q_weight=w, k_weight=w.bfloat16())
    refused("norm weights", call, q_weight=w[:16], k_weight=w[:16])
    for table in (torch.zeros(9, 34), torch.zeros(9, 7), torch.zeros(9, 0), torch.zeros(0, 32), torch.zeros(9, 32).bfloat16(), torch.zeros(32, 9).t()):
        refused("rope_table", call, rope_table=table)
    refused("q_out", call, q_out=torch.zeros(3, 4, 32).bfloat16())
    refused("q_out", call, q_out=torch.zeros(3, 4, 16))
    refused("CUDA device", call)
    for bad in (c._replace(k=c.k.int()), c._replace(v=c.v[:3]), c._replace(steps=c.steps.float()), c._replace(steps=c.steps[..., :2]), c._replace(k=c.k.transpose(1, 2)),
                c._replace(k=c.k[..., ::2], v=c.v[..., ::2])):
        refused("a cache in 4 bits", call, cache=bad)


def test_restore_refuses():
    refused("float32 or bfloat16", ops.kv4_restore, cache(), I(2), torch.float16)
    refused("pages", ops.kv4_restore, cache(), I(2).long(), torch.float32)
    refused("CUDA device", ops.kv4_restore, cache(), I(2), torch.float32)


def test_attention_refuses():
    c, q = cache(), torch.zeros(3, 4, 32)
    ok = dict(kv_len=I(3), block_table=I(3, 4), scale=0.1)
    call = lambda x=q, out=None, **kw: ops.kv4_attention(x, torch.empty_like(x) if out is None else out, kw.pop("cache", c), **{**ok, **kw})      # noqa: E731
    refused("q and out", call, x=q.half())
    refused("q and out", call, x=q[0])
    refused("q and out", call, out=q.bfloat16())
    refused("q and out", call, x=q.transpose(0, 1))
    refused("query heads", call, x=torch.zeros(3, 4, 16))
    refused("query heads", call, x=torch.zeros(3, 3, 32))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused("scale", call, scale=scale)
    refused("window", call, window=-1)
    refused("block_table", call, block_table=I(3, 4).long())
    refused("block_table", call, block_table=I(3, 0))
    refused("kv_len", call, kv_len=I(4))
    refused("kv_len", call, kv_len=I(6)[::2])
    refused("3 tokens of 2 requests", call, kv_len=I(2), block_table=I(2, 4))
    refused("2\\^30 tokens", call, block_table=torch.empty(3, 1 << 26, dtype=torch.int32))
    lens = dict(q_start=I(4), q_lens=[1, 1, 1], kv_lens=[1, 1, 1])
    refused("q_lens", call, **{**lens, "kv_lens": None})
    refused("q_lens", call, **{**lens, "q_start": None})
    refused("q_lens", call, **{**lens, "q_lens": [1, 1]})
    refused("q_start", call, **{**lens, "q_start": I(3)})
    refused("tokens of all", call, **{**lens, "q_lens": [1, 2, 1], "kv_lens": [9, 9, 9]})
    refused("tokens of all", call, **{**lens, "q_lens": [1, -1, 1]})
    refused("block table holds", call, **{**lens, "kv_lens": [1, 65, 1]})
    refused("block table holds", call, **{**lens, "kv_lens": [1, 0, 1]})
    refused("CUDA device", call)
    refused("CUDA device", call, **lens)
    refused("a cache in 4 bits", call, cache=c._replace(v=c.v.float()))
