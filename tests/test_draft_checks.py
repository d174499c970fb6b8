"""What the kernels of drafted tokens refuse, without a GPU: every argument is looked at before the device is."""
import pytest
import torch

from mini_sglang_b200 import ops

I = lambda *s: torch.zeros(s, dtype=torch.int32)      # noqa: E731, E741


def refused(match, call, *args, **kw):
    with pytest.raises(ops.KernelError, match=match):
        call(*args, **kw)


def test_plan_refuses():
    ok = dict(page_size=16, max_draft=8)
    refused("parents", ops.draft_plan, I(4).long(), I(2), I(2), I(2, 3), **ok)
    refused("draft_lens", ops.draft_plan, I(4), I(3), I(2), I(2, 3), **ok)
    refused("cached", ops.draft_plan, I(4), I(2), I(4)[::2], I(2, 3), **ok)
    refused("block_table", ops.draft_plan, I(4), I(2), I(2), I(3, 2).t(), **ok)
    refused("block_table", ops.draft_plan, I(4), I(2), I(2), I(2, 0), **ok)
    for n in (0, 257):
        refused("max_draft", ops.draft_plan, I(4), I(2), I(2), I(2, 3), page_size=16, max_draft=n)
    refused("page_size", ops.draft_plan, I(4), I(2), I(2), I(2, 3), page_size=0, max_draft=4)
    refused("CUDA device", ops.draft_plan, I(4), I(2), I(2), I(2, 3), **ok)


def test_accept_refuses():
    f = ops.draft_accept
    refused("tokens", f, I(4).float(), I(4), I(4), I(2), max_draft=4)
    refused("parents", f, I(4), I(5), I(4), I(2), max_draft=4)
    refused("following", f, I(4), I(4), I(3), I(2), max_draft=4)
    refused("q_start", f, I(4), I(4), I(4), I(0), max_draft=4)
    refused("max_draft", f, I(4), I(4), I(4), I(2), max_draft=300)
    cache = torch.zeros(5, 2, 16, 8)
    refused("kv_len and block_table", f, I(4), I(4), I(4), I(2), max_draft=4, caches=[cache])
    more = dict(max_draft=4, kv_len=I(1), block_table=I(1, 3))
    refused("kv_len", f, I(4), I(4), I(4), I(2), max_draft=4, kv_len=I(2), block_table=I(1, 3), caches=[cache])
    refused("a cache", f, I(4), I(4), I(4), I(2), caches=[cache.transpose(1, 2)], **more)
    refused("a cache", f, I(4), I(4), I(4), I(2), caches=[cache, torch.zeros(5, 2, 8, 8)], **more)
    refused("a cache", f, I(4), I(4), I(4), I(2), caches=[cache[0]], **more)
    refused("CUDA device", f, I(4), I(4), I(4), I(2), caches=[cache], **more)


def test_logprobs_refuse():
    f, x = ops.token_logprobs, torch.zeros(3, 50)
    refused("logits", f, x.half(), I(3))
    refused("logits", f, x.t(), I(50))
    refused("logits", f, x[0], I(50))
    refused("tokens", f, x, I(4))
    refused("tokens", f, x, I(3).long())
    for top in (-1, 33):
        refused("top", f, x, I(3), top)
    refused("top", f, x[:, :4], I(3), 5)
    refused("top", f, x[:, :0], I(3), 0)
    refused("CUDA device", f, x, I(3), 5)
