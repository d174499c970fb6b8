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
    refused("draft_lens", ops.draft_plan, I(4), I(2).long(), I(2), I(2, 3), **ok)
    refused("cached", ops.draft_plan, I(4), I(3), I(2), I(2, 3), **ok)
    refused("block_table", ops.draft_plan, I(4), I(3), I(3), I(2, 3), **ok)
    refused("block_table", ops.draft_plan, I(4), I(3), I(3), I(3), **ok)
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


def test_accept_hands_over_every_cache_once(monkeypatch):
    """What the library is called with, without a GPU: the addresses of the caches are there while the call reads them, those alike in one
    launch, each once, and at most as many as a launch takes."""
    import ctypes
    calls = []

    class Library:
        @staticmethod
        def msgl_draft_accept(*a):
            calls.append((a[7], a[-7], a[-6], a[-5], list((ctypes.c_uint64 * a[-3]).from_address(a[-4]))))
            return 0

    monkeypatch.setattr(ops, "_drafts", Library)
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    monkeypatch.setattr(ops, "sm_count", lambda d: 148)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    alike = [torch.zeros(5, 3, 16, 128, dtype=torch.bfloat16) for _ in range(150)]
    other = [torch.zeros(5, 1, 16, 256, dtype=torch.bfloat16), torch.zeros(7, 1, 16, 20)]
    more = dict(max_draft=4, kv_len=I(1), block_table=I(1, 3))
    for given, groups in ((alike, [alike[:128], alike[128:]]), (alike[:56] + alike[:56], [alike[:56]]), (other[:1] + alike[:3] + other[1:], [other[:1], alike[:3], other[1:]])):
        for _ in range(20):
            calls.clear()
            ops.draft_accept(I(8), I(8), I(8), I(2), caches=given, **more)
            assert [c[4] for c in calls] == [[x.data_ptr() for x in g] for g in groups]
            assert [c[0] is not None for c in calls] == [True] + [False] * (len(groups) - 1)          # the path is written by one launch
            assert [c[1:4] for c in calls] == [(g[0].shape[0], g[0].shape[1], g[0].shape[3] * g[0].element_size()) for g in groups]


def test_tree_attention_refuses():
    f = ops.tree_attention
    q, c = torch.zeros(4, 8, 16), torch.zeros(5, 2, 16, 16)
    ok = dict(q_start=I(2), kv_len=I(1), block_table=I(1, 3), mask=I(4, 1), n_kv=2, page_size=16, scale=1.0, max_draft=4)
    refused("q and out", f, q, q[:3], c, c, **ok)
    refused("q and out", f, q, q.bfloat16(), c, c, **ok)
    refused("q and out", f, q.half(), q.half(), c, c, **ok)
    refused("q and out", f, q.transpose(1, 2), q.transpose(1, 2), c, c, **ok)
    refused("q and out", f, q[0], q[0], c, c, **ok)
    refused("caches", f, q, q, c, c[:, :, :8], **ok)
    refused("caches", f, q, q, c[0], c[0], **ok)
    refused("block_table", f, q, q, c, c, **dict(ok, block_table=I(3)))
    refused("caches", f, q, q, c.bfloat16(), c.bfloat16(), **ok)
    refused("caches", f, q, q, c, c, **dict(ok, page_size=8))
    refused("whole groups", f, torch.zeros(4, 7, 16), torch.zeros(4, 7, 16), c, c, **ok)
    wide = torch.zeros(5, 2, 16, 513)
    refused("sizes up to 512", f, torch.zeros(4, 8, 513), torch.zeros(4, 8, 513), wide, wide, **ok)
    refused("block_table", f, q, q, c, c, **dict(ok, block_table=I(1, 3).long()))
    refused("q_start", f, q, q, c, c, **dict(ok, q_start=I(3)))
    refused("kv_len", f, q, q, c, c, **dict(ok, kv_len=I(2)))
    refused("max_draft", f, q, q, c, c, **dict(ok, max_draft=257))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused("scale", f, q, q, c, c, **dict(ok, scale=scale))
    refused("a mask row", f, q, q, c, c, **dict(ok, max_draft=33))
    refused("a mask row", f, q, q, c, c, **dict(ok, mask=I(4)))
    refused("mask", f, q, q, c, c, **dict(ok, mask=I(3, 1)))
    refused("mask", f, q, q, c, c, **dict(ok, mask=I(4, 1).long()))
    refused("CUDA device", f, q, q, c, c, **ok)


def test_logprobs_of_sampling_params():
    from mini_sglang_b200 import SamplingParams
    assert SamplingParams.init_from_dict({}).logprobs is None
    for n in (0, 1, 32):
        assert SamplingParams.init_from_dict({"logprobs": n}).logprobs == n
    for n in (-1, 33):
        with pytest.raises(ValueError, match="logprobs"):
            SamplingParams.init_from_dict({"logprobs": n})


def test_unreserved_tokens_leave_the_pages_as_they_were():
    from mini_sglang_b200.cache import CacheManager, PagedKVNeed
    mgr = CacheManager({0: PagedKVNeed(2, 8)}, page_size=4, num_pages=12, max_reqs=2, max_context_len=64)
    slot = mgr.open()
    mgr.reserve(slot, 6)
    mgr.commit(slot, 6)
    for n, kept in ((9, 3), (5, 1), (12, 12)):
        before = mgr.owned_pages(slot)
        mgr.reserve(slot, n)
        assert mgr.owned_pages(slot)[:len(before)] == before
        held = mgr.owned_pages(slot)
        at = int(mgr.length[slot])
        mgr.commit(slot, kept)
        mgr.unreserve(slot)
        assert int(mgr.length[slot]) == int(mgr.reserved[slot]) == at + kept and mgr.owned_pages(slot) == held
        assert mgr.pages_needed(slot, 1) in ([0], (0,)) or at + kept == 4 * len(held)
    mgr.close(slot)
    mgr.check_idle()


def test_scores_reach_the_tokens_they_belong_to():
    """The scheduler hands every request that asked its own rows, cut to the number it asked for, in step with its tokens."""
    from mini_sglang_b200.engine.scheduler import Req, Scheduler, _InFlight
    from mini_sglang_b200.ops import TokenLogprobs
    from mini_sglang_b200.sampling import SamplingParams
    reqs = [Req(str(i), [1, 2, 3], SamplingParams(max_new_tokens=8, ignore_eos=True, logprobs=n), []) for i, n in enumerate((2, None, 0))]
    rows = [0, 2]
    scores = TokenLogprobs(torch.tensor([-1.0, -3.0]), torch.tensor([0.5, 0.25]), torch.tensor([[-0.5, -1.0], [-0.1, -3.0]]), torch.tensor([[7, 4], [9, 6]]))
    flight = _InFlight(reqs, torch.tensor([4, 5, 6]), None, None, (rows, scores))
    flight.dead.add("2")
    Scheduler._collect(None, flight, None)                   # (of the scheduler itself only what ends a request is used)
    assert reqs[0].logprobs == [(-1.0, 0.5, [(7, -0.5), (4, -1.0)])] and reqs[1].logprobs == [] and reqs[2].logprobs == []
