"""A cache in 4 bits on the host: which models may have one, what it weighs, the options that ask for it."""
import types

import pytest
import torch

from mini_sglang_b200 import ops
from mini_sglang_b200.cache import CacheManager, PagedKVNeed, StateNeed
from mini_sglang_b200.engine.args import EngineArgs
from mini_sglang_b200.engine.step import CacheStorage, ModelRunner, kv_bytes_per_page


def wants(dtype, needs, takes=True):
    layers = [types.SimpleNamespace(mixer=types.SimpleNamespace(cache_need=lambda n=n: n, takes_kv4=takes)) for n in needs.values()]
    r = ModelRunner.__new__(ModelRunner)
    r.model = types.SimpleNamespace(layers=layers)
    return r._wants_kv4(dtype, {c: n for c, n in needs.items() if not isinstance(n, tuple)})


def test_models_that_may_have_one():
    assert wants("int4", {0: PagedKVNeed(8, 128), 1: PagedKVNeed(2, 64, window=100), 2: StateNeed((3,))})
    assert not wants("auto", {0: PagedKVNeed(8, 100)}, takes=False)
    for needs, words in [({0: StateNeed((3,))}, "no keys and values"), ({0: PagedKVNeed(8, 100)}, "steps of 8"), ({0: PagedKVNeed(8, 520)}, "up to 512"),
                         ({0: PagedKVNeed(1, 64, shared_kv=True)}, "one head size"), ({0: PagedKVNeed(1, 64, v_head_dim=32)}, "one head size"),
                         ({0: PagedKVNeed(1, 64, chunk=32)}, "over all keys or a window"), ({0: PagedKVNeed(1, 64, window=32, keep_first=4)}, "over all keys or a window")]:
        with pytest.raises(ValueError, match=words):
            wants("int4", needs)
    with pytest.raises(ValueError, match="activations' type only"):
        wants("int4", {0: PagedKVNeed(8, 128)}, takes=False)
    with pytest.raises(ValueError, match="one of auto, int4"):
        wants("fp8", {0: PagedKVNeed(8, 128)})


def test_only_plain_paged_attention_takes_it():
    from mini_sglang_b200.parts import MIXERS
    assert [name for name, cls in MIXERS.items() if cls.takes_kv4] == ["paged_attention"]


def test_what_it_weighs():
    needs = {0: PagedKVNeed(8, 128), 1: PagedKVNeed(2, 64)}
    assert kv_bytes_per_page(needs, 16, torch.bfloat16) == 16 * 2 * 2 * (8 * 128 + 2 * 64)
    assert kv_bytes_per_page(needs, 16, torch.bfloat16, kv4=True) == 16 * (8 * 136 + 2 * 72) == kv_bytes_per_page(needs, 16, torch.float32, kv4=True)
    mgr = CacheManager(needs, page_size=16, num_pages=5, max_reqs=2, max_context_len=64)
    storage = CacheStorage(mgr, torch.bfloat16, "cpu", kv4=True)
    assert storage.bytes() == 6 * kv_bytes_per_page(needs, 16, torch.bfloat16, kv4=True) and not storage.kv
    assert isinstance(storage.kv4[1], ops.KV4Cache) and storage.kv4[1].k.shape == (6, 2, 16, 32)


def test_options(tmp_path):
    d = str(tmp_path)
    assert EngineArgs(model=d).kv_cache_dtype == "auto" and EngineArgs(model=d, kv_cache_dtype="int4").kv_cache_dtype == "int4"
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        EngineArgs(model=d, kv_cache_dtype="int8")


def test_drafts_are_refused():
    r = ModelRunner.__new__(ModelRunner)
    r.mgr, r.kv4 = CacheManager({0: PagedKVNeed(2, 8)}, page_size=4, num_pages=4, max_reqs=2, max_context_len=16), True
    assert not r.drafts_supported()
    with pytest.raises(ValueError, match="activations' type"):
        r.verify([], None)


def test_which_requests_read_codes_directly():
    """The middle lengths go where they are estimated to be faster: few of them leave the prefill kernel without work for all SMs, many fill it."""
    of = lambda n, kv, B=1, more=(): ops._kv4_middle([n] * B + [m for m, _ in more], [kv] * B + [k for _, k in more], 20, 8, 4, 148)      # noqa: E731
    assert of(20, 4000) == 20                                     # none between
    assert of(64, 4000) == 128 and of(96, 500) == 128             # one request: its codes
    assert of(32, 2000, B=32) == 20 and of(64, 8000, B=8) == 20   # many: restored
    assert of(64, 4000, more=[(4000, 4000)]) == 20                # beside a long portion's tiles
    assert of(200, 4000) == 20                                    # longer than the middle
