"""Whole models over a cache in 4 bits."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_kv4
import plain_qwen3 as P
from helpers import PAGE, TOL, make_runner, model_dir, play, weights
from test_kv4_gpu import bound
from tiny_models import CONFIGS, random_tokens

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def runner(name, dtype, graphs=True, window=None, **kw):
    from mini_sglang_b200.config import load_config
    from mini_sglang_b200.engine.step import ModelRunner
    from mini_sglang_b200.weights import CheckpointSource
    d = model_dir(name)
    _, spec = load_config(d)
    for i, layer in enumerate(spec.layers):
        if window and i % 2 == 0:          # every other layer sees a window
            layer.mixer.params["window"] = window
    kw = {"page_size": PAGE[name], "num_pages": 400, "max_reqs": 8, **kw}
    return ModelRunner(spec, lambda exp, dt, dev: CheckpointSource(d, exp, dt, dev), dtype=dtype, use_cuda_graph=graphs, kv_cache_dtype="int4", **kw)


def plain_logits(name, tokens, monkeypatch):
    """Every position's logits with keys and values as their codes stand for them, float32 on the CPU."""
    whole = P.causal_gqa_attention

    def coded(x):
        codes, step, base = plain_kv4.quantised(x)
        return base.float()[..., None] + codes.float() * step.float()[..., None]

    with monkeypatch.context() as m, torch.no_grad():
        m.setattr(P, "causal_gqa_attention", lambda q, k, v, *a, **kw: whole(q, coded(k), coded(v), *a, **kw))
        return P.forward_sequence(CONFIGS[name], weights(name), list(tokens), device="cpu")


def trace(name, base):
    """Prompts whole and in portions, single tokens beside portions, then single tokens only."""
    V = CONFIGS[name]["vocab_size"]
    seqs = {r: random_tokens(n, V, base + n) for r, n in (("a", 61), ("b", 75), ("c", 20))}
    cuts = {"a": [40, 1, 1, 3] + [1] * 16, "b": [0, 30, 33, 2] + [1] * 10, "c": [2, 1, 0, 10] + [1] * 7}
    steps, at = [], dict.fromkeys(seqs, 0)
    for k in range(20):
        entries = []
        for r in seqs:
            n = cuts[r][k] if k < len(cuts[r]) else 0
            if n:
                entries.append((r, seqs[r][at[r]:at[r] + n], list(range(n))))
                at[r] += n
        steps.append({"entries": entries})
    return seqs, steps


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_float32_equals_the_plain_model_over_codes(name, graphs, monkeypatch):
    seqs, steps = trace(name, 2000)
    got = play(runner(name, "float32", graphs), steps)
    assert len(got) == sum(map(len, (seqs["a"], seqs["b"], seqs["c"])))
    for r, tokens in seqs.items():
        want = plain_logits(name, tokens, monkeypatch)
        for pos in range(len(tokens)):
            torch.testing.assert_close(got[(r, pos)], want[pos], **TOL["float32"])


@pytest.mark.parametrize("window", [None, 7])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", ["A", "C"])
def test_every_layer_attends_to_what_it_wrote(name, dtype, window, monkeypatch):
    """Rows written are those of the formula, bit for bit, and every attention is that of 64 bits over the cache as it then is: through portions, single
    tokens, slots used again."""
    from mini_sglang_b200 import ops
    calls = dict(write=0, attend=0)
    write, attend = ops.qknorm_rope_kv4write, ops.kv4_attention

    def checked_write(qkv, positions, n_q, n_kv, d, *, q_weight, k_weight, eps, rope_table, out_loc, cache, interleaved=False, attention_next=False):
        want = tuple(t.clone() for t in cache)
        q = write(qkv, positions, n_q, n_kv, d, q_weight=q_weight, k_weight=k_weight, eps=eps, rope_table=rope_table, out_loc=out_loc, cache=cache, interleaved=interleaved)
        q_plain = plain_kv4.append(qkv, positions, n_q, n_kv, d, q_weight, k_weight, eps, rope_table, out_loc, want, interleaved)
        assert torch.equal(q, q_plain.to(q.dtype)) and all(torch.equal(a, b) for a, b in zip(cache, want))
        calls["write"] += 1
        return q

    def checked_attend(q, out, cache, *, kv_len, block_table, scale, window=0, q_start=None, q_lens=None, kv_lens=None, workspace=None, fields_ahead=False):
        attend(q, out, cache, kv_len=kv_len, block_table=block_table, scale=scale, window=window, q_start=q_start, q_lens=q_lens, kv_lens=kv_lens, workspace=workspace,
               fields_ahead=fields_ahead)
        lens, kvs = q_lens or [1] * len(kv_len), kv_len.tolist()
        assert kv_lens is None or kvs == list(kv_lens)
        starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
        assert q_start is None or q_start.tolist() == starts
        want, facts = plain_kv4.attention(q, cache, starts, lens, kvs, block_table, scale, window)
        d = q.shape[2]
        tol = torch.maximum(bound(facts, max(kvs), d, q.dtype, False), bound(facts, max(kvs), d, q.dtype, True))
        assert ((out.double() - want).abs() <= tol + torch.finfo(q.dtype).eps / 2 * (want.abs() + tol)).all()
        calls["attend"] += 1

    monkeypatch.setattr(ops, "qknorm_rope_kv4write", checked_write)
    monkeypatch.setattr(ops, "kv4_attention", checked_attend)
    r = runner(name, dtype, graphs=False, window=window, num_pages=-(-220 // PAGE[name]) + 4, max_reqs=4)
    for base in (2100, 2200):          # the second time on pages and slots that the first gave back
        seqs, steps = trace(name, base)
        play(r, [dict(s, end=list(seqs) if s is steps[-1] else []) for s in steps])
    layers = CONFIGS[name]["num_hidden_layers"]
    assert calls["write"] == calls["attend"] == 2 * 20 * layers


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("B", "bfloat16"), ("C", "bfloat16")])
def test_graphs_replay_what_is_launched(name, dtype):
    seqs, steps = trace(name, 2300)
    a, b = play(runner(name, dtype, True), steps), play(runner(name, dtype, False), steps)
    assert a.keys() == b.keys()
    for k in a:
        torch.testing.assert_close(a[k], b[k], rtol=1e-5, atol=1e-5) if dtype == "float32" else torch.testing.assert_close(a[k], b[k], rtol=0.05, atol=0.02)


def test_head_size_128_in_graphs_and_among_portions():
    """The kernels of head size 128 in a whole model: single tokens in graphs of several batch sizes against the same steps launched one by one, bit for bit."""
    from mini_sglang_b200.config import load_config
    from mini_sglang_b200.engine.step import ModelRunner, StepEntry
    cfg = dict(CONFIGS["C"], head_dim=128, num_hidden_layers=2)
    import tempfile
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "config.json"), "w") as f:
            json.dump(cfg, f)
        _, spec = load_config(d)
        rs = [ModelRunner.from_random(spec, 3, dtype="bfloat16", page_size=16, num_pages=300, max_reqs=8, use_cuda_graph=g, kv_cache_dtype="int4") for g in (True, False)]
        V, outs = cfg["vocab_size"], [[], []]
        for r, out in zip(rs, outs):
            slots = [r.open() for _ in range(8)]
            rng = np.random.RandomState(0)
            toks = lambda n: rng.randint(0, V, n).tolist()      # noqa: E731
            out.append(r.step([StepEntry(slots[i], toks(n), [n - 1]) for i, n in enumerate((300, 17, 1, 2, 64, 5, 100, 33))]))
            for b in (8, 1, 4, 8, 2):
                out.append(r.step([StepEntry(s, toks(1), [0]) for s in slots[:b]]).clone())          # (a graph writes its logits where it wrote them before)
                assert r.last_step_used_graph == (r is rs[0])
            out.append(r.step([StepEntry(slots[0], toks(1), [0]), StepEntry(slots[1], toks(90), [89]), StepEntry(slots[2], toks(7), [6])]))
        from mini_sglang_b200 import ops
        ops.check_kernel_status()
        for x, y in zip(*outs):
            assert torch.isfinite(x).all() and torch.equal(x, y)


def make_engine(name, dtype, **kw):
    from mini_sglang_b200 import Engine, EngineArgs
    return Engine(EngineArgs(**{**dict(model=model_dir(name), dtype=dtype, page_size=PAGE[name], num_pages=256, max_num_reqs=8, random_seed=0, log_level="WARNING", kv_cache_dtype="int4"),
                                **kw}))


def test_generation_does_not_depend_on_the_batch_or_the_pool():
    """Shared prefixes, portions, retraction: float32 tokens are those of each request alone."""
    name, cfg = "B", CONFIGS["B"]
    shared = random_tokens(24, cfg["vocab_size"], 2400)
    prompts = [shared + random_tokens(n, cfg["vocab_size"], 2400 + n) for n in (3, 9, 17, 5, 30, 12)]
    sp = {"temperature": 0.0, "max_new_tokens": 12, "ignore_eos": True}
    alone = [make_engine(name, "float32").generate(input_ids=p, sampling_params=sp)["token_ids"] for p in prompts]
    for kw in (dict(), dict(num_pages=40, chunk_size=16, max_prefill_tokens=32), dict(disable_radix_cache=True, schedule_policy="fcfs", disable_overlap=True)):
        eng = make_engine(name, "float32", **kw)
        assert [o["token_ids"] for o in eng.generate(input_ids=prompts, sampling_params=sp)] == alone
        eng.scheduler.check_idle_invariants()


def test_pages_come_from_the_bytes_of_codes():
    from mini_sglang_b200.engine.step import kv_bytes_per_page
    r = runner("A", "bfloat16")
    assert r.storage.bytes() == (400 + 1) * kv_bytes_per_page(r.mgr.needs, PAGE["A"], torch.bfloat16, kv4=True)
    assert not r.drafts_supported()


def test_trace_run_takes_the_option(tmp_path):
    lines = [{"step": 0, "entries": [{"id": "x", "tokens": [1, 2, 3, 4, 5], "want": [4]}], "end": []}, {"step": 1, "entries": [{"id": "x", "tokens": [6], "want": [0]}], "end": ["x"]}]
    outs = []
    for dtype in ("int4", "auto"):
        out = tmp_path / dtype
        subprocess.run([sys.executable, os.path.join(ROOT, "bin", "trace_run"), "--model", model_dir("B"), "--dtype", "float32", "--out", str(out), "--max-tokens", "64",
                        "--kv-cache-dtype", dtype], input="".join(json.dumps(x) + "\n" for x in lines), text=True, check=True, capture_output=True, timeout=600)
        outs.append([np.fromfile(out / f"{s}.f32", dtype="<f4") for s in (0, 1)])
    for a, b in zip(*outs):
        assert np.isfinite(a).all() and a.shape == b.shape and not np.array_equal(a, b)
