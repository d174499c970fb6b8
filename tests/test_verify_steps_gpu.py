"""Drafted trees through whole models beyond the small case: logits made in portions, bfloat16 models whose head sizes are the tensor cores'."""
import random

import pytest
import torch

from helpers import BF16_MAX_FACTOR, BF16_RMS_FRACTION, assert_row_close, make_runner
from test_drafts_engine_gpu import decode, guess, sampler
from tiny_models import CONFIGS, random_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_logits_are_made_in_portions(temperature, monkeypatch):
    """No more logits at a time than the bound has room for; the tokens stay those of plain decoding."""
    from mini_sglang_b200.engine import DraftEntry, step
    V, rows = CONFIGS["B"]["vocab_size"], 7
    runner = make_runner("B", "float32", num_pages=400)
    smp, rng, seen, whole = sampler(runner), random.Random(3), [], runner.model.head.forward

    def head(h):
        seen.append(h.shape[0])
        return whole(h)

    monkeypatch.setattr(step, "VERIFY_LOGITS_BYTES", 4 * V * rows + 100)
    prompts, want, got, slots = [random_tokens(n, V, n) for n in (9, 20)], [], [], []
    for i, p in enumerate(prompts):
        slot = runner.open()
        want.append(decode(runner, slot, p, 30, smp, temperature, i))
        runner.close(slot)
    for i, p in enumerate(prompts):
        slots.append(runner.open())
        got.append([int(smp.sample(runner.step([step.StepEntry(slots[i], p, [len(p) - 1])]), [temperature], [i], [0])[0])])
    monkeypatch.setattr(runner.model.head, "forward", head)
    drafts = kept = 0
    while live := [i for i in range(2) if len(got[i]) < 16]:
        sizes = [rng.choice((3, 7, 13)) for _ in live]
        seen.clear()
        new = runner.verify([DraftEntry(slots[i], *guess(rng, want[i][len(got[i]) - 1:], n, V)) for i, n in zip(live, sizes)], smp, [temperature] * len(live), live,
                            [len(got[i]) for i in live])
        assert sum(seen) == sum(sizes) and max(seen) <= rows
        for i, more in zip(live, new):
            got[i].extend(more)
            kept += len(more)
        drafts += len(live)
    assert kept > drafts                                 # some drafts were accepted
    for g, w in zip(got, want):
        assert g == w[:len(g)]
    for s in slots:
        runner.close(s)


HEADS = {64: dict(num_attention_heads=4, num_key_value_heads=1), 128: dict(num_attention_heads=4, num_key_value_heads=2)}


@pytest.mark.parametrize("head_dim", [64, 128])
def test_verify_on_the_tensor_cores(head_dim, tmp_path, monkeypatch):
    """A bfloat16 model whose drafts are the plain model's own continuation among others: several tokens a round are kept, each (near-)best under the
    plain model, and the cache goes on as if they had been fed one by one."""
    import plain_qwen3
    from mini_sglang_b200 import ops
    from mini_sglang_b200.engine import DraftEntry, step
    from tiny_models import make_weights, write_model_dir
    cfg = dict(CONFIGS["B"], head_dim=head_dim, **HEADS[head_dim])
    weights, V = make_weights(cfg, 5), cfg["vocab_size"]
    write_model_dir(str(tmp_path), cfg, weights)
    runner = step.ModelRunner.from_model_dir(str(tmp_path), dtype="bfloat16", page_size=16, num_pages=64, max_reqs=2, max_context_len=512)
    lib, kinds = ops._draft_lib(), []

    class Library:
        def __getattr__(self, name):
            fn = getattr(lib, name)

            def attend(*a):
                kinds.append(a[-4])
                return fn(*a)
            return attend if name == "msgl_tree_attention" else fn

    monkeypatch.setattr(ops, "_drafts", Library())

    @torch.no_grad()
    def plain(seq):
        return plain_qwen3.forward_sequence(cfg, weights, list(seq), device="cpu")

    smp, rng, prompt = sampler(runner), random.Random(6), random_tokens(150, V, 8)
    slot = runner.open()
    got = [int(smp.sample(runner.step([step.StepEntry(slot, prompt, [149])]), [0.0], [0], [0])[0])]
    rounds = moved = 0
    while len(got) < 30:
        ahead = []                                       # what the plain model puts after the tokens so far
        for _ in range(5):
            ahead.append(int(plain(prompt + got + ahead)[-1].argmax()))
        toks, up = guess(rng, got[-1:] + ahead, 40, V)
        more = runner.verify([DraftEntry(slot, toks, up)], smp)[0]
        path = [0]
        for t in more[:-1]:
            path.append(next(i for i in range(len(up)) if up[i] == path[-1] and toks[i] == t))
        moved += path != list(range(len(path)))
        got.extend(more)
        rounds += 1
    assert len(got) - 1 > 2 * rounds and moved > 0       # several drafts a round were kept, not all where they lay
    ref = plain(prompt + got)
    for i, t in enumerate(got):
        row = ref[len(prompt) - 1 + i]
        # two logits of the row, each off by no more than the largest error that a bfloat16 row may have
        assert row[t] >= row.max() - 2 * BF16_MAX_FACTOR * BF16_RMS_FRACTION * row.pow(2).mean().sqrt(), (i, t)
    assert_row_close(runner.step([step.StepEntry(slot, [got[-1]], [0])]).float().cpu()[0], ref[-1], "bfloat16")
    assert set(kinds) == {ops._TREE_TC} and len(kinds) == rounds * cfg["num_hidden_layers"]
    runner.close(slot)
    runner.mgr.check_idle()
