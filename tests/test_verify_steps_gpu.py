"""Drafted trees through whole models beyond the small case: logits made in portions."""
import random

import pytest
import torch

from helpers import make_runner
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
