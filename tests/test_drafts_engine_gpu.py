"""Drafted trees through whole models: the tokens of plain decoding whatever the drafts, a cache that goes on as if they had been fed one by one, and
log probabilities of generated tokens."""
import math
import random

import pytest
import torch

from helpers import PAGE, make_runner, model_dir, plain_logits
from tiny_models import CONFIGS, random_tokens

pytestmark = pytest.mark.gpu


def sampler(runner, seed=3):
    from mini_sglang_b200.sampling import Sampler
    return Sampler(seed, runner.device)


def decode(runner, slot, prompt, n, smp, temperature, key):
    """n tokens one by one; the last is not fed."""
    from mini_sglang_b200.engine.step import StepEntry
    logits = runner.step([StepEntry(slot, prompt, [len(prompt) - 1])])
    out = []
    for i in range(n):
        out.append(int(smp.sample(logits, [temperature], [key], [i])[0]))
        if i + 1 < n:
            logits = runner.step([StepEntry(slot, [out[-1]], [0])])
    return out


def guess(rng, known, n, vocab):
    """A tree of n drafts behind known[0] that holds some of the tokens that follow, others beside them, in random places."""
    tokens, parents, right = [known[0]], [-1], [0]          # right: drafts on the true path
    while len(tokens) < n:
        if len(right) < len(known) and rng.random() < 0.6:
            parents.append(right[-1])
            tokens.append(known[len(right)])
            right.append(len(tokens) - 1)
        else:
            parents.append(rng.randrange(len(tokens)))
            tokens.append(rng.randrange(vocab))
    return tokens, parents


@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_verified_drafts_give_the_tokens_of_plain_decoding(name, temperature):
    from mini_sglang_b200.engine import DraftEntry
    from mini_sglang_b200.engine.step import StepEntry
    V, N = CONFIGS[name]["vocab_size"], 24
    runner = make_runner(name, "float32", num_pages=400, max_reqs=8)
    smp, rng = sampler(runner), random.Random(5)
    prompts = [random_tokens(n, V, 700 + n) for n in (5, 17, 30)]
    want = []
    for i, p in enumerate(prompts):
        slot = runner.open()
        want.append(decode(runner, slot, p, N, smp, temperature, 10 + i))
        runner.close(slot)
    slots = [runner.open() for _ in prompts]
    first = runner.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)])
    got = [[int(t)] for t in smp.sample(first, [temperature] * 3, [10, 11, 12], [0] * 3)]
    assert [g[0] for g in got] == [w[0] for w in want]
    rounds = kept = 0
    while min(map(len, got)) < N:
        live = [i for i in range(3) if len(got[i]) < N]
        entries = []
        for i in live:
            toks, up = guess(rng, want[i][len(got[i]) - 1:], rng.choice((1, 2, 6, 13)), V)
            entries.append(DraftEntry(slots[i], toks, up))
        new = runner.verify(entries, smp, [temperature] * len(live), [10 + i for i in live], [len(got[i]) for i in live])
        for i, more in zip(live, new):
            assert 1 <= len(more)
            got[i].extend(more)
            kept += len(more)
        rounds += len(live)
    assert kept > rounds                                     # some drafts were accepted
    for g, w in zip(got, want):
        assert g[:N] == w
    # the cache goes on: the next logits are those of the whole sequence
    for i, s in enumerate(slots):
        seq = prompts[i] + got[i]
        assert int(runner.mgr.length[s]) == len(seq) - 1
        row = runner.step([StepEntry(s, [got[i][-1]], [0])]).float().cpu()[0]
        ref = plain_logits(name, seq)[-1]
        torch.testing.assert_close(row, ref, rtol=1e-4, atol=5e-5)
    for s in slots:
        runner.close(s)
    runner.mgr.check_idle()


def test_verify_in_bfloat16_follows_the_plain_model():
    """bfloat16 on the tensor cores' head size: every token kept is (near-)best under the plain model."""
    from mini_sglang_b200.engine import DraftEntry
    from mini_sglang_b200.engine.step import StepEntry
    name = next((n for n in ("A", "B", "C") if CONFIGS[n].get("head_dim") in (64, 128)), "A")
    V = CONFIGS[name]["vocab_size"]
    runner = make_runner(name, "bfloat16", num_pages=400, page_size=16)
    smp, rng = sampler(runner), random.Random(1)
    prompt = random_tokens(40, V, 77)
    slot = runner.open()
    got = [int(smp.sample(runner.step([StepEntry(slot, prompt, [39])]), [0.0], [0], [0])[0])]
    while len(got) < 20:
        up = [-1] + [rng.randrange(i) for i in range(1, 30)]
        toks = [got[-1]] + [rng.randrange(V) for _ in range(29)]
        got.extend(runner.verify([DraftEntry(slot, toks, up)], smp)[0])
    ref = plain_logits(name, prompt + got)
    for i, t in enumerate(got):
        row = ref[len(prompt) - 1 + i]
        assert row[t] >= row.max() - 0.05, (i, t)
    runner.close(slot)


def test_verify_refuses():
    from mini_sglang_b200.cache import OutOfPages
    from mini_sglang_b200.engine import DraftEntry
    runner = make_runner("B", "float32", num_pages=3)
    smp, slot = sampler(runner), runner.open()
    for bad, match in ((DraftEntry(slot, []), "drafted tokens"), (DraftEntry(slot, [1, 2], [-1]), "drafted tokens"), (DraftEntry(slot, [1, 2], [-1, 1]), "earlier"),
                       (DraftEntry(slot, [1, 2], [0, 0]), "earlier"), (DraftEntry(slot, [1, 10 ** 9]), "token id"), (DraftEntry(slot, [1] * 257), "drafted tokens")):
        with pytest.raises(ValueError, match=match):
            runner.verify([bad], smp)
    with pytest.raises(ValueError, match="one tree"):
        runner.verify([DraftEntry(slot, [1]), DraftEntry(slot, [2])], smp)
    with pytest.raises(OutOfPages):
        runner.verify([DraftEntry(slot, [1] * 200)], smp)
    assert int(runner.mgr.reserved[slot]) == 0 and runner.verify([], smp) == []
    assert len(runner.verify([DraftEntry(slot, [1, 2, 3])], smp)[0]) >= 1
    assert int(runner.mgr.reserved[slot]) == int(runner.mgr.length[slot])
    runner.close(slot)
    runner.mgr.check_idle()


def test_models_with_windows_or_states_are_refused():
    import tempfile

    from mini_sglang_b200.engine import DraftEntry
    from mini_sglang_b200.engine.step import ModelRunner
    from tiny_models import write_model_dir
    from tiny_vekurax import CONFIGS_V, config_json, make_weights
    with tempfile.TemporaryDirectory() as d:
        write_model_dir(d, config_json(CONFIGS_V["VA"]), make_weights(CONFIGS_V["VA"], 3))
        runner = ModelRunner.from_model_dir(d, dtype="float32", page_size=4, num_pages=32, max_reqs=2, max_context_len=64)
        slot = runner.open()
        assert not runner.drafts_supported()
        with pytest.raises(ValueError, match="all keys"):
            runner.verify([DraftEntry(slot, [1, 2])], sampler(runner))


def make_engine(dtype="float32", **kw):
    from mini_sglang_b200 import Engine, EngineArgs
    return Engine(EngineArgs(**dict(dict(model=model_dir("B"), dtype=dtype, page_size=PAGE["B"], num_pages=256, max_num_reqs=8, random_seed=0, log_level="WARNING"), **kw)))


@pytest.mark.parametrize("overlap", [True, False])
def test_logprobs_of_generated_tokens(overlap):
    """Of every token of the requests that ask, and of no others; the tokens stay what they were."""
    V = CONFIGS["B"]["vocab_size"]
    prompts = [random_tokens(n, V, 40 + n) for n in (7, 16, 23)]
    base = {"temperature": 0.7, "max_new_tokens": 9, "ignore_eos": True}
    plain = make_engine(disable_overlap=not overlap).generate(input_ids=prompts, sampling_params=base)
    eng = make_engine(disable_overlap=not overlap)
    outs = eng.generate(input_ids=prompts, sampling_params=[dict(base, logprobs=4), base, dict(base, logprobs=0)])
    assert [o["token_ids"] for o in outs] == [o["token_ids"] for o in plain] and "logprobs" not in outs[1]
    for p, o, n in ((prompts[0], outs[0], 4), (prompts[2], outs[2], 0)):
        toks = o["token_ids"]
        lp = torch.log_softmax(plain_logits("B", p + toks).double(), -1)
        assert len(o["logprobs"]) == len(toks) == 9
        for i, e in enumerate(o["logprobs"]):
            row = lp[len(p) - 1 + i]
            assert e["token"] == toks[i] and len(e["top"]) == n
            # the logits are off by up to 1e-4 of their size and 5e-5 (the float32 path's bound), a log probability by twice that, an entropy by that
            # times the spread of the log probabilities
            assert math.isclose(e["logprob"], float(row[toks[i]]), rel_tol=2e-4, abs_tol=2e-4)
            assert math.isclose(e["entropy"], float(-(row.exp() * row).sum()), rel_tol=2e-3, abs_tol=2e-3)
            for a, b in zip(e["top"], row.topk(n).values.tolist()):
                assert math.isclose(a["logprob"], b, rel_tol=2e-4, abs_tol=2e-4) and math.isclose(float(row[a["token"]]), b, rel_tol=4e-4, abs_tol=4e-4)
    eng.scheduler.check_idle_invariants()


def test_logprobs_refused():
    eng = make_engine()
    from mini_sglang_b200 import SamplingParams
    for bad in (-1, 33):
        with pytest.raises(ValueError, match="logprobs"):
            eng.generate(input_ids=[1, 2], sampling_params={"logprobs": bad})
        with pytest.raises(ValueError, match="logprobs"):
            eng.generate(input_ids=[1, 2], sampling_params=SamplingParams(logprobs=bad))


def pokatar_runner(layers, tmp, **kw):
    from mini_sglang_b200.engine.step import ModelRunner
    from tiny_models import write_model_dir
    from tiny_pokatar import make_weights, model
    cfg = model(64, 97, 1e-5, layers)
    weights = make_weights(cfg, 8)
    write_model_dir(str(tmp), cfg, weights)
    return cfg, weights, ModelRunner.from_model_dir(str(tmp), dtype="float32", page_size=4, num_pages=200, max_reqs=4, max_context_len=256, **kw)


def test_verify_over_caches_whose_values_lie_in_the_key_rows(tmp_path):
    """Latent attention keeps one array a cache: its rows move once.  Drafts of the plain model's own tokens beside wrong ones."""
    import plain_pokatar as pk
    from mini_sglang_b200.engine import DraftEntry
    from mini_sglang_b200.engine.step import StepEntry
    from tiny_pokatar import dense, latent, layer
    cfg, weights, runner = pokatar_runner([layer(latent(3, 24, 16, 20, 40, base=500.0), dense(56)), layer(latent(2, 64, 32, 64, 96), None)], tmp_path)
    assert runner.drafts_supported()
    smp, rng, prompt = sampler(runner), random.Random(2), random_tokens(21, 97, 5)
    slot = runner.open()
    want = decode(runner, slot, prompt, 40, smp, 0.0, 0)
    runner.close(slot)
    slot = runner.open()
    got = [int(smp.sample(runner.step([StepEntry(slot, prompt, [20])]), [0.0], [0], [0])[0])]
    rounds = 0
    while len(got) < 30:
        toks, up = guess(rng, want[len(got) - 1:], 12, 97)
        got.extend(runner.verify([DraftEntry(slot, toks, up)], smp)[0])
        rounds += 1
    assert got[:30] == want[:30] and rounds < 20
    row = runner.step([StepEntry(slot, [got[-1]], [0])]).float().cpu()[0]
    ref = pk.forward_sequence(cfg, weights, prompt + got, dtype=torch.float64).float()[-1]
    torch.testing.assert_close(row, ref, rtol=1e-4, atol=5e-5)
    runner.close(slot)


def test_attention_with_a_further_term_is_refused(tmp_path):
    from mini_sglang_b200.engine import DraftEntry
    from tiny_pokatar import att, dense, layer
    _, _, runner = pokatar_runner([layer(att(4, 2, 32, 32), dense(56))], tmp_path)
    assert not runner.drafts_supported()
    with pytest.raises(ValueError, match="all keys"):
        runner.verify([DraftEntry(runner.open(), [1, 2])], sampler(runner))


def test_verify_wants_one_value_an_entry():
    from mini_sglang_b200.engine import DraftEntry
    runner = make_runner("B", "float32", num_pages=8)
    slot = runner.open()
    for kw in ({"temperatures": [0.0, 0.0]}, {"row_keys": []}, {"steps": [1, 2]}):
        with pytest.raises(ValueError, match="one value an entry"):
            runner.verify([DraftEntry(slot, [1, 2])], sampler(runner), **kw)
    assert int(runner.mgr.reserved[slot]) == 0
