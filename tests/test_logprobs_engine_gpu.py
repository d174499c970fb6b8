"""Log probabilities through the Engine where a request's way is not the plain one: none of the alternatives asked for, streamed, beside a request that is
refused, taken back and computed again."""
import math

import numpy as np
import pytest
import torch

from helpers import plain_logits
from test_drafts_engine_gpu import make_engine
from tiny_models import CONFIGS, random_tokens

pytestmark = pytest.mark.gpu
V = CONFIGS["B"]["vocab_size"]


def check(prompt, out, n):
    toks = out["token_ids"]
    lp = torch.log_softmax(plain_logits("B", prompt + toks).double(), -1)
    assert len(out["logprobs"]) == len(toks)
    for i, e in enumerate(out["logprobs"]):
        row = lp[len(prompt) - 1 + i]
        # the logits are off by up to 1e-4 of their size and 5e-5 (the float32 path's bound), a log probability by twice that
        assert e["token"] == toks[i] and len(e["top"]) == n
        assert math.isclose(e["logprob"], float(row[toks[i]]), rel_tol=2e-4, abs_tol=2e-4)
        for a, b in zip(e["top"], row.topk(n).values.tolist()):
            assert math.isclose(a["logprob"], b, rel_tol=2e-4, abs_tol=2e-4)


@pytest.mark.parametrize("overlap", [True, False])
@pytest.mark.parametrize("n", [0, 32, np.int64(3)])
def test_one_number_of_alternatives_for_all(n, overlap):
    eng = make_engine(disable_overlap=not overlap)
    prompts = [random_tokens(k, V, k) for k in (5, 12)]
    for p, o in zip(prompts, eng.generate(input_ids=prompts, sampling_params={"max_new_tokens": 6, "ignore_eos": True, "logprobs": n})):
        check(p, o, n)


def test_streamed():
    eng, prompt = make_engine(), random_tokens(9, V, 1)
    seen = 0
    for o in eng.generate(input_ids=prompt, sampling_params={"max_new_tokens": 7, "ignore_eos": True, "temperature": 0.9, "logprobs": 2}, stream=True):
        assert len(o["logprobs"]) == len(o["token_ids"]) >= seen
        seen = len(o["token_ids"])
    check(prompt, o, 2)
    assert seen == 7


def test_a_refused_request_leaves_the_others_alone():
    eng, prompt = make_engine(), random_tokens(9, V, 2)
    req = eng.add_request(input_ids=prompt, sampling_params={"max_new_tokens": 12, "ignore_eos": True, "logprobs": 1})
    for bad in (2.5, True, "3", 40):
        eng.step()
        with pytest.raises(ValueError, match="logprobs"):
            eng.add_request(input_ids=prompt, sampling_params={"logprobs": bad})
    eng._run_until([req])
    check(prompt, eng._result(req, 0.0), 1)
    eng.scheduler.check_idle_invariants()


@pytest.mark.parametrize("overlap", [True, False])
def test_requests_taken_back_and_computed_again(overlap):
    """Every generated token has its entry once, whichever step computed it."""
    prompts = [random_tokens(8 + k, V, 60 + k) for k in range(4)]
    eng = make_engine(disable_overlap=not overlap, num_pages=34, init_new_token_ratio=0.05, min_new_token_ratio_factor=0.05, disable_radix_cache=True, schedule_policy="fcfs")
    outs = eng.generate(input_ids=prompts, sampling_params={"max_new_tokens": 40, "ignore_eos": True, "logprobs": 2})
    assert eng.scheduler.stats["retractions"] > 0
    for p, o in zip(prompts, outs):
        assert len(o["token_ids"]) == 40
        check(p, o, 2)
    eng.scheduler.check_idle_invariants()
