"""Values of the right range and the wrong kind, without a GPU: refused where a user gives them, not inside a step that other requests share."""
import numpy as np
import pytest
import torch

from mini_sglang_b200 import SamplingParams, ops


@pytest.mark.parametrize("n", [2.5, 5.0, float("nan"), True, False, "5", [5], torch.tensor(2.0)])
def test_logprobs_is_a_whole_number(n):
    with pytest.raises(ValueError, match="logprobs"):
        SamplingParams.init_from_dict({"logprobs": n})
    with pytest.raises(ValueError, match="logprobs"):
        SamplingParams(logprobs=n).check_logprobs()


@pytest.mark.parametrize("n", [0, 5, 32, np.int64(7)])
def test_whole_numbers_are_taken(n):
    assert SamplingParams.init_from_dict({"logprobs": n}).logprobs == n


@pytest.mark.parametrize("top", [2.5, 2.0, True, "2", None])
def test_top_is_a_whole_number(top):
    with pytest.raises(ops.KernelError, match="top"):
        ops.token_logprobs(torch.zeros(3, 50), torch.zeros(3, dtype=torch.int32), top)


def test_whole_numbers_of_numpy_are_taken_as_top():
    with pytest.raises(ops.KernelError, match="CUDA device"):          # (nothing but the device is wrong)
        ops.token_logprobs(torch.zeros(3, 50), torch.zeros(3, dtype=torch.int32), np.int64(3))
