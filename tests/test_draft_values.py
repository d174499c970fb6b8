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


def test_tables_whose_rows_lie_beyond_32_bits_are_refused():
    """The kernels take the distance of a table's rows as 32 bits: a longer one would be cut and other rows read."""
    I = lambda *s: torch.zeros(s, dtype=torch.int32)      # noqa: E731, E741
    far = torch.empty_strided((2, 3), (2 ** 31, 1), dtype=torch.int32, device="meta")
    with pytest.raises(ops.KernelError, match="block_table"):
        ops.draft_plan(I(4), I(2), I(2), far, page_size=16, max_draft=4)
    cache = torch.zeros(5, 2, 16, 16)
    with pytest.raises(ops.KernelError, match="block_table"):
        ops.draft_accept(I(4), I(4), I(4), I(3), max_draft=4, kv_len=I(2), block_table=far, caches=[cache])
    q = torch.zeros(4, 8, 16)
    with pytest.raises(ops.KernelError, match="block_table"):
        ops.tree_attention(q, q, cache, cache, q_start=I(3), kv_len=I(2), block_table=far, mask=I(4, 1), n_kv=2, page_size=16, scale=1.0, max_draft=4)


def test_accept_takes_no_more_columns_than_its_counter_has_room_for():
    """A block's threads step over the columns of all caches with a 32-bit counter: sizes where it would pass its end are refused before a launch."""
    import ctypes
    lib = ops._draft_lib()
    there = torch.zeros(64, dtype=torch.uint8)

    def call(n_caches, row_bytes):
        addresses = (ctypes.c_void_p * n_caches)(*[there.data_ptr() // 16 * 16 + 2] * n_caches)          # (2 bytes a column)
        return lib.msgl_draft_accept(None, None, None, None, 0 if n_caches == 1 else 1, 0, 4, None, None, None, there.data_ptr(), there.data_ptr(), 1, 1, 16, 1, 1, row_bytes,
                                     addresses, n_caches, 1, None)
    assert call(1, 64) == 0                              # (no request: nothing to do)
    assert call(2, 2 ** 31 - 256) == 2                   # (2^31 - 256 columns, and a block steps by 256)
