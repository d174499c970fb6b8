"""Places of drafts on pages that a table does not have: slot 0, the page for padding, never a slot in front of the caches."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page", [1, 3, 16])
def test_page_numbers_that_are_none(page):
    from mini_sglang_b200 import ops
    far = 2 ** 31 - 1
    table = [[4, -1, 7, -2 ** 31, far, 2]]
    n = 6 * page
    plan = ops.draft_plan(i32([-1] + list(range(n - 1))), i32([n]), i32([0]), i32(table), page_size=page, max_draft=n)
    want = [t * page + i if t >= 0 and t * page + i < 2 ** 31 else 0 for t in table[0] for i in range(page)]
    assert plan.out_loc.tolist() == want and plan.positions.tolist() == list(range(n))
