"""The comparison that the tests of the row operators go by refuses what is not a number."""
import pytest
import torch

import indexed_util as iu


def test_check_passes_what_lies_within_the_bound():
    exact = torch.tensor([[1.0, -2.0, 0.0]], dtype=torch.float64)
    iu.check(exact.float(), exact, torch.zeros_like(exact))
    iu.check(exact.bfloat16(), exact, exact.abs() * iu.U32)
    with pytest.raises(AssertionError, match="1 of 3 values"):
        iu.check(torch.tensor([[1.0, -2.0, 1e-6]]), exact, torch.zeros_like(exact))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", iu.FLOATS)
def test_check_rejects_results_that_are_not_finite(value, dtype):
    exact = torch.ones(2, 3, dtype=torch.float64)
    got = torch.ones(2, 3, dtype=dtype)
    got[1, 2] = value
    with pytest.raises(AssertionError, match="first at .1, 2."):
        iu.check(got, exact, torch.zeros_like(exact))


def test_check_refuses_a_definition_or_a_bound_that_is_not_finite():
    one = torch.ones(1, 1, dtype=torch.float64)
    for exact, before in ((one * float("nan"), one), (one * float("inf"), one), (one, one * float("inf"))):
        with pytest.raises(AssertionError, match="finite"):
            iu.check(one.float(), exact, before)
