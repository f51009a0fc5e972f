"""The accuracy check itself: it passes what is within, and fails on NaN, inf and anything off."""

import math

import pytest
import torch

from strict import assert_within


def test_passes_what_is_within():
    want = torch.linspace(-3, 3, 60, dtype=torch.float64).view(4, 15)
    assert_within(want.float(), want, 2.0 ** -24 * want.abs())
    assert_within(want + 0.5, want, torch.tensor(0.5))
    assert_within(torch.empty(0, 3), torch.empty(0, 3, dtype=torch.float64), torch.tensor(0.0))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 1.001])
@pytest.mark.parametrize("where", [(0, 0), (3, 14)])
def test_fails_on_one_wrong_element(bad, where):
    want = torch.zeros((4, 15), dtype=torch.float64)
    got = want.clone()
    got[where] = bad
    with pytest.raises(AssertionError, match="1 of 60"):
        assert_within(got, want, torch.ones(4, 15))


def test_fails_where_the_value_or_the_room_is_no_number():
    want = torch.zeros(3, dtype=torch.float64)
    nan = torch.tensor([0, math.nan, 0], dtype=torch.float64)
    for args in ((want, nan, torch.ones(3)), (want, want, nan), (nan, nan, torch.ones(3))):
        with pytest.raises(AssertionError):
            assert_within(*args)
    with pytest.raises(AssertionError):
        assert_within(torch.full((3,), math.inf), torch.full((3,), math.inf), torch.ones(3))
    with pytest.raises(AssertionError):
        assert_within(want[:2], want, torch.ones(3))
