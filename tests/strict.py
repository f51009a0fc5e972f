"""The check that the accuracy tests share: every element a number, and within its own room."""

import torch


def assert_within(got, want, room, what=""):
    """|got - want| <= room everywhere.  Stated positively: a NaN in any of the three fails."""
    assert got.shape == want.shape
    off = (got.double() - want.double()).abs()
    ok = off <= room
    if not bool(ok.all()):
        bad = (~ok).nonzero()
        first = tuple(bad[0].tolist())
        raise AssertionError(f"{what}: {len(bad)} of {ok.numel()} elements off, the first at {first}: "
                             f"{got[first].item()} for {want[first].item()}")
    assert torch.isfinite(got).all(), what
