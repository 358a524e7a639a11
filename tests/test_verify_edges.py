"""Verification of drafts at the ends of float32's range; the tolerance is the one that test_shared_prefix.py derives."""
import pytest
import torch

from test_shared_prefix import check_verify, verify, verify_case

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("heat", [1e-45, 1e-40, 1e-39, 2.9e-39, 1.2e-38, 1e-30, 1e-6, 1e6, 3e38, 1e39, 1e300])
@pytest.mark.parametrize("probs", [False, True])
def test_temperatures_at_the_ends_of_float32(heat, probs):
    """Next to nothing, where one over the temperature is no number of float32 any more, and next to no difference between tokens."""
    c = verify_case(21, 3000, [3, 0, 2, 4], 0.5, probs)
    c["heat"] = heat
    check_verify(c)
    assert not torch.isnan(verify(c)[2]).any()
