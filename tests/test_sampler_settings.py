"""What a sampler refuses when it is made: a repetition that the operator divides by."""
import math

import pytest
import torch

from dynakv_amd.model import Sampler


@pytest.mark.parametrize("bad", [0.0, -1.0, math.nan, math.inf, torch.tensor([1.1, 0.0]),
                                 torch.tensor([-2.0, 1.0]), torch.tensor([math.nan, 1.0]),
                                 torch.tensor([1.0, math.inf])])
def test_repetition_must_be_positive(bad):
    with pytest.raises(ValueError, match="repetition must be positive and finite"):
        Sampler(device="cpu", repetition=bad)


def test_repetition_that_may_be():
    for good in (0.5, 1e-30, 3e38, torch.tensor([1.0, 0.7]), torch.empty(0)):
        assert "repetition" in Sampler(device="cpu", repetition=good).penalties
