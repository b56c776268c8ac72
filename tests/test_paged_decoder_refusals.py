"""What PagedDecoder refuses before it touches a device."""
import pytest
import torch

from bitstack_b200.serving import PagedDecoder


@pytest.mark.parametrize("steps", [0, -1])
def test_generate_makes_at_least_one_token(steps):
    d = PagedDecoder.__new__(PagedDecoder)             # refused before the decoder is looked at
    with pytest.raises(ValueError, match="at least 1"):
        d.generate([torch.tensor([1, 2])], steps=steps)
