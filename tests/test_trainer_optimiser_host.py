"""Numbers of the configuration that the named optimiser would not look at are refused, not passed by."""
import pytest
import torch

from conftest import pkg_module


@pytest.mark.parametrize("numbers", [{"weight_decay": 0.01}, {"state_bits": 8}, {"weight_decay": 0.01, "state_bits": 8}])
def test_adam_refuses_the_other_optimisers_numbers(numbers):
    tr = pkg_module("trainer")
    params = [torch.zeros(3, requires_grad=True)]
    with pytest.raises(ValueError):
        tr.make_optimizer(params, 1e-3, tr.PPOConfig(**numbers))
    assert isinstance(tr.make_optimizer(params, 1e-3, tr.PPOConfig(weight_decay=0.0, state_bits=32)), torch.optim.Adam)
