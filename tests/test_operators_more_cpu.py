"""Refusals of the layer norm's wrappers that need no GPU."""
import pytest
import torch

import iadmm_path  # noqa: F401
from iadmm import ops


def test_arguments_of_the_gradients():
    x, m = torch.zeros(3, 8), torch.zeros(3)
    for wdtype in (torch.float64, torch.int8, "float32"):
        with pytest.raises(TypeError, match="wdtype"):
            ops.layer_norm_bwd(x, x, m, m, wdtype=wdtype)
    for need in ((), (True,), (True, True, True, True)):
        with pytest.raises(ValueError, match="need"):
            ops.layer_norm_bwd(x, x, m, m, need=need)
