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


def test_a_trace_does_not_take_results_for_constants():
    """The refusal comes before the tensors are looked at (here: that they are on no GPU)."""
    from iadmm import autograd
    x, m = torch.ones(3, 8), torch.ones(3)
    for f in (ops.layer_norm, autograd.layer_norm, lambda s: ops.layer_norm_bwd(s, s, m, m)[0], lambda s: ops.grad_norm([s]),
              lambda s: ops.adamw_step([s], [s], [s], [s], 1)):
        with pytest.raises(RuntimeError, match="cannot record"):
            torch.jit.trace(f, (x,))
