"""iadmm.optim.AdamW and the command line around it without a GPU."""
import copy
import pickle

import pytest
import torch

import iadmm_path  # noqa: F401
from iadmm.optim import AdamW

SETTINGS = dict(lr=0.5, betas=(0.8, 0.95), eps=1e-4, weight_decay=0.2, state_bits=8, max_norm=3.0, seed=11, capturable=True)


def parameter(*shape):
    return torch.nn.Parameter(torch.zeros(*shape or (3,)))


@pytest.mark.parametrize("copied", [copy.copy, copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_a_copied_optimizer_has_its_settings_and_steps(copied):
    opt = AdamW([parameter()], **SETTINGS)
    other = copied(opt)
    for k in ("state_bits", "max_norm", "seed", "capturable", "norm"):
        assert getattr(other, k) == getattr(opt, k), k
    assert all(other.defaults[k] == v for k, v in opt.defaults.items())
    assert other.step(lambda: 7.0) == 7.0  # no gradient: nothing to do
    other.param_groups[0]["params"][0].grad = torch.ones(3)
    with pytest.raises(ValueError, match="no CPU fallback"):
        other.step()
