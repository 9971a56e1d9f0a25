"""iadmm.optim.AdamW as a program handles it around its steps: copied, pickled, regrouped, clipped inside a window."""
import copy
import pickle

import pytest
import torch

import iadmm_path  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def params(seed=0, dtype=torch.float32, shapes=((40, 40), (40,), (2, 40), (1,), (100, 1))):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((0.1 * torch.randn(*s, generator=g)).to(dtype).cuda()) for s in shapes]


def set_grads(ps, seed, scale=1.0):
    g = torch.Generator().manual_seed(1000 + seed)
    for p in ps:
        p.grad = (scale * torch.randn(*p.shape, generator=g)).to(p.dtype).cuda()


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_a_copy_goes_on_as_its_original(copied, bits, capturable):
    """The same bits: a copy has the same state, settings and counts."""
    from iadmm.optim import AdamW
    a = params()
    opt = AdamW([dict(params=a[:2]), dict(params=a[2:], lr=3e-3)], lr=1e-2, state_bits=bits, seed=5, max_norm=1.0,
                capturable=capturable)
    for t in range(3):
        set_grads(a, t)
        opt.step()
    other = copied(opt)
    b = [p for g in other.param_groups for p in g["params"]]
    assert all(p is not q and torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(opt.norm, other.norm)
    for t in range(3, 5):
        for ps, o in ((a, opt), (b, other)):
            set_grads(ps, t)
            o.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    for p, q in zip(a, b):
        assert int(opt.state[p]["step"]) == int(other.state[q]["step"]) == 5
        assert all(torch.equal(x, y) for x, y in zip(opt.moments(p), other.moments(q)))
