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


def test_counts_follow_the_parameters_not_their_place():
    """Counts on the device after the groups changed places, and beside a shallow copy that steps the same parameters:
    the same bits as an optimizer that counts on the host, whose counts are the parameters' own."""
    from iadmm.optim import AdamW
    ends = []
    for capturable in (False, True):
        a = params()
        opt = AdamW([dict(params=a[:1]), dict(params=a[1:2])], lr=1e-2, betas=(0.5, 0.75), capturable=capturable)
        set_grads(a[:1], 0)
        opt.step()
        for t in range(1, 6):
            set_grads(a[:2], t)
            opt.step()
            if t == 2:
                opt.param_groups.reverse()
            if t == 3:
                shallow = copy.copy(opt)
                shallow.step()
        assert [int(opt.state[p]["step"]) for p in a[:2]] == [7, 6]
        ends.append([p.detach().clone() for p in a[:2]])
    for p, q in zip(*ends):  # (the corrections of the two kinds of counts are rounded apart: 2 u of an update, 7 updates)
        assert bool(((p - q).abs() <= 7 * 2.0 ** -24 * (4 * p.abs() + 24 * 2e-2)).all())


def test_gradients_that_are_negated_views():
    from iadmm.optim import AdamW
    a, b = params(), params()
    set_grads(a, 0)
    for p, q in zip(a, b):
        q.grad = torch._neg_view(-p.grad)
    one, two = AdamW(a, max_norm=1.0), AdamW(b, max_norm=1.0)
    one.step()
    two.step()
    assert torch.equal(one.norm, two.norm) and all(torch.equal(p, q) for p, q in zip(a, b))


def test_numbers_on_the_device_that_lie_in_what_is_written_are_refused():
    """norm, lr and the steps' counts: every workgroup reads the first two while others write, and writes the third once."""
    from iadmm import ops
    buf = torch.rand(1000, device="cuda") + 0.5
    keep = buf.clone()
    p, g, m, v = buf[:300], torch.randn(300, device="cuda"), buf[300:600], buf[600:900]
    counts = torch.zeros(1, dtype=torch.int64, device="cuda")
    inside = buf[298:300].view(torch.int64)
    for kw in (dict(step=1, norm=p[7], max_norm=1.0), dict(step=1, norm=m[299], max_norm=1.0), dict(step=counts, lr=v[:1]),
               dict(step=inside), dict(step=counts, lr=counts.view(torch.float32)[1:]),
               dict(step=counts, norm=counts.view(torch.float32)[0], max_norm=1.0)):
        with pytest.raises(ValueError, match="overlaps"):
            ops.adamw_step([p], [g], [m], [v], **kw)
    torch.cuda.synchronize()
    assert torch.equal(buf, keep) and int(counts) == 0
    ops.adamw_step([p], [g], [m], [v], counts, lr=buf[900:901], norm=g[5].abs(), max_norm=1.0)  # side by side
    ops.adamw_step([p], [g], [m], [v], 2, norm=g[5:6], max_norm=1.0)                            # a gradient is only read
    assert int(counts) == 1 and torch.equal(buf[900:], keep[900:]) and not torch.equal(p, keep[:300])
