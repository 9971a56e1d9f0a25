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


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_inside_a_training_window(bits):
    """tbptt_batch's steps with a max_norm of half the gradients' norm: parameters and moments have the bits of an optimizer
    without it that is given the gradients times the clipping factor, and no parameter moves by more than lr |m| / sqrt(v),
    corrected: 1 at the first step; at the second m weighs the two gradients by (0.4737, 0.5263) and v their squares by
    (0.49975, 0.50025), so at most sqrt(0.4737^2 / 0.49975 + 0.5263^2 / 0.50025) = 1.0014, with 24 roundings in all."""
    from models.lstm import LSTM
    from iadmm import data, ops, train
    from iadmm.optim import AdamW

    class Recorded(AdamW):
        def step(self, closure=None):
            ps = [p for g in self.param_groups for p in g["params"]]
            grads = [None if p.grad is None else p.grad.clone() for p in ps]
            out = super().step(closure)
            self.seen.append((grads, self.norm.clone(), [p.detach().clone() for p in ps],
                              [[m.clone() for m in self.moments(p)] for p in ps]))
            return out

    raw = data.make_qp_batch(40, 14, 6, 4, first_index=2, device="cuda")
    d = dict(zip(("Q", "p", "A0", "zl", "zu"), ops.ruiz_scale(raw["Q"], raw["p"], raw["A0"], raw["zl"], raw["zu"], 10)[:5]))
    T, lr = 6, 1e-3

    def run(max_norm):
        torch.manual_seed(3)
        model = LSTM(20, 2, 48, T, "cuda", layer_norm=True)
        start = [p.detach().clone() for p in model.parameters()]
        opt = Recorded(model.parameters(), lr=lr, weight_decay=0.0, state_bits=bits, max_norm=max_norm, seed=9)
        opt.seen = []
        train.tbptt_batch(model, d, 14, 6, 2 * T, T, 6e-6, opt, micro_batch=2)
        return start, opt.seen

    _, free = run(1e9)
    most = 0.5 * min(float(norm) for _, norm, _, _ in free)
    start, seen = run(most)
    assert len(seen) == len(free) == 2
    own = [torch.nn.Parameter(p.clone()) for p in start]
    plain = AdamW(own, lr=lr, weight_decay=0.0, state_bits=bits, seed=9)
    before = start
    for k, (grads, norm, after, moments) in enumerate(seen):
        assert float(norm) > 1.5 * most
        factor = torch.tensor(most, device="cuda") / (norm + 1e-6)
        for p, g in zip(own, grads):
            p.grad = None if g is None else g * factor
        plain.step()
        assert sum(g is not None for g in grads) >= 18
        for p, old, new, ms in zip(own, before, after, moments):
            assert torch.equal(p, new) and all(torch.equal(a, b) for a, b in zip(plain.moments(p), ms)), k
            if bits == 32:
                assert bool(((new - old).abs() <= (1.0 if k == 0 else 1.0014) * lr * (1 + 24 * 2.0 ** -24) + 2.0 ** -23 * old.abs()).all())
        before = after


def test_a_captured_step_counts_on_after_the_counts_were_gathered_again():
    """Groups that changed places and a shallow copy's steps between the replays: the replays use and raise the parameters' own
    counts, in the memory that they were captured with."""
    from iadmm.optim import AdamW
    a, b = params(), params()
    groups = lambda ps: [dict(params=ps[:2]), dict(params=ps[2:], lr=3e-3)]  # noqa: E731
    mine = AdamW(groups(a), lr=1e-2, betas=(0.5, 0.75), capturable=True)
    host = AdamW(groups(b), lr=1e-2, betas=(0.5, 0.75))
    set_grads(a[2:], 0)  # the groups' counts are apart
    set_grads(b[2:], 0)
    mine.step()
    host.step()

    def both(t, step):
        set_grads(b, t)
        for p, q in zip(a, b):
            p.grad.copy_(q.grad)
        step()
        host.step()

    set_grads(a, 1)
    both(1, mine.step)
    where = [mine.state[p]["step"].data_ptr() for p in a]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mine.step()
    shallow = copy.copy(mine)
    for t, step in enumerate((graph.replay, shallow.step, mine.step, graph.replay, mine.step, graph.replay), 2):
        if t == 6:
            mine.param_groups.reverse()
        both(t, step)
        torch.cuda.synchronize()
        for p, q in zip(a, b):  # (counts of the two kinds: corrections rounded apart, 2 u of an update)
            assert bool(((p - q).abs() <= (t + 1) * 2.0 ** -24 * (4 * p.abs() + 24 * 2e-2)).all()), t
    assert [int(mine.state[p]["step"]) for p in a] == [host.state[p]["step"] for p in b] == [7, 7, 8, 8, 8]
    assert [mine.state[p]["step"].data_ptr() for p in a] == where
