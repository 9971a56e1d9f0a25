"""autograd.layer_norm as part of a program: views that torch negates on reading, checkpoints, hooks on saved tensors,
transforms that it refuses, captured graphs, long columns."""
import pytest
import torch

import iadmm_path  # noqa: F401

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def inputs(rows, cols, t=F32, seed=0):
    """x, dy, weight, bias; the first and the last two leaves."""
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 1009 + cols)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, dy = ((r(rows, cols) + 0.3).to(t).cuda() for _ in range(2))
    w, b = (1 + 0.3 * r(cols)).cuda(), (0.2 * r(cols)).cuda()
    return x.requires_grad_(), dy, w.requires_grad_(), b.requires_grad_()


def gradients(x, w, b, dy, run=None):
    from iadmm import autograd
    y = (run or autograd.layer_norm)(x, w, b)
    return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]


def same(got, want):
    return all(torch.equal(a, c) for a, c in zip(got, want))


def test_negated_views():
    """As an input and as the gradient that arrives: the bits of their negated copies."""
    from iadmm import autograd
    x, dy, w, b = inputs(9, 65)
    want = gradients((-x).detach().requires_grad_(), w, b, -dy)
    y = autograd.layer_norm(torch._neg_view(x), w, b)
    got = torch.autograd.grad(y, (x, w, b), torch._neg_view(dy), retain_graph=True)
    assert torch.equal(y, want[0]) and torch.equal(got[0], -want[1]) and same(got[1:], want[2:])
    y.register_hook(lambda g: torch._neg_view(g))
    assert same(torch.autograd.grad(y, (x, w, b), dy), got)


def test_captured_backward_pass():
    """Replays, with eager passes over leaves of their own between them, give the eager bits.  A capture beside a graph of
    the same leaves that is still alive is refused, and leaves that graph usable."""
    from iadmm import autograd
    x, dy, w, b = inputs(333, 800)
    leaves = (x, w, b)

    def captured():
        for t in leaves:
            t.grad = None
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = autograd.layer_norm(x, w, b)
            y.backward(dy)
        return g, y.detach()

    alive = autograd.layer_norm(x, w, b)
    for t in leaves:
        t.grad = None
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="still alive"):
            autograd.layer_norm(x, w, b).backward(dy)
        with pytest.raises(RuntimeError, match="still alive"):
            torch.autograd.grad(autograd.layer_norm(x, w, b), (w,), dy)
    assert all(t.grad is None for t in leaves)
    assert same(torch.autograd.grad(alive, leaves, dy), gradients(x, w, b, dy)[1:])
    del alive
    torch.cuda.synchronize()
    graph, y = captured()
    grads = [t.grad for t in leaves]
    for k in range(4):
        x2, dy2, w2, b2 = inputs(333, 800, seed=k + 1)
        with torch.no_grad():
            for t, s in ((x, x2), (dy, dy2), (w, w2), (b, b2)):
                t.copy_(s)
        want = gradients(x2, w2, b2, dy2)
        graph.replay()
        torch.cuda.synchronize()
        assert same([y, *grads], want), k


@pytest.mark.parametrize("t", [F32, BF16])
def test_many_long_rows(t):
    """A column of a few thousand rows has at most 48 + rows / 32 roundings of u = 2^-24 in its sums also where a row is so long that
    only two workgroups share a column.  dy repeats one number in each column, chosen so that a chain in fp32 rounds
    the same way each time: half a thousand times by 0.45 of a last place in the sum's last binade (208 roundings in all);
    in bf16 it is exact."""
    from iadmm import ops
    rows, cols = 2048, 524291 if t == F32 else 2 * 524291
    value = 1 + 0.9 * 2.0 ** -15 if t == F32 else 1 + 2.0 ** -7
    x = torch.empty(rows, cols, dtype=t, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(3))
    dy = torch.full((rows, cols), value, dtype=t, device="cuda")
    _, mean, rstd = ops.layer_norm(x, stats=True)
    _, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, need=(False, True, True))
    u, roundings = 2.0 ** -24, 48 + rows / 32
    want = rows * float(dy[0, 0])
    assert float((db.double() - want).abs().max()) <= (roundings + 1) * u * want
    for c in range(0, cols, 65536):
        part = slice(c, min(c + 65536, cols))
        terms = (x[:, part].double() - mean.double()[:, None]) * rstd.double()[:, None] * float(dy[0, 0])
        off = (dw[part].double() - terms.sum(0)).abs()
        assert bool((off <= roundings * u * terms.abs().sum(0) + u * terms.sum(0).abs()).all()), c


@pytest.mark.parametrize("t", [F32, F16])
def test_checkpoints_and_hooks_on_saved_tensors(t):
    """What is saved may be made again or lie elsewhere until the backward pass: the same bits."""
    from torch.utils.checkpoint import checkpoint
    from iadmm import autograd
    x, dy, w, b = inputs(70, 801, t)
    want = gradients(x, w, b, dy)
    for reentrant in (False, True):
        for p in (x, w, b):
            p.grad = None
        y = checkpoint(autograd.layer_norm, x, w, b, use_reentrant=reentrant)
        y.backward(dy)
        assert same([y.detach(), x.grad, w.grad, b.grad], want)
    with torch.autograd.graph.save_on_cpu():
        y = autograd.layer_norm(x, w, b)
    assert same(torch.autograd.grad(y, (x, w, b), dy), want[1:])
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda s: seen.append(s) or s.clone(), lambda s: s):
        y = autograd.layer_norm(x, w, b)
    assert same(torch.autograd.grad(y, (x, w, b), dy), want[1:]) and len(seen) == 4


def test_transforms_are_refused():
    """Batched, functional and forward-mode tensors: an error, nothing computed.  A compiled caller runs the call as it is."""
    import torch.autograd.forward_ad as forward_ad
    from iadmm import autograd, ops
    x, dy, w, b = inputs(6, 40)
    d = x.detach()
    for call in (lambda: torch.func.vmap(lambda r: autograd.layer_norm(r))(d.view(2, 3, 40)),
                 lambda: torch.func.vmap(lambda r: ops.layer_norm(r))(d.view(2, 3, 40)),
                 lambda: torch.func.vmap(lambda v: ops.layer_norm(d, v))(w.detach().expand(3, 40).contiguous()),
                 lambda: torch.func.grad(lambda s: autograd.layer_norm(s, w, b).sum())(d),
                 lambda: torch.func.jvp(lambda s: autograd.layer_norm(s), (d,), (d,)),
                 lambda: torch.autograd.functional.jacobian(autograd.layer_norm, d, vectorize=True)):
        with pytest.raises(RuntimeError):
            call()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            autograd.layer_norm(forward_ad.make_dual(d, dy), w, b)
    y = torch.compile(lambda s: autograd.layer_norm(s + 0, w, b) + 0, backend="eager")(x)
    assert same([y.detach(), *torch.autograd.grad(y, (x, w, b), dy)], gradients(x, w, b, dy))


def test_tensors_without_memory_are_refused():
    """A fake tensor says that it is on the device and has no address: none may stand for an operand that is left out."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from iadmm import _abi, autograd, ops
    x, dy, w, b = (p.detach() for p in inputs(6, 40))
    mode = FakeTensorMode()
    fx, fw, one = mode.from_tensor(x), mode.from_tensor(w), mode.from_tensor(w[:1].clone())
    _, mean, rstd = ops.layer_norm(x, stats=True)
    m, v = torch.zeros_like(x), torch.zeros_like(x)
    keep = x.clone()
    counts = torch.zeros(1, dtype=torch.int64, device="cuda")
    for call in (lambda: ops.layer_norm(fx), lambda: ops.layer_norm(x, fw), lambda: ops.layer_norm(x, w, fw), lambda: autograd.layer_norm(x, fw),
                 lambda: ops.layer_norm_bwd(dy, x, mean, rstd, fw), lambda: ops.layer_norm_bwd(fx, x, mean, rstd),
                 lambda: ops.grad_norm([fx]), lambda: ops.adamw_step([x], [fx], [m], [v], 1),
                 lambda: ops.adamw_step([x], [dy], [m], [v], 1, norm=one, max_norm=1.0),
                 lambda: ops.adamw_step([x], [dy], [m], [v], counts, lr=one)):
        with pytest.raises((RuntimeError, ValueError, _abi.IadmmError)):
            call()
    torch.cuda.synchronize()
    assert torch.equal(x, keep) and int(counts) == 0


def test_graphed_callable():
    """torch.cuda.make_graphed_callables: forward and backward captured apart; a training loop's bits are the eager ones."""
    from iadmm import autograd

    class Norm(torch.nn.Module):
        def __init__(self, w, b):
            super().__init__()
            self.w, self.b = (torch.nn.Parameter(p.detach().clone()) for p in (w, b))

        def forward(self, x):
            return autograd.layer_norm(x, self.w, self.b)

    x, dy, w, b = inputs(333, 800)
    plain, graphed = Norm(w, b), Norm(w, b)
    call = torch.cuda.make_graphed_callables(graphed, (torch.zeros_like(x).requires_grad_(),))
    for k in range(4):
        x, dy, _, _ = inputs(333, 800, seed=k)
        ends = []
        for f, m in ((plain, plain), (call, graphed)):
            for p in (x, m.w, m.b):
                p.grad = None
            y = f(x)
            y.backward(dy)
            ends.append([t.clone() for t in (y.detach(), x.grad, m.w.grad, m.b.grad)])
            with torch.no_grad():
                m.w -= 0.01 * m.w.grad
        assert same(*ends), k
