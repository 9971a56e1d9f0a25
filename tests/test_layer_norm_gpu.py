"""Layer norm (csrc/layernorm.hip) against the formulas in 64 bits.

Tolerances, element by element, with u = 2^-24 (half a step of fp32) and e = half a step of the result's type.
A sum over a row of n has at most K = 32 + n / 256 roundings on any path (of a thread 8 + 8 elements and vectors forward,
16 elements backward, or 24 from n = 1025 on; 6 over a wave, 4 over its waves; rows above 16384 add n / 1024), so with xh = (x - mu) r, q = dy w:
  |mu error| <= K u mean|x|;  r's relative error <= (K / 2 + 8) u;  xh is off by  u (K r mean|x| + (K + 16) |xh|)
  y:   |w| times that, 3 u (|xh w| + |b|) for the last fma and product, and e |y|
  dx (mean and rstd are inputs): r u (K mean|q| + K |xh| mean|q xh| + 8 (|q| + |mean q| + |xh mean(q xh)|)) + e |dx|
  dw, db: a column's sum has at most K' = 48 + rows / 32 roundings: u K' sum|dy xh| (and sum|dy|), and e |dw|
The spacing of the type's subnormal numbers is added, for results that small."""
import pytest
import torch

import iadmm_path  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def inputs(rows, cols, t, wt, seed=0, loc=0.5):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 1009 + cols)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (r(rows, cols) * (0.2 + r(rows, 1).abs()) + loc * r(rows, 1)).to(t).cuda()
    dy = r(rows, cols).to(t).cuda()
    w, b = (1 + 0.3 * r(cols)).to(wt).cuda(), (0.2 * r(cols)).to(wt).cuda()
    return x, dy, w, b


def half_step(t):
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps


def forward64(x, w, b, eps):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    r = 1 / ((x - mu).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mu) * r
    w = torch.ones_like(x[0]) if w is None else w.double()
    b = torch.zeros_like(x[0]) if b is None else b.double()
    y = xh * w + b
    K = 32 + x.shape[-1] / 256
    off = U * (K * r * x.abs().mean(-1, keepdim=True) + (K + 16) * xh.abs())
    return y, mu, r, w.abs() * off + 3 * U * ((xh * w).abs() + b.abs())


def backward64(dy, x, mean, rstd, w):
    x, dy = x.double(), dy.double()
    mu, r = mean.double().unsqueeze(-1), rstd.double().unsqueeze(-1)
    xh = (x - mu) * r
    q = dy if w is None else dy * w.double()
    s0, s1 = q.mean(-1, keepdim=True), (q * xh).mean(-1, keepdim=True)
    dx = r * (q - s0 - xh * s1)
    K = 32 + x.shape[-1] / 256
    tol = r * U * (K * q.abs().mean(-1, keepdim=True) + K * xh.abs() * (q * xh).abs().mean(-1, keepdim=True) +
                   8 * (q.abs() + s0.abs() + (xh * s1).abs()))
    Kc = 48 + x.shape[0] / 32
    return (dx, tol), ((dy * xh).sum(0), U * Kc * (dy * xh).abs().sum(0)), (dy.sum(0), U * Kc * dy.abs().sum(0))


def close(got, want, tol, what):
    e, tiny = half_step(got.dtype)
    off = (got.double() - want).abs()
    over = off - (tol + e * want.abs() + tiny)
    assert bool((over <= 0).all()), f"{what}: off by {float(off.max()):.3g}, {float(over.max()):.3g} more than allowed"


SHAPES = [(16, 800), (17, 800), (32, 1000), (128, 40), (129, 40), (127, 3), (4, 2100), (1, 12000), (2, 12000), (1, 1), (3, 2), (5, 40), (7, 127), (1, 200), (9, 129), (4, 256), (130, 257), (65, 800), (6, 1000),
          (33, 1025), (300, 7), (1000, 64), (5, 2049), (9, 4097), (3, 9001), (3, 16384), (2, 16385), (5, 20003),
          (9, 33), (70, 129), (7, 500), (200, 513), (6, 641), (35, 769), (40, 1100), (4, 1536), (19, 1537), (33, 2048), (3, 4095),
          (600, 2500), (7, 5000), (2, 8192), (3, 8193), (2, 30001), (2, 40000), (2, 70001)]
TYPES = [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)]


@pytest.mark.parametrize("t,wt", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_gradients(rows, cols, t, wt):
    from iadmm import ops
    x, dy, w, b = inputs(rows, cols, t, wt)
    y, mean, rstd = ops.layer_norm(x, w, b, 1e-5, stats=True)
    want, mu, r, tol = forward64(x, w, b, 1e-5)
    assert y.dtype == t and mean.dtype == rstd.dtype == F32 and mean.shape == rstd.shape == (rows,)
    close(y, want, tol, "y")
    close(mean.unsqueeze(-1), mu, (32 + cols / 256) * U * x.double().abs().mean(-1, keepdim=True), "mean")
    # (r's error grows by the mean's share of the spread: (mu's error r)^2 / 2, below its first-order term here)
    close(rstd.unsqueeze(-1), r, ((32 + cols / 256) / 2 + 8) * U * r + r * (r * (32 + cols / 256) * U *
          x.double().abs().mean(-1, keepdim=True)) ** 2, "rstd")
    got = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    for name, a, (want, tol) in zip(("dx", "dw", "db"), got, backward64(dy, x, mean, rstd, w)):
        close(a, want, tol, name)
    assert got[1].dtype == got[2].dtype == wt
    plain = ops.layer_norm(x)  # neither weight nor bias
    want, _, _, tol = forward64(x, None, None, 1e-5)
    close(plain, want, tol, "y without weights")
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd)
    for name, a, (want, tol) in zip(("dx", "dw", "db"), (dx, dw, db), backward64(dy, x, mean, rstd, None)):
        close(a, want, tol, name + " without weights")
    assert dw.dtype == F32


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [7, 43, 133, 521, 1029, 2051, 5003])
@pytest.mark.parametrize("where", ["first", "last"])
def test_infinities_stay_in_their_place(t, cols, where):
    """A row's last vector overlaps its neighbour: an infinite weight or gradient in the part held twice makes the same
    infinities and NaN as the formulas, and an infinite x its own row's alone."""
    from iadmm import ops
    x, dy, w, b = inputs(5, cols, t, F32)
    at = 0 if where == "first" else cols - min(cols, 6)
    _, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    wi = w.clone()
    wi[at] = float("inf")
    got = ops.layer_norm_bwd(dy, x, mean, rstd, wi)
    want = backward64(dy, x, mean, rstd, wi)
    assert torch.equal(got[0].isnan(), want[0][0].isnan()) and torch.equal(got[0].isinf(), want[0][0].isinf())
    plain = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    assert torch.equal(got[1], plain[1]) and torch.equal(got[2], plain[2])
    y, clean = ops.layer_norm(x, wi, b), ops.layer_norm(x, w, b)
    assert bool(y[:, at].isinf().all()) and torch.equal(torch.cat((y[:, :at], y[:, at + 1:]), 1), torch.cat((clean[:, :at], clean[:, at + 1:]), 1))
    di = dy.clone()
    di[2, at] = float("inf")
    dx, dw, db = ops.layer_norm_bwd(di, x, mean, rstd, w)
    rest = [0, 1, 3, 4]
    assert torch.equal(dx[rest], plain[0][rest]) and not bool(dx[2].isfinite().any())
    others = torch.arange(cols, device="cuda") != at
    assert torch.equal(dw[others], plain[1][others]) and torch.equal(db[others], plain[2][others])
    assert bool(db[at].isinf()) and not bool(dw[at].isfinite())
    xi = x.clone()
    xi[2, at] = float("inf")
    y, mean, rstd = ops.layer_norm(xi, w, b, stats=True)
    assert torch.equal(y[rest], clean[rest]) and bool(y[2].isnan().all())


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("cols,ld,shift", [(800, 801, 1), (37, 64, 3), (1025, 1031, 5), (17000, 17001, 1)])
def test_strided_rows_at_any_address(t, cols, ld, shift):
    """Rows of a wider buffer that start at an odd element: same bits as from a contiguous copy, and nothing
    beside the result is written."""
    from iadmm import ops
    rows = 11
    x, dy, w, b = inputs(rows, cols, t, F32)
    wide = torch.full((2, rows * ld + shift), 7.0, dtype=t, device="cuda")
    xs, dys = (wide[i, shift:].view(rows, ld)[:, :cols] for i in range(2))
    xs.copy_(x)
    dys.copy_(dy)
    assert xs.data_ptr() % 16 and not xs.is_contiguous()
    y0, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    y1, mean1, rstd1 = ops.layer_norm(xs, w, b, stats=True)
    assert torch.equal(y0, y1) and torch.equal(mean, mean1) and torch.equal(rstd, rstd1)
    for a, c in zip(ops.layer_norm_bwd(dy, x, mean, rstd, w), ops.layer_norm_bwd(dys, xs, mean, rstd, w)):
        assert torch.equal(a, c)
    around = torch.full((rows * cols + 8 + shift,), 7.0, dtype=t, device="cuda")
    out = around[shift:shift + rows * cols].view(rows, cols)
    assert ops.layer_norm(x, w, b, out=out) is out
    assert torch.equal(out, y0) and bool((around[:shift] == 7).all()) and bool((around[shift + rows * cols:] == 7).all())
    again = x.clone()
    assert torch.equal(ops.layer_norm(again, w, b, out=again), y0)  # in place


@pytest.mark.parametrize("cols", [40, 800, 4097, 20003])
def test_special_rows(cols):
    """Constant rows, rows with a mean far above their spread, rows with infinity or NaN: each alone."""
    from iadmm import ops
    x, dy, w, b = inputs(9, cols, F32, F32, loc=0.0)
    clean, mean0, rstd0 = ops.layer_norm(x, w, b, stats=True)
    dx0, _, db0 = ops.layer_norm_bwd(dy, x, mean0, rstd0, w)
    x = x.clone()
    x[1] = 3.0                     # no spread: y = b, rstd = 1 / sqrt(eps)
    x[3] += 4096.0                 # mean 4096, spread about 1
    x[5, cols // 2] = float("inf")
    x[7, cols - 1] = float("nan")
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    assert torch.equal(y[1], b) and abs(float(rstd[1]) * 1e-5 ** 0.5 - 1) < 1e-6
    want, _, r, tol = forward64(x[3:4], w, b, 1e-5)
    tol = tol + w.double().abs() * (r * (32 + cols / 256) * U * 4097) ** 2 * (x[3].double() - 4096).abs() * r
    close(y[3:4], want, tol, "row with a far mean")
    assert bool(torch.isnan(y[5]).all()) and bool(torch.isnan(y[7]).all())
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    for k in (0, 2, 4, 6, 8):
        assert torch.equal(y[k], clean[k]) and torch.equal(dx[k], dx0[k])
    assert bool(torch.isfinite(dx[1]).all())
    assert bool(torch.isnan(dx[7]).all()) and bool(torch.isnan(dw).all()) and torch.equal(db, db0)


def test_no_rows_and_refusals():
    from iadmm import _abi, ops
    x = torch.zeros(0, 33, device="cuda")
    y, mean, rstd = ops.layer_norm(x, stats=True)
    assert y.shape == (0, 33) and mean.shape == (0,)
    dx, dw, db = ops.layer_norm_bwd(x, x, mean, rstd)
    assert dx.shape == (0, 33) and bool((dw == 0).all()) and bool((db == 0).all())
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    bad = [dict(x=x.double()), dict(x=x.t()), dict(x=x[:, :0]), dict(x=torch.zeros((), device="cuda")), dict(x=x, weight=w[:7]),
           dict(x=x, weight=w.half()), dict(x=x, weight=w.cpu()), dict(x=x.half(), weight=w, bias=w.half()),
           dict(x=x, eps=-1.0), dict(x=x, eps=float("nan")), dict(x=x, out=x.half()), dict(x=x, out=x[:2]),
           dict(x=x[:1].expand(4, 8)), dict(x=x.cpu()), dict(x=x[:3], out=x[1:]), dict(x=x[:1], weight=w, out=w.view(1, 8)),
           dict(x=torch.zeros(4, 9, device="cuda")[:, :8], out=torch.zeros(4, 9, device="cuda").view(-1)[:32].view(8, 4))]
    wide = torch.zeros(4, 9, device="cuda")
    bad.append(dict(x=wide[:, :8], out=wide.view(-1)[:32].view(4, 8)))
    for kw in bad:
        with pytest.raises((TypeError, ValueError, _abi.IadmmError)):
            ops.layer_norm(**kw)
    m = torch.zeros(4, device="cuda")
    for args in [(x, x.half(), m, m), (x[:3], x, m, m), (x, x, m[:3], m), (x, x, m, m.double()), (x, x, m, m, w[:7])]:
        with pytest.raises((TypeError, ValueError)):
            ops.layer_norm_bwd(*args)


def test_same_bits_again_and_for_any_batch():
    """Fixed order: a call repeated gives the same bits, and a row's result does not depend on the others."""
    from iadmm import ops
    for cols in (40, 800, 2000, 9000):
        x, dy, w, b = inputs(700, cols, F32, F32)
        y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
        first = ops.layer_norm_bwd(dy, x, mean, rstd, w)
        for a, c in zip(first, ops.layer_norm_bwd(dy, x, mean, rstd, w)):
            assert torch.equal(a, c)
        part, m1, r1 = ops.layer_norm(x[311:320], w, b, stats=True)
        assert torch.equal(part, y[311:320]) and torch.equal(m1, mean[311:320])
        assert torch.equal(ops.layer_norm_bwd(dy[311:320], x[311:320], m1, r1, w)[0], first[0][311:320])


def test_parts_of_the_gradient():
    from iadmm import ops
    for cols in (100, 20000):
        x, dy, w, b = inputs(50, cols, BF16, F32)
        _, mean, rstd = ops.layer_norm(x, w, b, stats=True)
        full = ops.layer_norm_bwd(dy, x, mean, rstd, w)
        for need in [(True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, False)]:
            for a, c, on in zip(full, ops.layer_norm_bwd(dy, x, mean, rstd, w, need=need), need):
                assert (c is None) == (not on) and (c is None or torch.equal(a, c))


@pytest.mark.parametrize("t,wt", [(F32, F32), (BF16, F32), (F16, F16)])
def test_autograd_matches_formula_and_differences(t, wt):
    from iadmm import autograd
    rows, cols = 12, 800
    x, dy, w, b = inputs(rows, cols, t, wt)
    x3, w_, b_ = x.view(3, 4, cols).requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = autograd.layer_norm(x3, w_, b_)
    dx, dw, db = torch.autograd.grad(y, (x3, w_, b_), dy.view(3, 4, cols), retain_graph=True)
    xd = x.detach()
    _, mu, r, _ = forward64(xd, w.detach(), b.detach(), 1e-5)
    from iadmm import ops
    _, mean, rstd = ops.layer_norm(xd, w.detach(), b.detach(), stats=True)
    for a, (want, tol) in zip((dx.reshape(rows, cols), dw, db), backward64(dy, xd, mean, rstd, w.detach())):
        close(a, want, tol, "gradient")
    # differences of the 64-bit forward along a direction: its error ~ h^2 times third derivatives, below 1e-7 of
    # the sum's terms at h = 1e-4; the kernel's gradient adds half a step of its type to each term
    g = torch.Generator().manual_seed(5)
    d = torch.randn(rows, cols, generator=g).cuda().double()
    f = lambda s: float((forward64(xd.double() + s * d, w.detach(), b.detach(), 1e-5)[0] * dy.double()).sum())  # noqa: E731
    slope = (f(1e-4) - f(-1e-4)) / 2e-4
    mine = float((dx.reshape(rows, cols).double() * d).sum())
    size = float((dx.reshape(rows, cols).double() * d).abs().sum())
    assert abs(slope - mine) <= (half_step(t)[0] + 1e-5) * size
    # a sum's gradient is expanded, not stored; a transposed input is copied
    s, = torch.autograd.grad(y.float().sum(), b_)
    assert torch.equal(s, torch.full_like(s, rows))
    xt = torch.randn(cols, rows, generator=g).to(t).cuda().t().requires_grad_(True)
    gx, = torch.autograd.grad(autograd.layer_norm(xt, w_, b_), xt, dy)
    gc, = torch.autograd.grad(autograd.layer_norm(xt.detach().contiguous().requires_grad_(True), w_, b_).mul(1), w_, dy)
    assert gx.shape == xt.shape and bool(torch.isfinite(gx).all()) and bool(torch.isfinite(gc).all())


def test_frozen_parts_get_no_gradient():
    from iadmm import autograd
    x, dy, w, b = inputs(6, 96, F32, F32)
    y = autograd.layer_norm(x.requires_grad_(True), w, None)
    y.backward(dy)
    assert x.grad is not None and w.grad is None
    y = autograd.layer_norm(x.detach(), w.requires_grad_(True), b)
    y.backward(dy)
    assert w.grad is not None and b.grad is None
    full = torch.autograd.grad(autograd.layer_norm(x, w, b.requires_grad_(True)), (x, w, b), dy)
    only, = torch.autograd.grad(autograd.layer_norm(x.detach(), None, b), b, dy)
    assert torch.equal(only, full[2]) and torch.equal(w.grad, full[1]) and not autograd.layer_norm(x.detach()).requires_grad
    with torch.no_grad():
        assert not autograd.layer_norm(x, w, b).requires_grad


def test_writing_into_a_saved_tensor_is_noticed():
    """An out that a graph has saved: its backward refuses, as with torch's own in-place operations."""
    from iadmm import autograd, ops
    x, dy, w, b = inputs(5, 64, F32, F32)
    w.requires_grad_(True)
    y = autograd.layer_norm(x, w, b)
    ops.layer_norm(x, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_gradients_without_rows():
    from iadmm import autograd
    x, w = torch.zeros(0, 3, 40, device="cuda", requires_grad=True), torch.ones(40, device="cuda", requires_grad=True)
    dx, dw = torch.autograd.grad(autograd.layer_norm(x, w).sum(), (x, w))
    assert dx.shape == x.shape and bool((dw == 0).all())


def test_two_threads_on_two_streams():
    """Forward and gradients from two Python threads at once, each on its own stream: the bits of one after the other."""
    import threading
    from iadmm import autograd
    cases = [inputs(2000, 800, F32, F32, seed=s) for s in (1, 2)]

    def run(c):
        x, w, b = (t.detach().clone().requires_grad_(True) for t in (c[0], c[2], c[3]))
        y = autograd.layer_norm(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), c[1]))

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = run(cases[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, c in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_gradient_of_the_gradient_is_refused():
    from iadmm import autograd
    x, dy, w, b = inputs(4, 50, F32, F32)
    x.requires_grad_(True)
    g, = torch.autograd.grad(autograd.layer_norm(x, w, b), x, dy, create_graph=True)
    assert bool(torch.isfinite(g).all())
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(g.sum(), x)


def test_other_stream_and_replayed_graph():
    from iadmm import ops
    x, dy, w, b = inputs(333, 800, F32, F32)

    def both(x, dy):
        y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
        return (y, *ops.layer_norm_bwd(dy, x, mean, rstd, w))

    want = both(x, dy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = both(x, dy)
        graphs, outs = [], []
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    xs, dys = x.clone(), dy.clone()
    for _ in range(2):  # two graphs, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both(xs, dys))
        graphs.append(g)
    for k in range(4):
        x2, dy2, _, _ = inputs(333, 800, F32, F32, seed=k + 1)
        xs.copy_(x2)
        dys.copy_(dy2)
        want = both(x2, dy2)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, c) for a, c in zip(o, want)), k


def test_offsets_beyond_32_bits():
    """4.4e9 elements: the last rows, with byte and element offsets past 2^32, as if alone."""
    from iadmm import ops
    cols = 8192
    rows = (1 << 32) // cols + 1000
    x = torch.empty(rows, cols, dtype=F16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w = torch.linspace(0.5, 1.5, cols, device="cuda")
    y, mean, rstd = ops.layer_norm(x, w, stats=True)
    tail = slice(rows - 700, rows)
    yt, mt, rt = ops.layer_norm(x[tail], w, stats=True)
    assert torch.equal(y[tail], yt) and torch.equal(mean[tail], mt) and torch.equal(rstd[tail], rt)
    dx, dw, db = ops.layer_norm_bwd(y, x, mean, rstd, w)
    assert torch.equal(dx[tail], ops.layer_norm_bwd(y[tail], x[tail], mt, rt, w)[0])
    # db = sum y, a column's terms about w in size: K' u sum|y|, K' = 48 + rows / 32
    want, size = y.sum(0, dtype=torch.float64), y.abs().sum(0, dtype=torch.float64)
    assert bool(((db.double() - want).abs() <= (48 + rows / 32) * U * size).all())
