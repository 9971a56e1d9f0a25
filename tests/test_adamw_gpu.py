"""The AdamW step and the gradients' norm (csrc/adamw.hip).

The oracle steps in numpy's fp32 with the kernel's order of products and sums, each rounded by itself, so moments,
codes and exponents have to be equal bit for bit.  Of the parameters, the quotient m / (sqrt(v) c + eps) may be off
by 8 u of itself (u = 2^-24: two hardware approximations of 1 ulp each, two products and a sum), and the product
with the step size, the decay and the difference each round once:  4 u |p| + 10 u |update|.  A bf16 parameter is
the random cut of some fp32 value in that range.  The tests of the formula itself use 64 bits."""
import math

import numpy as np
import pytest
import torch

import iadmm_path  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
B = 256


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# ------------------------------------------------------------------------------------------------- the oracle
def mix(x):
    with np.errstate(over="ignore"):
        x = np.asarray(x, dtype=np.uint32)
        x = x ^ (x >> np.uint32(16))
        x = x * np.uint32(0xDEFBD895)
        x = x ^ (x >> np.uint32(15))
        x = x * np.uint32(0x066B4493)
        return x ^ (x >> np.uint32(16))


def random_bits(n, seed, step, slot):
    k = mix(((seed & 0xFFFFFFFF) + 0x9E3779B9) & 0xFFFFFFFF)
    k = mix(k ^ np.uint32(seed >> 32))
    k = mix((int(k) + step) & 0xFFFFFFFF)
    return mix(np.arange(n, dtype=np.uint32) ^ mix(k ^ np.uint32(slot)))


def values(codes, low):
    """What codes with three mantissa bits stand for: ``low`` is the exponent of the smallest normal one."""
    c = codes.astype(np.int64)
    e, n = c >> 3, c & 7
    return np.where(e == 0, n * 2.0 ** (low - 3), (8 + n) * np.exp2(np.maximum(e, 1) - 1.0 + low - 3))


def spread(e, n):
    return np.repeat(e.astype(np.float64), B)[:n]


def decode(m8, v8, e):
    n = len(m8)
    mag = np.where((m8 & 127) == 127, np.nan, values(m8 & 127, -6))
    m = np.where(m8 > 127, -mag, mag) * np.exp2(spread(e[:, 0], n))
    v = np.where(v8 == 255, np.inf, values(v8, -30) * np.exp2(spread(e[:, 1], n)))
    with np.errstate(over="ignore"):
        return m.astype(np.float32), v.astype(np.float32)


def exponents(x, shift, low, high):
    pad = np.zeros(-(-len(x) // B) * B, dtype=np.float32)
    pad[:len(x)] = np.where(np.isfinite(x), np.abs(x), 0)
    top = pad.reshape(-1, B).max(1)
    e = ((top.view(np.int32).astype(np.int64) + 0x200000) >> 23) - 127 - shift
    return np.clip(e, low, high)


def codes(x, e, low, noise, most):
    with np.errstate(invalid="ignore", over="ignore"):
        r = np.where(np.isfinite(x), np.abs(x), 0).astype(np.float64) * np.exp2(-spread(e, len(x)))
    k = np.maximum(np.frexp(r)[1] - 1, low)
    k = np.where(r == 0, low, k)
    n = (np.rint(r * np.exp2(20.0 + 3 - k)).astype(np.int64) + noise) >> 20
    return np.minimum(8 * (k - low) + n, most)


def encode(m, v, bits):
    em, ev = exponents(m, 8, -117, 120), exponents(v, 0, -93, 127)
    b = bits.astype(np.int64)
    cm = np.where(np.isfinite(m), codes(m, em, -6, (b >> 20) << 8, 126), 127) + 128 * (m < 0)
    cv = codes(v, ev, -30, b & 0xFFFFF, 254)
    cv = np.where((v > 0) & (cv == 0), 1, cv)
    cv = np.where(np.isfinite(v), cv, 255)
    return cm.astype(np.uint8), cv.astype(np.uint8), np.stack([em, ev], 1).astype(np.int8)


def step32(p, g, m, v, t, lr, betas, eps, wd, clip=None):
    """(p', |update|, m', v') of fp32 arrays, in fp32."""
    f = np.float32
    b1, b2 = betas
    with np.errstate(all="ignore"):
        g = g.astype(f) if clip is None else g.astype(f) * f(clip)
        m = f(b1) * m + f(1.0 - b1) * g
        v = f(b2) * v + f(1.0 - b2) * (g * g)
        d = np.sqrt(v) * f(1.0 / math.sqrt(1.0 - b2 ** t)) + f(eps)
        up = f(lr / (1.0 - b1 ** t)) * (m / d)
        return p.astype(f) * f(1.0 - lr * wd) - up, np.abs(up), m, v


def check_params(got, want, up, bits):
    want64, up = want.astype(np.float64), up.astype(np.float64)
    got32 = got.float().cpu().numpy().reshape(-1)
    assert np.array_equal(np.isnan(got32), np.isnan(want))
    fine = np.isfinite(want)
    tol = 4 * U * np.abs(want64) + 10 * U * np.nan_to_num(up) + 2.0 ** -148
    if got.dtype == torch.float32:
        assert np.all((np.abs(got32 - want64) <= tol)[fine])
        return

    def cut(x):
        b = x.astype(np.float32).view(np.uint32).astype(np.uint64)
        return ((((b + (bits >> np.uint32(16))) >> 16) << 16) & 0xFFFFFFFF).astype(np.uint32).view(np.float32)

    a, b = cut(want64 - tol), cut(want64 + tol)
    assert np.all(((np.minimum(a, b) <= got32) & (got32 <= np.maximum(a, b)))[fine])


def tensors(sizes, pdtype=torch.float32, gdtype=torch.float32, eight=False, seed=0, shift=0):
    """Parameters, gradients and moments with ``shift`` elements before each (an odd address)."""
    g = torch.Generator().manual_seed(seed)
    P, G, M, V, E = [], [], [], [], []
    place = lambda t: torch.cat([torch.zeros(shift, dtype=t.dtype), t.reshape(-1)]).cuda()[shift:]  # noqa: E731
    for n in sizes:
        scale = 10.0 ** (-4 + 3 * torch.rand(1, generator=g))
        P.append(place((0.05 * torch.randn(n, generator=g)).to(pdtype)))
        G.append(place((scale * torch.randn(n, generator=g)).to(gdtype)))
        m, v = 0.3 * scale * torch.randn(n, generator=g), (scale * (0.1 + torch.randn(n, generator=g).abs())) ** 2
        if eight:
            bits = np.full(n, 0x80080000, dtype=np.uint32)
            cm, cv, e = encode(m.numpy(), v.numpy(), bits)
            M.append(place(torch.from_numpy(cm)))
            V.append(place(torch.from_numpy(cv)))
            E.append(place(torch.from_numpy(e)).view(-1, 2))
        else:
            M.append(place(m))
            V.append(place(v))
    return P, G, M, V, E if eight else None


def to_np(t):
    return (t.float() if t.dtype == torch.bfloat16 else t).cpu().numpy().copy()


SIZES = [1, 2, 3, 5, 255, 256, 257, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 12289, 100003]
KINDS = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
         (torch.float32, torch.bfloat16)]


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("pdtype,gdtype", KINDS)
def test_step(pdtype, gdtype, eight, shift):
    """Two steps over tensors of every kind of size, at aligned and odd addresses, against the oracle."""
    from iadmm import ops
    P, G, M, V, E = tensors(SIZES, pdtype, gdtype, eight, seed=3, shift=shift)
    kw = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
    seed = 0x123456789ABCDEF
    for t in (7, 8):
        before = [[to_np(x) for x in L] for L in (P, G, M, V)] + ([[to_np(x) for x in E]] if eight else [])
        norm = ops.grad_norm(G) if t == 8 else None
        ops.adamw_step(P, G, M, V, t, exponents=E, seed=seed, norm=norm, max_norm=0.3 if t == 8 else None, **kw)
        torch.cuda.synchronize()
        clip = None
        if t == 8:
            clip = min(np.float32(1.0), np.float32(0.3) / (np.float32(norm.item()) + np.float32(1e-6)))
            assert clip < 1
        for i, n in enumerate(SIZES):
            p, g, m, v = (before[k][i] for k in range(4))
            if eight:
                m, v = decode(m, v, before[4][i])
            bits = random_bits(n, seed, t, i)
            want, up, m, v = step32(p, g, m, v, t, kw["lr"], kw["betas"], kw["eps"], kw["weight_decay"], clip)
            check_params(P[i], want, up, bits)
            if eight:
                cm, cv, e = encode(m, v, bits)
                assert np.array_equal(to_np(E[i]), e), n
                assert np.array_equal(to_np(M[i]) & 127, cm & 127) and np.array_equal(to_np(V[i]), cv), n
                assert np.array_equal(decode(to_np(M[i]), cv, e)[0], decode(cm, cv, e)[0])
            else:
                assert np.array_equal(to_np(M[i]), m) and np.array_equal(to_np(V[i]), v), n
            assert np.array_equal(to_np(G[i]), g)  # clipping leaves the gradients


def test_formula_in_64_bits():
    """32-bit moments, against torch's own AdamW in 64 bits over 20 steps from zero (each step's error is at most
    4 u |p| + 20 u |update| here, |update| <= lr / sqrt(1 - b2) in the worst case and about lr)."""
    from iadmm import ops
    g = torch.Generator().manual_seed(11)
    sizes = [(17, 5), (800,), (1,), (64, 64)]
    P = [torch.randn(*s, generator=g).cuda() for s in sizes]
    ref = [p.double().clone().requires_grad_(True) for p in P]
    opt = torch.optim.AdamW(ref, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    M, V = [torch.zeros_like(p) for p in P], [torch.zeros_like(p) for p in P]
    for t in range(1, 21):
        G = [torch.randn(*s, generator=g).cuda() for s in sizes]
        for r, x in zip(ref, G):
            r.grad = x.double()
        opt.step()
        ops.adamw_step(P, G, M, V, t, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    for p, r in zip(P, ref):
        assert bool(((p.double() - r).abs() <= 20 * U * (4 * r.abs() + 20 * 1e-2 * 2)).all())


@pytest.mark.parametrize("eight", [False, True])
def test_many_tensors_and_missing_gradients(eight):
    """More tensors than a launch takes, some empty, some without a gradient: the others as if alone in their
    place, the rest untouched."""
    from iadmm import ops
    sizes = [(37 * i * i) % 1500 for i in range(130)]
    P, G, M, V, E = tensors(sizes, eight=eight, seed=5)
    keep = [[x.clone() for x in L] for L in (P, M, V)]
    for i in range(3, 130, 7):
        G[i] = None
    ops.adamw_step(P, G, M, V, 4, exponents=E, seed=9, lr=1e-3)
    for i, n in enumerate(sizes):
        if G[i] is None:
            assert all(torch.equal(L[i], k[i]) for L, k in zip((P, M, V), keep))
            continue
        p, g, _, _ = (to_np(x) for x in (keep[0][i], G[i], M[i], V[i]))
        if eight:
            continue
        want, up, m, v = step32(p, g, to_np(keep[1][i]), to_np(keep[2][i]), 4, 1e-3, (0.9, 0.999), 1e-8, 0.01)
        check_params(P[i], want, up, None)
        assert np.array_equal(to_np(M[i]), m)
    if eight:  # one by one, each at its own place in the list: the same bits
        P2, G2, M2, V2, E2 = tensors(sizes, eight=eight, seed=5)
        for i in range(130):
            only = [x if k == i and G[k] is not None else None for k, x in enumerate(G2)]
            ops.adamw_step(P2, only, M2, V2, 4, exponents=E2, seed=9, lr=1e-3)
        for L, K in ((P, P2), (M, M2), (V, V2), (E, E2)):
            assert all(torch.equal(a, b) for a, b in zip(L, K))


@pytest.mark.parametrize("count", [48, 49, 64, 65, 4096, 4097, 9001])
def test_long_lists(count):
    """Every tensor of a list of any length is found, by its own workgroups: 1 to 3000 elements each, some empty."""
    from iadmm import ops
    sizes = np.array([(i * 7919) % 11 if i % 50 else (i * 31) % 3000 for i in range(count)])
    starts = np.concatenate([[0], np.cumsum(sizes)])
    n = int(starts[-1])
    g = torch.Generator(device="cuda").manual_seed(count)
    p, m = (torch.randn(n, device="cuda", generator=g) for _ in range(2))
    gr, v = 1e-2 * torch.randn(n, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
    cut = lambda t: [t[a:z] for a, z in zip(starts[:-1].tolist(), starts[1:].tolist())]  # noqa: E731
    want, up, wm, wv = step32(*(to_np(t) for t in (p, gr, m, v)), 5, 1e-3, (0.9, 0.999), 1e-8, 0.01)
    ops.adamw_step(cut(p), cut(gr), cut(m), cut(v), 5, lr=1e-3)
    check_params(p, want, up, None)
    assert np.array_equal(to_np(m), wm) and np.array_equal(to_np(v), wv)


def test_nothing_beside_a_tensor_is_written():
    from iadmm import ops
    for eight in (False, True):
        for n in (1, 5, 255, 257, 4099):
            P, G, M, V, E = tensors([n], torch.bfloat16, torch.bfloat16, eight, seed=n)
            bufs = []
            for L in (P, M, V) + ((E,) if eight else ()):
                t = L[0]
                buf = torch.full((t.numel() + 64,), 77, dtype=t.dtype, device="cuda")
                buf[32:32 + t.numel()] = t.reshape(-1)
                L[0] = buf[32:32 + t.numel()]
                bufs.append(buf)
            ops.adamw_step(P, G, M, V, 1, exponents=E)
            for buf in bufs:
                assert bool((buf[:32] == 77).all()) and bool((buf[-32:] == 77).all())


def test_random_rounding_keeps_the_mean():
    """4096 blocks of one value each, moved by less than half a code: the mean over the blocks moves with the
    values.  The mean of N cuts is off by at most 5 sigma <= 5 * step / (2 sqrt(N)) (chance 6e-7; the bits are
    fixed by the seed)."""
    from iadmm import ops
    N = 4096 * B
    m0, v0 = np.full(N, 1.07e-3, np.float32), np.full(N, 1.1e-6, np.float32)
    m0[::B], v0[::B] = 1.9e-3, 3.0e-6  # the blocks' largest
    cm, cv, e = encode(m0, v0, np.full(N, 0x80080000, np.uint32))
    M, V, E = ([torch.from_numpy(x).cuda()] for x in (cm, cv, e))
    P = [torch.full((N,), 0.2501, device="cuda").bfloat16()]
    G = [torch.full((N,), 1.2e-3, device="cuda")]
    m, v = decode(cm, cv, e)
    want_p, _, want_m, want_v = step32(to_np(P[0]), to_np(G[0]), m, v, 100, 1e-4, (0.9, 0.999), 1e-8, 0.01)
    ops.adamw_step(P, G, M, V, 100, exponents=E, lr=1e-4, seed=1)
    gm, gv = decode(to_np(M[0]), to_np(V[0]), to_np(E[0]))
    for got, want, step in ((gm, want_m, 2.0 ** -13), (gv, want_v, 2.0 ** -23), (to_np(P[0]), want_p, 2.0 ** -10)):
        inner = np.arange(N) % B != 0
        off = abs(got[inner].astype(np.float64).mean() - want[inner].astype(np.float64).mean())
        assert off <= 5 * step / (2 * math.sqrt(inner.sum())), (off, step)
        assert len(np.unique(got[inner])) == 2  # the two neighbours


def test_second_moment_follows_its_gradients():
    """200 steps of gradients four times as large as the moment stands for: nearest rounding would stay (0.1 %
    of 15 times the moment a step is 1.5 %, half a code is 3 to 6 %), the random one arrives where 32 bits do, to
    within 5 sigma of the mean of 65536 elements whose codes' steps are at most an eighth of them."""
    from iadmm import ops
    n = 65536
    P, G = [torch.zeros(n, device="cuda")], [torch.full((n,), 2e-3, device="cuda")]
    cm, cv, e = encode(np.zeros(n, np.float32), np.full(n, 1e-6, np.float32), np.full(n, 0x80080000, np.uint32))
    M, V, E = ([torch.from_numpy(x).cuda()] for x in (cm, cv, e))
    v = float(decode(cm, cv, e)[1][0])
    for t in range(1, 201):
        ops.adamw_step(P, G, M, V, t, exponents=E, lr=0.0, seed=2)
        v = 0.999 * v + 0.001 * 4e-6
    got = ops.adamw_decode8(M[0], V[0], E[0], torch.float32)[1].double().mean().item()
    # each step's rounding has sigma <= v / 16 an element; 200 of them add up to at most sqrt(200) / 16 = 0.9 v
    assert abs(got / v - 1) <= 5 * 0.9 / math.sqrt(n), (got, v)


def test_decode_every_code():
    from iadmm import ops
    cm = np.tile(np.arange(256, dtype=np.uint8), 6)
    e = np.array([[0, 0], [-117, -93], [119, 127], [-20, -30], [5, 7], [100, 1]], dtype=np.int8)
    m, v = decode(cm, cm, e)
    args = [torch.from_numpy(x).cuda() for x in (cm, cm, e)]
    gm, gv = ops.adamw_decode8(*args, dtype=torch.float32)
    assert np.array_equal(to_np(gm), m, equal_nan=True) and np.array_equal(to_np(gv), v)
    hm, hv = ops.adamw_decode8(*args)
    assert torch.equal(hm.float().nan_to_num(1.0), gm.nan_to_num(1.0)) and torch.equal(hv.float(), gv)
    gm, gv = ops.adamw_decode8(*[a[:1000] if a.dim() == 1 else a[:4] for a in args], dtype=torch.float32)
    assert np.array_equal(to_np(gv), v[:1000]) and gm.shape == (1000,)


@pytest.mark.parametrize("eight", [False, True])
def test_extreme_values(eight):
    """Infinite, NaN, huge, tiny and zero gradients, each in a block of ordinary ones, and whole blocks of them."""
    from iadmm import ops
    n = 8 * B
    P, G, M, V, E = tensors([n], eight=eight, seed=8)
    for block, x in enumerate((math.inf, -math.inf, math.nan, 3e38, 1e-42, 0.0)):
        G[0][block * B + 5] = x
    G[0][6 * B:7 * B] = 0.0
    for t, fill in ((M[0], 0), (V[0], 0)):
        t[6 * B:] = fill
    G[0][7 * B:] = 1e30
    before = [to_np(x[0]) for x in (P, G, M, V)] + ([to_np(E[0])] if eight else [])
    p, g, m, v = before[:4]
    for t in (3, 4):
        if eight:
            m, v = decode(m, v, before[4]) if t == 3 else decode(*got)
        bits = random_bits(n, 21, t, 0)
        ops.adamw_step(P, G, M, V, t, exponents=E, lr=1e-3, seed=21)
        want, up, m, v = step32(p, g, m, v, t, 1e-3, (0.9, 0.999), 1e-8, 0.01)
        check_params(P[0], want, up, bits)
        p = to_np(P[0])
        if eight:
            cm, cv, e = encode(m, v, bits)
            got = to_np(M[0]), to_np(V[0]), to_np(E[0])
            nan = np.isnan(decode(cm, cv, e)[0])
            assert np.array_equal(got[2], e) and np.array_equal(got[1], cv)
            assert np.array_equal((got[0] & 127)[~nan], (cm & 127)[~nan]) and np.all((got[0] & 127)[nan] == 127)
        else:
            assert np.array_equal(to_np(M[0]), m, equal_nan=True) and np.array_equal(to_np(V[0]), v, equal_nan=True)
        with np.errstate(invalid="ignore"):  # the sign of a product of NaN may differ: the values are what counts
            p = np.where(np.isnan(p), np.float32(np.nan), p)
    assert bool((P[0][6 * B:7 * B].cpu() != 0).any()) and bool(torch.isfinite(P[0][6 * B:]).all())


@pytest.mark.parametrize("eight", [False, True])
def test_counts_on_the_device(eight):
    """A step with its count on the device is the step with the same number (the powers are 64-bit on both sides:
    the fp32 factors may round apart by a step, 2 u of the update), eagerly and replayed from a graph with eager
    steps of other tensors in between; parameters without a gradient do not count."""
    from iadmm import ops
    sizes = [300, 1, 5000, 77] + [64] * 60
    A, C = (tensors(sizes, eight=eight, seed=6) for _ in range(2))
    counts = torch.arange(len(sizes), device="cuda")
    numbers = list(range(len(sizes)))
    lr = torch.tensor([2e-3], device="cuda")
    grads = [None if i == 3 else g for i, g in enumerate(C[1])]

    def device_step():
        ops.adamw_step(C[0], grads, *C[2:4], counts, exponents=C[4], lr=lr, seed=3, norm=norm, max_norm=0.5)

    def compare():
        for i in range(len(sizes)):
            tol = 4 * U * A[0][i].abs() + 24 * U * 2e-3 * 40 + 0.0
            assert bool(((A[0][i] - C[0][i]).abs() <= tol).all()), i
            assert torch.equal(A[2][i], C[2][i]) and torch.equal(A[3][i], C[3][i])
        assert counts.tolist() == numbers

    norm = ops.grad_norm(C[1])
    for k in range(5):
        if k == 1:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                device_step()
        if k:
            graph.replay()
        else:
            device_step()
        numbers = [x + (i != 3) for i, x in enumerate(numbers)]
        ops.adamw_step(A[0], [None if g is None else A[1][i] for i, g in enumerate(grads)], *A[2:4],
                       [max(x, 1) for x in numbers], exponents=A[4], lr=lr.item(), seed=3, norm=norm, max_norm=0.5)
        torch.cuda.synchronize()
        compare()
        lr.mul_(0.7)
        for x, y in zip(A[1], C[1]):
            y.mul_(1.1)
            x.copy_(y)
    with pytest.raises(RuntimeError, match="captured"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.adamw_step(*C[:4], 3, exponents=C[4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_norm(dtype):
    from iadmm import ops
    for sizes in ([300] * 16, [1024] * 32, [1024] * 31 + [1025], [0, 3, 0, 2049], [1] * 32, [1] * 33, [1], [5], [8192], [8193], [100003, 0, 3], [(i * 97) % 3000 for i in range(300)], [30_000_001],
                  [(i * 1931) % 40000 for i in range(240)], [8192] * 241, [5] * 480, [16384, 16383, 0, 16385, 2048, 600_000], [0, 0]):
        g = torch.Generator(device="cuda").manual_seed(len(sizes))
        G = [(10.0 ** (k % 7 - 3) * torch.randn(n, device="cuda", generator=g)).to(dtype) for k, n in enumerate(sizes)]
        want = math.sqrt(sum(float(x.double().square().sum()) for x in G))
        got = ops.grad_norm(G)
        assert got.shape == () and got.dtype == torch.float32
        # one rounding to fp32, and 64-bit sums of up to 3e7 positive terms in two orders
        assert abs(float(got) - want) <= (U + 1e-12) * want
        assert torch.equal(got, ops.grad_norm(G))
    odd = torch.randn(4100, device="cuda").to(dtype)[1:]
    assert abs(float(ops.grad_norm([odd, None])) - float(odd.double().norm())) <= (U + 1e-12) * float(odd.double().norm())
    big = torch.full((1000,), 1e30, device="cuda").to(dtype)
    assert abs(float(ops.grad_norm([big])) / (float(big[0]) * math.sqrt(1000)) - 1) <= 2 * U
    assert float(ops.grad_norm([torch.zeros(7, device="cuda")])) == 0.0
    odd[17] = math.inf
    assert float(ops.grad_norm([odd])) == math.inf
    odd[18] = math.nan
    assert math.isnan(float(ops.grad_norm([big, odd])))


def test_streams_and_graphs_of_the_norm():
    from iadmm import ops
    G = [torch.randn(n, device="cuda") for n in (10, 70000, 5)]
    want = ops.grad_norm(G)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.grad_norm(G)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.grad_norm(G)
        graphs.append((graph, out))
    for k in range(3):
        G[1].mul_(1.5)
        want = ops.grad_norm(G)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out in graphs)


def test_offsets_beyond_32_bits():
    """A bf16 tensor of 2^32 + 5000 elements with 8-bit moments: its last blocks by the oracle."""
    from iadmm import ops
    n = (1 << 32) + 5000
    P = torch.full((n,), 0.1, dtype=torch.bfloat16, device="cuda")
    G = torch.full((n,), 1e-3, dtype=torch.bfloat16, device="cuda")
    M, V = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    E = torch.zeros((n + B - 1) // B, 2, dtype=torch.int8, device="cuda")
    want = math.sqrt(n) * float(G[0])
    assert abs(float(ops.grad_norm([G])) / want - 1) <= 2 * U
    ops.adamw_step([P], [G], [M], [V], 1, exponents=[E], lr=1e-3, seed=4)
    at = (n - 4000) // B * B
    for a, z in ((0, 4 * B), (at, n)):
        idx = np.arange(a, z, dtype=np.uint64)
        k = mix(0x9E3779B9 + 4)
        k = mix(k)
        key = mix(mix((int(k) + 1) & 0xFFFFFFFF))
        with np.errstate(over="ignore"):
            low = (idx & np.uint64(0xFFFFFFFF)).astype(np.uint32) ^ (idx >> np.uint64(32)).astype(np.uint32) * np.uint32(0x9E3779B9)
        bits = mix(low ^ key)
        m = np.zeros(z - a, np.float32)
        p = np.full(z - a, float(torch.tensor(0.1).bfloat16()), np.float32)
        g = np.full(z - a, float(G[0]), np.float32)
        want, up, m, v = step32(p, g, m, m.copy(), 1, 1e-3, (0.9, 0.999), 1e-8, 0.01)
        check_params(P[a:z], want, up, bits)
        cm, cv, e = encode(m, v, bits)
        assert np.array_equal(to_np(M[a:z]), cm) and np.array_equal(to_np(V[a:z]), cv)
        assert np.array_equal(to_np(E[a // B:]) [:len(e)], e)


def test_refusals_change_nothing():
    from iadmm import ops
    P, G, M, V, _ = tensors([64, 65])
    _, _, M8, V8, E8 = tensors([64, 65], eight=True)
    keep = [x.clone() for x in P + M + V]
    nan = float("nan")
    norm = torch.ones((), device="cuda")
    bad = [
        dict(args=(P, G, M, [V[0], V[1][:64]], 1)), dict(args=(P, [G[0], G[1][:64]], M, V, 1)),
        dict(args=(P, G, M8, V8, 1)), dict(args=(P, G, M, V, 1), exponents=E8), dict(args=(P, G, M8, V8, 1), exponents=[E8[0], E8[0]]),
        dict(args=(P, G, M8, V8, 1), exponents=[E8[0], E8[1][:1, :1]]), dict(args=([P[0], P[0]], [G[0], G[0]], M, V, 1)),
        dict(args=(P, [G[0], G[1].view(5, 13)], M, V, 1)), dict(args=(P, G, M, V, 0)), dict(args=(P, G, M, V, [3, 0])),
        dict(args=(P, G, M, V, torch.ones(2, device="cuda"))), dict(args=(P, G, M, V, torch.ones(3, dtype=torch.int64, device="cuda"))),
        dict(args=(P, G, M, V, torch.ones(2, dtype=torch.int64))), dict(args=(P, G, M, V, 1), lr=torch.ones(1, device="cuda")),
        dict(args=(P, G, M, V, 1), lr=-1.0), dict(args=(P, G, M, V, 1), lr=nan), dict(args=(P, G, M, V, 1), betas=(1.0, 0.9)),
        dict(args=(P, G, M, V, 1), betas=(0.9, nan)), dict(args=(P, G, M, V, 1), eps=-1e-8),
        dict(args=(P, G, M, V, 1), weight_decay=nan), dict(args=(P, G, M, V, 1), norm=norm),
        dict(args=(P, G, M, V, 1), norm=norm, max_norm=0.0), dict(args=(P, G, M, V, 1), norm=norm.double(), max_norm=1.0),
        dict(args=(P, [g.double() for g in G], M, V, 1)), dict(args=(P, [g.cpu() for g in G], M, V, 1)),
        dict(args=(P, G, M, [M[0], V[1]], 1)),
    ]
    for kw in bad:
        args = kw.pop("args")
        with pytest.raises((TypeError, ValueError)):
            ops.adamw_step(*args, **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(keep, P + M + V))


def test_overlapping_tensors_are_refused():
    """Parts of one buffer that reach into each other, a gradient that reaches into what is written; parts side by side
    and gradients that share theirs (which is only read) are taken."""
    from iadmm import ops
    buf, g = torch.randn(1000, device="cuda"), torch.randn(400, device="cuda")
    m, v = ([torch.zeros(300, device="cuda") for _ in range(2)] for _ in range(2))
    keep = buf.clone()
    P = [buf[:300], buf[299:599]]
    with pytest.raises(ValueError, match="overlaps"):
        ops.adamw_step(P, [g[:300], g[:300]], m, v, 1)
    with pytest.raises(ValueError, match="overlaps"):
        ops.adamw_step([buf[:300], buf[300:600]], [buf[599:899], g[:300]], m, v, 1)
    with pytest.raises(ValueError, match="overlaps"):
        ops.adamw_step([buf[:300], buf[300:600]], [g[:300], g[:300]], [m[0], buf[500:800]], v, 1)
    torch.cuda.synchronize()
    assert torch.equal(buf, keep)
    ops.adamw_step([buf[:300], buf[300:600]], [buf[600:900], g[50:350]], m, v, 1)
    a, b = keep[:300].clone(), keep[300:600].clone()
    n, w = ([torch.zeros(300, device="cuda") for _ in range(2)] for _ in range(2))
    ops.adamw_step([a, b], [keep[600:900].clone(), g[50:350].clone()], n, w, 1)
    assert torch.equal(buf, torch.cat((a, b, keep[600:])))


def test_numbers_of_numpy():
    from iadmm import ops
    A, C = tensors([100]), tensors([100])
    ops.adamw_step(*A[:4], np.int64(3), lr=np.float64(1e-3))
    ops.adamw_step(*C[:4], [np.int32(3)], lr=1e-3)
    assert torch.equal(A[0][0], C[0][0])
    with pytest.raises((TypeError, ValueError)):
        ops.adamw_step(*A[:4], 3.5)
    neg = torch._neg_view(A[1][0])
    for call in (lambda: ops.adamw_step(A[0], [neg], A[2], A[3], 4), lambda: ops.grad_norm([neg])):
        with pytest.raises(ValueError):
            call()


def test_a_step_is_seen_by_the_version():
    """solver.PackedWeights goes by a parameter's version: a step has to raise it."""
    from iadmm import ops
    P, G, M, V, _ = tensors([10, 20])
    before = [p._version for p in P]
    ops.adamw_step(P, [G[0], None], M, V, 1)
    assert P[0]._version > before[0] and P[1]._version == before[1]
