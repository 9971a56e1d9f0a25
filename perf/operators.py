"""What the training-side operators are measured on: layer norm with its gradient, the norm of a set of
gradients, and the AdamW step over many tensors.

Each case is one pass through one operator (or through the ones that a training step calls together), as a
program calls it.  ``own`` chooses between the plain form -- elementary torch operations on the same buffers,
in 32 bits -- and the framework's kernels.

The tensors that an optimizer works on live in one flat buffer, each starting at a multiple of 256 elements
(the block of the 8-bit moments); the kernels get the tensors' views, the plain form works on the whole buffer
at once, and both return the buffers.
"""
import math

import numpy as np
import torch

own = False

ALIGN = 256  # elements that share the exponents of their 8-bit moments
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LR, BETAS, EPS, DECAY, MAX_NORM = 1e-4, (0.9, 0.999), 1e-8, 0.01, 1.0
LN_EPS = 1e-5


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one row of the hidden state, as a single coordinate's call: nothing but latency
        dict(name="ln_fwd_row_h200", op="ln", way="fwd", rows=1, cols=200, dtype="f32", wdtype="f32"),
        # the hidden state of a batch of two instances (n + m = 2000), h = 800, between two iterations of a solve
        dict(name="ln_fwd_batch2_h800", op="ln", way="fwd", rows=4000, cols=800, dtype="f32", wdtype="f32"),
        # long odd rows in half precision: nothing is aligned
        dict(name="ln_fwd_odd_f16", op="ln", way="fwd", rows=1021, cols=10007, dtype="f16", wdtype="f32"),
        # one iteration's normalisation in a training micro-batch of 128 instances: forward and gradients
        dict(name="ln_train_mb128_h800", op="ln", way="both", rows=256000, cols=800, dtype="f32", wdtype="f32"),
        # gradients alone, ordinary mixed-precision training: tokens by width
        dict(name="ln_bwd_bf16", op="ln", way="bwd", rows=8192, cols=4096, dtype="bf16", wdtype="bf16"),
        # gradients of a few narrow rows (hidden size 40 of the smallest test model)
        dict(name="ln_bwd_narrow_h40", op="ln", way="bwd", rows=1111, cols=40, dtype="f32", wdtype="f32"),
        # the cell's 16 parameter tensors: norm alone, as a training loop logs it
        dict(name="norm_model_h800", op="norm", layout="model", width=800, count=100, dtype="f32"),
        # the norm over a deep stack of odd-sized bf16 gradients
        dict(name="norm_stack_bf16", op="norm", layout="stack", width=1021, count=24, dtype="bf16"),
        # the smallest model of the configuration file (h = 200, 10 iterations): a step is all latency
        dict(name="adamw_model_h200", op="adamw", layout="model", width=200, count=10, pdtype="f32", gdtype="f32",
             bits=32, clip=False),
        # the benchmark's model, h = 800 and 100 iterations, with clipping by the global norm
        dict(name="adamw_model_h800_clip", op="adamw", layout="model", width=800, count=100, pdtype="f32",
             gdtype="f32", bits=32, clip=True),
        # a deep stack in bf16 with 8-bit moments and clipping
        dict(name="adamw8_stack_bf16_clip", op="adamw", layout="stack", width=1021, count=24, pdtype="bf16",
             gdtype="bf16", bits=8, clip=True),
        # the largest: a cell of 8192 units, 268 million parameters, everything in fp32
        dict(name="adamw_model_h8192", op="adamw", layout="model", width=8192, count=200, pdtype="f32",
             gdtype="f32", bits=32, clip=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ln", "ln", "adamw", "adamw", "norm"))
    if op == "ln":
        cols = _log(rng, 8, 12000)
        rows = _log(rng, 1, min(256000, 60_000_000 // cols))
        dtype = rng.choice(("f32", "bf16", "f16"))
        return dict(op="ln", way=rng.choice(("fwd", "bwd", "both")), rows=rows, cols=cols, dtype=dtype,
                    wdtype=rng.choice(("f32", dtype)))
    if rng.random() < 0.5:
        c = dict(layout="model", width=_log(rng, 8, 4096), count=rng.randint(1, 200))
    else:
        c = dict(layout="stack", width=_log(rng, 16, 1024), count=rng.randint(1, 24))
    if op == "norm":
        return dict(op="norm", dtype=rng.choice(("f32", "bf16")), **c)
    pdtype = rng.choice(("f32", "bf16"))
    return dict(op="adamw", pdtype=pdtype, gdtype=rng.choice(("f32", pdtype)), bits=rng.choice((32, 8)),
                clip=rng.random() < 0.5, **c)


def _sizes(case):
    """Elements of each tensor: the LSTM cell's 16 parameters (width units, count iterations), or a stack of
    ``count`` layers of four square matrices, four vectors and a scalar."""
    w, n = case["width"], case["count"]
    if case["layout"] == "model":
        return [s for _ in range(4) for s in (2 * w, w * w, w)] + [w, 1, n, n]
    return [s for _ in range(n) for s in (w, w * w, w * w, w * w, w, w * w, w, w, 1)]


def _places(sizes):
    """Where each tensor starts in the flat buffer, and the buffer's length."""
    at, starts = 0, []
    for s in sizes:
        starts.append(at)
        at += -(-s // ALIGN) * ALIGN
    return starts, at


def work(case):
    if case["op"] == "ln":
        e, es, ws = case["rows"] * case["cols"], _bytes(case["dtype"]), _bytes(case["wdtype"])
        vec = case["cols"] * ws
        passes = {"fwd": 2, "bwd": 3, "both": 4}[case["way"]]  # x, y / dy, x, dx / x, y, dy, dx
        flops = {"fwd": 8, "bwd": 14, "both": 22}[case["way"]]
        extra = {"fwd": 2, "bwd": 3, "both": 4}[case["way"]] * vec
        return {"bytes": passes * e * es + extra + (8 * case["rows"] if case["way"] == "bwd" else 0),
                "flops": flops * e}
    n = sum(_sizes(case))
    if case["op"] == "norm":
        return {"bytes": n * _bytes(case["dtype"]) + 4, "flops": 2 * n}
    p, g = _bytes(case["pdtype"]), _bytes(case["gdtype"])
    # the moments in and out; with 8 bits also their values in bf16, which the pass returns
    state = 16 if case["bits"] == 32 else 4 + 4 + 4 / ALIGN
    return {"bytes": n * (2 * p + g + state), "flops": n * (16 + 2 * case["clip"])}


def _bytes(d):
    return 4 if d == "f32" else 2


# ----------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "ln":
        rows, cols = case["rows"], case["cols"]
        t, wt = DTYPES[case["dtype"]], DTYPES[case["wdtype"]]
        # hidden states: each row with a mean and a spread of its own
        x = (normal(rows, cols) * (0.2 + normal(rows, 1).abs()) + 0.5 * normal(rows, 1)).to(t)
        s = dict(case=case, x=x, w=(1 + 0.1 * normal(cols)).to(wt), b=(0.1 * normal(cols)).to(wt))
        if case["way"] != "fwd":
            s["dy"] = normal(rows, cols).to(t)
        if case["way"] == "both":
            for k in "xwb":
                s[k].requires_grad_(True)
        if case["way"] == "bwd":
            x32 = x.float()
            s["mean"] = x32.mean(1)
            s["rstd"] = (x32.var(1, unbiased=False) + LN_EPS).rsqrt()
        return s
    sizes = _sizes(case)
    starts, total = _places(sizes)
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    lens = torch.tensor(sizes, device="cuda")
    padded = torch.tensor([-(-s // ALIGN) * ALIGN for s in sizes], device="cuda")
    first = torch.tensor(starts, device="cuda")
    which = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), padded, output_size=total)
    inside = torch.arange(total, device="cuda") - first[which] < lens[which]
    scale = 10 ** (torch.rand(len(sizes), device="cuda", generator=g) * 3 - 5)  # gradients differ by tensor
    scale = scale[which] * inside
    del which

    def views(flat):
        return [flat[a:a + s] for a, s in zip(starts, sizes)]

    if case["op"] == "norm":
        flat = (normal(total) * scale).to(DTYPES[case["dtype"]])
        return dict(case=case, flat=flat, grads=views(flat))
    P = (0.05 * normal(total) * inside).to(DTYPES[case["pdtype"]])
    G = (normal(total) * scale).to(DTYPES[case["gdtype"]])
    m = 0.3 * normal(total) * scale
    v = (scale * (0.3 + normal(total).abs())) ** 2
    s = dict(case=case, sizes=sizes, starts=starts, total=total, step=1000, seed=int(seed), P=P, G=G,
             params=views(P), grads=views(G))
    if case["bits"] == 32:
        s.update(M=m, V=v, E=None, m=views(m), v=views(v), e=None)
    else:
        half = torch.full((total,), 0x80080000, dtype=torch.int64, device="cuda")  # half a step for both: nearest
        M, V, E = _encode8(m, v, half)
        s.update(M=M, V=V, E=E, m=views(M), v=views(V),
                 e=[E[a // ALIGN:-(-(a + n) // ALIGN)] for a, n in zip(starts, sizes)])
    return s


# ------------------------------------------------------------------------------------------------- the pass
def run(s):
    op = s["case"]["op"]
    return _run_ln(s) if op == "ln" else _run_norm(s) if op == "norm" else _run_adamw(s)


def _run_ln(s):
    way = s["case"]["way"]
    if own:
        import iadmm_path  # noqa: F401
        from iadmm import autograd, ops
        if way == "fwd":
            return ops.layer_norm(s["x"], s["w"], s["b"], LN_EPS)
        if way == "bwd":
            return ops.layer_norm_bwd(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
        y = autograd.layer_norm(s["x"], s["w"], s["b"], LN_EPS)
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"]))
    x, w, b = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    if way == "bwd":
        mean, rstd = s["mean"][:, None], s["rstd"][:, None]
    else:
        mean = x.mean(1, keepdim=True)
        c = x - mean
        rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + LN_EPS)
    xhat = (x - mean) * rstd
    y = (xhat * w + b).to(s["x"].dtype) if way != "bwd" else None
    if way == "fwd":
        return y
    dy = s["dy"].float()
    wdy = dy * w
    dx = (wdy - wdy.mean(1, keepdim=True) - xhat * (wdy * xhat).mean(1, keepdim=True)) * rstd
    dw = (dy * xhat).sum(0, dtype=torch.float64)  # over up to 256000 rows
    db = dy.sum(0, dtype=torch.float64)
    grads = (dx.to(s["x"].dtype), dw.to(s["w"].dtype), db.to(s["b"].dtype))
    return grads if way == "bwd" else (y, *grads)


def _run_norm(s):
    if own:
        import iadmm_path  # noqa: F401
        from iadmm import ops
        return ops.grad_norm(s["grads"])
    return _norm(s["flat"])


def _norm(flat):
    d = flat.double()
    return (d * d).sum().sqrt().float()


def _run_adamw(s):
    case = s["case"]
    s["step"] += 1
    clip, eight = case["clip"], case["bits"] == 8
    if own:
        import iadmm_path  # noqa: F401
        from iadmm import ops
        norm = ops.grad_norm(s["grads"]) if clip else None
        ops.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], lr=LR, betas=BETAS, eps=EPS,
                       weight_decay=DECAY, exponents=s["e"], norm=norm, max_norm=MAX_NORM if clip else None,
                       seed=s["seed"])
        m, v = ops.adamw_decode8(s["M"], s["V"], s["E"]) if eight else (s["M"], s["V"])
    else:
        norm = _norm(s["G"]) if clip else None
        _plain_adamw(s, norm)
        m, v = s["M"], s["V"]
        if eight:
            m, v = (t.to(torch.bfloat16) for t in _decode8(s["M"], s["V"], s["E"]))
    return dict(p=s["P"], m=m, v=v, **({"norm": norm} if clip else {}))


def _plain_adamw(s, norm):
    """One AdamW step on the flat buffers, in place.

      g <- g min(1, max_norm / (norm + 1e-6));  m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g^2
      p <- p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    bf16 parameters and 8-bit moments are rounded up or down at random, by the bits of _random()."""
    b1, b2 = BETAS
    t = s["step"]
    g = s["G"].float()
    if norm is not None:
        g = g * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
    eight, half = s["E"] is not None, s["P"].dtype == torch.bfloat16
    m, v = _decode8(s["M"], s["V"], s["E"]) if eight else (s["M"], s["V"])
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    d = torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** t)) + EPS
    p = s["P"].float() * (1 - LR * DECAY) - (LR / (1 - b1 ** t)) * (m / d)
    bits = _random(s) if eight or half else None
    if half:
        up = (p.view(torch.int32).to(torch.int64) & 0xFFFFFFFF) + (bits >> 16)
        s["P"].copy_((up >> 16).to(torch.int16).view(torch.bfloat16))
    else:
        s["P"].copy_(p)
    if eight:
        for to, code in zip((s["M"], s["V"], s["E"]), _encode8(m, v, bits)):
            to.copy_(code)
    else:
        s["M"].copy_(m)
        s["V"].copy_(v)


def _mix(x):
    """32 random-looking bits of each 32-bit number (held in int64): two odd multipliers between shifts."""
    x = x ^ (x >> 16)
    x = (x * 0xDEFBD895) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x066B4493) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random(s):
    """The 32 bits of each element: of its place in its tensor, the tensor's place, the step and the seed."""
    dev = s["P"].device
    seed, step = s["seed"] & 0xFFFFFFFFFFFFFFFF, s["step"] & 0xFFFFFFFF
    k = _mix(((seed & 0xFFFFFFFF) + 0x9E3779B9) & 0xFFFFFFFF)
    k = _mix(k ^ (seed >> 32))
    k = _mix((k + step) & 0xFFFFFFFF)
    count = len(s["sizes"])
    padded = torch.tensor([-(-n // ALIGN) * ALIGN for n in s["sizes"]], device=dev)
    key = torch.repeat_interleave(_mix(torch.arange(count, device=dev) ^ k), padded, output_size=s["total"])
    first = torch.repeat_interleave(torch.tensor(s["starts"], device=dev), padded, output_size=s["total"])
    return _mix((torch.arange(s["total"], device=dev) - first) ^ key)


def _pow2(e):
    """2^e in 64 bits, exactly (e: whole numbers)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exponent(top, low, high, shift):
    """The exponent of a block whose largest magnitude is ``top``: from 1.75 times a power of two on, the next."""
    e = ((top.view(torch.int32) + 0x200000) >> 23) - 127 - shift
    return e.clamp(low, high)


def _code(r, low, noise):
    """A number's 8-bit code: a floating-point number with three bits of mantissa and ``low`` for the exponent of
    its smallest normal ones.  Bits below are kept to 20, ``noise`` (20 bits) is added, the rest is cut."""
    k = (torch.frexp(r).exponent.to(torch.int64) - 1).clamp(min=low)
    k = torch.where(r == 0, low, k)
    n = (torch.round(r * _pow2(20 + 3 - k)).to(torch.int64) + noise) >> 20
    return 8 * (k - low) + n


def _encode8(m, v, bits):
    """The 8-bit form of the two moments: codes (sign, 4 bits of exponent, 3 of mantissa for m; 5 and 3 for v,
    which has no sign) and the two exponents of each block of 256."""
    mb, vb = m.view(-1, ALIGN), v.view(-1, ALIGN)
    em = _exponent(mb.abs().amax(1), -117, 120, 8)
    ev = _exponent(vb.amax(1), -93, 127, 0)
    noise = bits.view(-1, ALIGN)
    cm = _code(mb.abs().double() * _pow2(-em)[:, None], -6, (noise >> 20) << 8).clamp(max=0x7E)
    cm = cm + 128 * (mb < 0)
    cv = _code(vb.double() * _pow2(-ev)[:, None], -30, noise & 0xFFFFF).clamp(max=254)
    cv = torch.where((vb > 0) & (cv == 0), 1, cv)  # a second moment that is not zero stays so
    return (cm.to(torch.uint8).view(-1), cv.to(torch.uint8).view(-1), torch.stack((em, ev), 1).to(torch.int8))


def _decode8(M, V, E):
    """The values (fp32) that the codes stand for."""
    c = torch.arange(256, device=M.device)

    def table(c, low):
        k = (c >> 3).clamp(min=1)
        n = torch.where(c >> 3 > 0, (c & 7) + 8, c & 7)
        return n.double() * _pow2(k - 1 + low - 3)

    tm = table(c & 127, -6) * torch.where(c > 127, -1.0, 1.0)
    tv = table(c, -30)
    m = tm[M.long()].view(-1, ALIGN) * _pow2(E[:, 0])[:, None]
    v = tv[V.long()].view(-1, ALIGN) * _pow2(E[:, 1])[:, None]
    return m.float().view(-1), v.float().view(-1)


# ------------------------------------------------------------------------------------- the values in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ln":
        return _exact_ln(s)
    if case["op"] == "norm":
        return torch.linalg.vector_norm(s["flat"].double())
    return _exact_adamw(s)


def _exact_ln(s):
    way = s["case"]["way"]
    x, w, b = (s[k].detach().double() for k in "xwb")
    if way == "bwd":
        z = (x - s["mean"].double()[:, None]) * s["rstd"].double()[:, None]
        r = s["rstd"].double()[:, None]
    else:
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        r = (var + LN_EPS).rsqrt()
        z = (x - mean) * r
    y = torch.addcmul(b, z, w) if way != "bwd" else None
    if way == "fwd":
        return y
    dy = s["dy"].double()
    q = dy * w
    inner = (q * z).sum(1, keepdim=True)
    dx = r / x.shape[1] * (x.shape[1] * q - q.sum(1, keepdim=True) - z * inner)
    dw, db = torch.mul(dy, z).sum(0), dy.sum(0)
    return (dx, dw, db) if way == "bwd" else (y, dx, dw, db)


def _exact_adamw(s):
    """The same step from the definition: moments as whole numbers of their steps, in numpy for the random bits."""
    case = s["case"]
    b1, b2 = BETAS
    t = s["step"] + 1
    g = s["G"].double()
    out = {}
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, MAX_NORM / (float(out["norm"]) + 1e-6))
    eight = case["bits"] == 8
    if eight:
        em, ev = (torch.repeat_interleave(s["E"][:, k].double(), ALIGN) for k in (0, 1))
        cm, cv = s["M"].double(), s["V"].double()
        sign = 1 - 2 * (cm >= 128).double()
        cm = cm % 128
        m = sign * _value(cm, -6) * torch.exp2(em)
        v = _value(cv, -30) * torch.exp2(ev)
    else:
        m, v = s["M"].double(), s["V"].double()
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g.square(), v, b2)
    p = s["P"].double()
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    if eight or case["pdtype"] == "bf16":
        u = torch.from_numpy(_exact_random(s["sizes"], s["starts"], s["total"], s["seed"], t)).to(p.device)
    out["p"] = p
    if case["pdtype"] == "bf16":
        step = torch.exp2(torch.floor(torch.log2(p.abs().clamp(min=2.0 ** -126))) - 7)
        low = torch.floor(p.abs() / step)
        part = torch.floor((p.abs() / step - low) * 65536 + 0.5) + torch.floor(u / 65536)
        out["p"] = torch.sign(p) * (low + (part >= 65536)) * step
    if eight:
        out["m"] = torch.sign(m) * _rounded(m.abs(), 448, -6, torch.floor(u / 2 ** 20) / 4096, 8)
        out["v"] = _rounded(v, 1.75, -30, torch.remainder(u, 2 ** 20) / 2 ** 20, 0)
    else:
        out["m"], out["v"] = m, v
    return out


def _value(c, low):
    e, n = torch.floor(c / 8), torch.remainder(c, 8)
    return torch.where(e == 0, n * 2.0 ** (low - 3), (8 + n) * torch.exp2(e - 1 + low - 3))


def _rounded(a, top, low, u, shift):
    """Magnitudes rounded to 8-bit floating point under their block's power of two, up with chance u's."""
    blocks = a.view(-1, ALIGN)
    most = blocks.amax(1, keepdim=True)
    floor = -93.0 if shift == 0 else -117.0
    e = torch.where(most > 0, torch.floor(torch.log2(most.clamp(min=1e-300))) - shift, floor)
    e = torch.where(most >= top * torch.exp2(e), e + 1, e).clamp(floor, 127.0 - 0.875 * shift)
    r = blocks * torch.exp2(-e)
    k = torch.where(r > 0, torch.floor(torch.log2(r.clamp(min=1e-300))), -1000.0).clamp(min=low)
    q = torch.exp2(k - 3)
    r = torch.floor(r / q + u.view(-1, ALIGN)) * q
    if shift == 0:
        r = torch.where((blocks > 0) & (r == 0), 2.0 ** (low - 3), r)
    return (r * torch.exp2(e)).view(-1)


def _exact_random(sizes, starts, total, seed, step):
    def scramble(x):
        with np.errstate(over="ignore"):
            x = x ^ (x >> np.uint32(16))
            x = x * np.uint32(0xDEFBD895)
            x = x ^ (x >> np.uint32(15))
            x = x * np.uint32(0x066B4493)
            return x ^ (x >> np.uint32(16))

    word = lambda a: np.array([a & 0xFFFFFFFF], dtype=np.uint32)  # noqa: E731
    key = scramble(word((seed & 0xFFFFFFFF) + 0x9E3779B9))
    key = scramble(key ^ word(seed >> 32))
    key = scramble(word(int(key[0]) + step))
    bits = np.empty(total, dtype=np.float64)
    for i, (a, n) in enumerate(zip(starts, sizes)):
        n = -(-n // ALIGN) * ALIGN
        bits[a:a + n] = scramble(np.arange(n, dtype=np.uint32) ^ scramble(key ^ word(i)))
    return bits
