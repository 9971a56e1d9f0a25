"""iadmm.optim.AdamW and the model's layer norm as the training loop and the CLI use them: norm of the gradients,
clipped step in 32 or 8 bits, normalised hidden state with its gradient, one after the other."""
import copy
import math

import pytest
import torch

import iadmm_path  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def params(seed=0, dtype=torch.float32, shapes=((40, 40), (40,), (2, 40), (1,), (100, 1))):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((0.1 * torch.randn(*s, generator=g)).to(dtype).cuda()) for s in shapes]


def set_grads(ps, seed, dtype=None, scale=1.0):
    g = torch.Generator().manual_seed(1000 + seed)
    for p in ps:
        p.grad = (scale * torch.randn(*p.shape, generator=g)).to(dtype or p.dtype).cuda()


def test_against_torch_in_64_bits():
    """Two groups, a parameter that joins late, clipping: torch.optim.AdamW and clip_grad_norm_ on fp64 copies.
    A step's error is at most 4 u |p| + 20 u |update|, |update| <= 2 lr here, and the clipping factor adds 4 u."""
    from iadmm.optim import AdamW
    a = params()
    b = [torch.nn.Parameter(p.detach().double()) for p in a]
    groups = lambda ps: [dict(params=ps[:2], lr=3e-3, weight_decay=0.1), dict(params=ps[2:], betas=(0.8, 0.99))]  # noqa: E731
    mine, ref = AdamW(groups(a), lr=1e-3, max_norm=5.0), torch.optim.AdamW(groups(b), lr=1e-3, weight_decay=0.01)
    for t in range(12):
        set_grads(a, t)
        if t < 4:
            a[3].grad = None
        for p, q in zip(a, b):
            q.grad = None if p.grad is None else p.grad.double()
        want = torch.nn.utils.clip_grad_norm_(b, 5.0)
        keep = [None if p.grad is None else p.grad.clone() for p in a]
        assert mine.step(lambda: 7.0) == 7.0
        ref.step()
        assert abs(float(mine.norm) / float(want) - 1) <= 2 * U
        assert all(p.grad is None if k is None else torch.equal(p.grad, k) for p, k in zip(a, keep))
        for p, q in zip(a, b):
            tol = (t + 1) * U * (4 * q.abs() + 24 * 2 * 3e-3)
            assert bool(((p.detach().double() - q.detach()).abs() <= tol).all())
    assert [mine.state[p]["step"] for p in a] == [12, 12, 12, 8, 12]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_and_loaded_run_goes_on_the_same(bits, dtype, tmp_path):
    from iadmm.optim import AdamW
    a = params(dtype=dtype)
    opt = AdamW(a, lr=1e-2, state_bits=bits, seed=5, max_norm=1.0)
    for t in range(3):
        set_grads(a, t)
        opt.step()
    torch.save({"o": opt.state_dict(), "p": [p.detach() for p in a]}, tmp_path / "s.pt")
    st = torch.load(tmp_path / "s.pt", weights_only=True)
    b = [torch.nn.Parameter(p) for p in st["p"]]
    other = AdamW(b, lr=1.0, state_bits=bits, seed=5, max_norm=1.0)
    other.load_state_dict(st["o"])
    for t in range(3, 6):
        for ps, o in ((a, opt), (b, other)):
            set_grads(ps, t)
            o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            w = other.state[q][k]
            assert torch.equal(v, w) and v.dtype == w.dtype if isinstance(v, torch.Tensor) else v == w
    kind = torch.uint8 if bits == 8 else torch.float32
    assert all(opt.state[p]["exp_avg"].dtype == kind for p in a)


def test_states_of_other_optimizers():
    from iadmm.optim import AdamW
    a = params()
    ref = torch.optim.Adam(a, lr=1e-2)
    set_grads(a, 0)
    ref.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    opt = AdamW(b, lr=1e-2, weight_decay=0.0)
    opt.load_state_dict(copy.deepcopy(ref.state_dict()))
    opt.param_groups[0]["weight_decay"] = 0.0
    for ps, o in ((a, ref), (b, opt)):
        set_grads(ps, 1)
        o.step()
    for p, q in zip(a, b):
        assert bool(((p - q).abs() <= 8 * U * p.abs() + 40 * U * 1e-2).all())
    eight = AdamW(params(), state_bits=8)
    with pytest.raises(ValueError, match="32 bits"):
        eight.load_state_dict(ref.state_dict())
    set_grads(eight.param_groups[0]["params"], 2)
    eight.step()
    wide = AdamW(params(), state_bits=32)
    wide.load_state_dict(eight.state_dict())
    for p, q in zip(eight.param_groups[0]["params"], wide.param_groups[0]["params"]):
        for x, y in zip(eight.moments(p), wide.moments(q)):
            assert torch.equal(x, y) and x.dtype == torch.float32
    with pytest.raises(ValueError, match="maximize"):
        up = torch.optim.AdamW(a, maximize=True)
        up.step()
        opt.load_state_dict(up.state_dict())
    with pytest.raises(ValueError, match="amsgrad"):
        ams = torch.optim.Adam(a, amsgrad=True)
        ams.step()
        opt.load_state_dict(ams.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """The captured step's replays, with eager work of the same kind between them, count on from the eager steps and
    equal the steps of an optimizer that counts on the host, but for the corrections' rounding (2 u of an update);
    8-bit moments are the same codes."""
    from iadmm.optim import AdamW
    a, b = params(), params()
    mine = AdamW(a, lr=1e-2, state_bits=bits, capturable=True, max_norm=2.0)
    host = AdamW(b, lr=1e-2, state_bits=bits, max_norm=2.0)
    with pytest.raises(RuntimeError, match="before the capture"):
        set_grads(a, 0)
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            mine.step()
    for t in range(2):
        for ps, o in ((a, mine), (b, host)):
            set_grads(ps, t)
            o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mine.step()
    for t in range(2, 7):
        set_grads(b, t, scale=0.3 * t)
        for p, q in zip(a, b):
            p.grad.copy_(q.grad)
        graph.replay()
        host.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert int(mine.state[p]["step"]) == host.state[q]["step"] == t + 1
            assert bool(((p - q).abs() <= (t + 1) * U * (4 * p.abs() + 24 * 2e-2)).all())
            assert torch.equal(mine.state[p]["exp_avg_sq"], host.state[q]["exp_avg_sq"])
    saved = mine.state_dict()
    c = [torch.nn.Parameter(p.detach().clone()) for p in a]
    again = AdamW(c, lr=1e-2, state_bits=bits, capturable=True, max_norm=2.0)
    again.load_state_dict(saved)
    for ps, o in ((a, mine), (c, again)):
        set_grads(ps, 9)
        o.step()
    assert all(torch.equal(p, q) and int(again.state[q]["step"]) == 8 for p, q in zip(a, c))


def small_problem(B=3, n=40, mi=14, me=6):
    from iadmm import data, ops
    raw = data.make_qp_batch(n, mi, me, B, first_index=2, device="cuda")
    sc = ops.ruiz_scale(raw["Q"], raw["p"], raw["A0"], raw["zl"], raw["zu"], 10)
    return dict(zip(("Q", "p", "A0", "zl", "zu"), sc[:5])), mi, me


def model_of(m, h, T, seed=3, **kw):
    from models.lstm import LSTM
    torch.manual_seed(seed)
    model = LSTM(m, 2, h, T, "cuda", **kw)
    with torch.no_grad():
        for q in model.parameters():
            q.mul_(3.0).add_(0.01)
    return model


def unroll(model, d, mi, me, T, normalise=None, H_of=lambda H: H):
    import utils
    B, n = d["Q"].shape[0], d["Q"].shape[1]
    m, h = mi + me, model.hidden_dim
    x, y, z = (torch.zeros(B, r, 1, device="cuda") for r in (n, m, m))
    xv = torch.zeros(B, n + m, 1, device="cuda")
    H, C = torch.zeros(B, n + m, h, device="cuda"), torch.zeros(B, n + m, h, device="cuda")
    loss = 0.0
    for t in range(T):
        H = H_of(H)
        if normalise is not None:
            H = normalise(H)
        x, y, z, xv, H, C, _, _, _ = model(t, mi, me, x, y, z, xv, 6e-6, H, C, lb=None, ub=None, **d)
        _, _, l = utils.primal_dual_loss(x, y, z, d["Q"], d["p"], d["A0"])
        loss = loss + l.mean() / T
    return loss, x, H


def test_model_with_layer_norm():
    """A model that normalises equals one that does not with torch's layer norm put before each iteration: the loss,
    the iterate and all gradients to 1e-5 (both sides in fp32, a layer norm apart by a few u; T = 6 iterations); and
    the window's shared gradient sums equal autograd's own (a cloned H starts a chain of its own) bit for bit."""
    d, mi, me = small_problem()
    h, T = 48, 6
    a, b = model_of(mi + me, h, T, layer_norm=True), model_of(mi + me, h, T)
    assert list(a.state_dict()) == list(b.state_dict()) + ["ln_w", "ln_b"]
    assert all(torch.equal(v, a.state_dict()[k]) for k, v in b.state_dict().items())
    w, bias = (torch.nn.Parameter(p.detach().clone()) for p in (a.ln_w, a.ln_b))
    loss_a, x_a, H_a = unroll(a, d, mi, me, T)
    loss_b, x_b, H_b = unroll(b, d, mi, me, T, lambda H: torch.nn.functional.layer_norm(H, (h,), w, bias, 1e-5))
    rel = lambda p, q: float((p.double() - q.double()).norm() / q.double().norm().clamp(min=1e-30))  # noqa: E731
    assert rel(x_a, x_b) < 1e-5 and rel(H_a, H_b) < 1e-5 and abs(float(loss_a) / float(loss_b) - 1) < 1e-5
    loss_a.backward()
    loss_b.backward()
    want = {k: p.grad for k, p in b.named_parameters()} | {"ln_w": w.grad, "ln_b": bias.grad}
    for k, p in a.named_parameters():
        assert rel(p.grad, want[k]) < 1e-5, k
    got = {k: p.grad.clone() for k, p in a.named_parameters()}
    a.zero_grad()
    unroll(a, d, mi, me, T, H_of=lambda H: H.clone())[0].backward()
    for k, p in a.named_parameters():
        assert torch.equal(p.grad, got[k]), k


def test_solver_runs_the_model_with_layer_norm():
    from iadmm import solver
    d, mi, me = small_problem(B=5)
    T = 5
    model = model_of(mi + me, 48, T, layer_norm=True)
    with torch.no_grad():
        _, x, H = unroll(model, d, mi, me, T)
        out = solver.solve(model, d["Q"], d["p"], d["A0"], d["zl"], d["zu"], mi, me, T, 6e-6, scaling=False)
        two = solver.solve(model, d["Q"], d["p"], d["A0"], d["zl"], d["zu"], mi, me, T, 6e-6, scaling=False, lanes=2)
        plain = solver.solve({k: v for k, v in solver.param_dict(model).items() if k in solver.PARAM_NAMES}, d["Q"], d["p"],
                             d["A0"], d["zl"], d["zu"], mi, me, T, 6e-6, scaling=False)
    assert torch.equal(out["x"], x) and torch.equal(out["H"], H)
    assert torch.equal(two["x"], x) and torch.equal(two["H"], H)
    assert not torch.equal(plain["x"], x)
    with pytest.raises(ValueError, match="layer_norm"):
        solver.solve(model, d["Q"], d["p"], d["A0"], d["zl"], d["zu"], mi, me, T, 6e-6, precision="f16x3")


@pytest.mark.parametrize("bits", [32, 8])
def test_training_window_end_to_end(bits):
    """tbptt_batch with the clipped multi-tensor step: every window's packed weights are the stepped ones (the
    parameters' versions rise), two runs end with the same bits, and a capped step moves less than lr each."""
    from iadmm import train
    from iadmm.optim import AdamW
    d, mi, me = small_problem(B=4)
    T = 6
    ends = []
    for _ in range(2):
        model = model_of(mi + me, 48, T, layer_norm=True)
        opt = AdamW(model.parameters(), lr=1e-3, weight_decay=0.0, state_bits=bits, max_norm=0.1)
        before = [p.detach().clone() for p in model.parameters()]
        loss = train.tbptt_batch(model, d, mi, me, 2 * T, T, 6e-6, opt, micro_batch=2)
        assert math.isfinite(loss) and float(opt.norm) > 0
        ends.append([p.detach().clone() for p in model.parameters()])
        assert any(not torch.equal(p, q) for p, q in zip(before, ends[-1]))
        with torch.no_grad():
            _, x, _ = unroll(model, d, mi, me, T)
            fresh = model_of(mi + me, 48, T, layer_norm=True)
            fresh.load_state_dict(model.state_dict())
            assert torch.equal(unroll(fresh, d, mi, me, T)[1], x)
    assert all(torch.equal(p, q) for p, q in zip(*ends))


@pytest.mark.parametrize("extra", [[], ["--state_bits", "8", "--layer_norm"]])
def test_command_trains_resumes_and_tests(extra, tmp_path, capsys):
    import main
    argv = ["--prob_type", "QP", "--num_var", "40", "--num_ineq", "16", "--num_eq", "8", "--outer_T", "6",
            "--truncated_length", "3", "--hidden_dim", "32", "--sigma", "6e-6", "--scaling", "--lr", "0.002",
            "--batch_size", "4", "--data_size", "20", "--val_frac", "0.1", "--test_frac", "0.1", "--eq_tol", "1e9",
            "--ineq_tol", "1e9", "--early_stop_mode", "min", "--synthetic", "--patience", "10", "--optimizer", "adamw",
            "--max_grad_norm", "1.0"] + extra
    whole = main.main(argv + ["--num_epoch", "3", "--save_dir", str(tmp_path / "a")])
    state = str(tmp_path / "resume.pt")
    first = main.main(argv + ["--num_epoch", "2", "--save_dir", str(tmp_path / "b"), "--resume", state])
    rest = main.main(argv + ["--num_epoch", "3", "--save_dir", str(tmp_path / "b"), "--resume", state])
    assert first + rest == whole and len(whole) == 3
    import shutil
    saved = tmp_path / "a" / "lstm" / "params"
    shutil.copy(saved / "QP_40_16_8_6_32.pth", saved / "QP_40_8_16_6_32.pth")  # (the two names of main.py:88, 557)
    reports, _ = main.main(argv + ["--test", "--test_outer_T", "6", "--test_batch_size", "2", "--save_dir", str(tmp_path / "a")])
    assert len(reports) == 1 and "Test_Obj" in capsys.readouterr().out
