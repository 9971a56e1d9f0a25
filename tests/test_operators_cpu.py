"""Layer norm and the optimizer's step without a GPU: what the entry points refuse before anything is launched."""
import array

import pytest
import torch

import iadmm_path  # noqa: F401
from iadmm import _abi, ops


def refused(match, name, *args):
    with pytest.raises(_abi.IadmmError, match=match):
        _abi.call(name, *args)


def test_layer_norm_arguments():
    f = "iadmm_layer_norm_fwd"
    refused("bad argument", f, 4, 0, 0, 0, 16, 8, None, None, 1e-5, 16, None, None, None)      # no columns
    refused("bad argument", f, 4, 8, 3, 3, 16, 8, None, None, 1e-5, 16, None, None, None)      # unknown type
    refused("bad argument", f, 4, 8, 0, 1, 16, 8, None, None, 1e-5, 16, None, None, None)      # bf16 weights, fp32 rows
    refused("bad argument", f, 4, 8, 0, 0, 16, 7, None, None, 1e-5, 16, None, None, None)      # overlapping rows
    refused("bad argument", f, 4, 8, 0, 0, None, 8, None, None, 1e-5, 16, None, None, None)
    refused("bad argument", f, 4, 8, 0, 0, 16, 8, None, None, float("nan"), 16, None, None, None)
    refused("size beyond", f, 1, (1 << 24) + 1, 0, 0, 16, 1 << 40, None, None, 1e-5, 16, None, None, None)
    _abi.call(f, 0, 8, 0, 0, None, 8, None, None, 1e-5, None, None, None, None)                # no rows: nothing to do
    b = "iadmm_layer_norm_bwd"
    need = _abi.lib().iadmm_layer_norm_bwd_ws_bytes(100, 800, 0)
    assert need == 13 * 2 * 800 * 4                                   # 8 rows a workgroup, dw and db of each
    assert _abi.lib().iadmm_layer_norm_bwd_ws_bytes(10 ** 6, 800, 0) == 256 * 2 * 800 * 4
    assert _abi.lib().iadmm_layer_norm_bwd_ws_bytes(0, 800, 0) == 0
    assert _abi.lib().iadmm_layer_norm_bwd_ws_bytes(16, 800, 0) == 0  # one workgroup has all rows
    assert _abi.lib().iadmm_layer_norm_bwd_ws_bytes(17, 800, 0) == 3 * 2 * 800 * 4
    refused("bad argument", b, 100, 800, 0, 0, 16, 800, 16, 800, 16, 16, None, 16, 16, 16, 16, need - 4, None)
    refused("bad argument", b, 100, 800, 0, 0, 16, 800, 16, 800, 16, 16, None, 16, 16, 16, None, need, None)
    refused("misaligned", b, 100, 800, 0, 0, 16, 800, 16, 800, 16, 16, None, 16, 16, 16, 20, need, None)
    refused("bad argument", b, 100, 800, 0, 0, 16, 799, 16, 800, 16, 16, None, 16, 16, 16, 16, need, None)


def record(p=16, g=16, m=16, v=16, e=16, n=4, step=1, slot=0, dtype=0, gdtype=0):
    return array.array("q", [p, g, m, v, e, n, step, slot | dtype << 32 | gdtype << 48])


ALIVE = []  # the records that a call reads by address


def step_args(rec, bits=32, lr=1e-3, lr_dev=None, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, norm=None, most=0.0, steps=None,
              ws=None, nbytes=0):
    ALIVE.append(rec)
    return (len(rec) // 8, rec.buffer_info()[0], bits, lr, lr_dev, b1, b2, eps, wd, norm, most, 0, steps, ws, nbytes, None)


def test_adamw_arguments():
    f, nan = "iadmm_adamw_step", float("nan")
    for rec in (record(p=0), record(g=0), record(m=0), record(v=0), record(n=-1), record(step=0), record(dtype=2),
                record(gdtype=2), record(slot=1 << 31)):
        refused("bad argument", f, *step_args(rec))
    refused("bad argument", f, *step_args(record(e=0), bits=8))
    refused("size beyond", f, *step_args(record(n=(1 << 40) + 1)))
    refused("size beyond", f, *step_args(record(n=1 << 36) + record(n=1)))
    refused("bad argument", f, *step_args(sum((record() for _ in range(49)), array.array("q"))))  # no workspace
    for kw in (dict(bits=16), dict(lr=-1.0), dict(lr=nan), dict(b1=1.0), dict(b2=nan), dict(eps=-1.0), dict(wd=-0.1),
               dict(norm=16, most=0.0), dict(lr_dev=16), dict(steps=16), dict(steps=16, ws=16, nbytes=64)):
        refused("bad argument", f, *step_args(record(), **kw))
    refused("misaligned", f, *step_args(record(), steps=16, ws=20, nbytes=72))
    _abi.call(f, *step_args(record(p=0, g=0, m=0, v=0, n=0)))  # an empty tensor: nothing to do
    n = "iadmm_grad_norm"
    grad = array.array("q", [16, 4, 0])
    need = _abi.lib().iadmm_grad_norm_ws_bytes(1)
    for rec in (array.array("q", [0, 4, 0]), array.array("q", [16, -1, 0]), array.array("q", [16, 4, 2])):
        refused("bad argument", n, 1, rec.buffer_info()[0], 16, 16, need, None)
    refused("bad argument", n, 1, grad.buffer_info()[0], None, 16, need, None)
    refused("bad argument", n, 1, grad.buffer_info()[0], 16, 16, need - 8, None)
    refused("misaligned", n, 1, grad.buffer_info()[0], 16, 24, need, None)
    refused("bad argument", "iadmm_adamw_decode8", 4, 16, 16, 16, 2, 16, 16, None)
    refused("bad argument", "iadmm_adamw_decode8", 4, 16, None, 16, 0, 16, 16, None)


def test_no_cpu_path():
    x = torch.zeros(3, 8)
    for call in (lambda: ops.layer_norm(x), lambda: ops.layer_norm_bwd(x, x, x[:, 0], x[:, 0]), lambda: ops.grad_norm([x]),
                 lambda: ops.adamw_step([x], [x.clone()], [x.clone()], [x.clone()], 1),
                 lambda: ops.adamw_decode8(x.byte(), x.byte(), torch.zeros(1, 2, dtype=torch.int8))):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()


def test_lists_are_checked():
    x = torch.zeros(3, 8)
    for args, error in ((([x], [x], [x], [], 1), ValueError), (([x.half()], [x], [x], [x], 1), TypeError)):
        with pytest.raises(error):
            ops.adamw_step(*args)
    with pytest.raises(ValueError, match="belong together"):
        ops.adamw_step([x], [x], [x], [x], 1, max_norm=1.0)
    with pytest.raises(ValueError, match="at least one"):
        ops.grad_norm([None])
    with pytest.raises(TypeError):
        ops.grad_norm([x.half()])
    with pytest.raises(ValueError, match="contiguous"):
        ops.grad_norm([x.t()])
    ops.adamw_step([x], [None], [x], [x], 1)  # no gradient: nothing to do


def test_optimizer_arguments():
    from iadmm.optim import AdamW
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in (dict(state_bits=16), dict(max_norm=0.0), dict(lr=-1.0), dict(lr=torch.tensor(1.0)), dict(betas=(1.0, 0.9)),
               dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            AdamW(p, **kw)
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float16))])
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([torch.nn.Parameter(torch.zeros(3, 4).t())])
    opt = AdamW(p)
    assert opt.step() is None and not opt.state  # no gradient: nothing to do
    p[0].grad = torch.ones(3)
    with pytest.raises(ValueError, match="no CPU fallback"):
        opt.step()


def test_command_line_options():
    import main
    base = ["--lr", "0.1"]
    args = main.parse_args(base)
    assert args.optimizer == "adam" and not args.layer_norm
    p = [torch.nn.Parameter(torch.zeros(3))]
    assert type(main.make_optimizer(args, p)) is torch.optim.Adam
    args = main.parse_args(base + ["--optimizer", "adamw", "--state_bits", "8", "--max_grad_norm", "2", "--weight_decay", "0.1"])
    opt = main.make_optimizer(args, p)
    assert (opt.state_bits, opt.max_norm, opt.defaults["lr"], opt.defaults["weight_decay"]) == (8, 2.0, 0.1, 0.1)
    for extra in (["--state_bits", "8"], ["--max_grad_norm", "1"]):
        with pytest.raises(SystemExit):
            main.make_optimizer(main.parse_args(base + extra), p)


def test_model_parameters_with_layer_norm():
    """The reference's 16 parameters are drawn the same with and without; without, the model is the reference's."""
    from models.lstm import LSTM
    from iadmm import solver
    models = []
    for on in (False, True):
        torch.manual_seed(1)
        models.append(LSTM(4, 2, 8, 3, "cpu", layer_norm=on))
    plain, normed = models
    assert list(normed.state_dict()) == list(plain.state_dict()) + ["ln_w", "ln_b"]
    assert all(torch.equal(v, normed.state_dict()[k]) for k, v in plain.state_dict().items())
    assert list(solver.param_dict(plain)) == list(solver.PARAM_NAMES)
    assert list(solver.param_dict(normed)) == list(solver.PARAM_NAMES) + list(solver.LN_NAMES)
    assert list(solver.param_dict(dict(solver.param_dict(normed)))) == list(solver.PARAM_NAMES) + list(solver.LN_NAMES)
