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


@pytest.mark.parametrize("bad,error", [(lambda: torch.nn.Parameter(torch.zeros(3, dtype=torch.float16)), TypeError),
                                       (lambda: torch.nn.Parameter(torch.zeros(3, 4).t()), ValueError)])
def test_a_refused_group_is_not_added(bad, error):
    opt = AdamW([parameter()])
    p = bad()
    with pytest.raises(error):
        opt.add_param_group(dict(params=(q for q in (parameter(2), p))))
    assert len(opt.param_groups) == 1
    p.grad = torch.ones_like(p)
    assert opt.step() is None                       # the refused parameter is not the optimizer's
    opt.add_param_group(dict(params=[parameter(2)], lr=0.1))
    assert [g["lr"] for g in opt.param_groups] == [1e-3, 0.1]


def stepped(kind, **kw):
    """A torch optimizer after one step, and a copy of its parameter."""
    p = parameter()
    opt = kind([p], **kw)
    p.grad = torch.ones(3)
    opt.step()
    return opt, torch.nn.Parameter(p.detach().clone())


def test_a_decay_inside_the_gradient_does_not_become_a_decoupled_one():
    """torch.optim.Adam's weight decay enters the moments; AdamW's does not."""
    ref, p = stepped(torch.optim.Adam, weight_decay=0.1)
    opt = AdamW([p], lr=0.25)
    with pytest.raises(ValueError, match="decoupled"):
        opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and not opt.state
    for kind, kw in ((torch.optim.Adam, {}), (torch.optim.Adam, dict(weight_decay=0.1, decoupled_weight_decay=True)),
                     (torch.optim.AdamW, dict(weight_decay=0.1))):
        ref, p = stepped(kind, **kw)
        opt = AdamW([p], lr=0.25)
        opt.load_state_dict(ref.state_dict())
        assert opt.param_groups[0]["weight_decay"] == kw.get("weight_decay", 0.0)
        assert torch.equal(opt.state[p]["exp_avg"], next(iter(ref.state.values()))["exp_avg"]) and opt.state[p]["step"] == 1
        opt.param_groups[0]["weight_decay"] = 0.3  # what a program sets from here on is AdamW's, and loads again
        again = AdamW([torch.nn.Parameter(p.detach().clone())])
        again.load_state_dict(opt.state_dict())
        assert again.param_groups[0]["weight_decay"] == 0.3


@pytest.mark.parametrize("bits", [8, 32])
def test_codes_that_are_none_are_refused_before_anything_is_loaded(bits):
    def state(codes=torch.uint8, exps=torch.int8, blocks=2):
        one = dict(step=3, exp_avg=torch.zeros(300, dtype=codes), exp_avg_sq=torch.zeros(300, dtype=codes),
                   exponents=torch.zeros(blocks, 2, dtype=exps))
        return dict(state={0: one}, param_groups=[dict(opt.param_groups[0], params=[0], lr=0.5)])
    opt = AdamW([parameter(300)], state_bits=bits)
    for kw in (dict(codes=torch.float32), dict(exps=torch.float32), dict(blocks=1), dict(blocks=3)):
        with pytest.raises(ValueError, match="8-bit moments"):
            opt.load_state_dict(state(**kw))
        assert not opt.state and opt.param_groups[0]["lr"] == 1e-3
    if bits == 8:
        opt.load_state_dict(state())
        assert opt.state[opt.param_groups[0]["params"][0]]["exponents"].shape == (2, 2)


def optimizer_of(kind, bits):
    """main.make_optimizer's, with a state as after one step."""
    import main
    args = main.parse_args(["--lr", "0.1", "--optimizer", kind, "--state_bits", str(bits)])
    opt = main.make_optimizer(args, [parameter()])
    p = opt.param_groups[0]["params"][0]
    if kind == "adamw":
        opt._state(p)["step"] = 1
    else:
        p.grad = torch.ones(3)
        opt.step()
    return opt


@pytest.mark.parametrize("older", [False, True])
@pytest.mark.parametrize("wrote", [("adam", 32), ("adamw", 32), ("adamw", 8)])
@pytest.mark.parametrize("reads", [("adam", 32), ("adamw", 32), ("adamw", 8)])
def test_resume_goes_on_with_the_optimizer_that_wrote_the_state(wrote, reads, older, tmp_path):
    """``older``: a file from before the optimizer was named in it, where Adam's entries alone tell nothing."""
    import main
    from utils import EarlyStopping
    path = str(tmp_path / "resume.pt")
    main.save_resume_state(path, torch.nn.Linear(1, 1), optimizer_of(*wrote), 0, EarlyStopping(str(tmp_path / "m.pth")))
    st = torch.load(path, weights_only=True)
    if older:
        del st["optimizer_kind"]
    if wrote == reads or (older and wrote[0] == "adam"):
        main.check_resumed_optimizer(path, st, optimizer_of(*reads))
    else:
        with pytest.raises(SystemExit, match=f"--optimizer {wrote[0]} --state_bits {wrote[1]}"):
            main.check_resumed_optimizer(path, st, optimizer_of(*reads))


def weights_file(path, layer_norm):
    from models.lstm import LSTM
    path.parent.mkdir(parents=True, exist_ok=True)
    torch.save(LSTM(4, 2, 8, 3, "cpu", layer_norm=layer_norm).state_dict(), path)


@pytest.mark.parametrize("held", [False, True])
def test_weights_of_the_other_kind_of_model_are_not_written_over(held, tmp_path):
    """The file names are the reference's for both kinds: the run ends before it touches a device or the file."""
    import main
    argv = ["--prob_type", "QP", "--num_var", "5", "--num_ineq", "3", "--num_eq", "1", "--outer_T", "3", "--hidden_dim", "8",
            "--lr", "0.1", "--synthetic", "--save_dir", str(tmp_path)]
    other = [] if held else ["--layer_norm"]
    path = tmp_path / "lstm" / "params" / "QP_5_3_1_3_8.pth"
    weights_file(path, held)
    before = path.read_bytes()
    with pytest.raises(SystemExit, match="without --layer_norm" if not held else "with --layer_norm"):
        main.main(argv + other)
    assert path.read_bytes() == before
    args = main.parse_args(argv)
    assert main.train_path(args) == str(path)
    main.check_weights_kind(str(path), held)                      # its own kind goes on over it
    for kind in (False, True):
        main.check_weights_kind(str(tmp_path / "none.pth"), kind)
        (tmp_path / "cut.pth").write_bytes(before[:100])          # what an interrupted run left
        main.check_weights_kind(str(tmp_path / "cut.pth"), kind)
