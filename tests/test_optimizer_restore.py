"""What a checkpoint's optimizer state may be loaded into (no GPU needed: nothing is stepped)."""
import pytest
import torch

from cafe_amd import train


def optimizer(name, lr=0.1, n=3):
    return train.make_optimizer(name, [torch.nn.Parameter(torch.zeros(4)) for _ in range(n)], lr)


def stepped(name, **kw):
    """As after a step, without one."""
    opt = optimizer(name, **kw)
    for p in opt.param_groups[0]["params"]:
        if name == "sgd":
            opt.state[p] = {}
        else:
            opt._init_state(p, opt.param_groups[0])["step"] = 5
            opt.state[p]["master"] = torch.full((4,), 7.0)
    return opt


@pytest.mark.parametrize("name", ["adamw", "adamw8bit"])
def test_its_own(name):
    opt = optimizer(name)
    train.restore_optimizer(opt, stepped(name).state_dict())
    assert all(s["step"] == 5 and (s["master"] == 7).all() for s in opt.state.values()) and len(opt.state) == 3


@pytest.mark.parametrize("saved,into", [("adamw", "sgd"), ("adamw8bit", "adamw"), ("adamw", "adamw8bit")])
def test_another_ones(saved, into):
    with pytest.raises(ValueError, match="another"):
        train.restore_optimizer(optimizer(into), stepped(saved).state_dict())


def test_other_parameters():
    with pytest.raises(ValueError, match="another"):
        train.restore_optimizer(optimizer("adamw"), stepped("adamw", n=4).state_dict())


def test_none():
    """The parameters were loaded: masters and moments of others are dropped."""
    for name in ("adamw", "adamw8bit", "sgd"):
        opt = stepped(name)
        train.restore_optimizer(opt, None)
        assert not opt.state


@pytest.mark.gpu
def test_a_resumed_run_steps_as_the_command_line_says(tmp_path):
    common = ["--model", "wdl", "--workload", "cfg5", "--mini-batch-size", "128", "--dense-ops", "hip", "--optimizer", "adamw"]
    path = str(tmp_path / "ck.pt")
    train.main(common + ["--num-batches", "2", "--dense-learning-rate", "0.01", "--save-model", path])
    seen = []
    make = train.make_optimizer

    def spy(*args):
        seen.append(make(*args))
        return seen[-1]
    train.make_optimizer = spy
    try:
        train.main(common + ["--num-batches", "3", "--dense-learning-rate", "0.002", "--weight-decay", "0.03", "--load-model", path])
    finally:
        train.make_optimizer = make
    g, = seen[0].param_groups
    assert (g["lr"], g["weight_decay"]) == (0.002, 0.03) and {s["step"] for s in seen[0].state.values()} == {3}
