"""run_mlp refuses modules whose call is more than their class's formula, instead of computing something else (no GPU needed:
what is allowed gets as far as asking for one)."""
import pytest
import torch
import torch.nn as nn

from cafe_amd import _lib
from cafe_amd.linear import run_mlp

X = torch.zeros(3, 5)


def layers():
    return nn.Sequential(nn.Linear(5, 7), nn.ReLU(), nn.Linear(7, 2), nn.Sigmoid())


class Scaled(nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


class Loud(nn.Sequential):
    def forward(self, x):
        return super().forward(x) + 1


class LeakyReLU(nn.ReLU):
    def forward(self, x):
        return nn.functional.leaky_relu(x)


def own_forward(m):
    m.forward = lambda x: x
    return m


def hooked(m, register):
    getattr(m, register)(lambda *a: None)
    return m


CASES = {
    "weight_norm": lambda: nn.Sequential(torch.nn.utils.weight_norm(nn.Linear(5, 7)), nn.ReLU()),
    "parametrized weight_norm": lambda: nn.Sequential(torch.nn.utils.parametrizations.weight_norm(nn.Linear(5, 7)), nn.ReLU()),
    "subclass of Linear": lambda: nn.Sequential(Scaled(5, 7), nn.ReLU()),
    "subclass of an activation": lambda: nn.Sequential(nn.Linear(5, 7), LeakyReLU()),
    "subclass of Sequential": lambda: Loud(nn.Linear(5, 7)),
    "another container": lambda: nn.ModuleList(layers()),
    "forward on a Linear": lambda: nn.Sequential(own_forward(nn.Linear(5, 7))),
    "forward on the Sequential": lambda: own_forward(layers()),
    "forward hook": lambda: nn.Sequential(hooked(nn.Linear(5, 7), "register_forward_hook")),
    "pre-hook": lambda: nn.Sequential(hooked(nn.Linear(5, 7), "register_forward_pre_hook")),
    "backward hook": lambda: nn.Sequential(hooked(nn.Linear(5, 7), "register_full_backward_hook")),
    "hook of an activation": lambda: nn.Sequential(nn.Linear(5, 7), hooked(nn.ReLU(), "register_forward_hook")),
    "a function": lambda: [nn.Linear(5, 7), torch.relu],
    "a gap": lambda: [nn.Linear(5, 7), None],
    "hook of the Sequential": lambda: hooked(layers(), "register_forward_hook"),
}


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("kind", list(CASES))
def test_refused(kind):
    with pytest.raises(ValueError):
        run_mlp(CASES[kind](), X)


def test_global_hooks():
    handle = nn.modules.module.register_module_forward_hook(lambda *a: None)
    try:
        with pytest.raises(ValueError, match="hooks"):
            run_mlp(layers(), X)
    finally:
        handle.remove()


def test_allowed():
    for mods in (layers(), list(layers()), layers()[:-1], nn.Sequential(nn.Linear(5, 7), nn.GELU())):
        with pytest.raises(_lib.CafeError, match="GPU"):
            run_mlp(mods, X)


def test_layers_beside_the_stacks():
    """WDL's wide layer and DCN's last one are modules too."""
    from cafe_amd.ctr_models import CafeCTRHead
    head = CafeCTRHead("wdl", 4, 8, 13, dense_ops="hip")
    hooked(head.wide, "register_forward_pre_hook")
    with pytest.raises(ValueError, match="hooks"):
        head(torch.rand(6, 13), torch.randn(4, 6, 8))


@pytest.mark.gpu
def test_last_layer_of_dcn():
    from cafe_amd.ctr_models import CafeCTRHead
    head = CafeCTRHead("dcn", 4, 8, 13, dense_ops="hip").cuda()
    hooked(head.last_layer, "register_forward_hook")
    for call in (head, head.logits):
        with pytest.raises(ValueError, match="hooks"):
            call(torch.rand(6, 13, device="cuda"), torch.randn(4, 6, 8, device="cuda"))
