"""cafe_amd.interact and cafe_amd.adamw refuse what they have no kernel for before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

from cafe_amd import _lib
from cafe_amd.adamw import AdamW, Moment8, adamw_step, adamw_tick, moment8_values
from cafe_amd.interact import dot_interaction

EMB, X = torch.zeros(3, 4, 8), torch.zeros(4, 8)


@pytest.mark.parametrize("x,emb,kw", [
    (X, EMB[0], {}),                                            # not [F, B, D]
    (torch.zeros(5, 8), EMB, {}),                               # another batch
    (torch.zeros(4, 9), EMB, {}),                               # another width
    (X.double(), EMB, {}),
    (X, EMB.half(), {}),                                        # rows narrower than the result
    (X.half(), EMB.bfloat16(), {}),
    (None, EMB, dict(dtype=torch.int32)),
    (X, EMB, dict(dtype=torch.float16)),                        # x is not of the result's type
    (None, torch.zeros(0, 4, 8), {}),                           # no rows
    (None, torch.zeros(129, 1, 1), {}),                         # too many
    (torch.zeros(1, 1), torch.zeros(128, 1, 1), {}),
])
def test_interaction_arguments(x, emb, kw):
    with pytest.raises(ValueError):
        dot_interaction(x, emb, **kw)


def test_no_cpu_path():
    with pytest.raises(_lib.CafeError):
        dot_interaction(X, EMB)
    p = torch.zeros(5)
    with pytest.raises(_lib.CafeError):
        adamw_step([p], [p.clone()], [p.clone()], [p.clone()], step=1, lr=0.1)
    with pytest.raises(_lib.CafeError):
        moment8_values([Moment8.zeros(5, "cpu")], [])
    with pytest.raises(_lib.CafeError):
        adamw_tick(torch.zeros(1, dtype=torch.int64), torch.zeros(3), lr=0.1)
    q = torch.nn.Parameter(torch.zeros(5))
    q.grad = torch.zeros(5)
    with pytest.raises(_lib.CafeError):
        AdamW([q]).step()


def _lists(n=2, shape=(4, 3), dtype=torch.float32):
    return [[torch.zeros(shape, dtype=dtype if k < 2 else torch.float32) for _ in range(n)] for k in range(4)]


def test_adamw_lists():
    p, g, m, v = _lists()
    e = Moment8.zeros(12, "cpu")
    bad = [
        (p, g[:1], m, v, {}),                                               # lengths
        (p, g, m, v, dict(masters=p[:1])),
        ([p[0], p[0]], g, m, v, {}),                                        # the same parameter twice
        ([p[0], p[1].double()], g, m, v, {}),                               # mixed types
        (p, [g[0], g[1].half()], m, v, {}),
        (p, [g[0], g[1].t()], m, v, {}),                                    # another shape
        (p, [g[0], g[1].to_sparse()], m, v, {}),
        ([p[0], torch.zeros(3, 4).t()], g, m, v, {}),                       # not contiguous
        (p, g, [m[0], m[1].half()], v, {}),
        (p, g, m, [v[0], v[1][:2]], {}),
        (p, g, [e, m[1]], v, {}),                                           # 8 and 32 bits mixed
        (p, g, [m[0], e], v, {}),
        (p, g, m, [e, e], {}),
        (p, g, [e, Moment8.zeros(13, "cpu")], [e, e], {}),                  # wrong number of codes
        (p, g, [e, Moment8(e.codes, torch.ones(2, dtype=torch.uint8))], [e, e], {}),
        (p, g, m, v, dict(masters=[p[0].clone(), p[1].half()])),
        ([t.double() for t in p], [t.double() for t in g], m, v, {}),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            adamw_step(*args[:4], step=1, lr=0.1, **args[4])
    assert adamw_step([], [], [], [], step=1, lr=0.1) is None
    assert moment8_values([], []) == ([], [])


def test_optimizer_arguments():
    q = torch.nn.Parameter(torch.zeros(5))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)),
               dict(betas=(0.9,)), dict(lr=torch.tensor(0.1))):
        with pytest.raises(ValueError):
            AdamW([q], **kw)
    q.grad = torch.zeros(5).to_sparse()
    with pytest.raises(ValueError):
        AdamW([q]).step()


def test_c_entry_points():
    """Bad sizes, codes, strides and null pointers come back as errors before any HIP call."""
    L = _lib.load()
    p = ctypes.c_void_p(4096)                                   # never read

    def fwd(x=p, ldx=8, emb=p, sf=32, sb=8, batch=4, fields=3, dim=8, te=0, t=0, out=p, ldo=14):
        return L.cafe_interact_fwd_dev(x, ldx, emb, sf, sb, batch, fields, dim, 0, te, t, out, ldo, None)

    for kw in (dict(emb=None), dict(out=None), dict(ldo=13), dict(batch=-1), dict(dim=-1), dict(fields=-1), dict(fields=128),
               dict(x=None, fields=0), dict(x=None, fields=1 << 20), dict(te=1), dict(te=3), dict(t=-1), dict(ldx=-1), dict(sf=-1), dict(sb=-1)):
        assert fwd(**kw) != 0, kw
        assert L.cafe_last_error()
    assert fwd(batch=0, out=None, emb=None) == 0

    def bwd(dout=p, x=p, emb=p, batch=4, fields=3, dim=8, te=0, t=0, dx=p, lddx=8, demb=p, dsb=8):
        return L.cafe_interact_bwd_dev(dout, 14, x, 8, emb, 32, 8, batch, fields, dim, 0, te, t, dx, lddx, demb, 32, dsb, None)

    for kw in (dict(dout=None), dict(emb=None), dict(x=None), dict(lddx=7), dict(dsb=7), dict(fields=200), dict(batch=-2), dict(te=2, t=1)):
        assert bwd(**kw) != 0, kw
    assert bwd(x=None, dx=None, demb=None) == 0

    def adam(cols, count=1, t=0, bits=32, lr=0.1, b1=0.9, b2=0.99, eps=0.0, wd=0.0, step=1):
        table = (ctypes.c_int64 * len(cols))(*cols) if cols is not None else None
        return L.cafe_adamw_dev(table, count, t, bits, lr, b1, b2, eps, wd, step, None, None)

    ok = [4096, 4096, 4096, 4096, 0, 0, 0, 0]                   # no values: nothing to do
    assert adam(ok) == 0
    for kw in (dict(count=-1), dict(t=3), dict(bits=16), dict(lr=-1.0), dict(lr=float("nan")), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0),
               dict(wd=-1.0), dict(step=0)):
        assert adam(ok, **kw) != 0, kw
    assert adam(None) != 0
    assert adam([0, 4096, 4096, 4096, 0, 0, 0, 5]) != 0         # null pointers, negative size
    assert adam([4096, 4096, 4096, 4096, 0, 0, 0, 5], bits=8) != 0
    assert adam([4096, 4096, 4096, 4096, 0, 0, 0, -5]) != 0
    assert L.cafe_adamw_tick_dev(None, None, 0.1, 0.9, 0.99, 0.0, p, None) != 0
    assert L.cafe_adamw_tick_dev(p, None, 0.1, 1.5, 0.99, 0.0, p, None) != 0
    assert L.cafe_moment8_values_dev(None, 1, None) != 0
    assert L.cafe_moment8_values_dev((ctypes.c_int64 * 5)(0, 4096, 4096, 3, 0), 1, None) != 0
    assert L.cafe_moment8_values_dev((ctypes.c_int64 * 5)(4096, 4096, 4096, -3, 0), 1, None) != 0


def test_nothing_is_listed_twice():
    z = lambda: torch.zeros(5)                                                         # noqa: E731
    p, m = z(), z()
    for lists in (([p, p], [z(), z()], [z(), z()], [z(), z()]), ([z(), z()], [z(), z()], [m, m], [z(), z()]),
                  ([z(), z()], [z(), z()], [m, z()], [z(), m])):
        with pytest.raises(ValueError, match="twice"):
            adamw_step(*lists, step=1, lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([z(), z()], [z(), z()], [z(), z()], [z(), z()], step=1, lr=0.1, masters=[m, m])


def test_the_step_count_follows_a_group_to_another_device():
    opt = AdamW([torch.nn.Parameter(torch.zeros(3))], capturable=True)
    saved = opt.state_dict()
    saved["param_groups"][0]["device_step"] = {"cuda:5": 7}
    opt.load_state_dict(saved)
    assert list(opt.param_groups[0]["device_step"]) == ["cpu"]
    assert opt.state_dict()["param_groups"][0]["device_step"] == {"cpu": 7}
