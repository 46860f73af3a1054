"""What a copied, pickled or loaded diffrast.optim.AdamW goes on with."""

import copy
import io
import pickle

import pytest
import torch


def seeds(opt):
    return [g["seed"] for g in opt.param_groups]


def saved(o):
    """o through torch.save: plain pickle does not read float8 tensors back, whoever made them."""
    b = io.BytesIO()
    torch.save(o, b)
    b.seek(0)
    return torch.load(b, weights_only=False)


def make(seed, second=None):
    from diffrast import optim

    a, b = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.ones(4))
    return optim.AdamW([dict(params=[a]), dict(params=[b]) if second is None else dict(params=[b], seed=second)], state_bits=8, seed=seed)


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))], ids=["copied", "pickled"])
def test_a_copy_has_the_seed(copied):
    opt = copied(make(7, 9))
    assert opt.seed == 7 and seeds(opt) == [7, 9]
    assert opt.step() is None  # no gradients: nothing


def test_a_state_dict_has_the_seed():
    opt = make(5)
    opt.load_state_dict(make(7, 9).state_dict())
    assert seeds(opt) == [7, 9]
    saved = make(7).state_dict()
    for g in saved["param_groups"]:
        del g["seed"]  # one that was saved without
    opt = make(5)
    opt.load_state_dict(saved)
    assert seeds(opt) == [5, 5]


@pytest.mark.gpu
@pytest.mark.parametrize("copied", [copy.deepcopy, saved, None], ids=["copied", "saved", "loaded"])
def test_a_copy_steps_as_the_original(copied):
    from diffrast import optim

    g = torch.Generator("cuda").manual_seed(0)
    net = torch.nn.Linear(70, 30).cuda()

    def step(net, opt, g):
        for p in net.parameters():
            p.grad = torch.randn(p.shape, device="cuda", generator=g)
        opt.step()

    opt = optim.AdamW(net.parameters(), lr=0.1, state_bits=8, seed=3)
    step(net, opt, g)
    if copied:
        net2, opt2 = copied((net, opt))
    else:
        net2 = copy.deepcopy(net)
        opt2 = optim.AdamW(net2.parameters(), lr=0.1, state_bits=8, seed=4)
        opt2.load_state_dict(opt.state_dict())
    for _ in range(3):
        same = torch.Generator("cuda")
        same.set_state(g.get_state())
        step(net, opt, g)
        step(net2, opt2, same)
    for p, q in zip(net.parameters(), net2.parameters()):
        assert p.data_ptr() != q.data_ptr() and bool(torch.equal(p, q))
        for k in ("exp_avg", "exp_avg_sq"):
            assert bool(torch.equal(opt.state[p][k].view(torch.uint8), opt2.state[q][k].view(torch.uint8)))


def test_load_hooks_see_and_change_what_is_loaded():
    """Pre-hooks' dictionary is what is loaded, in the states' own types, before post-hooks run."""
    from diffrast import optim

    def opt_of(value):
        p = torch.nn.Parameter(torch.zeros(5, dtype=torch.bfloat16))
        opt = optim.AdamW([p])
        opt.state[p] = dict(step=torch.tensor(3), exp_avg=torch.full((5,), value), exp_avg_sq=torch.full((5,), value))
        return opt, p

    source, q = opt_of(1 + 2.0**-20)
    opt, p = opt_of(7.0)
    seen = []

    def doubled(o, d):
        d = copy.deepcopy(d)
        d["state"][0]["exp_avg"] *= 2
        d["param_groups"][0]["lr"] = 0.5
        return d

    opt.register_load_state_dict_pre_hook(doubled)
    opt.register_load_state_dict_post_hook(lambda o: seen.append(o.state[p]["exp_avg"].clone()))
    for _ in range(2):  # nothing of the first load is left for the second
        opt.load_state_dict(source.state_dict())
        s = opt.state[p]
        assert opt.param_groups[0]["lr"] == 0.5 and s["exp_avg"].dtype == torch.float32 and int(s["step"]) == 3
        assert torch.equal(s["exp_avg"], 2 * source.state[q]["exp_avg"]) and torch.equal(s["exp_avg_sq"], source.state[q]["exp_avg_sq"])
        assert s["exp_avg_sq"].data_ptr() != source.state[q]["exp_avg_sq"].data_ptr()
        assert torch.equal(seen.pop(), s["exp_avg"])
    bad = source.state_dict()
    bad["param_groups"][0]["params"] = [0, 1]
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)


@pytest.mark.parametrize("bad", [dict(state_bits=16), dict(seed=-1), dict(seed=1 << 63), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0),
                                 dict(weight_decay=float("nan"))])
def test_a_groups_own_numbers_are_checked(bad):
    """As the optimizer's are, before there are states by them."""
    from diffrast import optim

    t = lambda: torch.nn.Parameter(torch.zeros(3))  # noqa: E731
    with pytest.raises(ValueError):
        optim.AdamW([dict(params=[t()]), dict(params=[t()], **bad)])
    opt = optim.AdamW([t()])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[t()], **bad))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[t()], state_bits=8, lr=torch.tensor(0.5)))
    assert len(opt.param_groups) == 2 and seeds(opt) == [0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_states_under_another_default_type(bits, default):
    from diffrast import optim

    p = torch.nn.Parameter(torch.ones(300, device="cuda", dtype=torch.float32))
    p.grad = torch.ones_like(p)
    opt = optim.AdamW([p], state_bits=bits)
    was = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        opt.step()
    finally:
        torch.set_default_dtype(was)
    kinds = {k: v.dtype for k, v in opt.state[p].items()}
    assert kinds.pop("step") == torch.int64 and bool((p < 1).all())
    assert set(kinds.values()) == ({torch.float32} if bits == 32 else {torch.float32, torch.float8_e4m3fn})
