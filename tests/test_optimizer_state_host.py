"""CPU-only checks of what ``train.AdamW`` does with saved states: what fits is taken over whole, what does
not is refused before anything of the optimizer is replaced.  Nothing here takes a step."""

import copy

import pytest
import torch

SIZES = [(6, 50), (7,)]


@pytest.fixture(scope="module")
def AdamW(built_lib):
    from unirl_amd.train import AdamW

    return AdamW


def params(dtype=torch.float32, device="cpu"):
    return [torch.nn.Parameter(torch.zeros(s, dtype=dtype, device=device)) for s in SIZES]


def saved_state(opt, steps, bits=32, master=False):
    """A state as ``opt`` would have it after ``steps`` (one number per parameter, None: never a gradient)."""
    sd = copy.deepcopy(opt.state_dict())
    base = 0
    for i, (p, n) in enumerate(zip([p for g in opt.param_groups for p in g["params"]], steps)):
        blocks = -(-p.numel() // 256)
        if n is not None:
            dtype = torch.float32 if bits == 32 else torch.uint8
            s = {"step": n, "index_base": base}
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.arange(p.numel()).view(p.shape).to(dtype)
                if bits == 8:
                    s[name + "_scale"] = torch.full((blocks,), 100, dtype=torch.uint8)
            if master:
                s["master"] = torch.full(p.shape, 0.5)
            sd["state"][i] = s
        base += 256 * blocks
    return sd


def same(a, b):
    if isinstance(a, dict):
        return isinstance(b, dict) and a.keys() == b.keys() and all(same(a[k], b[k]) for k in a)
    if isinstance(a, (list, tuple)):
        return len(a) == len(b) and all(same(x, y) for x, y in zip(a, b))
    if isinstance(a, torch.Tensor):
        return isinstance(b, torch.Tensor) and a.dtype == b.dtype and torch.equal(a, b)
    return a == b


def test_a_fitting_state_is_taken_over_whole(AdamW):
    for bits in (32, 8):
        opt = AdamW(params(torch.bfloat16), state_bits=bits, master_weights=True)
        sd = saved_state(opt, [4, None], bits, master=True)
        sd["param_groups"][0]["lr"] = 0.25
        opt.load_state_dict(sd)
        assert same(opt.state_dict(), sd)
        assert all(t.dtype == sd["state"][0][k].dtype and t is not sd["state"][0][k]
                   for k, t in opt.state[opt.param_groups[0]["params"][0]].items() if isinstance(t, torch.Tensor))
        assert opt._next_base == 512


def test_hooks_see_and_change_what_is_loaded(AdamW):
    opt = AdamW(params())
    called = []

    def before(o, sd):
        sd = copy.deepcopy(sd)
        sd["state"][0]["step"] = 9
        return sd

    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(lambda o: called.append(dict(o.state[o.param_groups[0]["params"][0]])))
    opt.load_state_dict(saved_state(opt, [4, 4]))
    assert called[0]["step"] == 9 and opt.state[opt.param_groups[0]["params"][0]]["step"] == 9


def refused(sd):
    """Variants of ``sd`` that do not fit, by name."""
    def change(f):
        c = copy.deepcopy(sd)
        f(c)
        return c

    def pop(key):
        return lambda c: c["state"][1].pop(key)

    def put(key, value):
        return lambda c: c["state"][1].update({key: value})

    return {
        "no index_base": change(pop("index_base")), "no step": change(pop("step")), "no second moment": change(pop("exp_avg_sq")),
        "another shape": change(put("exp_avg_sq", torch.zeros(8))), "another dtype": change(put("exp_avg", torch.zeros(7).bfloat16())),
        "not a tensor": change(put("exp_avg", 0.0)), "unaligned base": change(put("index_base", 100)),
        "a master of another shape": change(put("master", torch.zeros(8))),
        "a group less": change(lambda c: c["param_groups"].pop()),
        "a parameter less": change(lambda c: c["param_groups"][0]["params"].pop()),
        "no seed": change(lambda c: c["param_groups"][0].pop("seed")),
        "betas out of range": change(lambda c: c["param_groups"][0].update(betas=(1.0, 0.9))),
    }


def test_a_refused_state_leaves_the_optimizer_as_it_was(AdamW):
    ps = params()
    opt = AdamW(ps, lr=1e-2)
    opt.load_state_dict(saved_state(opt, [3, 3]))
    before = copy.deepcopy(opt.state_dict())
    sd = saved_state(opt, [5, 5])
    sd["param_groups"][0]["lr"] = 1.0
    plain = torch.optim.AdamW(params())
    for p in plain.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    plain.step()
    for name, bad in {**refused(sd), "torch's AdamW": plain.state_dict()}.items():
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
            pytest.fail(f"{name} was not refused")
        assert same(opt.state_dict(), before), name
        assert [p is q for p, q in zip(opt.param_groups[0]["params"], ps)] == [True, True]
    eight = AdamW(params(), state_bits=8)
    with pytest.raises(ValueError, match="saved moments"):
        eight.load_state_dict(sd)
    short = saved_state(eight, [1, 1], 8)
    short["state"][0]["exp_avg_scale"] = torch.zeros(1, dtype=torch.uint8)
    with pytest.raises(ValueError, match="exp_avg_scale"):
        eight.load_state_dict(short)
    assert not eight.state


def test_the_count_of_steps_moves_between_host_and_device(AdamW):
    """Without ``capturable`` each parameter counts, with it the group does, on the device: a state saved
    one way and loaded the other goes on counting."""
    host, dev = AdamW(params()), AdamW(params(), capturable=True)
    dev.load_state_dict(saved_state(host, [5, 5]))
    step = dev.param_groups[0]["step"]
    assert step.dtype == torch.int64 and step.shape == () and int(step) == 5
    assert [dev.state[p]["step"] for p in dev.param_groups[0]["params"]] == [0, 0]  # one call for all of a group
    back = AdamW(params())
    back.load_state_dict(dev.state_dict())
    assert back.param_groups[0]["step"] is None
    assert [back.state[p]["step"] for p in back.param_groups[0]["params"]] == [5, 5]
    # the same way round nothing changes, and the copy counts alone
    again = AdamW(params(), capturable=True)
    again.load_state_dict(dev.state_dict())
    step.add_(1)
    assert int(again.param_groups[0]["step"]) == 5
    one = AdamW(params())
    one.load_state_dict(saved_state(one, [5, 2]))
    assert [one.state[p]["step"] for p in one.param_groups[0]["params"]] == [5, 2]


def test_counts_that_one_number_cannot_hold(AdamW):
    dev = AdamW(params(), capturable=True)
    with pytest.raises(ValueError, match="number of steps per group"):
        dev.load_state_dict(saved_state(AdamW(params()), [5, 2]))
    assert not dev.state and dev.param_groups[0]["step"] is None
    # a parameter that never had a gradient has no state, and groups count apart
    dev.load_state_dict(saved_state(AdamW(params()), [5, None]))
    assert int(dev.param_groups[0]["step"]) == 5
    def two(**kw):
        return AdamW([{"params": [p]} for p in params()], **kw)
    dev = two(capturable=True)
    dev.load_state_dict(saved_state(two(), [5, 2]))
    assert [int(g["step"]) for g in dev.param_groups] == [5, 2]
    fresh = two(capturable=True)
    fresh.load_state_dict(saved_state(two(), [None, None]))
    assert [g["step"] for g in fresh.param_groups] == [None, None]


def test_how_a_state_is_held_stays_the_optimizers_choice(AdamW):
    """Bits and masters that differ are refused where a state has them, and never overwritten."""
    def build(**kw):
        return AdamW(params(torch.bfloat16), **kw)
    for mine, theirs in ((True, False), (False, True)):
        opt = build(master_weights=mine)
        with pytest.raises(ValueError, match="master"):
            opt.load_state_dict(saved_state(build(master_weights=theirs), [2, 2], master=theirs))
        assert opt.param_groups[0]["master_weights"] is mine and not opt.state
    # before its first step an optimizer has no state that could differ
    opt = build(master_weights=True, state_bits=8)
    opt.load_state_dict(build(lr=0.5).state_dict())
    assert (opt.param_groups[0]["master_weights"], opt.param_groups[0]["state_bits"], opt.param_groups[0]["lr"]) == (True, 8, 0.5)
    # fp32 parameters have no masters under either setting
    opt = AdamW(params(), master_weights=True)
    opt.load_state_dict(saved_state(AdamW(params()), [2, 2]))
    assert opt.param_groups[0]["master_weights"] is True and len(opt.state) == 2


def test_a_tensor_rate_comes_to_the_parameters(AdamW):
    """A checkpoint mapped to the CPU holds its rate there; the step needs it where the parameters are.
    (The meta device stands for another one.)"""
    for capturable in (True, False):
        opt = AdamW(params(device="meta"), capturable=capturable)
        sd = copy.deepcopy(opt.state_dict())
        sd["param_groups"][0]["lr"] = torch.tensor(0.5)
        opt.load_state_dict(sd)
        lr = opt.param_groups[0]["lr"]
        if capturable:
            assert lr.device.type == "meta" and lr.dtype == torch.float32
        else:
            assert lr == 0.5 and isinstance(lr, float)


def held(opt):
    """Every tensor that a captured step of ``opt`` would read or write beside parameters and gradients."""
    return [t for p in opt.param_groups[0]["params"] for t in opt.state[p].values() if isinstance(t, torch.Tensor)] + [
        g[k] for g in opt.param_groups for k in ("step", "lr") if isinstance(g[k], torch.Tensor)] + list(opt._controls.values())


def test_what_a_captured_step_holds_is_written_in_place(AdamW):
    lr = torch.tensor(0.25)
    opt = AdamW(params(torch.bfloat16), lr=lr, state_bits=8, master_weights=True, capturable=True)
    opt._controls[0] = torch.zeros(32, dtype=torch.uint8)
    opt.load_state_dict(saved_state(opt, [3, 3], 8, master=True))
    before = held(opt)
    assert len(before) == 2 * 5 + 3
    sd = saved_state(opt, [4, 4], 8, master=True)
    sd["param_groups"][0].update(lr=torch.tensor(0.125), step=torch.tensor(7))
    sd["state"][1]["exp_avg"] += 1
    opt.load_state_dict(sd)
    assert all(a is b for a, b in zip(held(opt), before)) and lr == 0.125
    assert int(opt.param_groups[0]["step"]) == 7
    assert torch.equal(opt.state[opt.param_groups[0]["params"][1]]["exp_avg"], sd["state"][1]["exp_avg"])
    # its own tensors, the two parameters' masters exchanged: read before they are written
    ps = opt.param_groups[0]["params"]
    a = AdamW([ps[0], torch.nn.Parameter(ps[0].detach().clone())], capturable=True, master_weights=True)
    a.load_state_dict(saved_state(a, [1, 1], master=True))
    mine = a.state_dict()
    mine["state"][1]["master"].fill_(9.0)
    mine["state"] = {0: dict(mine["state"][1]), 1: dict(mine["state"][0])}
    a.load_state_dict(mine)
    assert [float(a.state[p]["master"].mean()) for p in a.param_groups[0]["params"]] == [9.0, 0.5]
    # a state from before the first step: zeros, and masters as the parameters are
    with torch.no_grad():
        ps[0].fill_(2.0)
    before = held(opt)
    opt.load_state_dict(AdamW(params(torch.bfloat16), lr=0.5, state_bits=8, master_weights=True, capturable=True).state_dict())
    assert all(a is b for a, b in zip(held(opt), before)) and lr == 0.5
    s = opt.state[ps[0]]
    assert int(opt.param_groups[0]["step"]) == 0 and bool((s["master"] == 2.0).all())
    assert not any(s[k].any() for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"))
    bases = [opt.state[p]["index_base"] for p in ps]
    assert len(set(bases)) == 2 and opt._next_base == 512 + 256


def test_groups_that_share_a_tensor_rate_load_rates_of_their_own(AdamW):
    lr = torch.tensor(0.25)
    opt = AdamW([{"params": [p]} for p in params()], lr=lr, capturable=True)
    sd = copy.deepcopy(opt.state_dict())
    sd["param_groups"][0]["lr"], sd["param_groups"][1]["lr"] = 0.5, torch.tensor(0.125)
    opt.load_state_dict(sd)
    assert [float(g["lr"]) for g in opt.param_groups] == [0.5, 0.125] and lr == 0.25
    assert all(isinstance(g["lr"], torch.Tensor) for g in opt.param_groups)


def test_moments_of_a_parameter_without_a_state(AdamW):
    """Asking leaves nothing behind: an empty entry would be saved with the others."""
    ps = params()
    opt = AdamW(ps)
    with pytest.raises(ValueError, match="no state"):
        opt.moments(ps[0])
    assert not opt.state and opt.state_dict()["state"] == {}


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate parameters")
def test_a_refused_group_is_not_added(AdamW):
    opt = AdamW(params())
    p = torch.nn.Parameter(torch.zeros(4, 6))
    for bad in (dict(params=[p], state_bits=4), dict(params=[p], betas=(1.0, 0.9)), dict(params=[p, p]),
                dict(params=[torch.nn.Parameter(torch.zeros(6, 4).t())])):
        with pytest.raises(ValueError):
            opt.add_param_group(bad)
        assert len(opt.param_groups) == 1
    with pytest.raises(TypeError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2, dtype=torch.float64))]))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[p]))
    assert len(opt.param_groups) == 2


def test_a_group_on_two_devices_is_refused(AdamW):
    ps = [torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4, device="meta"))]
    opt = AdamW(ps)
    for p in ps:
        p.grad = torch.zeros_like(p)
    with pytest.raises(ValueError, match="one device"):
        opt.step()
    assert not opt.state


def test_a_group_saved_without_its_empty_count(AdamW):
    """Tools that drop entries that are None leave out the group's count where the states have theirs."""
    for capturable in (False, True):
        opt = AdamW(params(), capturable=capturable)
        sd = saved_state(opt, [5, 5])
        del sd["param_groups"][0]["step"]
        opt.load_state_dict(sd)
        got = opt.param_groups[0]["step"]
        assert int(got) == 5 if capturable else got is None
