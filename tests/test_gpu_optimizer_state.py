"""``train.AdamW`` on the device: states saved and loaded across settings, in the middle of training."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def model(dtype, dev):
    g = torch.Generator().manual_seed(0)
    return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dtype).to(dev)) for s in ((33, 20), (20,), ())]


def set_grads(params, seed):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = torch.randn(p.shape, generator=g).to(p.dtype).to(p.device)


def copied(params):
    return [torch.nn.Parameter(p.detach().clone()) for p in params]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("first", [False, True])
def test_a_state_moves_between_host_and_device_counts(dev, bits, first):
    """Three steps, then saved, loaded into an optimizer that counts in the other place, and two steps more: the
    same bytes as two more steps of the first.  (Both work the step's scalars out in fp64 and round them once.)"""
    from unirl_amd.train import AdamW

    kw = dict(lr=1e-2, state_bits=bits, master_weights=True, max_grad_norm=1.0, seed=3)
    ours = model(torch.bfloat16, dev)
    a = AdamW(ours, capturable=first, **kw)
    for k in range(3):
        set_grads(ours, k)
        a.step()
    twin = copied(ours)
    b = AdamW(twin, capturable=not first, **kw)
    b.load_state_dict(a.state_dict())
    for k in range(3, 5):
        for ps, opt in ((ours, a), (twin, b)):
            set_grads(ps, k)
            opt.step()
        for p, q in zip(ours, twin):
            assert torch.equal(p, q), k
            for name in ("exp_avg", "exp_avg_sq", "master"):
                assert torch.equal(a.state[p][name], b.state[q][name]), (k, name)
    assert not math.isnan(float(b.grad_norm))


def test_a_checkpoint_mapped_to_the_cpu(dev):
    """Saved with a tensor rate, read back onto the CPU: the step goes on where the parameters are."""
    import io

    from unirl_amd.train import AdamW

    def build(ps):
        return AdamW(ps, lr=torch.tensor(1e-2, device=dev), capturable=True, state_bits=8)

    ours = model(torch.float32, dev)
    a = build(ours)
    set_grads(ours, 0)
    a.step()
    twin = copied(ours)
    buf = io.BytesIO()
    torch.save(a.state_dict(), buf)
    buf.seek(0)
    b = build(twin)
    b.load_state_dict(torch.load(buf, map_location="cpu", weights_only=True))
    for ps, opt in ((ours, a), (twin, b)):
        set_grads(ps, 1)
        opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ours, twin))


def test_a_captured_step_goes_on_with_a_loaded_state(dev):
    """Captured, trained on, then set back to a state saved before: every replay gives what an optimizer that was
    loaded with that state and never captured gives."""
    import copy

    from unirl_amd.train import AdamW

    kw = dict(state_bits=8, master_weights=True, max_grad_norm=1.0, capturable=True, seed=3)
    lr = torch.tensor(1e-2, device=dev)
    ours = model(torch.bfloat16, dev)
    a = AdamW(ours, lr=lr, **kw)
    set_grads(ours, 0)
    grads = [p.grad for p in ours]
    a.step()
    saved = copy.deepcopy(a.state_dict())
    twin = copied(ours)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.step()
    lr.fill_(3e-2)
    for _ in range(2):
        graph.replay()
    a.load_state_dict(saved)
    assert float(lr) == float(torch.tensor(1e-2))
    with torch.no_grad():
        for p, q in zip(ours, twin):
            p.copy_(q)
    b = AdamW(twin, lr=torch.tensor(1e-2, device=dev), **kw)
    b.load_state_dict(saved)
    junk = [torch.full((1 << 16,), 255, dtype=torch.uint8, device=dev) for _ in range(16)]  # takes what was freed
    for k in range(1, 5):
        set_grads(twin, k)
        for g, q in zip(grads, twin):
            g.copy_(q.grad)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for p, q in zip(ours, twin):
            assert torch.equal(p, q), k
    assert all(bool((j == 255).all()) for j in junk)
    assert int(a.param_groups[0]["step"]) == int(b.param_groups[0]["step"]) == 5


@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_leaves_every_group_as_it_was(dev, capturable):
    """The second group lies on the CPU, where there is no kernel: the first is not stepped either."""
    from unirl_amd.train import AdamW

    ours = model(torch.float32, dev)
    other = torch.nn.Parameter(torch.zeros(4))
    opt = AdamW([dict(params=ours), dict(params=[other])], capturable=capturable)
    set_grads(ours, 0)
    before = [p.detach().clone() for p in ours]
    other.grad = torch.ones_like(other)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ours, before))
    other.grad = None
    twin = AdamW([dict(params=copied(ours))], capturable=capturable)
    set_grads(twin.param_groups[0]["params"], 0)
    opt.step()
    twin.step()
    assert all(torch.equal(p, q) for p, q in zip(ours, twin.param_groups[0]["params"]))


def test_parameters_made_in_inference_mode(dev):
    """Weights loaded under inference mode have no version to raise: the step counts once, like any other."""
    from unirl_amd import ops

    def step(p):
        m, v = torch.zeros(300, device=dev), torch.zeros(300, device=dev)
        ops.adamw_step([p], [torch.ones(300, device=dev)], [m], [v], lr=1e-2, step=1)
        return p

    with torch.inference_mode():
        p = torch.ones(300, device=dev)
    assert p.is_inference()
    assert torch.equal(step(p), step(torch.ones(300, device=dev)))
