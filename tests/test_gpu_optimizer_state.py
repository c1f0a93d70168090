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
