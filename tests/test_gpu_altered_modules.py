"""``chunked_replay_logp`` with heads and norms whose call a user's program has changed."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(dev, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(4)
    hidden = torch.randn(2, 12, 64, generator=g).to(dtype).to(dev)
    tokens = torch.randint(0, 333, (2, 12), generator=g).to(dev)
    return hidden, tokens


@pytest.mark.parametrize("kind", [torch.nn.RMSNorm, torch.nn.LayerNorm])
def test_a_norm_with_a_forward_of_its_own_is_called(dev, kind):
    """A replaced ``forward`` that doubles the output: the replay has to see doubled states."""
    from unirl_amd import models

    hidden, tokens = inputs(dev)
    head = torch.nn.Linear(64, 333, bias=False, device=dev, dtype=torch.bfloat16)
    norm = kind(64).to(dev, torch.bfloat16)
    called, plain = [], norm.forward

    def twice(x):
        called.append(tuple(x.shape))
        return plain(x) * 2

    norm.forward = twice
    with torch.no_grad():
        out = models.chunked_replay_logp(head, hidden, tokens, final_norm=norm)
        want = models.chunked_replay_logp(head, plain(hidden) * 2, tokens)
    assert called == [(2, 12, 64)] and torch.equal(out, want)


@pytest.mark.parametrize("trains", [False, True])
def test_a_head_whose_weight_is_made_in_front_of_the_call(dev, trains):
    """A hook in front writes the weight that the forward reads (as the older weight norm does), or the forward
    is replaced: log-probs and gradients are those of the changed head."""
    from unirl_amd import models

    hidden, tokens = inputs(dev)
    base = torch.randn(333, 64, device=dev).bfloat16() / 8
    plain = torch.nn.Linear(64, 333, bias=False, device=dev, dtype=torch.bfloat16)

    def hooked():
        head = torch.nn.Linear(64, 333, bias=False, device=dev, dtype=torch.bfloat16)

        def make(m, args):
            with torch.no_grad():
                m.weight.copy_(base * 2)

        head.register_forward_pre_hook(make)
        return head

    def replaced():
        head = torch.nn.Linear(64, 333, bias=False, device=dev, dtype=torch.bfloat16)
        with torch.no_grad():
            head.weight.copy_(base)
        head.forward = lambda h: torch.nn.functional.linear(h, head.weight * 2)
        return head

    with torch.no_grad():
        plain.weight.copy_(base * 2)
    for build in (hooked, replaced):
        h = hidden.clone().requires_grad_(trains)
        out = models.chunked_replay_logp(build(), h, tokens, keep_logits=True if trains else None, fused_head=False)
        want = models.chunked_replay_logp(plain, hidden, tokens, fused_head=False)
        # the same library product in both, and the same kernel behind it
        assert torch.allclose(out, want, rtol=1e-5, atol=1e-5)
        if trains:
            g, = torch.autograd.grad(out.sum(), h)
            hh = hidden.clone().requires_grad_(True)
            w, = torch.autograd.grad(models.chunked_replay_logp(plain, hh, tokens, keep_logits=True, fused_head=False).sum(), hh)
            assert float((g.float() - w.float()).abs().max()) <= 2.0**-7 * float(w.float().abs().max())
