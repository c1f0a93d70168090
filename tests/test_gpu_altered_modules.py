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
