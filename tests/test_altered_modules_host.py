"""CPU-only checks of when ``chunked_replay_logp`` may compute a module's values itself instead of calling it."""

import pytest
import torch


@pytest.fixture(scope="module")
def ar_logp(built_lib):
    from unirl_amd.models import ar_logp

    return ar_logp


def alterations():
    """Ways in which a user's program changes what a call of one module does."""
    def own_forward(m):
        plain = m.forward
        m.forward = lambda *args: plain(*args)
    return {
        "a forward of its own": own_forward,
        "a forward hook": lambda m: m.register_forward_hook(lambda *a: None),
        "a forward hook with keywords": lambda m: m.register_forward_hook(lambda *a: None, with_kwargs=True),
        "a hook in front": lambda m: m.register_forward_pre_hook(lambda *a: None),
        "a backward hook": lambda m: m.register_full_backward_hook(lambda *a: None),
        "a hook in front of the backward": lambda m: m.register_full_backward_pre_hook(lambda *a: None),
    }


@pytest.mark.parametrize("how", alterations())
def test_an_altered_module_is_called(ar_logp, how):
    for build in (lambda: torch.nn.RMSNorm(8), lambda: torch.nn.LayerNorm(8), lambda: torch.nn.Linear(8, 8)):
        module = build()
        assert not ar_logp._is_altered(module)
        alterations()[how](module)
        assert ar_logp._is_altered(module)
    handle = torch.nn.modules.module.register_module_forward_pre_hook(lambda *a: None)
    try:
        assert ar_logp._is_altered(torch.nn.RMSNorm(8))
    finally:
        handle.remove()
    assert not ar_logp._is_altered(torch.nn.RMSNorm(8))


@pytest.mark.parametrize("how", alterations())
def test_an_altered_linear_is_not_plain(ar_logp, how):
    head = torch.nn.Linear(8, 8)
    assert ar_logp._is_plain_linear(head)
    alterations()[how](head)
    assert not ar_logp._is_plain_linear(head)
