"""Model-side pieces of the hot path: the log-prob arithmetic and the norms in front of a policy's
output (no model forwards)."""

from .ar_logp import ARLogprobStep, chunked_replay_logp, token_entropy, token_logp, token_logp_entropy
from .norm import layer_norm, modulated_layer_norm, rms_norm

__all__ = [
    "ARLogprobStep",
    "chunked_replay_logp",
    "layer_norm",
    "modulated_layer_norm",
    "rms_norm",
    "token_entropy",
    "token_logp",
    "token_logp_entropy",
]
