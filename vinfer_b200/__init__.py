"""vinfer_b200: a B200-native (sm_100a) token sampler for vinfer.

One fused, memory-bound CUDA pass per batch of logits rows (penalties, temperature, top-k,
softmax, top-p, min-p, inverse-CDF draw), reached through a C ABI
(``include/vinfer_sampler.h``) and registered as the ``b200`` backend of a ``sampler`` op
family with the same registry contract as vinfer's kernel registry. Beside it, over the same rows
of logits: beam search (``vinfer_b200.beam``) and distillation from top log-probabilities
(``vinfer_b200.distill``).
"""

from vinfer_b200.kernels.sampler import SAMPLER, B200Sampler, SamplerBackend
from vinfer_b200.registry import BackendContext, BackendRegistry
from vinfer_b200.sampling import (
    BeamStep,
    DecodeStates,
    RowParams,
    SamplingParams,
    SlotHistogram,
    TokenHistogram,
    position_seed,
    position_uniform,
)

__all__ = [
    "SAMPLER",
    "B200Sampler",
    "BackendContext",
    "BackendRegistry",
    "BeamStep",
    "DecodeStates",
    "RowParams",
    "SamplerBackend",
    "SamplingParams",
    "SlotHistogram",
    "TokenHistogram",
    "position_seed",
    "position_uniform",
]
