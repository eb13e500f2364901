"""epure (MI355X build) -- the fused codebook dequant-matmul behind every
packed linear, on hand-written gfx950 HIP kernels, and what a served batch
needs between the linears (rotary positions, a paged key-value cache, attention,
drafted tokens verified).

Public names follow the reference package (epure/__init__.py:31-37) for the
parts this build covers: the packed store, linear and embedding, the fine-tuning
helpers, and the ``epure.kernels`` backend contract.
"""
from . import container
from .drafts import verify_draft
from .finetune import (
    ScaleTuner,
    make_trainable,
    packed_weights,
    snapshot_indices,
    trainable_forward,
    verify_frozen,
)
from .paged import PagedKVCache, Rotary, rope_frequencies
from .runtime import (
    ExpertHolder,
    PackedEmbedding,
    PackedExperts,
    PackedLinear,
    PackedWeight,
    apply_packed,
    tie_packed_lm_head,
)

__version__ = "0.2.4+mi355x"

__all__ = [
    "PackedWeight", "PackedLinear", "PackedEmbedding", "PackedExperts", "ExpertHolder",
    "apply_packed", "tie_packed_lm_head",
    "make_trainable", "packed_weights", "snapshot_indices", "verify_frozen",
    "trainable_forward", "ScaleTuner", "container",
    "Rotary", "rope_frequencies", "PagedKVCache", "verify_draft",
    "__version__",
]
