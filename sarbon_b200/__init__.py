"""sarbon_b200: B200-native temporal block-sparse stem engine for Sarbon.

Public API (mirrors ``sarbon.sparse``):

* :class:`FusedSparseEngine` -- the engine (CUDA library ``libsarbon_sparse.so``).
* :class:`LocalBackbone`, :func:`stem_to_local`, :func:`fold` -- stem topology and BN folding.
* :func:`budget_buckets` -- the reference's budget schedule.
* :func:`cell_active_blocks` -- cell-level gating (``gating.py``) on the GPU.
* :func:`ms_deform_attn_core` -- the detector's deformable-attention core as one kernel.
* :func:`cross_attention`, :func:`rope_axes`, :func:`gated_norm` and their gradients -- a transformer
  block that reads an encoder's memory (:mod:`sarbon_b200.memory_ops`).

Importing the package does not load the CUDA library; constructing an engine does, and
raises :class:`SarbonLibraryError` when it is missing.
"""
from ._lib import SarbonLibraryError
from .fused_engine import FusedSparseEngine, budget_buckets, fuse_layers
from .gating import boxes_to_block_mask, boxes_to_block_masks, cell_active_blocks
from .deform_attn import ms_deform_attn_core
from .local import LocalBackbone, Node, fold, stem_to_local
from .memory_ops import (cross_attention, cross_attention_backward, gated_norm, gated_norm_backward, grid_positions,
                         rope_axes, rope_table)

__all__ = ["FusedSparseEngine", "LocalBackbone", "Node", "SarbonLibraryError", "budget_buckets",
           "boxes_to_block_mask", "boxes_to_block_masks", "cell_active_blocks", "cross_attention",
           "cross_attention_backward", "fold", "fuse_layers", "gated_norm", "gated_norm_backward", "grid_positions",
           "ms_deform_attn_core", "rope_axes", "rope_table", "stem_to_local"]
