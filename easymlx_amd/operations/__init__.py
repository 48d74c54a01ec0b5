"""Attention operations (plugin boundary + the paged attention op)."""

from ._base_operation import (
    AttentionOutput,
    BaseOperation,
    CacheType,
    ExecutionMode,
    MetadataField,
    Operation,
    OperationRegistry,
    OperationRequirements,
    RequirementsBuilder,
)
from .tree_attention import TreeAccept, tree_accept, tree_attention
from .unified_attention import UnifiedAttention, UnifiedAttnMetadata, paged_attention

__all__ = (
    "AttentionOutput",
    "BaseOperation",
    "CacheType",
    "ExecutionMode",
    "MetadataField",
    "Operation",
    "OperationRegistry",
    "OperationRequirements",
    "RequirementsBuilder",
    "TreeAccept",
    "UnifiedAttention",
    "UnifiedAttnMetadata",
    "paged_attention",
    "tree_accept",
    "tree_attention",
)
