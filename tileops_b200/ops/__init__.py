from .gqa import (
    GroupedQueryAttentionDecodePagedFp8KVCacheFwdOp,
    GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp,
    GroupedQueryAttentionDecodePagedWithKVCacheFwdOp,
    GroupedQueryAttentionDecodeWithKVCacheFwdOp,
    GroupedQueryAttentionFwdOp,
    GroupedQueryAttentionPrefillFwdOp,
    GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp,
    GroupedQueryAttentionPrefillPagedWithKVCacheFwdOp,
    GroupedQueryAttentionPrefillVarlenFwdOp,
    GroupedQueryAttentionSlidingWindowFwdOp,
    GroupedQueryAttentionSlidingWindowVarlenFwdOp,
)
from .mha import MultiHeadAttentionDecodePagedWithKVCacheFwdOp, MultiHeadAttentionDecodeWithKVCacheFwdOp
from .op_base import Op
from .paged_kv import (
    Int4KVCacheAppendFwdOp,
    Int4KVCacheGatherFwdOp,
    PagedKVCachePlanFwdOp,
    PagedKVCacheReleaseFwdOp,
    QKNormRopeFwdOp,
    QKNormRopeInt4KVCacheAppendFwdOp,
    QKNormRopeKVCacheAppendFwdOp,
)

__all__ = [
    "Op",
    "GroupedQueryAttentionFwdOp",
    "GroupedQueryAttentionPrefillFwdOp",
    "GroupedQueryAttentionPrefillVarlenFwdOp",
    "GroupedQueryAttentionPrefillPagedWithKVCacheFwdOp",
    "GroupedQueryAttentionSlidingWindowFwdOp",
    "GroupedQueryAttentionSlidingWindowVarlenFwdOp",
    "GroupedQueryAttentionDecodeWithKVCacheFwdOp",
    "GroupedQueryAttentionDecodePagedWithKVCacheFwdOp",
    "GroupedQueryAttentionDecodePagedFp8KVCacheFwdOp",
    "MultiHeadAttentionDecodeWithKVCacheFwdOp",
    "MultiHeadAttentionDecodePagedWithKVCacheFwdOp",
    "GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp",
    "GroupedQueryAttentionPrefillPagedInt4KVCacheFwdOp",
    "PagedKVCachePlanFwdOp",
    "PagedKVCacheReleaseFwdOp",
    "QKNormRopeFwdOp",
    "QKNormRopeKVCacheAppendFwdOp",
    "QKNormRopeInt4KVCacheAppendFwdOp",
    "Int4KVCacheAppendFwdOp",
    "Int4KVCacheGatherFwdOp",
]
