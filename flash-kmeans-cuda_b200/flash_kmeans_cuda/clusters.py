"""What a model does with the labels and centroids of a clustering.

``batch_kmeans_Euclid`` returns ids (B, N) and centroids (B, K, D) of batched rows. The
operators here read them:

* ``cluster_order`` groups the positions of each row of ids by cluster;
* ``cluster_lookup`` reads centroids (or any table of rows, such as a token embedding)
  back by id, with the gradient of the table;
* ``cluster_select`` picks the clusters whose centroids score best against a query;
* ``cluster_attention`` attends to the keys of the selected clusters only, with its
  gradients.

For attention the clustered rows are keys: a cache (batch, kv_heads, n_keys, head_dim) is
clustered as ``k.reshape(batch * kv_heads, n_keys, head_dim)``, so row ``b * kv_heads + h`` of
ids, order, offsets, centroids and sel belongs to kv head h of sequence b. Query head h reads kv
head ``h // (q_heads // kv_heads)``, and the query heads of one kv head share their selection.

All calls run on the current stream of their inputs' device, take their scratch memory from
PyTorch's caching allocator, never synchronise and can be captured into CUDA graphs. Two runs
on the same inputs give the same bits. A tensor that is not on a CUDA device raises
``ValueError``, any other bad argument ``RuntimeError``. (No reference counterpart.)
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _C


def cluster_order(ids: torch.Tensor, n_clusters: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Positions grouped by cluster.

    ``ids`` is (B, N), int32 or int64. Returns int32 ``order`` (B, N) and ``offsets``
    (B, n_clusters + 1): ``order[b, offsets[b, c] : offsets[b, c + 1]]`` are the positions n with
    ``ids[b, n] == c``, ascending. An id outside [0, n_clusters), such as -1 for padding, belongs
    to no cluster; ``order`` holds -1 from ``offsets[b, n_clusters]`` on.
    """
    return _C.cluster_order(ids, n_clusters)


def cluster_lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]``: rows of a table by id, differentiable in the table.

    ``table`` is (K, D) with ids of any shape, giving ids.shape + (D,), or (B, K, D) with ids
    (B, N), giving (B, N, D): float16, bfloat16 or float32. ids are int32 or int64; one outside
    [0, K) gives a row of zeros and no gradient. The product is formed in float32 and rounded
    once; the gradient ``dtable[k] = scale * sum of dy[n] where ids[n] == k`` is summed in float32
    (in ascending n, of large clusters block by block) and rounded once. The gradient itself has no
    graph: a backward pass with ``create_graph=True`` raises ``RuntimeError``, and so does a table with
    a forward-mode tangent.
    """
    return _C.cluster_lookup(table, ids, scale)


def cluster_select(
    q: torch.Tensor,
    centroids: torch.Tensor,
    offsets: torch.Tensor,
    top_k: int,
    *,
    order: Optional[torch.Tensor] = None,
    q_pos: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """The ``top_k`` clusters that score best for each query, for ``cluster_attention``.

    ``score = scale * max over the group's query heads of q . centroid + bias``, with ``q``
    (batch, q_heads, n_queries, head_dim) and ``centroids`` (batch * kv_heads, n_clusters,
    head_dim), both float16 or both bfloat16, head_dim a multiple of 8 up to 128, at most 16384
    clusters and top_k at most 1024. ``scale`` is head_dim ** -0.5 unless given; ``bias`` is
    (batch * kv_heads, n_clusters) float32, for instance the log of the cluster sizes; +inf
    forces a cluster in, -inf keeps it out.

    Returns int32 (batch * kv_heads, n_queries, top_k): cluster indices in ascending order,
    then -1. Ties go to the lowest index, and the choice is that of exact arithmetic, not of a
    rounded sum. Clusters without positions are never selected. With ``q_pos`` (batch, n_queries)
    int32, the last position each query sees, neither are clusters whose first position lies
    behind it; that needs ``order``. The result has no gradient.
    """
    return _C.cluster_select(q, centroids, offsets, top_k, order, q_pos, bias, scale)


def cluster_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    sel: torch.Tensor,
    order: torch.Tensor,
    offsets: torch.Tensor,
    *,
    q_pos: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of each query over the keys of its selected clusters.

    ``q`` is (batch, q_heads, n_queries, head_dim), ``k`` and ``v`` (batch, kv_heads, n_keys,
    head_dim): float16 or bfloat16, head_dim a multiple of 8 up to 128, any strides (tensors
    whose last dimension is not dense, or whose rows are not 16-byte aligned, are copied).
    ``sel`` (batch * kv_heads, n_queries, top_k) is what ``cluster_select`` gives; entries
    outside [0, n_clusters) select nothing, a cluster listed twice counts twice. ``order`` and
    ``offsets`` come from ``cluster_order``. ``q_pos`` (batch, n_queries) int32 is the last
    position that a query sees: ``n_keys - n_queries + i`` is the causal mask, -1 sees nothing,
    None everything. ``scale`` is head_dim ** -0.5 unless given.

    Returns out like q (contiguous) and, with ``return_lse``, the float32 log of each row's sum of
    exponentials (batch, q_heads, n_queries), which joins attention over several sets of keys. A
    query that sees no key gets zeros and -inf. Differentiable in q, k and v, but not through lse: such
    a join has no gradient. The gradient itself has no graph: a backward pass with
    ``create_graph=True`` raises ``RuntimeError``, and so does an input with a forward-mode tangent.
    """
    out, lse = _C.cluster_attention(q, k, v, sel, order, offsets, q_pos, scale)
    return (out, lse) if return_lse else out
