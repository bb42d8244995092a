"""Training losses over a base of embeddings.

``softmax_cross_entropy(queries, database, targets)`` is the retrieval loss of
a query encoder (and, where they are trained, of the stored rows): every row of
the database is a class, the logits are ``scale * queries @ database.T``, and
``targets[b]`` is the row that query b should retrieve.  The [batch, n] logits
are never kept: the forward pass streams the rows through the tensor cores with
a running softmax, the backward pass recomputes them piece by piece (kernels in
csrc/xent.cu).  The reference has no training beyond its k-means declaration
(csrc/include/rapidadb/clustering/kmeans.h:9-24).
"""
from __future__ import annotations

import torch

from rapidadb_b200._lib import C

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def softmax_cross_entropy(queries: torch.Tensor, database: torch.Tensor, targets: torch.Tensor,
                          scale: float = 1.0, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of ``queries`` against every row of ``database``.

    ``loss[b] = logsumexp_n(scale * <q_b, x_n>) - scale * <q_b, x_targets[b]>``

    Args:
        queries:      [batch, dim] CUDA tensor, float32 / float16 / bfloat16.
        database:     [n, dim], same device and dtype, n >= 1 (e.g. the rows of
                      an index, or a batch of positives for in-batch negatives).
        targets:      [batch] int64 or int32 row numbers.  A query whose target
                      is ``ignore_index`` has loss 0 and no gradient, whatever
                      it holds; any other target outside [0, n) gives NaN.
        scale:        inverse temperature, positive and finite.  (A learnable
                      one: pass ``queries * temperature`` and ``scale=1``.)
        reduction:    "mean" over the queries that are not ignored (NaN when
                      all are), "sum" or "none" ([batch] losses).

    The loss is float32; gradients have their tensor's dtype.  Sums are held in
    float32.  16-bit gradients are rounded twice before their final rounding, the
    matrix of probabilities and (for the rows' gradient) the weighted queries, each
    to the operands' type: in norm about 1.1 (queries) and 1.4 times (rows) as far
    from the exact value as the final rounding alone.  float32 operands are
    multiplied as three bfloat16 planes; gradients are within 4e-6 in norm, and
    infinities in operands give NaN.  The backward pass keeps no logits; its
    workspace is the probabilities of a piece of the rows (512 MB, up to 2 GB for
    very many queries) and a few values per element of the queries.

    Gradients are computed only for the inputs that require them, in a fixed order
    of sums (the same call gives the same bits), and once: a backward pass with
    ``create_graph=True`` raises.  To capture a step into a CUDA graph, run it
    once before, and take the gradients with ``torch.autograd.grad`` of leaves
    made inside the capture.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}")
    return C().softmax_cross_entropy_loss(queries, database, targets, scale, ignore_index, _REDUCTIONS[reduction])
