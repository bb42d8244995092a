"""``rapidadb.losses`` alias: training losses over a base of embeddings."""
from rapidadb_b200.losses import softmax_cross_entropy  # noqa: F401
