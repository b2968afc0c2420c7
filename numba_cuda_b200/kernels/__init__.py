"""Library kernels: ``reduction`` (cuda.reduce), ``transpose``, ``headnorm`` (norm and
rotation of queries and keys) and ``kvcache`` (quantised paged cache)."""
