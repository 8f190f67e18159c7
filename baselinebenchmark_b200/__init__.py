"""B200-native MoBA (Mixture of Block Attention) causal prefill.

Drop-in for the package the reference loads by path
(backends/_mthreads/ops/moba/__init__.py:2-3 exports ``parallel_moba``)."""
from .paged import PagedKV, paged_append, paged_attention, paged_load, paged_store
from .parallel import moba_attn_varlen, moba_forward, parallel_moba

__all__ = ["parallel_moba", "moba_attn_varlen", "moba_forward",
           "PagedKV", "paged_store", "paged_load", "paged_attention", "paged_append"]
