"""B200 (sm_100a) gated-delta-rule kernels behind the contest's GDN ``run`` API.

* ``gdn_decode.run(q, k, v, state, A_log, a, dt_bias, b, scale)``
* ``gdn_prefill.run(q, k, v, state, A_log, a, dt_bias, b, cu_seqlens, scale)``
* ``gdn_mtp.run(q, k, v, initial_state, initial_state_indices, A_log, a, dt_bias,
  b, scale, intermediate_states_buffer=None)`` and flashinfer's
  ``gdn_mtp.gated_delta_rule_mtp(...)`` (pool-indexed multi-token decode)

Linear attention with a decay per head, the same states without the delta rule:

* ``decay_prefill.run(q, k, v, state, log_decay, cu_seqlens, scale)``
* ``decay_decode.run(q, k, v, state, log_decay, scale)`` and, over a pool of states,
  ``decay_decode.run_pool(q, k, v, pool, indices, log_decay, scale)``
* ``decay_tree.run(q, k, v, pool, indices, parents, log_decay, scale)`` (trees of
  drafted tokens) and ``decay_tree.commit(...)`` (the accepted path)

Pool slots of either recurrence parked in 8 bits:

* ``state_cache.empty(...)``, ``state_cache.store(...)``, ``state_cache.load(...)``

All call hand-written CUDA kernels through the C ABI in ``include/gdn_b200.h``
and ``include/gdn_decay_b200.h``
(``libgdn_b200.so``, built by ``python -m rocm_flashinfer_contest_b200.build``).
"""
from . import decay_decode, decay_prefill, decay_tree, gdn_decode, gdn_mtp, gdn_prefill, state_cache  # noqa: F401
from ._lib import GDNError, LIB_PATH  # noqa: F401

__all__ = ["decay_decode", "decay_prefill", "decay_tree", "gdn_decode", "gdn_mtp", "gdn_prefill", "state_cache",
           "GDNError", "LIB_PATH"]
