"""CPU oracle for the chain-flow drafting hot path (TEST INFRASTRUCTURE ONLY).

This package is a plain-torch, fp32, CPU restatement of the reference algorithm, written
from the reference's behaviour (each function cites the reference file:line it follows).
It exists to CHECK the CUDA product path, never to BE it:

* only ``tests/``, ``__graft_entry__.smoke()`` and ``bench.py``'s CPU-baseline / reference
  arm may import it;
* the product package ``chain_flow_b200`` never imports it and has no CPU fallback.

Pinning: ``tests/test_oracle_golden.py`` checks every function here against golden vectors
that ``tests/golden/make_golden.py`` generated by importing and running the reference's own
classes (``TreeFlowDrafter``, ``FlowDrafterProposer._beam_chains`` / ``_beam_tree``,
``kernels/tree_scan.tree_gated_delta_scan``) in the build container, and the context ring
against ``tests/golden/ring.npz`` (``tests/golden/make_ring_golden.py``: the reference's
``FlowDrafterProposer._ring_write`` / ``_ring_gather``).
"""
from .flow import (FlowConfig, layer_norm, mha, flow_block, expert_velocity, integrate,
                   path_residual, markov_bias)
from .beam import beam_chains, beam_tree, head_logprobs, twopass_candidates, twopass_logprobs
from .gdn import tree_gdn_scan, path_gdn_output, tree_gdn_verify, tree_gdn_factor, gdn_sequence
from .ring import ring_write, ring_gather
from .vae import vae_encode, vae_decode, predict_hidden_vae
from .tree_attn import tree_attn_merge, attention_over
from .tree_verify import tree_verify_greedy
from .paged import kv_quantise, kv_values, paged_attention

__all__ = [
    "FlowConfig", "layer_norm", "mha", "flow_block", "expert_velocity", "integrate",
    "path_residual", "markov_bias", "beam_chains", "beam_tree", "head_logprobs", "twopass_candidates",
    "twopass_logprobs",
    "tree_gdn_scan", "path_gdn_output", "tree_gdn_verify", "tree_gdn_factor", "ring_write", "ring_gather",
    "vae_encode", "vae_decode", "predict_hidden_vae", "tree_attn_merge", "attention_over", "tree_verify_greedy",
    "gdn_sequence", "kv_quantise", "kv_values", "paged_attention",
]
