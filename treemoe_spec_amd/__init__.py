"""treemoe_spec_amd — MI355X (gfx950) implementation of TreeMoE-Spec's
verification hot path: op1 (tree-aware grouped MoE with op3 budget routing)
and op4 (greedy tree verify + paged KV commit).

Module layout mirrors the reference package:
  treemoe_spec_amd.kernels.op1_tree_moe   tree_moe_forward, route_experts, Routing, ...
  treemoe_spec_amd.kernels.op4_commit     fused_verify_commit, VerifyResult
  treemoe_spec_amd.kernels.tree_attention    tree_attention
  treemoe_spec_amd.kernels.rms_norm          rms_norm, rms_norm_fp8
  treemoe_spec_amd.kernels.rotary            RotaryPlan, rotary_embed, rotary_append
  treemoe_spec_amd.kernels.prompt_attention  PromptPlan, prompt_attention, prompt_attention_cached
  treemoe_spec_amd.kernels.sample_tokens     sample_tokens
  treemoe_spec_amd.kernels.branch_attention  BranchPlan, branch_attention
  treemoe_spec_amd.kernels.beam_search       beam_select, reorder_rows
  treemoe_spec_amd.kernels.cache_eviction    attention_mass, evict
  treemoe_spec_amd.kv_cache               PagedKVCache (page size configurable), BranchCache
The GPU work lives in libtreemoe_amd.so (C ABI: include/treemoe_amd.h).
"""

__version__ = "0.1.0"

NUM_LAYERS = 32
NUM_EXPERTS = 8
TOP_K = 2
HIDDEN_DIM = 4096
INTERMEDIATE_DIM = 14336
VOCAB_SIZE = 32000
TREE_SIZE = 64
TREE_MAX_DEPTH = 6
