"""MI355X-native (gfx950) Gated DeltaNet layer path of nano-vllm-extend.

The GDN kernels of the Qwen3.5 hybrid model -- varlen / decode / padded
causal conv + SiLU, fused g/beta, chunked gated delta rule, recurrent
decode (single- and multi-token), gated RMSNorm, the projection GEMMs with the
requests' low-rank adapters, the norms around the mixer -- as hand-written HIP for
gfx950 behind the C ABI of include/gdn_mi355x.h, with Python wrappers that
keep the reference's call signatures (ops), a host mirror of the layer
dispatch (gdn_layer), the slot-pool bookkeeping (state_pool) and the hook
that installs the kernels into the reference model module (integration).
"""
from . import _lib, ops, state_pool, gdn_layer, integration  # noqa: F401
from .ops import (  # noqa: F401
    LoraPool,
    Qwen3_5RMSNormGated,
    adapter_rows,
    add_rms_norm,
    add_rms_norm_fp8,
    causal_conv_silu,
    causal_conv_silu_varlen,
    causal_conv_silu_varlen_parts,
    chunk_gated_delta_rule,
    chunk_gated_delta_rule_varlen,
    commit_states,
    commit_tree,
    conv_decode_step,
    conv_tree_step,
    fused_g_beta,
    linear,
    linear_fp8,
    linear_fp8_lora,
    linear_lora,
    quantize_fp8,
    quantize_weight_fp8,
    recurrent_gated_delta_rule,
    recurrent_gdn_inplace,
    recurrent_gdn_multitoken,
    recurrent_gdn_tree,
    recurrent_tree_fused,
    rms_norm_gated,
    rms_norm_gated_fp8,
)
from .gdn_layer import GatedDeltaNetBlock, GatedDeltaNetCore, GatedDeltaNetLayer, Switches, TreeStep  # noqa: F401
from .state_pool import LinearStatePool, allocate_state_pools, reset_linear_states, varlen_meta  # noqa: F401
