"""Torch ops of the cache operators (``fastdecisions_cache::``): one node each under ``torch.compile``, capturable in a HIP graph.

They wrap ``paged_kv_write``, ``paged_kv_read`` (``paged_kv_kernel``), ``paged_gqa_attention``
(``paged_gqa_kernel``), ``prep_qkv_state`` (``packed_conv_kernel``) and
``recurrent_gated_delta_rule`` (``gated_delta_kernel``) in the forms the cached layers call;
caches and states are updated in place and declared so.  ``gated_delta_rule_states`` is the chunked
rule (``chunk_gated_delta_rule``) from and to states that the caller gathers and scatters."""
from __future__ import annotations

from typing import Optional

import torch

from .gated_delta_kernel import chunk_gated_delta_rule, recurrent_gated_delta_rule
from .packed_conv_kernel import prep_qkv_state
from .paged_gqa_kernel import paged_gqa_attention
from .paged_kv_kernel import paged_kv_read, paged_kv_write


@torch.library.custom_op("fastdecisions_cache::paged_kv_write", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"),
                         device_types="cuda")
def paged_kv_write_op(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      page_table: torch.Tensor, cache_lens: torch.Tensor, k_scale: Optional[torch.Tensor],
                      v_scale: Optional[torch.Tensor], cu_seqlens: Optional[torch.Tensor]) -> None:
    paged_kv_write(key, value, k_cache, v_cache, page_table, cache_lens, k_scale=k_scale, v_scale=v_scale,
                   cu_seqlens=cu_seqlens)


@paged_kv_write_op.register_fake
def _paged_kv_write_fake(key, value, k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, cu_seqlens):
    return None


@torch.library.custom_op("fastdecisions_cache::paged_kv_read", mutates_args=(), device_types="cuda")
def paged_kv_read_op(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
                     total: int, k_scale: Optional[torch.Tensor],
                     v_scale: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    return paged_kv_read(k_cache, v_cache, page_table, cu_seqlens, total, k_scale=k_scale, v_scale=v_scale)


@paged_kv_read_op.register_fake
def _paged_kv_read_fake(k_cache, v_cache, page_table, cu_seqlens, total, k_scale, v_scale):
    _, h, _, d = k_cache.shape
    return tuple(k_cache.new_empty((1, total, h, d), dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))


@torch.library.custom_op("fastdecisions_cache::paged_gqa", mutates_args=(), device_types="cuda")
def paged_gqa_op(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                 cache_lens: torch.Tensor, k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor],
                 gate: Optional[torch.Tensor], cu_seqlens: Optional[torch.Tensor], max_seqlen: int) -> torch.Tensor:
    return paged_gqa_attention(q, k_cache, v_cache, page_table, cache_lens, k_scale=k_scale, v_scale=v_scale, gate=gate,
                               cu_seqlens=cu_seqlens, max_seqlen=max_seqlen)


@paged_gqa_op.register_fake
def _paged_gqa_fake(q, k_cache, v_cache, page_table, cache_lens, k_scale, v_scale, gate, cu_seqlens, max_seqlen):
    b, h, t, d = q.shape
    return q.new_empty((b, t, h, d)).permute(0, 2, 1, 3)


@torch.library.custom_op("fastdecisions_cache::packed_conv_state", mutates_args=("conv_state",), device_types="cuda")
def packed_conv_state_op(x: torch.Tensor, weight: torch.Tensor, conv_state: torch.Tensor,
                         cu_seqlens: Optional[torch.Tensor],
                         state_indices: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return prep_qkv_state(x, weight, conv_state, cu_seqlens=cu_seqlens, state_indices=state_indices)


@packed_conv_state_op.register_fake
def _packed_conv_state_fake(x, weight, conv_state, cu_seqlens, state_indices):
    batch, seq, channels = x.shape
    shape = (batch, seq, channels // 3 // 128, 128)
    return tuple(x.new_empty(shape) for _ in range(3))


@torch.library.custom_op("fastdecisions_cache::gated_delta_step", mutates_args=("state",), device_types="cuda")
def gated_delta_step_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                        state: torch.Tensor, cu_seqlens: Optional[torch.Tensor],
                        state_indices: torch.Tensor) -> torch.Tensor:
    """The rule with q and k normalised, the states of ``state_indices`` updated in place."""
    return recurrent_gated_delta_rule(q, k, v, g, beta, initial_state=state, use_qk_l2norm_in_kernel=True,
                                      cu_seqlens=cu_seqlens, state_indices=state_indices)[0]


@gated_delta_step_op.register_fake
def _gated_delta_step_fake(q, k, v, g, beta, state, cu_seqlens, state_indices):
    return v.new_empty(v.shape)


def gated_delta_rule_states(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                            initial_state: torch.Tensor,
                            cu_seqlens: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    """The chunked rule with q and k normalised: (out, final states)."""
    return chunk_gated_delta_rule(q, k, v, g, beta, initial_state=initial_state, output_final_state=True,
                                  use_qk_l2norm_in_kernel=True, cu_seqlens=cu_seqlens)


gated_delta_rule_states_op = torch.library.custom_op("fastdecisions_cache::gated_delta_rule_states",
                                                     gated_delta_rule_states, mutates_args=(), device_types="cuda")


@gated_delta_rule_states_op.register_fake
def _gated_delta_rule_states_fake(q, k, v, g, beta, initial_state, cu_seqlens):
    return v.new_empty(v.shape), initial_state.new_empty(initial_state.shape, dtype=torch.float32)
