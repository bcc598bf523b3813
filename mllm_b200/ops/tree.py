"""Operators for drafted token trees: one round of speculative decoding over the paged cache.

A draft is a tree of tokens per request.  Its nodes are rows of one batch: request b has ``seq_lens[b] - prefix_lens[b]`` of them from
row ``q_start_loc[b]`` on, behind ``prefix_lens[b]`` cached tokens, and node j owns the cache slot
``req_to_token[req_pool_indices[b], prefix_lens[b] + j]``.  ``parents[row]`` is the node (counted within the request) that a row's node
continues, in front of it, or -1: node 0, the request's last token, and every other node that continues the cached text directly.  A
node's position is the number of cached tokens and of its ancestors.

    q = tree_qk_norm_rope_kv_write(qkv, ...)        per layer: norms, rotation, keys and values to the cache
    o = attention_tree(q, ...)                      per layer: cached tokens, ancestors, itself
    path, tokens, counts = tree_speculative_sample(logits, ...)
    tree_kv_compact(store, ..., path, counts)       the accepted nodes' cache rows, all layers

Index tensors are contiguous int32 tensors on the device of the data.  Nothing here reads them on the host, so a round can be captured
in a CUDA graph; numbers that point outside the tensors are recorded (:func:`mllm_b200.ops.check_status`) and what they describe is left out.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import reference as ref


def _ops():
    from .. import ops

    return ops


def _check_index(what: str, rows: int, device, req_to_token, parents, *per_request) -> None:
    """Shapes, types and devices of the index tensors of a batch of trees."""
    if req_to_token.dim() != 2 or req_to_token.dtype != torch.int32 or req_to_token.stride(1) != 1 or req_to_token.device != device:
        raise ValueError(f"{what}: req_to_token must be a two-dimensional int32 tensor with unit inner stride on {device}")
    batch = per_request[0].numel()
    for t, n in ((parents, rows), *((t, batch) for t in per_request)):
        if t.dim() != 1 or t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{what}: parents [{rows}] and one number per request [{batch}] must be contiguous int32 vectors on {device}")


def _check_caches(what: str, k_cache, v_cache, heads: int, dim: int, dtype, device) -> None:
    if (k_cache.dim() != 3 or k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride() or k_cache.dtype != v_cache.dtype
            or k_cache.shape[1] != heads or k_cache.shape[2] != dim or k_cache.stride(2) != 1
            or k_cache.dtype not in (dtype, torch.float8_e4m3fn, torch.float8_e5m2) or k_cache.device != device or v_cache.device != device):
        raise ValueError(f"{what}: the caches must be [slots, {heads}, {dim}] views of one layout, of {dtype} or an 8-bit float, on {device}")


def attention_tree(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, parents, scale: float,
                   out: Optional[torch.Tensor] = None, window: Optional[int] = None, logit_cap: float = 0.0,
                   sink: Optional[torch.Tensor] = None, chunk: Optional[int] = None) -> torch.Tensor:
    """Attention of drafted nodes ``q`` [T, Hq, D] (heads of a node contiguous): each sees the cached tokens, its ancestors and itself.
    ``window``, ``logit_cap``, ``sink`` and ``chunk`` as for :func:`mllm_b200.ops.attention_prefill`, by positions: siblings share theirs.
    Heads of 64, 128 and 256 features, 16-bit, over caches of their type or of unscaled 8-bit floats.  Rows of ``out`` that belong to no
    request keep what they hold.  A value in the cache that is no number reaches the nodes that see it and no others."""
    if q.dim() != 3 or k_cache.dim() != 3 or q.stride(2) != 1 or q.stride(1) != q.shape[2]:
        raise ValueError("attention_tree: q must be [T, heads, features] with the heads of a node contiguous")
    hkv = k_cache.shape[1]
    _check_caches("attention_tree", k_cache, v_cache, hkv, q.shape[2], q.dtype, q.device)
    _check_index("attention_tree", q.shape[0], q.device, req_to_token, parents, req_pool_indices, seq_lens, prefix_lens, q_start_loc)
    if hkv == 0 or q.shape[1] % hkv or q.shape[1] > 128 * hkv:
        raise ValueError(f"attention_tree: {q.shape[1]} query heads over {hkv} key heads")
    if window is not None and window < 0 or chunk is not None and chunk < 0 or (window and chunk):
        raise ValueError("attention_tree: either a sliding window or chunks, of positive lengths")
    if sink is not None and (sink.dtype != torch.float32 or sink.shape != (q.shape[1],) or sink.device != q.device):
        raise ValueError(f"attention_tree: sink must be fp32 [{q.shape[1]}] on {q.device}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1
                            or out.stride(1) != out.shape[2]):
        raise ValueError("attention_tree: out must be like q, with the heads of a node contiguous")
    ops = _ops()
    if not ops.use_kernels(q):
        return ref.attention_tree(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, parents, scale, out,
                                  window, logit_cap, sink, chunk)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ops.ext().attention_tree(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, parents, float(scale), out,
                             int(window or 0), float(logit_cap or 0.0), None if sink is None else sink.contiguous(), int(chunk or 0))
    return out
