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


_front = None


def _ops():
    """The package that this module is part of; it is not complete while this one is imported."""
    global _front
    if _front is None:
        from .. import ops as _front
    return _front


def tree_kernels_cover(head_dim: int, cache_dtype, act_dtype) -> bool:
    """Whether :func:`tree_qk_norm_rope_kv_write` and :func:`attention_tree` have kernels for such heads, rows and caches; on the GPU they refuse
    others."""
    return (head_dim in (64, 128, 256) and act_dtype in (torch.bfloat16, torch.float16)
            and cache_dtype in (act_dtype, torch.float8_e4m3fn, torch.float8_e5m2))


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


def tree_qk_norm_rope_kv_write(qkv, q_weight, k_weight, parents, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, inv_freq,
                               k_cache, v_cache, num_q_heads: int, num_kv_heads: int, head_dim: int, eps: float,
                               position_delta: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Prologue of :func:`attention_tree`: ``qkv`` [T, (Hq + 2 Hkv) * D] -> queries [T, Hq, D]; keys and values go to the nodes' slots.
    Query and key heads are divided by their root mean square and multiplied by ``q_weight`` / ``k_weight`` [D] (None: left as they are), then
    the first ``2 * inv_freq.numel()`` features turn (feature i with the one half of them on) by ``inv_freq`` (fp32) times the node's
    position: cached tokens, ancestors, and ``position_delta`` [requests] int32 where text positions do not count from 0.  Heads of 64, 128
    and 256 features on the GPU, a multiple of 16 of them rotated; rows and weights begin on 16-byte boundaries there.  ``qkv`` is left as it
    is; results are rounded once; queries of rows that belong to no request are zero."""
    args = (parents, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, inv_freq, k_cache, v_cache, num_q_heads, num_kv_heads,
            head_dim, float(eps), position_delta)
    ops = _ops()
    if ops.use_kernels(qkv):        # the binding makes the same checks
        return ops.ext().tree_qk_norm_rope_kv_write(qkv, q_weight, k_weight, *args)
    what = "tree_qk_norm_rope_kv_write"
    if num_q_heads < 1 or num_kv_heads < 1:
        raise ValueError(f"{what}: {num_q_heads} query heads and {num_kv_heads} key heads")
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.shape[1] != (num_q_heads + 2 * num_kv_heads) * head_dim:
        raise ValueError(f"{what}: qkv must be [T, {(num_q_heads + 2 * num_kv_heads) * head_dim}] with unit inner stride")
    _check_caches(what, k_cache, v_cache, num_kv_heads, head_dim, qkv.dtype, qkv.device)
    _check_index(what, qkv.shape[0], qkv.device, req_to_token, parents, req_pool_indices, seq_lens, prefix_lens, q_start_loc,
                 *(() if position_delta is None else (position_delta,)))
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or inv_freq.numel() * 2 > head_dim or inv_freq.device != qkv.device:
        raise ValueError(f"{what}: inv_freq must be an fp32 vector, one number per rotated pair of {head_dim} features, on {qkv.device}")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (head_dim,) or w.dtype != qkv.dtype or w.device != qkv.device):
            raise ValueError(f"{what}: weights must be vectors of {head_dim} like qkv")
    return ref.tree_qk_norm_rope_kv_write(qkv, q_weight, k_weight, *args)


def attention_tree(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, parents, scale: float,
                   out: Optional[torch.Tensor] = None, window: Optional[int] = None, logit_cap: float = 0.0,
                   sink: Optional[torch.Tensor] = None, chunk: Optional[int] = None) -> torch.Tensor:
    """Attention of drafted nodes ``q`` [T, Hq, D] (heads of a node contiguous): each sees the cached tokens, its ancestors and itself.
    ``scale`` is positive; ``window``, ``logit_cap``, ``sink`` and ``chunk`` as for :func:`mllm_b200.ops.attention_prefill`, by positions:
    siblings share theirs.  Heads of 64, 128 and 256 features, 16-bit, over caches of their type or of unscaled 8-bit
    floats.  Rows of ``out`` that belong to no request keep what they hold.  A value in the cache that is no number reaches the nodes that see it and
    no others.  On the GPU a token whose slot lies outside the cache is seen by none, and a node that sees nothing has a row of zeros."""
    ops = _ops()
    if ops.use_kernels(q):          # the binding makes the same checks
        return ops.ext().attention_tree(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, parents,
                                        float(scale), out, int(window or 0), float(logit_cap or 0.0), sink, int(chunk or 0))
    if q.dim() != 3 or k_cache.dim() != 3 or q.stride(2) != 1 or q.stride(1) != q.shape[2]:
        raise ValueError("attention_tree: q must be [T, heads, features] with the heads of a node contiguous")
    hkv = k_cache.shape[1]
    _check_caches("attention_tree", k_cache, v_cache, hkv, q.shape[2], q.dtype, q.device)
    _check_index("attention_tree", q.shape[0], q.device, req_to_token, parents, req_pool_indices, seq_lens, prefix_lens, q_start_loc)
    if hkv == 0 or q.shape[1] == 0 or q.shape[1] % hkv or q.shape[1] > 128 * hkv:
        raise ValueError(f"attention_tree: {q.shape[1]} query heads over {hkv} key heads")
    if window is not None and window < 0 or chunk is not None and chunk < 0 or (window and chunk):
        raise ValueError("attention_tree: either a sliding window or chunks, of positive lengths")
    if not torch.finfo(torch.float32).tiny <= scale <= torch.finfo(torch.float32).max:
        raise ValueError(f"attention_tree: scale must be positive and finite, not {scale}")
    if sink is not None and (sink.dtype != torch.float32 or sink.shape != (q.shape[1],) or sink.device != q.device):
        raise ValueError(f"attention_tree: sink must be fp32 [{q.shape[1]}] on {q.device}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1
                            or out.stride(1) != out.shape[2]):
        raise ValueError("attention_tree: out must be like q, with the heads of a node contiguous")
    return ref.attention_tree(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, parents, scale, out,
                              window, logit_cap, sink, chunk)


def tree_speculative_sample(logits, tokens, parents, tree_lens, q_start_loc, temperature, top_k, top_p, min_p, uniform, uniform_final,
                            max_steps: int, draft_probs: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Walks each request's tree from node 0 with the target's distribution and emits tokens that are distributed as the target's own.

    ``logits`` [T, vocab] of all nodes, ``tokens`` [T] int64 and ``parents`` [T] of the ``tree_lens[b]`` nodes from row ``q_start_loc[b]`` on.
    At a node the distribution p is that of :func:`mllm_b200.ops.top_k_top_p_min_p_sample` (temperature up to 1e-6: the most likely token;
    ``top_k`` below 1 and ``top_p`` of 1 and more do not filter; every filter looks at the whole distribution, and ties at a cut are kept).
    The node's children, in order, up to 64 of them: child c with token x is taken if ``uniform[c] * q(x) < p(x)``, otherwise
    ``p <- max(p - q, 0)``, scaled to 1 (left as it is where nothing remains).  q is row ``draft_probs[node]``, the distribution that each of
    the node's children was drawn from, independently of the others (with replacement), or without ``draft_probs`` all of x: candidates that
    were picked, not drawn.  Where no child is taken, or ``max_steps`` nodes are reached, the walk ends with the first token whose running sum of
    p in the order of the ids passes ``uniform_final[b]``.  Random numbers are from [0, 1).  A logit that is no number counts as minus infinity,
    a row without a finite logit gives its first token, and infinite logits share the mass.

    Returns ``path`` [requests, max_steps] int32, the nodes of the walk from node 0 on (whose cache rows are now valid), ``tokens``
    [requests, max_steps] int64, the emitted tokens (those of ``path[:, 1:]`` and one more), both -1 behind ``counts`` [requests] int32."""
    ops = _ops()
    if ops.use_kernels(logits):     # the binding makes the same checks
        f32 = lambda x: x if x is None or x.dtype == torch.float32 and x.is_contiguous() else x.float().contiguous()  # noqa: E731
        if top_k.dtype != torch.int32 or not top_k.is_contiguous():
            top_k = top_k.to(torch.int32).contiguous()
        return ops.ext().tree_speculative_sample(logits, tokens, parents, tree_lens, q_start_loc, f32(temperature), top_k, f32(top_p), f32(min_p),
                                                 f32(uniform), f32(uniform_final), int(max_steps), draft_probs)
    what = "tree_speculative_sample"
    if logits.dim() != 2 or logits.stride(1) != 1 or logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"{what}: logits must be [T, vocab] in 16 or 32 bits with unit inner stride")
    T, dev, batch = logits.shape[0], logits.device, tree_lens.numel()
    if tokens.shape != (T,) or tokens.dtype != torch.int64 or tokens.device != dev or not tokens.is_contiguous():
        raise ValueError(f"{what}: tokens must be a contiguous int64 vector of {T} on {dev}")
    for t, n in ((parents, T), (tree_lens, batch), (q_start_loc, batch)):
        if t.shape != (n,) or t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
            raise ValueError(f"{what}: parents [{T}], tree_lens and q_start_loc [{batch}] must be contiguous int32 vectors on {dev}")
    for t, n in ((temperature, batch), (top_k, batch), (top_p, batch), (min_p, batch), (uniform, T), (uniform_final, batch)):
        if t is not None and (t.shape != (n,) or t.device != dev):
            raise ValueError(f"{what}: temperature, top_k, top_p, min_p and uniform_final have {batch} numbers, uniform {T}, all on {dev}")
    if draft_probs is not None and (draft_probs.shape != logits.shape or draft_probs.dtype != torch.float32 or draft_probs.device != dev
                                    or draft_probs.stride(1) != 1):
        raise ValueError(f"{what}: draft_probs must be fp32 [T, vocab] like logits, with unit inner stride")
    if max_steps < 1 or logits.shape[1] < 1:
        raise ValueError(f"{what}: max_steps and the vocabulary must be at least 1")
    return ref.tree_speculative_sample(logits, tokens, parents, tree_lens, q_start_loc, temperature, top_k, top_p, min_p, uniform, uniform_final,
                                       max_steps, draft_probs)


def tree_kv_compact(store, req_to_token, req_pool_indices, prefix_lens, path, counts) -> None:
    """Brings the cache rows of accepted nodes together, in place and in every plane of ``store`` [.., slots, features] (contiguous; a pool's
    storage of all layers): for i below ``counts[b]``, what node ``path[b, i]`` of request b has in its slot goes to the slot of node i.
    ``path`` [requests, steps] and ``counts`` [requests] are those of :func:`tree_speculative_sample`: a path rises from node 0 on, what
    stands behind ``counts`` is not read.  The request then holds ``prefix_lens + counts`` tokens.  A request appears once in a call, and no two
    nodes share a slot."""
    ops = _ops()
    if ops.use_kernels(store):      # the binding makes the same checks
        return ops.ext().tree_kv_compact(store, req_to_token, req_pool_indices, prefix_lens, path, counts)
    what = "tree_kv_compact"
    if store.dim() < 2 or not store.is_contiguous() or store.shape[-1] * store.element_size() % 16:
        raise ValueError(f"{what}: store must be contiguous [.., slots, features] with rows of a multiple of 16 bytes")
    _check_index(what, counts.numel(), store.device, req_to_token, counts, req_pool_indices, prefix_lens)
    if path.dim() != 2 or path.shape[0] != counts.numel() or path.dtype != torch.int32 or not path.is_contiguous() or path.device != store.device:
        raise ValueError(f"{what}: path must be a contiguous int32 tensor [{counts.numel()}, steps] on {store.device}")
    if counts.numel() != req_pool_indices.numel():
        raise ValueError(f"{what}: counts must have one number per request")
    ref.tree_kv_compact(store, req_to_token, req_pool_indices, prefix_lens, path, counts)
