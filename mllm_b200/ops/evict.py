"""Operators that shorten requests in the paged cache: what is attended to stays, the rest makes room.

Each kv head of each layer has a sum of attention weights per cached token, ``sums[row of the request table, kv head, cache index]`` in fp32
(of all layers: one dimension in front).  The token at cache index i of request b owns the slot
``req_to_token[req_pool_indices[b], i]``.  Keys are cached with their positions turned in and attention does not ask which position a cache row
is of, so each head may keep tokens of its own: the request gets shorter, and its next token's *position* goes on counting.

    attention_prefill_weights(q, ...)                     per layer, behind a prompt's attention: what its last queries looked at
    keep, counts = cache_select(sums, ..., budgets)       all layers: the last tokens, the first ones, the largest sums
    cache_evict(store, sums, ..., keep, counts)           their rows and sums to the front, in order; the request has ``counts`` tokens now
    o = attention_decode_weights(q, ...)                  per layer: decode attention, and the weights added to the sums

Index tensors are contiguous int32 tensors on the device of the data.  Nothing here reads them on the host, so a step can be captured in a
CUDA graph; numbers that point outside the tensors are recorded (:func:`mllm_b200.ops.check_status`) and what they describe is left out.  A
request appears once in a call (a row of the table whose sums nobody reads may appear more often, as padded rows of a batch do), and
requests that share slots cannot be shortened.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import reference as ref

_front = None
_FP32 = torch.finfo(torch.float32)


def _ops():
    """The package that this module is part of; it is not complete while this one is imported."""
    global _front
    if _front is None:
        from .. import ops as _front
    return _front


def cache_weights_cover(head_dim: int, group: int, cache_dtype, act_dtype) -> bool:
    """Whether :func:`attention_decode_weights` and :func:`attention_prefill_weights` have kernels for such heads (``group`` query heads to a
    key head), rows and caches; on the GPU they refuse others."""
    return (head_dim in (64, 128, 256) and 1 <= group <= (16 if head_dim == 256 else 32) and act_dtype in (torch.bfloat16, torch.float16)
            and cache_dtype in (act_dtype, torch.float8_e4m3fn, torch.float8_e5m2))


def _check_ints(what: str, device, n: int, **vectors) -> None:
    for name, t in vectors.items():
        if t.shape != (n,) or t.dtype != torch.int32 or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{what}: {name} must be a contiguous int32 vector of {n} on {device}")


def _check_table(what: str, device, req_to_token) -> None:
    if req_to_token.dim() != 2 or req_to_token.dtype != torch.int32 or req_to_token.stride(1) != 1 or req_to_token.device != device:
        raise ValueError(f"{what}: req_to_token must be a two-dimensional int32 tensor with unit inner stride on {device}")


def _check_sums(what: str, device, sums, dims: int, heads: int) -> None:
    if (sums.dim() != dims or sums.dtype != torch.float32 or sums.shape[-2] != heads or (sums.stride(-1) != 1 and sums.shape[-1] != 1)
            or sums.device != device):
        raise ValueError(f"{what}: sums must be fp32 [{'layers, ' if dims == 4 else ''}requests, {heads}, tokens] with unit inner stride on {device}")


def _apart(t) -> bool:
    """Whether no element of a tensor that is written lies where another does (an expanded tensor's do)."""
    span = 1
    for stride, size in sorted((t.stride(i), t.shape[i]) for i in range(t.dim()) if t.shape[i] > 1):
        if stride < span:
            return t.numel() == 0
        span += stride * (size - 1)
    return True


def _check_written_sums(what: str, device, sums, dims: int, heads: int) -> None:
    _check_sums(what, device, sums, dims, heads)
    if not _apart(sums):
        raise ValueError(f"{what}: sums are written: their rows and heads must not overlap")


def _check_rows(what: str, q, caches, scale: float, logit_cap: float, sink) -> int:
    """Checks queries, caches and what makes scores of them; the number of kv heads."""
    if q.dim() != 3 or q.stride(2) != 1 or q.stride(1) != q.shape[2]:
        raise ValueError(f"{what}: q must be [rows, heads, features] with the heads of a row contiguous")
    for c in caches:
        if (c.dim() != 3 or c.shape != caches[0].shape or c.stride() != caches[0].stride() or c.dtype != caches[0].dtype or c.shape[2] != q.shape[2]
                or c.stride(2) != 1 or c.dtype not in (q.dtype, torch.float8_e4m3fn, torch.float8_e5m2) or c.device != q.device):
            raise ValueError(f"{what}: caches must be [slots, heads, {q.shape[2]}] views of one layout, of {q.dtype} or an 8-bit float, on {q.device}")
    hkv = caches[0].shape[1]
    if hkv == 0 or q.shape[1] == 0 or q.shape[1] % hkv:
        raise ValueError(f"{what}: {q.shape[1]} query heads over {hkv} key heads")
    most = _FP32.max / 2        # times log2 e it is finite still
    if not _FP32.tiny <= scale <= most:
        raise ValueError(f"{what}: scale must be positive and at most {most:.3g}, not {scale}")
    if logit_cap != 0 and not _FP32.tiny <= logit_cap <= most:
        raise ValueError(f"{what}: logit_cap must be 0, or positive and at most {most:.3g}, not {logit_cap}")
    if sink is not None and (sink.dtype != torch.float32 or sink.shape != (q.shape[1],) or not sink.is_contiguous() or sink.device != q.device):
        raise ValueError(f"{what}: sink must be fp32 [{q.shape[1]}] on {q.device}")
    return hkv


def attention_decode_weights(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, scale: float, sums, decay: float = 1.0,
                             out: Optional[torch.Tensor] = None, logit_cap: float = 0.0, sink: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`mllm_b200.ops.attention_decode` that adds up what is looked at: ``q`` [requests, Hq, D] -> [requests, Hq, D], and for the tokens of
    request b, in row ``req_pool_indices[b]`` of ``sums`` [rows, Hkv, tokens], ``sums <- decay * sums + weights``, the weights of a group's
    heads added up.  The sum of the newest token, at index ``seq_lens[b] - 1``, begins with its weights.  ``decay`` is from 0 to 1; ``sink`` joins
    the normaliser and has no sum.  Sums are made of unrounded weights in fp32.  Heads of 64, 128 (up to 32 query heads to a key head) and
    256 features (up to 16), 16-bit, over caches of their type or of unscaled 8-bit floats.  On the GPU a token whose slot lies outside the cache is
    seen by none and its weight is 0; a request that sees nothing has a row of zeros."""
    ops = _ops()
    if ops.use_kernels(q):          # the binding makes the same checks
        return ops.ext().attention_decode_weights(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, float(scale), sums, float(decay), out,
                                                  float(logit_cap or 0.0), sink)
    what = "attention_decode_weights"
    hkv = _check_rows(what, q, (k_cache, v_cache), scale, logit_cap, sink)
    _check_table(what, q.device, req_to_token)
    _check_ints(what, q.device, q.shape[0], req_pool_indices=req_pool_indices, seq_lens=seq_lens)
    _check_written_sums(what, q.device, sums, 3, hkv)
    if not 0.0 <= decay <= 1.0:
        raise ValueError(f"{what}: decay must be from 0 to 1, not {decay}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1 or out.stride(1) != out.shape[2]
                            or not _apart(out)):
        raise ValueError(f"{what}: out must be like q, with the heads of a row contiguous and rows apart")
    return ref.attention_decode_weights(q, k_cache, v_cache, req_to_token, req_pool_indices, seq_lens, scale, sums, decay, out, logit_cap, sink)


def attention_prefill_weights(q, k_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, scale: float, sums, last: int = 0,
                              add: bool = False, logit_cap: float = 0.0, sink: Optional[torch.Tensor] = None) -> None:
    """The weights that new tokens of prompts give to the cached tokens, for queries and keys as :func:`mllm_b200.ops.attention_prefill` takes them
    (call it behind the prologue; the attention itself is that function's).  Of request b's ``n = seq_lens[b] - prefix_lens[b]`` new rows, from
    ``q_start_loc[b]`` on, the last ``last`` are observed, all of them where that is 0 or more than n.  Every cached token's sum becomes what the
    observed queries behind it and at it give it, all heads of a group; with ``add``, tokens in front of the new ones (index below
    ``prefix_lens[b]``) keep what they have and get that on top.  A request without new rows is left as it is; no row of ``q`` is two requests'.
    Sizes and types as for :func:`attention_decode_weights`; a group has up to 32 heads at each of them, a batch up to 65535 requests."""
    ops = _ops()
    if ops.use_kernels(q):          # the binding makes the same checks
        return ops.ext().attention_prefill_weights(q, k_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, float(scale), sums,
                                                   int(last), bool(add), float(logit_cap or 0.0), sink)
    what = "attention_prefill_weights"
    hkv = _check_rows(what, q, (k_cache,), scale, logit_cap, sink)
    _check_table(what, q.device, req_to_token)
    _check_ints(what, q.device, req_pool_indices.numel(), req_pool_indices=req_pool_indices, seq_lens=seq_lens, prefix_lens=prefix_lens,
                q_start_loc=q_start_loc)
    _check_written_sums(what, q.device, sums, 3, hkv)
    if last < 0:
        raise ValueError(f"{what}: last must be 0 (all new tokens) or positive, not {last}")
    ref.attention_prefill_weights(q, k_cache, req_to_token, req_pool_indices, seq_lens, prefix_lens, q_start_loc, scale, sums, int(last), bool(add),
                                  logit_cap, sink)


def cache_select(sums, req_pool_indices, seq_lens, budgets, max_budget: int, first: int = 4, recent: int = 32, pool: int = 1
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which tokens stay: ``(keep [layers, requests, Hkv, max_budget], counts [requests])``, int32.  ``counts[b]`` is ``budgets[b]``, at most
    ``max_budget`` and the request's ``seq_lens[b]``.  Of every list of ``sums`` [layers, rows, Hkv, tokens] stay the last ``recent`` tokens, then of
    the others the first ``first``, then those with the largest scores until there are ``counts[b]``; a score is the largest of the ``pool`` sums
    (odd, up to 63) around the token (of the request's tokens, the first and the last ones among them, so that the ``pool // 2`` beside those
    inherit theirs), ties go to the lowest index, NaN counts as minus infinity.  The kept tokens' cache indices rise; behind them
    stands -1."""
    ops = _ops()
    if ops.use_kernels(sums):       # the binding makes the same checks
        return tuple(ops.ext().cache_select(sums, req_pool_indices, seq_lens, budgets, int(max_budget), int(first), int(recent), int(pool)))
    what = "cache_select"
    if sums.dim() != 4:
        raise ValueError(f"{what}: sums must be [layers, requests, heads, tokens]")
    _check_sums(what, sums.device, sums, 4, sums.shape[2])
    _check_ints(what, sums.device, req_pool_indices.numel(), req_pool_indices=req_pool_indices, seq_lens=seq_lens, budgets=budgets)
    if not 0 <= max_budget <= sums.shape[3]:
        raise ValueError(f"{what}: max_budget must be from 0 to the {sums.shape[3]} tokens of the sums, not {max_budget}")
    if first < 0 or recent < 0:
        raise ValueError(f"{what}: first and recent are numbers of tokens, not {first} and {recent}")
    if pool < 1 or pool > 63 or pool % 2 == 0:
        raise ValueError(f"{what}: pool must be odd and from 1 to 63, not {pool}")
    return ref.cache_select(sums, req_pool_indices, seq_lens, budgets, int(max_budget), int(first), int(recent), int(pool))


def cache_evict(store, sums, req_to_token, req_pool_indices, keep, counts) -> None:
    """Moves what stays to the front, in place: for i below ``counts[b]``, what the token at cache index ``keep[layer, b, head, i]`` has in ``store``
    [layers, 2, Hkv, slots, features] (contiguous; :class:`mllm_b200.mem_cache.memory_pool.KVPool`'s storage) and in ``sums`` [layers, rows, Hkv,
    tokens] (or None) goes to index i.  ``keep`` and ``counts`` are those of :func:`cache_select`; no index may be smaller than its place, and none
    is read behind ``counts``.  The request then has ``counts[b]`` tokens, and nothing is kept in its slots from there on (a paged allocator takes
    pages back: :meth:`mllm_b200.mem_cache.memory_pool.TokenToKVPoolAllocator.free_behind`)."""
    ops = _ops()
    if ops.use_kernels(store):      # the binding makes the same checks
        return ops.ext().cache_evict(store, sums, req_to_token, req_pool_indices, keep, counts)
    what = "cache_evict"
    if store.dim() != 5 or store.shape[1] != 2 or not store.is_contiguous() or store.shape[4] * store.element_size() % 16:
        raise ValueError(f"{what}: store must be contiguous [layers, 2, heads, slots, features] with rows of 16-byte multiples")
    batch, dev = req_pool_indices.numel(), store.device
    _check_table(what, dev, req_to_token)
    _check_ints(what, dev, batch, req_pool_indices=req_pool_indices, counts=counts)
    if (keep.dim() != 4 or keep.shape[:3] != (store.shape[0], batch, store.shape[2]) or keep.dtype != torch.int32 or not keep.is_contiguous()
            or keep.device != dev):
        raise ValueError(f"{what}: keep must be contiguous int32 [{store.shape[0]}, {batch}, {store.shape[2]}, tokens] on {dev}")
    if sums is not None:
        _check_written_sums(what, dev, sums, 4, store.shape[2])
        if sums.shape[0] != store.shape[0]:
            raise ValueError(f"{what}: sums of {sums.shape[0]} layers, and a store of {store.shape[0]}")
    ref.cache_evict(store, sums, req_to_token, req_pool_indices, keep, counts)
