"""Serving operators on torch tensors: what a serving loop needs beside the one-token greedy step.

* ``tree_attention``  attention of drafted tokens (one token tree per sequence) over the KV cache
* ``tree_masks``      masks and depths of token trees from parent indices (host side)
* ``cache_commit``    the accepted path of each tree moved into place in the KV cache
* ``lora_apply``      low-rank adapters of many requests at once beside a shared projection
* ``route_experts``   experts from softmax / sigmoid scores with a balancing bias, groups, renormalised weights
                      (``MoEBlock.forward_routed`` runs the expert GEMMs on the result)
* ``status``          whether the calls so far ran as they should (synchronises)

Each call runs on the device of its tensors, asynchronously on ``stream`` (default: that device's current stream); scratch
comes from torch's allocator, so calls on different streams and captured graphs have their own.  As with torch's own
operators, a tensor that belongs to another stream than the one it is used on is the caller's to keep alive and to order
(``record_stream``, ``wait_stream``); what a call returns belongs to the stream it ran on.  Refused arguments and failed launches
raise ``GptossError``; a wait on the GPU that gives up (its results mean nothing then) is noted there, and ``status`` raises it.
Nothing else is kept between calls.  There is no backward pass: tensors that require a gradient are refused while gradients are
recorded (they pass under ``torch.no_grad()``).

The calls are short on the GPU (from 2 us), so their host side counts: csrc/serving_torch.cpp looks the tensors over,
allocates and calls the C ABI (3 to 5 us a call; in Python that was 8 to 13).
"""
from __future__ import annotations

import contextlib
import ctypes as C
import importlib.util

import numpy as np
import torch

from . import capi
from .moe import GptossError

TREE_MAX_NODES = 256
_SCORING = {"softmax": 0, "sigmoid": 1}
_binding = None


def _bind():
    """The compiled binding, with the C functions of the loaded library."""
    global _binding
    if capi.TORCH_LIB_PATH is None or not capi.TORCH_LIB_PATH.exists():
        raise RuntimeError(f"{capi.TORCH_LIB_PATH or 'the binding to torch'} is missing: run `python -c 'import __graft_entry__ as e; e.build()'` first")
    lib = capi.load()
    spec = importlib.util.spec_from_file_location("_serving_torch", capi.TORCH_LIB_PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.bind(GptossError, *[C.cast(getattr(lib, "gptoss_" + f), C.c_void_p).value for f in (
        "tree_attention", "tree_attention_workspace", "cache_commit", "lora_apply", "lora_workspace", "expert_choice",
        "serving_last_error")])
    _binding = mod
    return mod


def _bad(message):
    raise GptossError(capi.ERR_BAD_ARG, message)


def _on(stream, t, call, *args):
    """call(t, *args) with `stream`, of t's device, as torch's current one."""
    if isinstance(t, torch.Tensor) and t.device != stream.device:
        _bad("the stream belongs to another device than the tensors")
    with torch.cuda.stream(stream):
        return call(t, *args)


def status(device=None):
    """Waits for all work of a device (default: the current one) and raises GptossError if a kernel of these operators gave up on a
    bounded wait since the last such call, or if the device reports an error."""
    lib = capi.load()
    with contextlib.nullcontext() if device is None else torch.cuda.device(device):
        rc = lib.gptoss_serving_status()
    if rc != capi.OK:
        raise GptossError(rc, lib.gptoss_serving_last_error().decode())


def tree_masks(parents, max_nodes=None):
    """parents: per sequence the parent of each drafted token (an earlier index of the same tree, or -1 for a token that
    follows the last cached one).  Returns numpy int32 arrays (offsets [B+1], mask [n_tokens, words], depth [n_tokens]) in
    which every token sees its ancestors and itself."""
    offsets = np.zeros(len(parents) + 1, np.int32)
    for b, p in enumerate(parents):
        offsets[b + 1] = offsets[b] + len(p)
    widest = max((len(p) for p in parents), default=0)
    if widest > TREE_MAX_NODES:
        _bad(f"more than {TREE_MAX_NODES} drafted tokens in a sequence")
    words = max(1, (max(widest, max_nodes or 0) + 31) // 32)
    mask = np.zeros((int(offsets[-1]), words), np.uint32)
    depth = np.zeros(int(offsets[-1]), np.int32)
    for b, ps in enumerate(parents):
        for i, p in enumerate(ps):
            if not -1 <= p < i:
                _bad(f"sequence {b}: the parent of token {i} must be -1 or an earlier token")
            t = offsets[b] + i
            if p >= 0:
                mask[t] = mask[offsets[b] + p]
                depth[t] = depth[offsets[b] + p] + 1
            mask[t, i >> 5] |= np.uint32(1 << (i & 31))
    return offsets, mask.view(np.int32), depth


def tree_attention(q, k_cache, v_cache, offsets, ctx_len, mask, depth=None, *, max_nodes, max_ctx, sinks=None, cache_rows=None,
                   window=0, scale=None, out=None, stream=None):
    """Attention of drafted tokens over the cache (``gptoss_tree_attention`` in the C header says what it computes).

    q [n_tokens, n_q_heads, head_dim] bf16 (the token stride is free), caches [rows, n_kv_heads, max_seq, head_dim] bf16,
    offsets int32 [B+1], ctx_len int32 [B], mask int32 [n_tokens, words], depth int32 [n_tokens] (with a window), sinks fp32
    [n_q_heads], cache_rows int32 [B].  max_nodes / max_ctx: upper bounds of the drafted / cached tokens of a sequence.
    Returns out like q (bf16); rows behind the last sequence are not written."""
    call = (_binding or _bind()).tree_attention
    if stream is None:
        return call(q, k_cache, v_cache, offsets, ctx_len, mask, depth, max_nodes, max_ctx, sinks, cache_rows, window, scale, out)
    return _on(stream, q, call, k_cache, v_cache, offsets, ctx_len, mask, depth, max_nodes, max_ctx, sinks, cache_rows, window, scale, out)


def cache_commit(k_cache, v_cache, ctx_len, offsets, path, *, max_path, cache_rows=None, stream=None):
    """Moves the accepted path of each tree into place, in the caches [layers, rows, n_kv_heads, max_seq, head_dim] (or
    without the layers), bf16.  path int32: the accepted drafted tokens of all sequences, ascending within one; sequence b
    has path[offsets[b]:offsets[b+1]], at most max_path.  ``gptoss_cache_commit`` in the C header."""
    call = (_binding or _bind()).cache_commit
    if stream is None:
        call(k_cache, v_cache, ctx_len, offsets, path, max_path, cache_rows)
    else:
        _on(stream, k_cache, call, v_cache, ctx_len, offsets, path, max_path, cache_rows)


def lora_apply(x, a, b, ids, y, *, scale=None, out=None, stream=None):
    """out[t] = y[t] + scale[ids[t]] * b[ids[t]] (a[ids[t]] x[t]); a token whose id is outside [0, n_adapters) keeps y[t].

    x [T, K] bf16, a [n_adapters, rank, K] bf16, b [n_adapters, n_out, rank] bf16, ids int32 [T], y fp32 [T, n_out], scale
    fp32 [n_adapters].  out: y itself by default (in place).  ``gptoss_lora_apply`` in the C header."""
    call = (_binding or _bind()).lora_apply
    if stream is None:
        return call(x, a, b, ids, y, scale, out)
    return _on(stream, x, call, a, b, ids, y, scale, out)


def route_experts(logits, top_k, *, scoring="softmax", bias=None, n_groups=1, topk_groups=1, group_top=1, renormalize=True,
                  weight_scale=1.0, stream=None):
    """Experts of each token from router logits [T, E] fp32: (weights fp32 [T, top_k], ids int32 [T, top_k]) in descending
    order of the choice.  ``gptoss_expert_choice`` in the C header says how they are chosen."""
    call = (_binding or _bind()).route_experts
    if scoring not in _SCORING:
        _bad("scoring must be 'softmax' or 'sigmoid'")
    args = (top_k, _SCORING[scoring], bias, n_groups, topk_groups, group_top, renormalize, weight_scale)
    if stream is None:
        return call(logits, *args)
    return _on(stream, logits, call, *args)
