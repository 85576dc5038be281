"""Serving operators on torch tensors: what a serving loop needs beside the one-token greedy step.

* ``tree_attention``  attention of drafted tokens (one token tree per sequence) over the KV cache
* ``tree_masks``      masks and depths of token trees from parent indices (host side)
* ``cache_commit``    the accepted path of each tree moved into place in the KV cache
* ``lora_apply``      low-rank adapters of many requests at once beside a shared projection
* ``route_experts``   experts from softmax / sigmoid scores with a balancing bias, groups, renormalised weights
                      (``MoEBlock.forward_routed`` runs the expert GEMMs on the result)

Each call runs on the device of its tensors, asynchronously on ``stream`` (default: that device's current stream); scratch
comes from torch's allocator, so calls on different streams and captured graphs have their own.  Errors raise
``GptossError``.  Nothing is kept between calls.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import capi
from .moe import GptossError

TREE_MAX_NODES = 256
_SCORING = {"softmax": 0, "sigmoid": 1}


def _check(rc):
    if rc != capi.OK:
        raise GptossError(rc, capi.load().gptoss_serving_last_error().decode())


def _bad(message):
    raise GptossError(capi.ERR_BAD_ARG, message)


def _need(name, t, dtype, ndim, device=None):
    """t is a cuda tensor of that type and rank, contiguous in its last dimension, on `device`."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != ndim:
        _bad(f"{name} must be a {dtype} tensor of {ndim} dimensions")
    if not t.is_cuda:
        _bad(f"{name} must be a cuda tensor")
    if device is not None and t.device != device:
        _bad(f"{name} is on {t.device}, expected {device}")


def _dense(name, t, dtype, ndim, device):
    _need(name, t, dtype, ndim, device)
    if not t.is_contiguous():
        _bad(f"{name} must be contiguous")


def _launch(device, stream, call):
    """call(stream handle) with `device` current and, for what it allocates, `stream` as torch's current stream."""
    with torch.cuda.device(device):
        if stream is None:
            return call(C.c_void_p(torch.cuda.current_stream().cuda_stream))
        with torch.cuda.stream(stream):
            return call(C.c_void_p(stream.cuda_stream))


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
    _need("q", q, torch.bfloat16, 3)
    dev = q.device
    n_tokens, nq, hd = q.shape
    if q.stride(2) != 1 or q.stride(1) != hd:
        _bad("q: heads of a token must be contiguous")
    _dense("k_cache", k_cache, torch.bfloat16, 4, dev)
    _dense("v_cache", v_cache, torch.bfloat16, 4, dev)
    if k_cache.shape != v_cache.shape or k_cache.shape[3] != hd:
        _bad("k_cache and v_cache must have the same shape and q's head_dim")
    _dense("offsets", offsets, torch.int32, 1, dev)
    _dense("ctx_len", ctx_len, torch.int32, 1, dev)
    _dense("mask", mask, torch.int32, 2, dev)
    n_seqs = ctx_len.shape[0]
    if offsets.shape[0] != n_seqs + 1 or mask.shape[0] < n_tokens:
        _bad("offsets needs one more entry than ctx_len, mask a row per token")
    if depth is not None:
        _dense("depth", depth, torch.int32, 1, dev)
        if depth.shape[0] < n_tokens:
            _bad("depth needs an entry per token")
    if sinks is not None:
        _dense("sinks", sinks, torch.float32, 1, dev)
        if sinks.shape[0] != nq:
            _bad("sinks needs an entry per query head")
    if cache_rows is not None:
        _dense("cache_rows", cache_rows, torch.int32, 1, dev)
        if cache_rows.shape[0] != n_seqs:
            _bad("cache_rows needs an entry per sequence")
    if out is not None:
        _need("out", out, torch.bfloat16, 3, dev)
        if out.shape != q.shape or out.stride(2) != 1 or out.stride(1) != hd:
            _bad("out must have q's shape and contiguous heads")
    rows, nkv, max_seq, _ = k_cache.shape
    stride = lambda t: t.stride(0) if n_tokens > 1 else nq * hd  # noqa: E731
    args = capi.TreeAttentionArgs(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), None, offsets.data_ptr(), ctx_len.data_ptr(),
        None if cache_rows is None else cache_rows.data_ptr(), mask.data_ptr(), None if depth is None else depth.data_ptr(),
        None if sinks is None else sinks.data_ptr(), None, 0, stride(q), 0, n_tokens, n_seqs, max_nodes, max_ctx,
        mask.shape[1], rows, max_seq, nq, nkv, hd, window, hd ** -0.5 if scale is None else scale)

    def call(s):
        nonlocal out
        if out is None:
            out = torch.empty((n_tokens, nq, hd), dtype=torch.bfloat16, device=dev)
        args.out, args.out_stride = out.data_ptr(), stride(out)
        lib = capi.load()
        need = lib.gptoss_tree_attention_workspace(C.byref(args))
        if need:
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            args.workspace, args.workspace_bytes = work.data_ptr(), need
        _check(lib.gptoss_tree_attention(C.byref(args), s))

    _launch(dev, stream, call)
    return out


def cache_commit(k_cache, v_cache, ctx_len, offsets, path, *, max_path, cache_rows=None, stream=None):
    """Moves the accepted path of each tree into place, in the caches [layers, rows, n_kv_heads, max_seq, head_dim] (or
    without the layers), bf16.  path int32: the accepted drafted tokens of all sequences, ascending within one; sequence b
    has path[offsets[b]:offsets[b+1]], at most max_path.  ``gptoss_cache_commit`` in the C header."""
    if isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4 and isinstance(v_cache, torch.Tensor):
        k_cache, v_cache = k_cache[None], v_cache[None]
    _need("k_cache", k_cache, torch.bfloat16, 5)
    dev = k_cache.device
    _dense("k_cache", k_cache, torch.bfloat16, 5, dev)
    _dense("v_cache", v_cache, torch.bfloat16, 5, dev)
    if k_cache.shape != v_cache.shape:
        _bad("k_cache and v_cache must have the same shape")
    _dense("ctx_len", ctx_len, torch.int32, 1, dev)
    _dense("offsets", offsets, torch.int32, 1, dev)
    _dense("path", path, torch.int32, 1, dev)
    n_seqs = ctx_len.shape[0]
    if offsets.shape[0] != n_seqs + 1:
        _bad("offsets needs one more entry than ctx_len")
    if cache_rows is not None:
        _dense("cache_rows", cache_rows, torch.int32, 1, dev)
        if cache_rows.shape[0] != n_seqs:
            _bad("cache_rows needs an entry per sequence")
    layers, rows, nkv, max_seq, hd = k_cache.shape
    _launch(dev, stream, lambda s: _check(capi.load().gptoss_cache_commit(
        k_cache.data_ptr(), v_cache.data_ptr(), layers, rows, nkv, max_seq, hd, n_seqs,
        None if cache_rows is None else cache_rows.data_ptr(), ctx_len.data_ptr(), offsets.data_ptr(), path.data_ptr(),
        max_path if path.shape[0] else 0, s)))


def lora_apply(x, a, b, ids, y, *, scale=None, out=None, stream=None):
    """out[t] = y[t] + scale[ids[t]] * b[ids[t]] (a[ids[t]] x[t]); a token whose id is outside [0, n_adapters) keeps y[t].

    x [T, K] bf16, a [n_adapters, rank, K] bf16, b [n_adapters, n_out, rank] bf16, ids int32 [T], y fp32 [T, n_out], scale
    fp32 [n_adapters].  out: y itself by default (in place).  ``gptoss_lora_apply`` in the C header."""
    _need("x", x, torch.bfloat16, 2)
    dev = x.device
    T, K = x.shape
    _dense("a", a, torch.bfloat16, 3, dev)
    _dense("b", b, torch.bfloat16, 3, dev)
    n, rank, _ = a.shape
    n_out = b.shape[1]
    if a.shape[2] != K or b.shape[0] != n or b.shape[2] != rank:
        _bad("a must be [n_adapters, rank, K] and b [n_adapters, n_out, rank]")
    _dense("ids", ids, torch.int32, 1, dev)
    out = y if out is None else out
    for name, t in (("y", y), ("out", out)):
        _need(name, t, torch.float32, 2, dev)
        if t.shape != (T, n_out) or (n_out > 1 and t.stride(1) != 1):
            _bad(f"{name} must be [T, n_out] with contiguous rows")
    if ids.shape[0] != T or (K > 1 and x.stride(1) != 1):
        _bad("ids needs an entry per token, x contiguous rows")
    if scale is not None:
        _dense("scale", scale, torch.float32, 1, dev)
        if scale.shape[0] != n:
            _bad("scale needs an entry per adapter")
    one = T <= 1
    args = capi.LoraArgs(x.data_ptr(), a.data_ptr(), b.data_ptr(), None if scale is None else scale.data_ptr(), ids.data_ptr(),
                         y.data_ptr(), out.data_ptr(), None, 0, K if one else x.stride(0), n_out if one else y.stride(0),
                         n_out if one else out.stride(0), T, K, n_out, rank, n)

    def call(s):
        lib = capi.load()
        need = lib.gptoss_lora_workspace(C.byref(args))
        if need:
            work = torch.empty(need, dtype=torch.uint8, device=dev)
            args.workspace, args.workspace_bytes = work.data_ptr(), need
        _check(lib.gptoss_lora_apply(C.byref(args), s))

    _launch(dev, stream, call)
    return out


def route_experts(logits, top_k, *, scoring="softmax", bias=None, n_groups=1, topk_groups=1, group_top=1, renormalize=True,
                  weight_scale=1.0, stream=None):
    """Experts of each token from router logits [T, E] fp32: (weights fp32 [T, top_k], ids int32 [T, top_k]) in descending
    order of the choice.  ``gptoss_expert_choice`` in the C header says how they are chosen."""
    _need("logits", logits, torch.float32, 2)
    dev = logits.device
    T, E = logits.shape
    if E > 1 and logits.stride(1) != 1:
        _bad("logits must have contiguous rows")
    if bias is not None:
        _dense("bias", bias, torch.float32, 1, dev)
        if bias.shape[0] != E:
            _bad("bias needs an entry per expert")
    if scoring not in _SCORING:
        _bad("scoring must be 'softmax' or 'sigmoid'")
    if not 1 <= top_k <= 8:
        _bad("top_k must be 1..8")

    def call(s):
        w = torch.empty((T, top_k), dtype=torch.float32, device=dev)
        ids = torch.empty((T, top_k), dtype=torch.int32, device=dev)
        args = capi.ExpertChoiceArgs(logits.data_ptr(), None if bias is None else bias.data_ptr(), w.data_ptr(), ids.data_ptr(),
                                     logits.stride(0) if T > 1 else E, T, E, top_k, _SCORING[scoring], n_groups, topk_groups,
                                     group_top, int(renormalize), weight_scale)
        _check(capi.load().gptoss_expert_choice(C.byref(args), s))
        return w, ids

    return _launch(dev, stream, call)
