"""Serving operators on torch tensors: what a serving loop needs beside the one-token greedy step.

* ``tree_attention``  attention of drafted tokens (one token tree per sequence) over the KV cache
* ``tree_masks``      masks and depths of token trees from parent indices (host side)
* ``cache_commit``    the accepted path of each tree moved into place in the KV cache
* ``lora_apply``      low-rank adapters of many requests at once beside a shared projection
* ``route_experts``   experts from softmax / sigmoid scores with a balancing bias, groups, renormalised weights
                      (``MoEBlock.forward_routed`` runs the expert GEMMs on the result)

Each call runs on the device of its tensors, asynchronously on ``stream`` (default: that device's current stream); scratch
comes from torch's allocator, so calls on different streams and captured graphs have their own.  As with torch's own
operators, a tensor that belongs to another stream than the one it is used on is the caller's to keep alive and to order
(``record_stream``, ``wait_stream``); what a call returns belongs to the stream it ran on.  Errors raise ``GptossError``.
Nothing is kept between calls.

The calls are short on the GPU (from 2 us), so their host side counts: what a call is given is looked over in one
expression, and only where that fails are the arguments gone through one by one for the message; the raw stream handle is
asked for directly (a ``torch.cuda.Stream`` object costs 3 us, a device context 1.4 us).
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import capi
from .moe import GptossError

TREE_MAX_NODES = 256
_SCORING = {"softmax": 0, "sigmoid": 1}
_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _check(rc):
    if rc:
        raise GptossError(rc, capi.load().gptoss_serving_last_error().decode())


def _bad(message):
    raise GptossError(capi.ERR_BAD_ARG, message)


def _view(name, t, dtype, ndim, dev=None):
    """t is a tensor of that type and number of dimensions on cuda device `dev` (default: any); returns its device."""
    try:
        at = t.get_device()
        if t.dtype is dtype and t.dim() == ndim and at >= 0 and (dev is None or at == dev):
            return at
    except AttributeError:
        pass
    where = "a cuda device" if dev is None else f"cuda:{dev}"
    _bad(f"{name} must be a {dtype} tensor of {ndim} dimensions on {where}")


def _dense(name, t, dtype, ndim, dev):
    _view(name, t, dtype, ndim, dev)
    if not t.is_contiguous():
        _bad(f"{name} must be contiguous")


def _launch(dev, stream, call, *args):
    """call(stream handle, *args) with device `dev` current and, for what it allocates, `stream` as torch's current one."""
    if stream is None and _current_device() == dev:
        return call(_raw_stream(dev), *args)
    with torch.cuda.device(dev):
        if stream is None:
            return call(_raw_stream(dev), *args)
        with torch.cuda.stream(stream):
            return call(stream.cuda_stream, *args)


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
    try:
        dev = q.get_device()
        plain = (
            q.dtype is _BF16 is k_cache.dtype is v_cache.dtype and offsets.dtype is _I32 is ctx_len.dtype is mask.dtype
            and q.dim() == 3 and k_cache.dim() == 4 and mask.dim() == 2 and offsets.dim() == 1 == ctx_len.dim()
            and 0 <= dev == k_cache.get_device() == v_cache.get_device() == offsets.get_device() == ctx_len.get_device() == mask.get_device()
            and k_cache.is_contiguous() and v_cache.is_contiguous() and offsets.is_contiguous() and ctx_len.is_contiguous()
            and mask.is_contiguous()
            and (depth is None or depth.dtype is _I32 and depth.dim() == 1 and depth.get_device() == dev and depth.is_contiguous())
            and (sinks is None or sinks.dtype is _F32 and sinks.dim() == 1 and sinks.get_device() == dev and sinks.is_contiguous())
            and (cache_rows is None or cache_rows.dtype is _I32 and cache_rows.dim() == 1 and cache_rows.get_device() == dev
                 and cache_rows.is_contiguous()))
    except AttributeError:
        plain = False
    if not plain:
        dev = _view("q", q, _BF16, 3)
        _dense("k_cache", k_cache, _BF16, 4, dev)
        _dense("v_cache", v_cache, _BF16, 4, dev)
        _dense("offsets", offsets, _I32, 1, dev)
        _dense("ctx_len", ctx_len, _I32, 1, dev)
        _dense("mask", mask, _I32, 2, dev)
        for name, t, dtype in (("depth", depth, _I32), ("sinks", sinks, _F32), ("cache_rows", cache_rows, _I32)):
            if t is not None:
                _dense(name, t, dtype, 1, dev)
    n_tokens, nq, hd = q.shape
    token_stride, head_stride, last = q.stride()
    if last != 1 or (head_stride != hd and nq > 1):
        _bad("q: heads of a token must be contiguous")
    rows, nkv, max_seq, cache_hd = k_cache.shape
    if v_cache.shape != k_cache.shape or cache_hd != hd:
        _bad("k_cache and v_cache must have the same shape and q's head_dim")
    n_seqs = ctx_len.shape[0]
    mask_rows, words = mask.shape
    if offsets.shape[0] != n_seqs + 1 or mask_rows < n_tokens:
        _bad("offsets needs one more entry than ctx_len, mask a row per token")
    depth_at = sinks_at = rows_at = None
    if depth is not None:
        if depth.shape[0] < n_tokens:
            _bad("depth needs an entry per token")
        depth_at = depth.data_ptr()
    if sinks is not None:
        if sinks.shape[0] != nq:
            _bad("sinks needs an entry per query head")
        sinks_at = sinks.data_ptr()
    if cache_rows is not None:
        if cache_rows.shape[0] != n_seqs:
            _bad("cache_rows needs an entry per sequence")
        rows_at = cache_rows.data_ptr()
    if out is not None:
        _view("out", out, _BF16, 3, dev)
        if out.shape != q.shape or out.stride(2) != 1 or (out.stride(1) != hd and nq > 1):
            _bad("out must have q's shape and contiguous heads")
    if n_tokens <= 1:
        token_stride = nq * hd
    args = capi.TreeAttentionArgs(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), None, offsets.data_ptr(), ctx_len.data_ptr(), rows_at,
        mask.data_ptr(), depth_at, sinks_at, None, 0, token_stride, 0, n_tokens, n_seqs, max_nodes, max_ctx, words, rows, max_seq,
        nq, nkv, hd, window, hd ** -0.5 if scale is None else scale)
    return _launch(dev, stream, _tree_attention, args, q, out)


def _tree_attention(s, args, q, out):
    lib = capi.load()
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    args.out = out.data_ptr()
    args.out_stride = out.stride(0) if args.n_tokens > 1 else args.n_q_heads * args.head_dim
    need = lib.gptoss_tree_attention_workspace(C.byref(args))
    if need:
        work = q.new_empty(need, dtype=torch.uint8)
        args.workspace, args.workspace_bytes = work.data_ptr(), need
    _check(lib.gptoss_tree_attention(C.byref(args), s))
    return out


def cache_commit(k_cache, v_cache, ctx_len, offsets, path, *, max_path, cache_rows=None, stream=None):
    """Moves the accepted path of each tree into place, in the caches [layers, rows, n_kv_heads, max_seq, head_dim] (or
    without the layers), bf16.  path int32: the accepted drafted tokens of all sequences, ascending within one; sequence b
    has path[offsets[b]:offsets[b+1]], at most max_path.  ``gptoss_cache_commit`` in the C header."""
    try:
        dev, ndim = k_cache.get_device(), k_cache.dim()
        plain = (
            k_cache.dtype is _BF16 is v_cache.dtype and ctx_len.dtype is _I32 is offsets.dtype is path.dtype and 4 <= ndim <= 5
            and ctx_len.dim() == 1 == offsets.dim() == path.dim()
            and 0 <= dev == v_cache.get_device() == ctx_len.get_device() == offsets.get_device() == path.get_device()
            and k_cache.is_contiguous() and v_cache.is_contiguous() and ctx_len.is_contiguous() and offsets.is_contiguous()
            and path.is_contiguous()
            and (cache_rows is None or cache_rows.dtype is _I32 and cache_rows.dim() == 1 and cache_rows.get_device() == dev
                 and cache_rows.is_contiguous()))
    except AttributeError:
        plain = False
    if not plain:
        ndim = 4 if isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4 else 5
        dev = _view("k_cache", k_cache, _BF16, ndim)
        _dense("k_cache", k_cache, _BF16, ndim, dev)
        _dense("v_cache", v_cache, _BF16, ndim, dev)
        _dense("ctx_len", ctx_len, _I32, 1, dev)
        _dense("offsets", offsets, _I32, 1, dev)
        _dense("path", path, _I32, 1, dev)
        if cache_rows is not None:
            _dense("cache_rows", cache_rows, _I32, 1, dev)
    shape = k_cache.shape
    if v_cache.shape != shape:
        _bad("k_cache and v_cache must have the same shape")
    n_seqs = ctx_len.shape[0]
    if offsets.shape[0] != n_seqs + 1:
        _bad("offsets needs one more entry than ctx_len")
    rows_at = None
    if cache_rows is not None:
        if cache_rows.shape[0] != n_seqs:
            _bad("cache_rows needs an entry per sequence")
        rows_at = cache_rows.data_ptr()
    layers = 1 if ndim == 4 else shape[0]
    rows, nkv, max_seq, hd = shape[-4:]
    _launch(dev, stream, _cache_commit, k_cache.data_ptr(), v_cache.data_ptr(), layers, rows, nkv, max_seq, hd, n_seqs, rows_at,
            ctx_len.data_ptr(), offsets.data_ptr(), path.data_ptr(), path.shape[0], max_path)


def _cache_commit(s, *args):
    _check(capi.load().gptoss_cache_commit(*args, s))


def lora_apply(x, a, b, ids, y, *, scale=None, out=None, stream=None):
    """out[t] = y[t] + scale[ids[t]] * b[ids[t]] (a[ids[t]] x[t]); a token whose id is outside [0, n_adapters) keeps y[t].

    x [T, K] bf16, a [n_adapters, rank, K] bf16, b [n_adapters, n_out, rank] bf16, ids int32 [T], y fp32 [T, n_out], scale
    fp32 [n_adapters].  out: y itself by default (in place).  ``gptoss_lora_apply`` in the C header."""
    if out is None:
        out = y
    try:
        dev = x.get_device()
        plain = (
            x.dtype is _BF16 is a.dtype is b.dtype and ids.dtype is _I32 and y.dtype is _F32 is out.dtype
            and x.dim() == 2 == y.dim() == out.dim() and a.dim() == 3 == b.dim() and ids.dim() == 1
            and 0 <= dev == a.get_device() == b.get_device() == ids.get_device() == y.get_device() == out.get_device()
            and a.is_contiguous() and b.is_contiguous() and ids.is_contiguous()
            and (scale is None or scale.dtype is _F32 and scale.dim() == 1 and scale.get_device() == dev and scale.is_contiguous()))
    except AttributeError:
        plain = False
    if not plain:
        dev = _view("x", x, _BF16, 2)
        _dense("a", a, _BF16, 3, dev)
        _dense("b", b, _BF16, 3, dev)
        _dense("ids", ids, _I32, 1, dev)
        _view("y", y, _F32, 2, dev)
        _view("out", out, _F32, 2, dev)
        if scale is not None:
            _dense("scale", scale, _F32, 1, dev)
    T, K = x.shape
    n, rank, a_k = a.shape
    b_n, n_out, b_rank = b.shape
    if a_k != K or b_n != n or b_rank != rank:
        _bad("a must be [n_adapters, rank, K] and b [n_adapters, n_out, rank]")
    x_stride, y_stride, out_stride = x.stride(), y.stride(), out.stride()
    if y.shape != (T, n_out) or out.shape != y.shape or y_stride[1] != 1 or out_stride[1] != 1:
        _bad("y and out must be [T, n_out] with contiguous rows")
    if ids.shape[0] != T or x_stride[1] != 1:
        _bad("ids needs an entry per token, x contiguous rows")
    scale_at = None
    if scale is not None:
        if scale.shape[0] != n:
            _bad("scale needs an entry per adapter")
        scale_at = scale.data_ptr()
    one = T <= 1
    args = capi.LoraArgs(x.data_ptr(), a.data_ptr(), b.data_ptr(), scale_at, ids.data_ptr(), y.data_ptr(), out.data_ptr(), None, 0,
                         K if one else x_stride[0], n_out if one else y_stride[0], n_out if one else out_stride[0], T, K, n_out,
                         rank, n)
    _launch(dev, stream, _lora_apply, args, x)
    return out


def _lora_apply(s, args, x):
    lib = capi.load()
    need = lib.gptoss_lora_workspace(C.byref(args))
    if need:
        work = x.new_empty(need, dtype=torch.uint8)
        args.workspace, args.workspace_bytes = work.data_ptr(), need
    _check(lib.gptoss_lora_apply(C.byref(args), s))


def route_experts(logits, top_k, *, scoring="softmax", bias=None, n_groups=1, topk_groups=1, group_top=1, renormalize=True,
                  weight_scale=1.0, stream=None):
    """Experts of each token from router logits [T, E] fp32: (weights fp32 [T, top_k], ids int32 [T, top_k]) in descending
    order of the choice.  ``gptoss_expert_choice`` in the C header says how they are chosen."""
    dev = _view("logits", logits, _F32, 2)
    T, E = logits.shape
    stride, last = logits.stride()
    if last != 1 and E > 1:
        _bad("logits must have contiguous rows")
    bias_at = None
    if bias is not None:
        _dense("bias", bias, _F32, 1, dev)
        if bias.shape[0] != E:
            _bad("bias needs an entry per expert")
        bias_at = bias.data_ptr()
    if scoring not in _SCORING:
        _bad("scoring must be 'softmax' or 'sigmoid'")
    if not 1 <= top_k <= 8:
        _bad("top_k must be 1..8")
    args = capi.ExpertChoiceArgs(logits.data_ptr(), bias_at, None, None, stride if T > 1 else E, T, E, top_k, _SCORING[scoring],
                                 n_groups, topk_groups, group_top, 1 if renormalize else 0, weight_scale)
    return _launch(dev, stream, _route_experts, args, logits)


def _route_experts(s, args, logits):
    w = logits.new_empty((args.T, args.k))
    ids = logits.new_empty((args.T, args.k), dtype=_I32)
    args.topk_w, args.topk_i = w.data_ptr(), ids.data_ptr()
    _check(capi.load().gptoss_expert_choice(C.byref(args), s))
    return w, ids
