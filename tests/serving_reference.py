"""Plain statements of the serving operators in 64 bits (torch, any device), and the error bounds of their kernels."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # rounding to nearest, relative


def tree_attention(q, k_cache, v_cache, offsets, ctx_len, mask, depth, sinks=None, cache_rows=None, window=0, scale=None):
    """(out, bound): out fp64 [n_tokens, nq, hd]; bound: how far a kernel may be off, element by element.

    Scores in fp32 from bf16 inputs: every product is exact, hd additions and the scaling are off by at most
    e = (hd + 4) 2^-24 scale sum|q||k| each.  The exponential turns that into a relative error 2e (its argument's, plus as
    much again for the maximum and the reduction of the argument) + 2^-18 (the function itself).  A weight rounded to bf16:
    2^-8; the same in the denominator.  The result is rounded to bf16 once more: 2^-8."""
    nq, hd = q.shape[1:]
    group = nq // k_cache.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    off, ctx = offsets.tolist(), ctx_len.tolist()
    rows = list(range(len(ctx))) if cache_rows is None else cache_rows.tolist()
    for b, c in enumerate(ctx):
        a, n = off[b], off[b + 1] - off[b]
        if n == 0:
            continue
        j = torch.arange(n, device=q.device)
        seen = torch.ones(n, c + n, dtype=torch.bool, device=q.device)
        seen[:, c:] = (mask[a:a + n].long()[:, j >> 5] >> (j & 31)[None]) & 1 != 0
        if window:
            d = depth[a:a + n].long()
            place = torch.cat([torch.arange(c, device=q.device), c + d])
            seen &= place[None] > (c + d)[:, None] - window
        k = k_cache[rows[b], :, :c + n].double().repeat_interleave(group, 0)
        v = v_cache[rows[b], :, :c + n].double().repeat_interleave(group, 0)
        used = seen.any(0)
        k[:, ~used], v[:, ~used] = 0, 0
        x = q[a:a + n].double().transpose(0, 1)
        s = x @ k.transpose(1, 2) * scale
        e = ((hd + 4) * 2.0 ** -24 * scale) * (x.abs() @ k.abs().transpose(1, 2)).masked_fill(~seen, 0).amax(2, keepdim=True)
        s = s.masked_fill(~seen, -math.inf)
        sink = torch.full((nq, n, 1), -math.inf, dtype=torch.float64, device=q.device)
        if sinks is not None:
            sink = sinks.double().view(nq, 1, 1).expand(nq, n, 1)
        top = torch.maximum(s.amax(2, keepdim=True), sink)
        top = top.masked_fill(top == -math.inf, 0)
        p = torch.exp(s - top)
        total = p.sum(2, keepdim=True) + torch.exp(sink - top)
        p = p / total.masked_fill(total == 0, 1)
        out[a:a + n] = (p @ v).transpose(0, 1)
        spread = (p @ v.abs()).transpose(0, 1)
        # one weight after another: an element that a masked value would spoil keeps what its own weights give
        bound[a:a + n] = HALF[torch.bfloat16] * out[a:a + n].abs() + (4 * e + 2.0 ** -17 + 2 * HALF[torch.bfloat16]).transpose(0, 1) * spread
    return out, bound


def lora(x, a, b, ids, y, scale=None):
    """(out, bound): out fp64; fp32 sums of exact products are off by at most (terms) 2^-23 of the sum of magnitudes
    (an accumulator that truncates: one step of the largest partial sum each), the final additions by 2^-23."""
    out = y.double().clone()
    bound = torch.zeros_like(out)
    K, rank = x.shape[1], a.shape[1]
    for i in range(a.shape[0]):
        who = (ids == i).nonzero()[:, 0]
        if not len(who):
            continue
        s = 1.0 if scale is None else float(scale[i])
        xa, aa, ba = x[who].double(), a[i].double(), b[i].double()
        u = xa @ aa.t()
        off_u = (K + 8) * 2.0 ** -23 * (xa.abs() @ aa.abs().t())
        out[who] += s * (u @ ba.t())
        bound[who] = abs(s) * ((off_u + (rank + 8) * 2.0 ** -23 * u.abs()) @ ba.abs().t())
    return out, bound + 2.0 ** -23 * (out.abs() + y.double().abs())


def route(logits, k, scoring="softmax", bias=None, n_groups=1, topk_groups=1, group_top=1, renormalize=True, weight_scale=1.0):
    """(weights fp64, ids): token by token, expert by expert."""
    T, E = logits.shape
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    if scoring == "softmax":
        top = x.amax(1, keepdim=True)  # of infinite logits only those equal to the largest count; a row of -inf scores 0
        score = torch.where(top.isinf(), (x == math.inf).double(), torch.exp(x - top.masked_fill(top.isinf(), 0)))
        total = score.sum(1, keepdim=True)
        score = score / total.masked_fill(total == 0, 1)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score + (0 if bias is None else bias.double().cpu())
    choice = torch.where(torch.isnan(choice), torch.full_like(choice, -math.inf), choice)
    size = E // n_groups
    ids, weights = torch.zeros(T, k, dtype=torch.int32), torch.zeros(T, k, dtype=torch.float64)
    for t in range(T):
        c = choice[t].tolist()
        worth = [sum(sorted(c[g * size:(g + 1) * size], reverse=True)[:group_top]) for g in range(n_groups)]
        kept = set(sorted(range(n_groups), key=lambda g: (-worth[g], g))[:topk_groups])
        best = sorted((e for e in range(E) if e // size in kept), key=lambda e: (-c[e], e))[:k]
        w = score[t, best]
        if renormalize:
            w = w / w.sum() if float(w.sum()) > 0 else w * 0
        ids[t], weights[t] = torch.tensor(best, dtype=torch.int32), w * weight_scale
    return weights, ids
