"""Inputs of the tree attention on which every slot of the cache shows in the result, and what the result has to be.

Over a long context the bound of serving_reference.tree_attention is wider than what a lost tile of slots changes.  Here weights are
powers of two (queries and keys with one element, small whole numbers; scale ln 2), and V is 1 in one dimension of each slot of a
block and 0 elsewhere: an output element is the sum of the weights of 16 neighbouring slots over the sum of all.  A slot that is
lost or counted twice moves it by at least 1/64 (the others of the 16 weigh at most 4 times as much), four times TOLERANCE: the rounding
of the output to bf16, 2^-8, and room for what 20 ln 2 in fp32 and the exponential are off by, 2^-16.  The weights themselves are
exact in bf16."""
import math

import torch

LN2 = math.log(2.0)
TOLERANCE = 2.0 ** -8 + 2.0 ** -16


def levels(slots, steps):
    """log2 of the weights.  steps: 0 to 2 among neighbours, 6 more or less from one third of the context to the next,
    so that the shares' largest scores differ; else 0 for all."""
    s = torch.arange(slots)
    return (s % 3 + 6 * ((s * 3) // slots % 2)).double() if steps else torch.zeros(slots, dtype=torch.float64)


def seen_by(offsets, ctx, mask, depth, window, slots):
    """bool [tokens, slots]: which slots each drafted token attends to."""
    out = torch.zeros(int(offsets[-1]), slots, dtype=torch.bool)
    for b, c in enumerate(ctx.tolist()):
        a, n = int(offsets[b]), int(offsets[b + 1] - offsets[b])
        j = torch.arange(n)
        row = torch.ones(n, c + n, dtype=torch.bool)
        row[:, c:] = (mask[a:a + n].long()[:, j >> 5] >> (j & 31)[None]) & 1 != 0
        if window:
            place = torch.cat([torch.arange(c), c + depth[a:a + n].long()])
            row &= place[None] > (c + depth[a:a + n].long())[:, None] - window
        out[a:a + n, :c + n] = row
    return out


def blocks(slots, hd):
    return [(a, min(a + 16 * hd, slots)) for a in range(0, slots, 16 * hd)]


def values(slots, hd, head, block):
    """V of one kv head: [slots, hd]."""
    v = torch.zeros(slots, hd)
    s = torch.arange(*block)
    v[s, ((s - block[0]) // 16 + 7 * head) % hd] = 1.0
    return v


def expected(seen, level, sink_log2, v, count=None):
    """[tokens, hd] in 64 bits.  count: how often each slot is counted (1), for mistakes that are planted."""
    w = seen.double() * (2.0 ** level)[None].to(seen.device)
    if count is not None:
        w = w * count[None]
    total = w.sum(1, keepdim=True) + (0.0 if sink_log2 is None else 2.0 ** sink_log2)
    return (w @ v.double().to(w.device)) / total.masked_fill(total == 0, 1)


def differs(got, want):
    return (got - want).abs() > TOLERANCE * want.abs()
