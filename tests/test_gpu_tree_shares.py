"""Contexts that are cut into shares: every slot is counted once, in every share (tree_shares.py)."""
import pytest

import tree_shares as sh

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("steps", [False, True])
@pytest.mark.parametrize("slots,hd", [(700, 32), (5000, 64), (30011, 64)])
def test_a_lost_or_doubled_slot_would_show(slots, hd, steps):
    """The mistakes are planted in the expectation: single slots around the ends of tiles, and whole tiles."""
    seen, level = torch.ones(1, slots, dtype=torch.bool), sh.levels(slots, steps)
    places = [range(t - 1, t + 1) for t in range(64, slots, 1216)] + [range(t, min(t + 64, slots)) for t in range(0, slots, 4096)]
    for block in sh.blocks(slots, hd):
        v = sh.values(slots, hd, 0, block)
        want = sh.expected(seen, level, 0.0, v)
        for place in places:
            if place[0] < block[0] or place[-1] >= block[1]:
                continue
            for times in (0.0, 2.0):
                for part in (place, place[:1]):
                    count = torch.ones(slots, dtype=torch.float64)
                    count[list(part)] = times
                    wrong = sh.expected(seen, level, 0.0, v, count)
                    # the output as a kernel rounds it
                    assert sh.differs(wrong.bfloat16().double(), want).any(), (block, part, times)


def run(nodes, ctx, nq, nkv, hd, window=0, max_ctx=None, sinks=True, steps=False, chain=True):
    import random
    from gptoss_b200 import serving
    rng = random.Random(len(ctx) * 1000 + ctx[0])
    parents = [[i - 1 if chain else rng.randrange(-1, i) for i in range(n)] for n in nodes]
    offsets, mask, depth = (torch.from_numpy(x) for x in serving.tree_masks(parents))
    ctx_len = torch.tensor(ctx, dtype=torch.int32)
    slots = max(c + n for c, n in zip(ctx, nodes))
    level, B = sh.levels(slots, steps), len(ctx)
    seen = sh.seen_by(offsets, ctx_len, mask, depth, window, slots).cuda()
    q = torch.zeros(int(offsets[-1]), nq, hd, dtype=torch.bfloat16, device="cuda")
    q[:, :, 3] = 1.0
    k = torch.full((B, nkv, slots + 5, hd), float("nan"), dtype=torch.bfloat16, device="cuda")
    for b, (c, n) in enumerate(zip(ctx, nodes)):  # behind a sequence's last slot anything may stand
        k[b, :, :c + n] = torch.randint(-3, 4, (nkv, c + n, hd), device="cuda").bfloat16()
        k[b, :, :c + n, 3] = level[:c + n].cuda().bfloat16()
    sink = torch.full((nq,), 4 * sh.LN2, device="cuda") if sinks else None
    size = torch.tensor([2.0 ** (b % 5) for b in range(B)], device="cuda")  # which sequence's cache row was read
    of = torch.repeat_interleave(torch.arange(B), (offsets[1:] - offsets[:-1]).long()).cuda()
    for block in sh.blocks(slots, hd):
        v = torch.zeros_like(k)
        v[:, :, slots:] = float("nan")
        for h in range(nkv):
            v[:, h, :slots] = (sh.values(slots, hd, h, block).cuda()[None] * size[:, None, None]).bfloat16()
        got = serving.tree_attention(q, k, v, offsets.cuda(), ctx_len.cuda(), mask.cuda(), depth.cuda(), max_nodes=max(nodes),
                                     max_ctx=max(ctx) if max_ctx is None else max_ctx, sinks=sink, window=window, scale=sh.LN2)
        for h in range(nkv):
            want = sh.expected(seen, level.cuda(), 4.0 if sinks else None, sh.values(slots, hd, h, block)) * size[of].double()[:, None]
            wrong = sh.differs(got[:, h * nq // nkv:(h + 1) * nq // nkv].double(), want[:, None])
            assert not wrong.any(), (block, h, wrong.nonzero()[:5].tolist())


gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("steps", [False, True])
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("B", [200, 148, 98, 74, 59, 49, 42, 37])  # 1 to 8 shares: as many as find room on 148 SMs, two on each
def test_shares_that_join_in_a_cluster(B, hd, steps):
    run([1 + b % 3 for b in range(B)], [2000 - 7 * (b % 150) for b in range(B)], 2, 1, hd, steps=steps)


@gpu
@pytest.mark.parametrize("steps", [False, True])
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("nodes,ctx,nq,nkv", [([13, 5, 2], [30011, 20999, 64], 2, 1), ([1], [9000], 1, 1), ([40, 7], [8000, 8191], 8, 1),
                                              ([3] * 2, [12345, 700], 16, 4), ([256], [6001], 8, 1)])
def test_shares_that_join_through_memory(nodes, ctx, nq, nkv, hd, steps):
    run(nodes, ctx, nq, nkv, hd, steps=steps)


@gpu
@pytest.mark.parametrize("max_ctx", [0, 1, 500, 4095, 20000, 1 << 30])
@pytest.mark.parametrize("nodes", [[3, 2, 1, 9], [40, 33, 64, 17]])
def test_any_bound_on_the_contexts(nodes, max_ctx):
    """A bound that is too small leaves the rest of a context to its last share, one that is too large leaves shares empty."""
    run(nodes, [6000, 4096, 1, 777], 8, 1, 64, max_ctx=max_ctx, steps=True)


@gpu
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("window", [1, 63, 64, 65, 1000, 3000])
def test_windows(window, sinks):
    """Tiles begin where the first token's window does, and every token has an edge of its own."""
    run([30, 4, 100], [5000, 2999, 200], 8, 2, 64, window=window, sinks=sinks, steps=True)
    run([30, 4, 100], [5000, 2999, 200], 4, 2, 32, window=window, sinks=sinks, steps=True, chain=False)


@gpu
@pytest.mark.parametrize("nodes", [[16] * 40, [64] * 10, [17] * 20])
def test_one_and_two_query_tiles(nodes):
    """8 query heads to a kv head: 16 tokens fill a query tile."""
    run(nodes, [1500 + 31 * b for b in range(len(nodes))], 16, 2, 64, steps=True, chain=False)
