"""The serving operators on the GPU against plain statements in 64 bits (serving_reference.py, which derives the bounds)."""
import math
import random

import numpy as np
import pytest

import serving_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def serving():
    from gptoss_b200 import serving
    return serving


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def random_parents(n, rng, chain=False):
    return [i - 1 if chain or rng.random() < 0.1 else rng.randrange(-1, i) for i in range(n)]


def tree_case(serving, nodes, ctx, nq=8, nkv=2, hd=64, S=None, rows=None, seed=0, chain=False, sd=1.0, sinks=True, max_nodes=None):
    g, rng = gen(seed), random.Random(seed)
    B = len(nodes)
    S = S or max(c + n for c, n in zip(ctx, nodes)) + 3
    off, mask, depth = serving.tree_masks([random_parents(n, rng, chain) for n in nodes], max_nodes)
    n_rows = rows or B
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(q=(r(int(off[-1]), nq, hd) * sd).bfloat16(), k_cache=r(n_rows, nkv, S, hd).bfloat16(),
                v_cache=r(n_rows, nkv, S, hd).bfloat16(), offsets=ints(off.tolist()), ctx_len=ints(ctx),
                mask=torch.from_numpy(mask).cuda(), depth=torch.from_numpy(depth).cuda(), sinks=r(nq) if sinks else None)


def check_tree(serving, c, max_nodes, max_ctx, **kw):
    got = serving.tree_attention(**c, **kw, max_nodes=max_nodes, max_ctx=max_ctx)
    want, bound = ref.tree_attention(**c, **kw)
    n = int(c["offsets"][-1])
    assert torch.isfinite(got[:n].float()).all()
    over = (got[:n].double() - want[:n]).abs() - bound[:n]
    assert float(over.max()) <= 0, (float(over.max()), int(over.argmax()))
    return got


@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (8, 1), (6, 2), (4, 2), (20, 4), (7, 7)])
def test_tree_attention_head_layouts(serving, hd, nq, nkv):
    nodes, ctx = [5, 1, 33, 17], [200, 0, 31, 129]
    check_tree(serving, tree_case(serving, nodes, ctx, nq, nkv, hd, seed=nq * 100 + hd), 33, 200)


@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("nodes,ctx", [(1, 0), (1, 1), (1, 127), (1, 128), (2, 126), (2, 127), (15, 113), (16, 112), (17, 112),
                                       (63, 65), (64, 64), (65, 63), (128, 0), (129, 255), (255, 1), (256, 700)])
def test_tree_attention_lengths_around_tiles(serving, hd, nodes, ctx):
    n, c = [nodes, max(1, nodes - 1), nodes], [ctx, ctx + 1, max(0, ctx - 1)]
    check_tree(serving, tree_case(serving, n, c, 8, 1, hd, seed=nodes + ctx, chain=nodes % 2 == 0), max(n), max(c))


@pytest.mark.parametrize("window", [1, 2, 16, 127, 128, 129, 1000])
def test_tree_attention_window(serving, window):
    nodes, ctx = [40, 3, 64], [500, 7, 128]
    c = tree_case(serving, nodes, ctx, 16, 2, seed=window, chain=True)
    check_tree(serving, c, 64, 500, window=window)
    check_tree(serving, tree_case(serving, nodes, ctx, 16, 2, seed=window), 64, 500, window=window)


def test_tree_attention_long_contexts_and_cache_rows(serving):
    nodes, ctx = [13, 4, 64], [30011, 517, 9000]
    c = tree_case(serving, nodes, ctx, 16, 2, rows=5, seed=3)
    rows = ints([4, 0, 2])
    a = check_tree(serving, c, 64, 30011, cache_rows=rows)
    # the bound on the contexts sizes the launch only: one that is too small gives the same numbers within the bound
    check_tree(serving, c, 64, 10, cache_rows=rows)
    check_tree(serving, c, 64, 0, cache_rows=rows, window=1234)
    assert torch.equal(a, serving.tree_attention(**c, cache_rows=rows, max_nodes=64, max_ctx=30011))  # same bits again


def test_tree_attention_sharp_and_flat_scores(serving):
    for sd in (0.0, 30.0):
        check_tree(serving, tree_case(serving, [19, 64], [700, 33], sd=sd, seed=int(sd)), 64, 700)
    c = tree_case(serving, [9], [50], seed=1)
    c["sinks"] = torch.tensor([-math.inf, 60.0, -60.0, 0.0, 5.0, -5.0, 1.0, 2.0], device="cuda")
    check_tree(serving, c, 9, 50)


@pytest.mark.parametrize("sinks", [True, False])
def test_tree_attention_rows_that_see_nothing_are_zero(serving, sinks):
    c = tree_case(serving, [6, 3, 0, 4], [0, 40, 10, 0], sinks=sinks, seed=8)
    c["mask"][1] = 0       # sequence without cached tokens, nothing drafted in sight
    c["mask"][3] = 1 << 5  # sees one later token only
    c["mask"][9:] = 0
    got = check_tree(serving, c, 6, 40)
    assert (got[1] == 0).all() and (got[9:] == 0).all()


def test_tree_attention_any_mask(serving):
    c = tree_case(serving, [70, 256, 31], [5, 130, 0], seed=4, max_nodes=256)
    bits = torch.randint(-2 ** 31, 2 ** 31, c["mask"].shape, generator=gen(9), device="cuda", dtype=torch.int64)
    c["mask"] = bits.to(torch.int32)  # bits behind a tree's last token are set too: they mean nothing
    check_tree(serving, c, 256, 130)
    check_tree(serving, c, 256, 130, window=40)


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("hd", [32, 64])
def test_tree_attention_what_is_masked_may_hold_anything(serving, poison, hd):
    nodes, ctx = [40, 7, 150], [300, 120, 1]
    c = tree_case(serving, nodes, ctx, 8, 1, hd, S=520, rows=4, seed=5)
    want = serving.tree_attention(**c, max_nodes=150, max_ctx=300, window=100)
    full = serving.tree_attention(**c, max_nodes=150, max_ctx=300)
    for b, (n, x) in enumerate(zip(nodes, ctx)):
        for cache in (c["k_cache"], c["v_cache"]):
            cache[b, :, x + n:] = poison
    for cache in (c["k_cache"], c["v_cache"]):
        cache[3] = poison
    assert torch.equal(full, serving.tree_attention(**c, max_nodes=150, max_ctx=300))
    # cached tokens that left the window of every drafted token
    c["k_cache"][0, :, :200], c["v_cache"][0, :, :200] = poison, poison
    assert torch.equal(want, serving.tree_attention(**c, max_nodes=150, max_ctx=300, window=100))
    # a drafted token spoils itself and its descendants, nobody else
    for b, i in ((0, 11), (2, 3), (2, 140)):
        c["k_cache"][b, :, ctx[b] + i], c["v_cache"][b, :, ctx[b] + i] = poison, poison
    got = serving.tree_attention(**c, max_nodes=150, max_ctx=300, window=100)
    off = c["offsets"].tolist()
    clean = torch.ones(off[-1], dtype=torch.bool)
    for b, i in ((0, 11), (2, 3), (2, 140)):
        for t in range(off[b], off[b + 1]):
            if int(c["mask"][t, i >> 5]) >> (i & 31) & 1:
                clean[t] = False
    clean = clean.cuda()
    assert 0 < int((~clean).sum()) < len(clean)
    assert torch.equal(got[clean], want[clean])
    if math.isnan(poison):
        assert got[~clean].isnan().all()


def test_tree_attention_a_spoiled_value_keeps_to_its_dims(serving):
    c = tree_case(serving, [40], [100], 8, 1, seed=15)
    want, bound = ref.tree_attention(**c)
    c["v_cache"][0, 0, 103, 7] = math.inf   # drafted token 3, one element
    got = serving.tree_attention(**c, max_nodes=40, max_ctx=100)
    sees = (c["mask"][:, 0] >> 3) & 1 != 0
    assert (got[sees][:, :, 7] == math.inf).all()
    keep = torch.ones(64, dtype=torch.bool)
    keep[7] = False
    assert float(((got.double() - want).abs() - bound)[:, :, keep.cuda()].max()) <= 0
    assert float(((got.double() - want).abs() - bound)[~sees].max()) <= 0


def test_tree_attention_strides_and_rows_behind(serving):
    c = tree_case(serving, [9, 20], [77, 140], 8, 2, seed=6)
    n = 29
    qkv = torch.randn(n + 5, (8 + 4) * 64, generator=gen(1), device="cuda").bfloat16()
    out = torch.full((n + 5, 3, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")[:, 1]
    c["q"] = qkv[:, 64:9 * 64].unflatten(1, (8, 64))
    mask = torch.full((n + 5, 1), -1, dtype=torch.int32, device="cuda")
    mask[:n] = c["mask"]
    c["mask"] = mask
    c["depth"] = torch.cat([c["depth"], torch.zeros(5, dtype=torch.int32, device="cuda")])
    serving.tree_attention(**c, max_nodes=20, max_ctx=140, out=out)
    want, bound = ref.tree_attention(**c)
    assert float(((out[:n].double() - want[:n]).abs() - bound[:n]).max()) <= 0
    assert (out[n:] == 7.0).all()
    assert (out.as_strided((n + 5, 64 * 8), (3 * 8 * 64, 1), 0) == 7.0).all()  # what lies beside out in its buffer


def test_tree_attention_full_cache_and_offsets_beyond_32_bits(serving):
    S, nkv, rows = 65536, 8, 66  # 2.2e9 elements per cache
    k = torch.empty(rows, nkv, S, 64, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    c = tree_case(serving, [10], [300], 16, nkv, S=310, seed=2)
    k[65, :, :310], v[65, :, :310] = c["k_cache"][0], c["v_cache"][0]
    want, bound = ref.tree_attention(**c)
    c["k_cache"], c["v_cache"] = k, v
    got = serving.tree_attention(**c, max_nodes=10, max_ctx=300, cache_rows=ints([65]))
    assert float(((got.double() - want).abs() - bound).max()) <= 0
    # a context that ends with the cache
    k[65, :, S - 310:], v[65, :, S - 310:] = k[65, :, :310].clone(), v[65, :, :310].clone()
    c["ctx_len"] = ints([S - 10])
    k[65, :, :S - 310] = 0
    v[65, :, :S - 310] = 0
    got = serving.tree_attention(**c, max_nodes=10, max_ctx=S - 10, cache_rows=ints([65]))
    want, bound = ref.tree_attention(**c, cache_rows=ints([65]))
    assert float(((got.double() - want).abs() - bound).max()) <= 0


def test_tree_attention_indices_outside_the_cache_reach_no_memory(serving):
    c = tree_case(serving, [4, 4, 4], [20, 20, 20], seed=7)
    want = serving.tree_attention(**c, max_nodes=4, max_ctx=20)
    got = serving.tree_attention(**c, max_nodes=4, max_ctx=20, cache_rows=ints([-1, 1, 3]))
    assert torch.equal(got[4:8], want[4:8])
    assert (got[:4] == 0).all() and (got[8:] == 0).all()  # rows outside the cache: nothing to attend to
    c["ctx_len"] = ints([-5, 20, 10 ** 9])
    got = serving.tree_attention(**c, max_nodes=4, max_ctx=20)
    assert torch.equal(got[4:8], want[4:8])


def test_tree_attention_graph_replay_and_streams(serving):
    c = tree_case(serving, [20, 9], [400, 77], S=700, seed=11, max_nodes=64)
    out = torch.empty_like(c["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    serving.tree_attention(**c, max_nodes=64, max_ctx=600, out=out, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serving.tree_attention(**c, max_nodes=64, max_ctx=600, out=out)
    for ctx in ([400, 77], [0, 600], [513, 1]):
        c["ctx_len"].copy_(ints(ctx))
        out.zero_()
        graph.replay()
        want, bound = ref.tree_attention(**c)
        assert float(((out.double() - want).abs() - bound).max()) <= 0


# ---- the accepted path ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,nkv,layers", [(64, 8, 3), (32, 1, 1), (64, 1, 2)])
@pytest.mark.parametrize("paths", [[[0], [1], []], [[0, 1, 2], [3, 5, 6], [63]], [list(range(64)), list(range(1, 64)), [0, 2, 4, 6, 8, 10, 12, 14, 16, 18]],
                                   [list(range(0, 64, 2)), list(range(50, 64)), [5]]])
def test_cache_commit(serving, hd, nkv, layers, paths):
    g = gen(len(paths[0]) + hd)
    S, rows = 200, 5
    k = torch.randn(layers, rows, nkv, S, hd, generator=g, device="cuda").bfloat16()
    v = torch.randn(layers, rows, nkv, S, hd, generator=g, device="cuda").bfloat16()
    ctx, row = [0, 136, 70], [3, 0, 4]
    want_k, want_v = k.clone(), v.clone()
    for b, p in enumerate(paths):
        for w, x in ((want_k, k), (want_v, v)):
            w[:, row[b], :, ctx[b]:ctx[b] + len(p)] = x[:, row[b], :, [ctx[b] + i for i in p]]
    off = np.cumsum([0] + [len(p) for p in paths]).tolist()
    serving.cache_commit(k, v, ints(ctx), ints(off), ints(sum(paths, [])), cache_rows=ints(row), max_path=64)
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_cache_commit_one_layer_without_rows_and_bad_indices(serving):
    k = torch.arange(2 * 1 * 16, device="cuda").view(2, 1, 16, 1).expand(2, 1, 16, 32).bfloat16().contiguous()
    v = -k
    before = k.clone()
    serving.cache_commit(k, v, ints([4, 12]), ints([0, 2, 4]), ints([1, 3, 2, 9]), max_path=4)
    want = before.clone()
    want[0, 0, 4], want[0, 0, 5] = before[0, 0, 5], before[0, 0, 7]
    want[1, 0, 12] = before[1, 0, 14]  # slot 12 + 9 lies behind the cache: not moved
    assert torch.equal(k, want) and torch.equal(v, -want)
    serving.cache_commit(k, v, ints([4, 99]), ints([0, 0, 1]), ints([1]), max_path=4)
    serving.cache_commit(k, v, ints([4, 4]), ints([1, 1000, 70]), ints([0]), max_path=64)  # offsets behind the path's end
    serving.cache_commit(k, v, ints([4, 4]), ints([0, 1, 2]), ints([1, 1]), cache_rows=ints([-1, 2]), max_path=4)
    assert torch.equal(k, want) and torch.equal(v, -want)


# ---- adapters ---------------------------------------------------------------------------------------------------------
def lora_case(T, K, n_out, rank, n, seed=0, ids=None):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if ids is None:
        ids = torch.randint(-1, n, (T,), generator=g, device="cuda", dtype=torch.int64).int()
    return dict(x=r(T, K).bfloat16(), a=(r(n, rank, K) * K ** -0.5).bfloat16(), b=r(n, n_out, rank).bfloat16(), ids=ids,
                y=r(T, n_out), scale=r(n))


def check_lora(serving, c, **kw):
    want, bound = ref.lora(**c)
    y0 = c["y"].clone()
    got = serving.lora_apply(**c, out=torch.full_like(c["y"], math.nan), **kw)
    assert torch.equal(c["y"], y0)
    assert float(((got.double() - want).abs() - bound).max()) <= 0
    idle = (c["ids"] < 0) | (c["ids"] >= c["a"].shape[0])
    assert torch.equal(got[idle], y0[idle])
    return got


@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("nodes,ctx", [([5], [20011]), ([1], [700]), ([130], [9000]), ([3, 2], [15000, 40])])
def test_tree_attention_many_shares(serving, nodes, ctx, hd):
    """One kv head: the context is cut into up to as many shares as the GPU has room for."""
    check_tree(serving, tree_case(serving, nodes, ctx, 2, 1, hd, seed=hd + ctx[0]), max(nodes), max(ctx))


@pytest.mark.parametrize("nodes,ctx,nq,nkv,window", [([24] * 6, [900] * 6, 16, 2, 128), ([13, 7], [9000, 4000], 8, 1, 0), ([64] * 8, [500] * 8, 64, 8, 0)])
def test_tree_attention_gives_the_same_bits_every_time(serving, nodes, ctx, nq, nkv, window):
    c = tree_case(serving, nodes, ctx, nq, nkv, 64, seed=77)
    c["v_cache"][:, :, ctx[0] + 2, 5] = math.nan  # a masked row for most of the tokens
    call = lambda: serving.tree_attention(**c, window=window, max_nodes=max(nodes), max_ctx=max(ctx))  # noqa: E731
    want = call()
    side, load = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
    outs = []
    for _ in range(40):
        with torch.cuda.stream(side):
            load = torch.sin(load)
        outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o.view(torch.int16), want.view(torch.int16)) for o in outs)


@pytest.mark.parametrize("T,K,n_out,rank,n", [
    (1, 2880, 5120, 16, 3), (1, 8, 8, 8, 1), (2, 64, 96, 8, 1), (3, 2880, 2880, 24, 5), (16, 72, 40, 128, 2), (17, 520, 1000, 40, 3),
    (31, 4096, 2880, 64, 40), (64, 2880, 5120, 32, 7), (257, 4096, 2880, 32, 48), (1000, 136, 264, 16, 1), (1025, 200, 2312, 8, 300),
    (4099, 256, 512, 64, 6), (129, 64, 64, 128, 129), (2048, 72, 1000, 128, 3), (2100, 1032, 40, 24, 90), (3001, 8, 8, 8, 1),
    (2500, 200, 328, 16, 2000), (5000, 64, 2048, 16, 4500), (2051, 64, 8, 64, 40), (9001, 64, 72, 8, 3), (17000, 32, 40, 8, 4000), (1536, 2880, 264, 16, 5), (1600, 3080, 72, 40, 3), (2400, 2000, 136, 16, 7), (400, 64, 96, 16, 1500), (300, 64, 96, 16, 1023), (32, 264, 136, 48, 4), (33, 264, 136, 48, 4)])
def test_lora(serving, T, K, n_out, rank, n):
    check_lora(serving, lora_case(T, K, n_out, rank, n, seed=T + rank))


def test_lora_orders_ids_and_in_place(serving):
    T, n = 700, 9
    for ids in ([5] * T, [-1] * T, sorted(i % n for i in range(T)), [0] * 300 + [-1] * 17 + [8] * 383,
                [n + 3 if i % 3 else 2 for i in range(T)]):
        check_lora(serving, lora_case(T, 128, 256, 16, n, seed=1, ids=ints(ids)))
    c = lora_case(T, 128, 256, 16, n, seed=2)
    want = serving.lora_apply(**c, out=torch.empty_like(c["y"]))
    c["scale"] = None
    check_lora(serving, c)
    c = lora_case(T, 128, 256, 16, n, seed=2)
    assert serving.lora_apply(**c) is c["y"] and torch.equal(c["y"], want)


@pytest.mark.parametrize("T", [33, 64, 65, 255, 256, 257, 300, 511, 512, 513, 767, 768, 1279, 1535, 2047, 2111])
def test_lora_groups_of_every_size(serving, T):
    """Runs of one adapter, one adapter for all, none at all, an adapter each, 64 and 65 tokens each; in place and not."""
    n = 70
    for i, ids in enumerate(([7] * T, [-1] * T, [t % n for t in range(T)], [t // 64 % n for t in range(T)], [t // 65 % n for t in range(T)],
                             [-1] * (T - 1) + [3], [n + 5] * 40 + [t % 2 for t in range(T - 40)] if T > 40 else [n] * T)):
        c = lora_case(T, 72, 136, 16, n, seed=T + i, ids=ints(ids))
        got = check_lora(serving, c)
        y = c["y"].clone()
        assert torch.equal(serving.lora_apply(**{**c, "y": y}), got)


@pytest.mark.parametrize("T,rank,n", [(20, 16, 2), (300, 32, 3), (567, 64, 3), (767, 16, 11), (1200, 16, 5), (1279, 128, 2), (700, 16, 1100), (3000, 32, 7)])
def test_lora_gives_the_same_bits_every_time(serving, T, rank, n):
    """Also when other work runs beside it, which changes the order in which the tokens' threads come."""
    c = lora_case(T, 1736, 520, rank, n, seed=T)
    if n > 1000:
        c["ids"] = torch.where(torch.arange(T, device="cuda") % 3 == 0, c["ids"], c["ids"] % 2)
    want = serving.lora_apply(**c, out=torch.empty_like(c["y"]))
    side, load = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
    outs = []
    for i in range(60):
        with torch.cuda.stream(side):
            load = torch.sin(load)
        outs.append(serving.lora_apply(**c, out=torch.empty_like(c["y"])))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_lora_strides_zeros_and_what_is_not_served(serving):
    c = lora_case(50, 128, 64, 16, 4, seed=3)
    wide = torch.randn(50, 256, generator=gen(4), device="cuda").bfloat16()
    c["x"] = wide[:, 64:192]
    big = torch.randn(50, 200, generator=gen(5), device="cuda")
    c["y"] = big[:, 8:72]
    out = torch.full((50, 80), 3.0, device="cuda")
    want, bound = ref.lora(**c)
    serving.lora_apply(**c, out=out[:, 4:68])
    assert float(((out[:, 4:68].double() - want).abs() - bound).max()) <= 0
    assert (out[:, :4] == 3).all() and (out[:, 68:] == 3).all()
    # an adapter nobody uses and tokens without one may hold anything
    c = lora_case(50, 128, 64, 16, 4, seed=6)
    c["ids"][c["ids"] == 2] = -1
    want = serving.lora_apply(**c, out=torch.empty_like(c["y"]))
    c["a"][2], c["b"][2], c["scale"][2] = math.nan, math.nan, math.nan
    c["x"][c["ids"] < 0] = math.nan
    assert torch.equal(serving.lora_apply(**c, out=torch.empty_like(c["y"])), want)
    # neither may one adapter spoil another's tokens
    c["a"][1, 3, 5], c["b"][1, 7, 2] = math.inf, math.nan
    got = serving.lora_apply(**c, out=torch.empty_like(c["y"]))
    assert torch.equal(got[c["ids"] != 1], want[c["ids"] != 1])


def test_lora_a_token_does_not_depend_on_its_neighbours_values(serving):
    c = lora_case(96, 512, 320, 16, 2, seed=12, ids=ints([0] * 50 + [1] * 46))
    want = serving.lora_apply(**c, out=torch.empty_like(c["y"]))
    c["x"][3], c["y"][60] = math.nan, math.inf
    got = serving.lora_apply(**c, out=torch.empty_like(c["y"]))
    keep = torch.ones(96, dtype=torch.bool)
    keep[3] = keep[60] = False
    assert torch.equal(got[keep.cuda()], want[keep.cuda()])
    assert got[3].isnan().all()


def test_lora_graph_replay_and_streams(serving):
    c = lora_case(200, 256, 512, 32, 5, seed=7)
    out = torch.empty_like(c["y"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    serving.lora_apply(**c, out=out, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serving.lora_apply(**c, out=out)
    for seed in range(3):
        c["ids"].copy_(torch.randint(-1, 5, (200,), generator=gen(seed), device="cuda").int())
        out.zero_()
        graph.replay()
        want, bound = ref.lora(**c)
        assert float(((out.double() - want).abs() - bound).max()) <= 0


# ---- choice of experts ------------------------------------------------------------------------------------------------
# weights: the argument of the exponential is off by 2^-24 of up to 16, the sums add as much again
W_TOL = 2.0 ** -19


def check_route(serving, logits, k, **kw):
    w, i = serving.route_experts(logits, k, **kw)
    want_w, want_i = ref.route(logits, k, **kw)
    assert torch.equal(i.cpu(), want_i)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=W_TOL, atol=1e-30)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,groups,kept,top", [
    (1, 1, 1, 1, 1, 1), (1, 128, 4, 1, 1, 1), (3, 32, 4, 1, 1, 1), (5, 40, 8, 1, 1, 1), (257, 256, 8, 8, 4, 2), (100, 160, 6, 8, 3, 1),
    (33, 96, 8, 32, 8, 2), (64, 8, 8, 8, 8, 1), (7, 64, 1, 2, 1, 2), (1000, 72, 5, 4, 2, 2), (9, 255, 8, 1, 1, 1), (2, 33, 3, 11, 2, 2)])
def test_route_experts(serving, scoring, T, E, k, groups, kept, top):
    g = gen(T * E)
    logits = torch.randn(T, E, generator=g, device="cuda") * 2
    bias = torch.randn(E, generator=g, device="cuda") * 0.1
    for b in (None, bias):
        for renorm in (True, False):
            check_route(serving, logits, k, scoring=scoring, bias=b, n_groups=groups, topk_groups=kept, group_top=top,
                        renormalize=renorm, weight_scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_experts_ties_take_the_lowest_index(serving, scoring):
    g = gen(3)
    logits = torch.randint(0, 3, (300, 64), generator=g, device="cuda").float()
    logits[0] = 1.0
    bias = torch.randint(0, 2, (64,), generator=g, device="cuda").float() * 0.5
    for b in (None, bias):
        check_route(serving, logits, 6, scoring=scoring, bias=b)
        check_route(serving, logits, 6, scoring=scoring, bias=b, n_groups=8, topk_groups=3, group_top=2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_experts_near_ties(serving, scoring):
    """Logits that differ in the last bits of fp32, and large ones."""
    g = gen(5)
    base = torch.randn(400, 1, generator=g, device="cuda")
    logits = base + torch.randint(0, 9, (400, 48), generator=g, device="cuda") * 1e-7
    check_route(serving, logits, 8, scoring=scoring)
    check_route(serving, logits, 8, scoring=scoring, bias=torch.linspace(0, 1e-6, 48, device="cuda"), n_groups=4, topk_groups=2, group_top=2)
    check_route(serving, logits * 12, 8, scoring=scoring)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_experts_infinities_and_nan(serving, scoring):
    logits = torch.randn(6, 32, generator=gen(6), device="cuda")
    logits[0, 3:] = -math.inf
    logits[1, 5] = math.inf
    logits[2, ::2] = math.nan
    logits[3] = -math.inf
    logits[4] = math.nan
    logits[5, 9] = -3e38
    check_route(serving, logits, 5, scoring=scoring)
    bias = torch.zeros(32, device="cuda")
    bias[4], bias[7], bias[8] = -math.inf, math.nan, 1e30
    check_route(serving, logits, 5, scoring=scoring, bias=bias)
    check_route(serving, logits, 5, scoring=scoring, n_groups=4, topk_groups=2, group_top=1)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_experts_scores_that_all_but_vanish(serving, scoring):
    logits = torch.randn(20, 64, generator=gen(12), device="cuda") - (150 if scoring == "sigmoid" else 0)
    logits[:, 40:] -= 150
    bias = torch.zeros(64, device="cuda")
    bias[40:] = torch.linspace(3, 2, 24, device="cuda")
    for renorm in (True, False):
        check_route(serving, logits, 6, scoring=scoring, bias=bias, renormalize=renorm)
        check_route(serving, logits, 3, scoring=scoring, bias=bias, renormalize=renorm, n_groups=8, topk_groups=2, group_top=2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_experts_scores_below_the_range_of_fp64_tie(serving, scoring, renorm):
    logits = torch.full((3, 40), -2000.0, device="cuda")
    logits[0, 1], logits[0, 7], logits[0, 9] = 0.0, -900.0, -800.0   # all but the first score 0 in fp64
    logits[1, 3], logits[1, 5], logits[1, 6] = 0.0, -690.0, -600.0   # these do not
    logits[2] -= torch.arange(40, device="cuda").flip(0)
    check_route(serving, logits, 4, scoring=scoring, renormalize=renorm)
    check_route(serving, logits[:, :2], 1, scoring=scoring, renormalize=renorm)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_experts_many_random_rows(serving, scoring):
    """Against the plain operator in 64 bits on the GPU: 20000 rows, so that near ties of every kind occur."""
    logits = torch.randn(20000, 256, generator=gen(13), device="cuda") * 1.5
    bias = torch.randn(256, generator=gen(14), device="cuda") * 0.1
    x = logits.double()
    score = torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)
    for b in (None, bias):
        choice = score if b is None else score + b.double()
        want = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :8]
        w, i = serving.route_experts(logits, 8, scoring=scoring, bias=b)
        assert torch.equal(i.long(), want)
        ww = torch.gather(score, 1, want)
        torch.testing.assert_close(w.double(), ww / ww.sum(1, keepdim=True), rtol=W_TOL, atol=0)


def test_route_experts_strided_rows_stream_and_graph(serving):
    wide = torch.randn(70, 100, generator=gen(8), device="cuda")
    check_route(serving, wide[:, 3:67], 4, scoring="sigmoid")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    w, i = serving.route_experts(wide[:, 3:67], 4, stream=side)
    side.synchronize()
    assert torch.equal(i, serving.route_experts(wide[:, 3:67], 4)[1])
    logits = wide[:, :64].contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, i = serving.route_experts(logits, 4)
    logits.copy_(torch.randn(70, 64, generator=gen(9), device="cuda"))
    graph.replay()
    assert torch.equal(i.cpu(), ref.route(logits, 4)[1])


def test_routed_block_matches_the_block_on_its_own_routing_and_the_oracle(serving, oracle):
    import oracle_lib
    from gptoss_b200 import moe, synth
    H, I, E, k, T = 256, 192, 16, 4, 200
    w = synth.MoELayerWeights(H, I, E, seed=7, sigma=0.05)
    t = synth.activations(7, T, H)
    blk = moe.MoEBlock(hidden=H, intermediate=I, n_experts=E, top_k=k, max_tokens=T)
    blk.upload_layer(0, w)
    t_dev = torch.from_numpy(synth.f32_to_bf16_bits(t).view(np.int16).reshape(T, H)).cuda().view(torch.bfloat16)
    x0 = torch.randn(T, H, generator=gen(1), device="cuda")
    a, b = x0.clone(), x0.clone()
    blk.forward(0, t_dev, a)
    blk.status()
    tw, ti = torch.from_numpy(blk.tap("topk_w", T)).cuda(), torch.from_numpy(blk.tap("topk_i", T)).cuda()
    blk.forward_routed(0, t_dev, tw, ti, b)
    blk.status()
    assert torch.equal(a, b)
    # another rule: grouped sigmoid scores with a bias; then some slots without an expert, and repeated experts
    scores = torch.from_numpy(blk.tap("scores", T)).cuda()
    rw, ri = serving.route_experts(scores, k, scoring="sigmoid", bias=torch.linspace(-0.1, 0.1, E, device="cuda"), n_groups=4,
                                   topk_groups=2, group_top=2, weight_scale=2.0)
    for ids in (ri, torch.where(torch.rand(ri.shape, generator=gen(2), device="cuda") < 0.3, -1, ri).int(),
                torch.full_like(ri, 5), torch.where(ri == 3, E + 4, ri).int()):
        x = torch.zeros(T, H, device="cuda")
        blk.forward_routed(0, t_dev, rw, ids.contiguous(), x)
        blk.status()
        inside = ((ids >= 0) & (ids < E)).cpu().numpy()
        want = np.zeros((T, H))
        for j in range(k):  # slot by slot: the oracle takes a full set of experts per token
            one_i = np.where(inside[:, j], ids[:, j].cpu().numpy(), 0).astype(np.int32)[:, None]
            one_w = np.where(inside[:, j], rw[:, j].cpu().numpy(), 0).astype(np.float32)[:, None]
            want += oracle.moe_block(t, one_w, one_i, w, mode=oracle_lib.MODE_GPU_BF16)
        got = x.cpu().numpy()
        assert np.linalg.norm(got - want) <= 1e-4 * np.linalg.norm(want)
    with pytest.raises(moe.GptossError):
        blk.forward_routed(1, t_dev, rw, ri, x)  # no such layer
    blk.close()


def test_arguments_that_the_python_layer_refuses(serving):
    """Types, shapes, layouts and devices, one at a time; nothing is launched."""
    from gptoss_b200 import capi, moe

    def refused(call, good, changes):
        call(**good)
        for name, value in changes:
            with pytest.raises(moe.GptossError) as e:
                call(**{**good, name: value})
            assert e.value.code == capi.ERR_BAD_ARG, name

    c = tree_case(serving, [3, 4], [5, 6], seed=1)
    good = {**c, "cache_rows": ints([0, 1]), "max_nodes": 4, "max_ctx": 6, "window": 3}
    refused(serving.tree_attention, good, [
        ("q", c["q"].float()), ("q", c["q"][0]), ("q", c["q"].cpu()), ("q", c["q"].transpose(0, 1)), ("q", None), ("k_cache", c["k_cache"].half()),
        ("v_cache", c["v_cache"][:, :1]), ("v_cache", c["v_cache"].transpose(1, 2)), ("offsets", c["offsets"].long()), ("offsets", c["offsets"][:2]),
        ("ctx_len", c["ctx_len"].cpu()), ("mask", c["mask"][:3]), ("mask", c["mask"].float()), ("depth", c["depth"][:2]), ("depth", None),
        ("depth", c["depth"].long()), ("sinks", c["sinks"][:3]), ("sinks", c["sinks"].bfloat16()), ("cache_rows", ints([0])), ("max_nodes", 300),
        ("max_nodes", 40), ("out", torch.empty(7, 8, 64, device="cuda")), ("out", torch.empty(6, 8, 64, device="cuda").bfloat16()), ("window", -1),
        ("scale", 0.0), ("scale", math.nan)])
    k = torch.zeros(2, 3, 2, 16, 32, dtype=torch.bfloat16, device="cuda")
    good = dict(k_cache=k, v_cache=k.clone(), ctx_len=ints([1, 2]), offsets=ints([0, 1, 2]), path=ints([0, 1]), max_path=2, cache_rows=ints([0, 2]))
    refused(serving.cache_commit, good, [
        ("k_cache", k.float()), ("k_cache", k[0, 0]), ("v_cache", k[:1]), ("v_cache", k.transpose(1, 2)), ("ctx_len", ints([1, 2]).long()),
        ("offsets", ints([0, 1])), ("path", ints([0, 1]).cpu()), ("cache_rows", ints([0])), ("max_path", -1), ("path", None)])
    c = lora_case(5, 64, 32, 8, 2)
    refused(serving.lora_apply, c, [
        ("x", c["x"].float()), ("x", c["x"][:, :60]), ("x", c["x"][:4]), ("a", c["a"][:1]), ("a", c["a"].transpose(1, 2)), ("b", c["b"][:, :, :4]),
        ("ids", c["ids"].long()), ("ids", c["ids"][:3]), ("y", c["y"].bfloat16()), ("y", c["y"][:, :24]), ("y", c["y"].t()), ("y", c["y"].cpu()),
        ("scale", c["scale"][:1]), ("scale", c["scale"].double()), ("out", c["y"][:4]), ("ids", None)])
    good = dict(logits=torch.zeros(3, 16, device="cuda"), top_k=2, bias=torch.zeros(16, device="cuda"))
    refused(serving.route_experts, good, [
        ("logits", good["logits"].half()), ("logits", good["logits"].t()), ("logits", good["logits"].cpu()), ("bias", good["bias"][:8]),
        ("bias", good["bias"].double()), ("top_k", 0), ("top_k", 9), ("scoring", "relu"), ("n_groups", 3), ("topk_groups", 2), ("group_top", 3)])


def test_python_layer_refuses_numbers(serving):
    """Numbers of the wrong kind or beyond 32 bits."""
    from gptoss_b200 import moe
    c = tree_case(serving, [3, 4], [5, 6], seed=2)
    for bad in (1 << 31, -(1 << 31), 1 << 40):
        with pytest.raises(moe.GptossError):
            serving.tree_attention(**c, max_nodes=bad, max_ctx=6)
    with pytest.raises(OverflowError):
        serving.tree_attention(**c, max_nodes=4, max_ctx=1 << 70)
    for name, value in (("max_nodes", 4.5), ("max_nodes", None), ("max_ctx", "6"), ("scale", "1")):
        with pytest.raises(TypeError):
            serving.tree_attention(**{**c, "max_nodes": 4, "max_ctx": 6, name: value})
    logits = torch.zeros(2, 8, device="cuda")
    with pytest.raises(moe.GptossError):
        serving.route_experts(logits, 2, scoring="relu")
    with pytest.raises(TypeError):
        serving.route_experts(logits, 2, weight_scale=None)
    got = serving.tree_attention(**c, max_nodes=np.int64(4), max_ctx=np.int32(6), scale=np.float32(0.125))
    assert torch.equal(got, serving.tree_attention(**c, max_nodes=4, max_ctx=6))


def test_what_a_call_returns(serving):
    """The given output itself, y in place, and on a side stream the same results."""
    c = tree_case(serving, [3, 4], [5, 6], seed=3)
    out = torch.empty_like(c["q"])
    assert serving.tree_attention(**c, max_nodes=4, max_ctx=6, out=out) is out
    lo = lora_case(40, 64, 32, 8, 2)
    want = serving.lora_apply(**{**lo, "out": torch.empty_like(lo["y"])})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = lo["y"].clone()
    side.wait_stream(torch.cuda.current_stream())
    assert serving.lora_apply(**{**lo, "y": y}, stream=side) is y
    side.synchronize()
    assert torch.equal(y, want)
