"""Cases of the serving operators (``gptoss_b200.serving``) in their plain form and as the framework's kernels.

    tree    attention of the drafted tokens of many sequences (a token tree per sequence) over the KV cache
    commit  the accepted path of each tree moved into place in the KV cache of every layer
    lora    low-rank adapters of many requests at once, added to the output of a shared projection
    route   experts chosen from softmax or sigmoid scores, with a balancing bias, groups and renormalised weights

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call, ``run`` is one call.  With
``own`` false, ``run`` computes the operator with elementary torch operations in 32 bits (64 where a comparison decides
an integer); with ``own`` true it calls the framework.
"""
import math
import random

import torch

own = False


# ---- cases ----------------------------------------------------------------------------------------------------------
def _tree(name, batch, nodes, ctx, shape="tree", q_heads=64, kv_heads=8, head_dim=64, window=0, sinks=True):
    return {"name": name, "op": "tree", "batch": batch, "nodes": nodes, "ctx": ctx, "shape": shape, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "window": window, "sinks": sinks}


def _commit(name, layers, batch, kv_heads, head_dim, slots, nodes, accepted):
    return {"name": name, "op": "commit", "layers": layers, "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim,
            "slots": slots, "nodes": nodes, "accepted": accepted}


def _lora(name, tokens, k, n_out, rank, adapters, order="mixed", without=0.1):
    return {"name": name, "op": "lora", "tokens": tokens, "k": k, "n_out": n_out, "rank": rank, "adapters": adapters,
            "order": order, "without": without}


def _route(name, tokens, experts, top_k, scoring, bias=False, groups=1, topk_groups=1, group_top=1, renormalize=True):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "scoring": scoring,
            "bias": bias, "groups": groups, "topk_groups": topk_groups, "group_top": group_top, "renormalize": renormalize}


def listed():
    return [
        # one user, a short chain from an n-gram drafter: latency of the verification step's attention
        _tree("tree_b1_chain4", 1, 4, 333, shape="chain"),
        # a batch in the middle of its answers, a windowed layer (window of the 20b and 120b configurations)
        _tree("tree_b16_n24_window", 16, 24, 1800, window=128),
        # few sequences over a long document: the context has to be split over the GPU
        _tree("tree_b3_n13_long", 3, 13, 30011),
        # a full serving batch with wide trees: the most arithmetic
        _tree("tree_b64_n64", 64, 64, 4096),
        # the small configuration's attention geometry (head_dim 32, 2 query heads on 1 kv head), no sinks
        _tree("tree_hd32_b9_n17", 9, 17, 501, q_heads=2, kv_heads=1, head_dim=32, sinks=False),
        # one user's accepted tokens, every layer of the 20b configuration
        _commit("commit_b1", 24, 1, 8, 64, 640, 16, 3),
        # a serving batch
        _commit("commit_b64", 24, 64, 8, 64, 384, 64, 6),
        # one decoded token with one adapter on the QKV projection of the 20b configuration
        _lora("lora_t1_r16", 1, 2880, 5120, 16, 4, without=0.0),
        # a decode step of many requests on the attention output projection, an adapter each, some without one
        _lora("lora_t257_r32", 257, 4096, 2880, 32, 48),
        # prompts of a few tenants in one batch, on the QKV projection
        _lora("lora_t8192_r64", 8192, 2880, 5120, 64, 6, order="runs"),
        # one decoded token through a softmax router of the 120b configuration's width
        _route("route_t1_e128", 1, 128, 4, "softmax"),
        # a prompt batch through a grouped sigmoid router with a balancing bias
        _route("route_t8192_e256", 8192, 256, 8, "sigmoid", bias=True, groups=8, topk_groups=4, group_top=2),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "commit", "lora", "lora", "route"])
    most = [work(c) for c in listed() if c["op"] == op]
    while True:
        case = _drawn(op, rng)
        if all(work(case)[x] <= max(w[x] for w in most) for x in ("bytes", "flops")):
            return case


def _drawn(op, rng):
    if op == "tree":
        head_dim = rng.choice([64, 64, 64, 32])
        kv_heads = rng.choice([1, 2, 4, 8])
        q_heads = kv_heads * rng.choice([1, 2, 4, 8, 8])
        nodes = _log_int(rng, 1, 256)
        batch = _log_int(rng, 1, 64)
        room = max(1, min(64 * 64 * 4096 // (batch * nodes), 64 * 4096 // batch, 60000))
        ctx = _log_int(rng, 1, room)
        return {"op": "tree", "batch": batch, "nodes": nodes, "ctx": ctx, "shape": rng.choice(["chain", "tree", "tree"]),
                "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "window": rng.choice([0, 0, 128, _log_int(rng, 1, 1000)]), "sinks": rng.random() < 0.7}
    if op == "commit":
        nodes = _log_int(rng, 2, 256)
        return {"op": "commit", "layers": _log_int(rng, 1, 36), "batch": _log_int(rng, 1, 64), "kv_heads": rng.choice([1, 2, 8]),
                "head_dim": rng.choice([32, 64]), "slots": nodes + _log_int(rng, 16, 128), "nodes": nodes,
                "accepted": rng.randint(1, min(nodes, 12))}
    if op == "lora":
        rank = rng.choice([8, 16, 16, 24, 32, 64, 128])
        return {"op": "lora", "tokens": _log_int(rng, 1, 8192), "k": 8 * _log_int(rng, 8, 512), "n_out": 8 * _log_int(rng, 8, 640),
                "rank": rank, "adapters": _log_int(rng, 1, 1024 // rank), "order": rng.choice(["mixed", "runs"]),
                "without": rng.choice([0.0, 0.1, 0.5])}
    groups = rng.choice([1, 1, 4, 8])
    experts = groups * _log_int(rng, 4, 256 // groups)
    topk_groups = rng.randint(1, groups)
    return {"op": "route", "tokens": _log_int(rng, 1, 8192), "experts": experts,
            "top_k": rng.randint(1, min(8, topk_groups * (experts // groups))), "scoring": rng.choice(["softmax", "sigmoid"]),
            "bias": rng.random() < 0.5, "groups": groups, "topk_groups": topk_groups,
            "group_top": rng.choice([1, 2]), "renormalize": rng.random() < 0.7}


# ---- sizes that follow from a case alone ----------------------------------------------------------------------------
def _spread(n, lo, hi):
    """n lengths between lo and hi, unequal, the first one hi."""
    return [hi - int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _tree_lengths(case):
    return _spread(case["batch"], case["ctx"] // 2, case["ctx"]), _spread(case["batch"], (case["nodes"] + 1) // 2, case["nodes"])


def _parents(n, shape, rng):
    """Parents of a tree of n drafted tokens in order of their depth (-1: follows the last cached token)."""
    if shape == "chain":
        return list(range(-1, n - 1))
    width = max(1, int(math.isqrt(n)))
    return [-1 if i < width else rng.randrange(max(0, (i - width) // 2), i) for i in range(n)]


# ---- what a program holds before the call ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2 + 1)
    rng = random.Random(seed)
    randn = lambda *shape, sd=1.0: torch.randn(*shape, generator=gen, device="cuda") * sd  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "tree":
        B, hd = case["batch"], case["head_dim"]
        ctx, nodes = _tree_lengths(case)
        order = list(range(B))
        rng.shuffle(order)
        ctx, nodes = [ctx[i] for i in order], [nodes[i] for i in order]
        offsets, depth, masks = [0], [], []
        words = (case["nodes"] + 31) // 32
        for n in nodes:
            depths, seen = [], []
            for i, p in enumerate(_parents(n, case["shape"], rng)):
                depths.append(0 if p < 0 else depths[p] + 1)
                seen.append((0 if p < 0 else seen[p]) | 1 << i)
            depth += depths
            masks += [[(m >> 32 * w & 0xFFFFFFFF) - (1 << 32 if m >> 32 * w & 0x80000000 else 0) for w in range(words)] for m in seen]
            offsets.append(len(depth))
        rows, slots = B + 2, (case["ctx"] + case["nodes"] + 15) // 16 * 16
        cache = (rows, case["kv_heads"], slots, hd)
        place = list(range(rows))
        rng.shuffle(place)
        return {"case": case, "q": randn(len(depth), case["q_heads"], hd, sd=1.5).bfloat16(), "k": randn(*cache, sd=1.2).bfloat16(),
                "v": randn(*cache).bfloat16(), "offsets": ints(offsets), "ctx": ints(ctx), "rows": ints(place[:B]),
                "mask": ints(masks), "depth": ints(depth), "sinks": randn(case["q_heads"]) if case["sinks"] else None}
    if case["op"] == "commit":
        B = case["batch"]
        accepted = _spread(B, 1, case["accepted"])
        rng.shuffle(accepted)
        offsets, path = [0], []
        for n in accepted:
            # the path's first node is node 0 or one behind the path's length, the others lie behind that length too
            # where the tree has room: the same call twice then moves the same rows
            first = 0 if rng.random() < 0.5 or case["nodes"] < 2 * n else rng.randint(n, case["nodes"] - n)
            behind = range(max(first + 1, n), case["nodes"])
            path += [first] + sorted(rng.sample(behind, n - 1)) if len(behind) >= n - 1 else range(n)
            offsets.append(len(path))
        cache = (case["layers"], B, case["kv_heads"], case["slots"], case["head_dim"])
        return {"case": case, "k": randn(*cache).bfloat16(), "v": randn(*cache).bfloat16(), "offsets": ints(offsets),
                "path": ints(path), "ctx": ints([rng.randrange(case["slots"] - case["nodes"] + 1) for _ in range(B)]),
                "rows": ints(rng.sample(range(B), B))}
    if case["op"] == "lora":
        T, n = case["tokens"], case["adapters"]
        if case["order"] == "runs":  # prompts one behind the other, a few per adapter
            cuts = sorted(rng.randrange(T) for _ in range(2 * n))
            runs = [rng.randrange(n) if rng.random() >= case["without"] else -1 for _ in range(2 * n + 1)]
            ids, at = [], 0
            for t in range(T):
                while at < 2 * n and t >= cuts[at]:
                    at += 1
                ids.append(runs[at])
        else:
            ids = [rng.randrange(n) if rng.random() >= case["without"] else -1 for _ in range(T)]
        return {"case": case, "x": randn(T, case["k"]).bfloat16(), "a": randn(n, case["rank"], case["k"], sd=case["k"] ** -0.5).bfloat16(),
                "b": randn(n, case["n_out"], case["rank"], sd=0.05).bfloat16(), "ids": ints(ids), "y": randn(T, case["n_out"]),
                "scale": torch.rand(n, generator=gen, device="cuda") + 0.5}
    E = case["experts"]
    return {"case": case, "logits": randn(case["tokens"], E, sd=1.5), "bias": randn(E, sd=0.1) if case["bias"] else None}


# ---- one call -------------------------------------------------------------------------------------------------------
def _serving():
    import __graft_entry__
    __graft_entry__.load_package()
    from gptoss_b200 import serving
    return serving


def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](case, state)


def _own_tree(case, s):
    return _serving().tree_attention(s["q"], s["k"], s["v"], s["offsets"], s["ctx"], s["mask"], s["depth"], sinks=s["sinks"],
                                     cache_rows=s["rows"], window=case["window"], max_nodes=case["nodes"], max_ctx=case["ctx"])


def _own_commit(case, s):
    _serving().cache_commit(s["k"], s["v"], s["ctx"], s["offsets"], s["path"], cache_rows=s["rows"], max_path=case["accepted"])
    return s["k"], s["v"]


def _own_lora(case, s):
    return _serving().lora_apply(s["x"], s["a"], s["b"], s["ids"], s["y"], scale=s["scale"], out=torch.empty_like(s["y"]))


def _own_route(case, s):
    return _serving().route_experts(s["logits"], case["top_k"], scoring=case["scoring"], bias=s["bias"], n_groups=case["groups"],
                                    topk_groups=case["topk_groups"], group_top=case["group_top"], renormalize=case["renormalize"])


_own = {"tree": _own_tree, "commit": _own_commit, "lora": _own_lora, "route": _own_route}


def _plain_tree(case, s):
    """Every sequence padded to the longest: scores, mask, softmax with the sink in the denominator, weighted sum."""
    N, nkv, hd, window = case["nodes"], case["kv_heads"], case["head_dim"], case["window"]
    group = case["q_heads"] // nkv
    L = case["ctx"] + N
    first, last, ctx, rows = s["offsets"][:-1].long(), s["offsets"][1:].long(), s["ctx"].long(), s["rows"].long()
    at = first[:, None] + torch.arange(N, device="cuda")                       # [B, N] rows of q, padded
    real = at < last[:, None]
    at = torch.where(real, at, torch.zeros_like(at))
    B = at.shape[0]
    q = s["q"].float()[at].view(B, N, nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, group * N, hd)
    k, v = s["k"][:, :, :L][rows].float(), s["v"][:, :, :L][rows].float()
    slot = torch.arange(L, device="cuda")
    draft = slot - ctx[:, None]                                                # [B, L] node behind a slot, negative: cached
    bits = s["mask"].long()[at]                                                # [B, N, words]
    node = draft.clamp(0, N - 1)[:, None, :].expand(B, N, L)
    bit = (torch.gather(bits, 2, node >> 5) >> (node & 31)) & 1
    seen = torch.where(draft[:, None] < 0, True, (bit != 0) & (draft < (last - first)[:, None])[:, None])
    if window:
        depth = s["depth"].long()[at]
        place = torch.where(draft < 0, slot.expand(B, L), ctx[:, None] + torch.gather(depth, 1, draft.clamp(0, N - 1)))
        seen = seen & (place[:, None] > (ctx[:, None] + depth)[:, :, None] - window)
    seen = seen[:, None, None].expand(B, 1, group, N, L).reshape(B, 1, group * N, L)
    scores = torch.matmul(q, k.transpose(2, 3)) * hd ** -0.5
    scores = scores.masked_fill(~seen, -math.inf)
    sink = torch.full((nkv, group, N), -math.inf, device="cuda")
    if s["sinks"] is not None:
        sink = s["sinks"].view(nkv, group, 1).expand(nkv, group, N)
    sink = sink.reshape(1, nkv, group * N, 1)
    top = torch.maximum(scores.amax(3, keepdim=True), sink)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(3, keepdim=True) + torch.exp(sink - top)
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.view(B, nkv, group, N, hd).permute(0, 3, 1, 2, 4).reshape(B, N, nkv * group, hd)
    return out[real].bfloat16()


def _plain_commit(case, s):
    ctx, rows, path = s["ctx"].long(), s["rows"].long(), s["path"].long()
    step = torch.arange(case["accepted"], device="cuda")
    at = s["offsets"][:-1].long()[:, None] + step
    real = at < s["offsets"][1:].long()[:, None]
    source = torch.where(real, path[torch.where(real, at, torch.zeros_like(at))], step.expand_as(at))
    source, target, row = (ctx[:, None] + source).flatten(), (ctx[:, None] + step).flatten(), rows[:, None].expand_as(at).flatten()
    s["k"][:, row, :, target] = s["k"][:, row, :, source]
    s["v"][:, row, :, target] = s["v"][:, row, :, source]
    return s["k"], s["v"]


def _plain_lora(case, s):
    """Both products over all adapters side by side; a token keeps the part of its own adapter."""
    T, n, rank = case["tokens"], case["adapters"], case["rank"]
    mine = (s["ids"].long()[:, None] == torch.arange(n, device="cuda")).float() * s["scale"]
    u = torch.matmul(s["x"].float(), s["a"].float().view(n * rank, -1).t()).view(T, n, rank) * mine[:, :, None]
    return s["y"] + torch.matmul(u.view(T, n * rank), s["b"].float().transpose(1, 2).reshape(n * rank, -1))


def _plain_route(case, s):
    """Scores and selection in 64 bits: a difference in the last of 32 bits would change an expert's place."""
    T, E, G = case["tokens"], case["experts"], case["groups"]
    logits = s["logits"].double()
    if case["scoring"] == "softmax":
        scores = torch.exp(logits - logits.amax(1, keepdim=True))
        scores = scores / scores.sum(1, keepdim=True)
    else:
        scores = 1.0 / (1.0 + torch.exp(-logits))
    choice = scores if s["bias"] is None else scores + s["bias"].double()
    if G > 1:
        best = torch.sort(choice.view(T, G, E // G), dim=2, descending=True).values[:, :, :case["group_top"]].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["topk_groups"]]
        open_groups = torch.zeros(T, G, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        choice = choice.masked_fill(~open_groups[:, :, None].expand(T, G, E // G).reshape(T, E), -math.inf)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    weights = torch.gather(scores, 1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    return weights.float(), ids.int()


_plain = {"tree": _plain_tree, "commit": _plain_commit, "lora": _plain_lora, "route": _plain_route}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "tree":
        group = case["q_heads"] // case["kv_heads"]
        slots, pairs, tokens = 0, 0, 0
        for ctx, n in zip(*_tree_lengths(case)):
            reach = min(ctx, case["window"] - 1) if case["window"] else ctx  # cached tokens that the tree's first token sees
            slots += reach + n
            pairs += n * (reach + (n + 1) // 2 if case["shape"] == "chain" else reach + math.isqrt(n))
            tokens += n
        row = case["head_dim"] * 2
        return {"bytes": slots * case["kv_heads"] * 2 * row + tokens * (case["q_heads"] * 2 * row + 4 * ((case["nodes"] + 31) // 32 + 1)),
                "flops": 4 * pairs * case["kv_heads"] * group * case["head_dim"]}
    if case["op"] == "commit":
        moved = sum(_spread(case["batch"], 1, case["accepted"]))
        return {"bytes": case["layers"] * moved * case["kv_heads"] * case["head_dim"] * 2 * 2 * 2, "flops": 0}
    if case["op"] == "lora":
        T, used = case["tokens"], min(case["adapters"], case["tokens"])
        served = T * (1 - case["without"])
        return {"bytes": T * case["n_out"] * 8 + served * case["k"] * 2 + used * case["rank"] * (case["k"] + case["n_out"]) * 2 + T * 4,
                "flops": 2 * served * case["rank"] * (case["k"] + case["n_out"])}
    return {"bytes": case["tokens"] * (case["experts"] * 4 + case["top_k"] * 8), "flops": case["tokens"] * case["experts"] * 8}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "commit":
        return None
    if case["op"] == "tree":
        group, hd = case["q_heads"] // case["kv_heads"], case["head_dim"]
        offsets, ctxs, rows, masks, depth = (s[x].tolist() for x in ("offsets", "ctx", "rows", "mask", "depth"))
        out = torch.empty(*s["q"].shape, dtype=torch.float64, device="cuda")
        for i, (c, row) in enumerate(zip(ctxs, rows)):
            a, z = offsets[i], offsets[i + 1]
            n = z - a
            places = list(range(c)) + [c + d for d in depth[a:z]]
            seen = torch.ones(n, c + n, dtype=torch.bool)
            seen[:, c:] = torch.tensor([[masks[a + r][j >> 5] >> (j & 31) & 1 for j in range(n)] for r in range(n)], dtype=torch.bool)
            if case["window"]:
                reach = torch.tensor(depth[a:z])[:, None] + c - torch.tensor(places)[None, :]
                seen &= reach < case["window"]
            k = s["k"][row, :, :c + n].double()
            v = s["v"][row, :, :c + n].double()
            q = s["q"][a:z].double().view(n, case["kv_heads"], group, hd).permute(1, 2, 0, 3)
            logit = torch.einsum("hgnd,hld->hgnl", q, k) / math.sqrt(hd)
            logit[:, :, ~seen.cuda()] = -math.inf
            if s["sinks"] is not None:
                extra = s["sinks"].double().view(case["kv_heads"], group, 1, 1).expand(-1, -1, n, 1)
                weight = torch.softmax(torch.cat([logit, extra], 3), 3)[..., :-1]
            else:
                weight = torch.softmax(logit, 3).nan_to_num(0.0)
            out[a:z] = torch.einsum("hgnl,hld->nhgd", weight, v).reshape(n, -1, hd)
        return out
    if case["op"] == "lora":
        out = s["y"].double()
        for adapter in range(case["adapters"]):
            who = (s["ids"] == adapter).nonzero()[:, 0]
            low = s["x"][who].double() @ s["a"][adapter].double().t()
            out[who] += float(s["scale"][adapter]) * (low @ s["b"][adapter].double().t())
        return out
    logits = s["logits"].cpu().double()
    score = torch.softmax(logits, 1) if case["scoring"] == "softmax" else torch.sigmoid(logits)
    pick = score if s["bias"] is None else score + s["bias"].cpu().double()
    size = case["experts"] // case["groups"]
    if case["groups"] > 1:
        rank = torch.topk(pick.view(-1, case["groups"], size), min(case["group_top"], size), dim=2).values.sum(2)
        floor = torch.topk(rank, case["topk_groups"], dim=1).values[:, -1:]
        pick = torch.where((rank >= floor).repeat_interleave(size, 1), pick, torch.full_like(pick, -math.inf))
    best = torch.topk(pick, case["top_k"], dim=1).indices
    weight = torch.gather(score, 1, best)
    if case["renormalize"]:
        weight = weight / weight.sum(1, keepdim=True)
    return weight.cuda(), None
