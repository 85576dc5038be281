"""The model's steps over drafted tokens and its adapters, against the fixtures of the reference's own forward() and against
the one-token steps.  Tolerances on logits are those of test_gpu_model.py (bf16 rounding of GEMM inputs and cache; the tree
attention adds one bf16 rounding of queries and one of weights, each of the size of the cache's)."""
import random
from pathlib import Path

import numpy as np
import pytest

from gptoss_b200 import binfmt, capi, synth

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DATA = Path(__file__).parent / "golden"
LOGIT_TOL, MARGIN_SAFE = 4e-3, 8e-3


@pytest.fixture(scope="module")
def golden():
    return np.load(DATA / "moe_7m_golden.npz")


@pytest.fixture(scope="module")
def checkpoint(golden, tmp_path_factory):
    p = tmp_path_factory.mktemp("ckpt") / "gpt-oss-7m-synth.bin"
    binfmt.write_synthetic(str(p), binfmt.config_7m(), int(golden["seed"]))
    return p


def chain(n):
    return list(range(-1, n - 1))


def with_siblings(ids, rng, vocab, extra):
    """The chain `ids` hidden in a tree: wrong tokens between its nodes, hanging from nodes before them.  Returns (tokens,
    parents, places of the chain)."""
    toks, pars, places, last = [], [], [], -1
    for t in ids:
        for _ in range(rng.randrange(extra + 1)):
            toks.append(rng.randrange(vocab))
            pars.append(rng.randrange(-1, len(toks) - 1))
        toks.append(int(t))
        pars.append(last)
        last = len(toks) - 1
        places.append(last)
    return toks, pars, places


@pytest.mark.parametrize("pieces,extra", [([95], 0), ([1, 2, 5, 17, 30, 40], 0), ([1, 4, 3, 9, 20, 8, 25, 25], 3)])
def test_drafted_tokens_match_reference_forward(golden, checkpoint, pieces, extra):
    from gptoss_b200 import model
    cfg = binfmt.config_7m()
    seq = np.concatenate([golden["prompt"], golden["generated"]]).astype(np.int32)
    n_pos, rng = len(golden["next_token"]), random.Random(extra)
    assert sum(pieces) == n_pos
    m = model.Model(cfg, max_batch=256, max_seq=384)
    m.load_bin(checkpoint)
    other = synth.uniform_ids(5, 9, n_pos, cfg.vocab_size).astype(np.int32)
    ctx, pos = np.array([0, 7], np.int32), 0  # a second sequence in another row, over tokens nobody put into its cache
    for n in pieces:
        toks, pars, places = with_siblings(seq[pos:pos + n], rng, cfg.vocab_size, extra)
        nxt, _ = m.step_tree([toks, other[pos:pos + n]], [pars, chain(n)], [3, 200], ctx)
        for j, at in enumerate(places):
            np.testing.assert_allclose(m.logits(at)[golden["probe_idx"]], golden["probe_logits"][pos + j], rtol=0, atol=LOGIT_TOL,
                                       err_msg=f"position {pos + j}")
            if golden["top2_margin"][pos + j] > MARGIN_SAFE:
                assert nxt[at] == golden["next_token"][pos + j], pos + j
        ctx = m.accept([3, 200], ctx, [places, list(range(n))])
        pos += n
        assert ctx.tolist() == [pos, 7 + pos]
    m.close()


@pytest.mark.parametrize("pieces,extra", [([200], 0), ([3, 1, 40, 60, 7, 89], 0), ([10, 30, 1, 60, 49, 50], 2)])
def test_drafted_tokens_hd64_gqa8_sliding_window_match_reference_forward(tmp_path, pieces, extra):
    import sys
    sys.path.insert(0, str(DATA))
    from make_golden import attn_config
    from gptoss_b200 import model
    g = np.load(DATA / "attn_hd64_golden.npz")
    cfg = attn_config()
    ckpt = tmp_path / "attn-hd64-synth.bin"
    binfmt.write_synthetic(str(ckpt), cfg, int(g["seed"]), sigma=float(g["sigma"]))
    ids, rng = g["ids"].astype(np.int32), random.Random(extra + 1)
    m = model.Model(cfg, max_batch=256, max_seq=256)
    m.load_bin(ckpt)
    tol = 0.02 * float(g["logit_std"].mean())
    ctx, pos = np.zeros(1, np.int32), 0
    for n in pieces:
        n = min(n, len(ids) - pos)
        toks, pars, places = with_siblings(ids[pos:pos + n], rng, cfg.vocab_size, extra if pos + n < 150 else 0)
        nxt, = m.step_tree([toks], [pars], [1], ctx)
        for j, at in enumerate(places):
            got = m.logits(at)[g["probe_idx"]]
            assert float(np.abs(got - g["probe_logits"][pos + j]).max()) <= tol, pos + j
            if g["top2_margin"][pos + j] > 4 * tol:
                assert nxt[at] == g["next_token"][pos + j]
        ctx = m.accept([1], ctx, [places])
        pos += n
    # the one-token step reads the cache that the trees left: it agrees with the tree's step on the same token
    last = m.step_seqs(ids[-1:], np.array([1], np.int32), ctx - 1)
    one = m.logits(0)[g["probe_idx"]]
    assert float(np.abs(one - g["probe_logits"][len(ids) - 1]).max()) <= tol and len(last) == 1
    m.close()


@pytest.mark.parametrize("drafter", ["none", "right", "mixed", "wrong"])
def test_drafted_greedy_decode_reproduces_the_reference(golden, checkpoint, drafter):
    """40 tokens of the reference's greedy continuation, whatever is drafted: those behind the first ten, from where on no
    top-2 gap is below MARGIN_SAFE (and no router gap anywhere near 1e-4, where a bf16 engine may choose another expert: the
    continuation of greedy_7m_golden.npz has one of 9.5e-5 at its 16th token and is of no use to a path that rounds
    differently)."""
    from gptoss_b200 import model
    g, first, n_new = golden, 10, 40
    assert float(g["top2_margin"][31 + first:31 + first + n_new].min()) > MARGIN_SAFE and float(g["route_gap"].min()) > 4e-4
    cfg = binfmt.config_7m()
    m = model.Model(cfg, max_batch=96, max_seq=160)
    m.load_bin(checkpoint)
    truth = g["prompt"].tolist() + g["generated"].tolist()
    rng = random.Random(1)
    steps = 0
    inner = m.step_tree

    def counted(*a, **k):
        nonlocal steps
        steps += 1
        return inner(*a, **k)

    m.step_tree = counted

    def draft(history):
        n = len(history)
        right = truth[n:n + 6] if history == truth[:n] else []
        if drafter == "none":
            return [], []
        if drafter == "right":
            return right, chain(len(right))
        toks, pars, _ = with_siblings(right if drafter == "mixed" else [], rng, cfg.vocab_size, 2)
        return toks + [rng.randrange(cfg.vocab_size) for _ in range(3)], pars + [-1, len(toks) - 1, -1]

    n = len(g["prompt"]) + first
    out = m.generate_drafted([truth[:n], synth.uniform_ids(3, 4, 41, cfg.vocab_size).tolist()], n_new, draft)
    assert out.shape == (2, n_new)
    assert out[0].tolist() == truth[n:n + n_new]
    if drafter in ("right", "mixed"):  # alone, the first sequence needs a step per seven tokens
        steps = 0
        out = m.generate_drafted([truth[:n]], n_new, draft)
        assert out[0].tolist() == truth[n:n + n_new] and steps <= 1 + (n_new + 6) // 7
    m.close()


def test_step_tree_refuses(checkpoint):
    from gptoss_b200 import model, moe
    m = model.Model(binfmt.config_7m(), max_batch=16, max_seq=32)
    with pytest.raises(moe.GptossError) as e:
        m.step_tree([[1]], [[-1]], [0], [0])  # no weights yet
    assert e.value.code == capi.ERR_STATE
    m.load_bin(checkpoint)
    with pytest.raises(moe.GptossError):
        m.accept([0], [0], [[0]])  # nothing drafted yet
    for bad in (([[1, 2]], [[-1, 1]], [0], [0]), ([[1, 2]], [[-1, -2]], [0], [0]), ([[1]], [[-1]], [16], [0]), ([[1]], [[-1]], [-1], [0]),
                ([[1], [2]], [[-1], [-1]], [3, 3], [0, 0]), ([[1]], [[-1]], [0], [32]), ([[1, 2]], [chain(2)], [0], [31]),
                ([[1]], [[-1]], [0], [-1]), ([list(range(17))], [chain(17)], [0], [0]), ([[]], [[]], [0], [0]),
                ([list(range(9)), list(range(8))], [chain(9), chain(8)], [0, 1], [0, 0])):
        with pytest.raises(moe.GptossError) as e:
            m.step_tree(*bad)
        assert e.value.code == capi.ERR_BAD_ARG
    m.step_tree([[1, 2, 3]], [chain(3)], [0], [29])
    for bad in (([0], [29], [[1, 0]]), ([0], [29], [[0, 0]]), ([0], [29], [[3]]), ([16], [0], [[0]]), ([0, 0], [0, 0], [[0], [0]]),
                ([0], [-1], [[0]]), ([0], [29], [[-1]])):
        with pytest.raises(moe.GptossError):
            m.accept(*bad)
    assert m.accept([0], [29], [[0, 2]]).tolist() == [31]
    assert m.accept([0], [29], [[]]).tolist() == [29]
    m.close()


# ---- adapters ----------------------------------------------------------------------------------------------------------
def random_adapter(cfg, rank, seed, sd=0.3):
    rng = np.random.default_rng(seed)
    qd, qkv = cfg.head_dim * cfg.n_attn_heads, cfg.head_dim * (cfg.n_attn_heads + 2 * cfg.n_kv_heads)
    r = lambda *s: (rng.standard_normal(s) * sd).astype(np.float32)  # noqa: E731
    return dict(a_qkv=r(rank, cfg.hidden_dim), b_qkv=r(qkv, rank), a_o=r(rank, qd), b_o=r(cfg.hidden_dim, rank))


def test_adapters_touch_only_the_rows_bound_to_them(checkpoint):
    from gptoss_b200 import model
    cfg = binfmt.config_7m()
    B, n_pos = 40, 12
    ids = synth.uniform_ids(7, 5, B * n_pos, cfg.vocab_size).reshape(n_pos, B).astype(np.int32)
    plain, m = model.Model(cfg, max_batch=B, max_seq=32), model.Model(cfg, max_batch=B, max_seq=32)
    for x in (plain, m):
        x.load_bin(checkpoint)
    m.lora_create(3, 8)
    for layer in range(cfg.n_layers):
        m.lora_load(0, layer, **random_adapter(cfg, 8, layer), scale=0.5)
        m.lora_load(2, layer, **random_adapter(cfg, 8, 10 + layer), scale=2.0)  # adapter 1 stays zero
    m.lora_bind(5, 0), m.lora_bind(9, 2), m.lora_bind(11, 1), m.lora_bind(30, 0)
    for pos in range(n_pos):
        plain.step(ids[pos], pos)
        if pos % 3 == 2:  # a compacted step: the bound rows keep their adapters
            m.step_rows(ids[pos], np.arange(B, dtype=np.int32), pos)
        else:
            m.step(ids[pos], pos)
        for row in (0, 4, 6, 11, 39):
            assert np.array_equal(m.logits(row), plain.logits(row)), (pos, row)
        for row in (5, 9, 30):
            assert float(np.abs(m.logits(row) - plain.logits(row)).max()) > 0.01, (pos, row)
    # a row's result does not depend on who shares the step, nor on the order of the rows
    want = m.logits(30)
    order = np.array([30, 9, 2], np.int32)
    m.step_rows(ids[n_pos - 1, order], order, n_pos - 1)
    assert np.array_equal(m.logits(0), want)
    m.lora_bind(30, -1), m.lora_bind(9, -1)
    p2 = np.array([n_pos - 1, 3, n_pos - 1], np.int32)
    m.step_seqs(ids[n_pos - 1, order], order, p2)
    assert not np.array_equal(m.logits(0), want)
    plain.close()
    m.close()


def test_adapters_equal_merged_weights(tmp_path):
    """An adapter whose rows of A pick one input each: B A is then a matrix of B's columns, exact in bf16.  On a checkpoint
    whose projections are zero, the model with the adapter and the model with the merged weights compute the same products;
    only the order of a few fp32 additions differs."""
    import sys
    sys.path.insert(0, str(DATA))
    from make_golden import attn_config
    from gptoss_b200 import model
    cfg, rank, scale = attn_config(), 16, 2.0
    base = tmp_path / "base.bin"
    binfmt.write_synthetic(str(base), cfg, 11, sigma=0.05)
    _, tensors = binfmt.read(str(base))
    rng = np.random.default_rng(2)
    ads = []
    for layer in range(cfg.n_layers):
        ad = random_adapter(cfg, rank, 20 + layer, sd=0.2)
        for k in ("a_qkv", "a_o"):
            pick = np.zeros_like(ad[k])
            pick[np.arange(rank), rng.permutation(pick.shape[1])[:rank]] = 1.0
            ad[k] = pick
        for k in ("b_qkv", "b_o"):
            ad[k] = synth.bf16_bits_to_f32(synth.f32_to_bf16_bits(ad[k].reshape(-1))).reshape(ad[k].shape)
        ads.append(ad)
    for name, merge in (("zero.bin", False), ("merged.bin", True)):
        with open(tmp_path / name, "wb") as f:
            f.write(cfg.pack())
            for t in binfmt.TENSOR_ORDER:
                v = np.array(tensors[t])
                if t in ("qkv_w", "attn_out_w"):
                    a, b = ("a_qkv", "b_qkv") if t == "qkv_w" else ("a_o", "b_o")
                    v = np.stack([scale * ads[x][b] @ ads[x][a] if merge else np.zeros_like(v[x]) for x in range(cfg.n_layers)])
                v.astype(np.float32).tofile(f)
    zero, merged = (model.Model(cfg, max_batch=64, max_seq=64) for _ in range(2))
    zero.load_bin(tmp_path / "zero.bin")
    merged.load_bin(tmp_path / "merged.bin")
    zero.lora_create(4, rank)
    for layer, ad in enumerate(ads):
        zero.lora_load(2, layer, **ad, scale=scale)
    B = 48  # beyond the size at which the tokens are sorted by adapter
    for row in range(B):
        zero.lora_bind(row, 2)
    ids = synth.uniform_ids(1, 2, 20 * B, cfg.vocab_size).reshape(20, B).astype(np.int32)
    for pos in range(20):
        zero.step(ids[pos], pos), merged.step(ids[pos], pos)
        a, b = zero.logits(17), merged.logits(17)
        assert float(np.abs(a - b).max()) <= 2e-3 * float(b.std()), pos
    # the same through drafted tokens
    t = ids[:6, 3].tolist()
    zero.step_tree([t], [chain(6)], [50], [0]), merged.step_tree([t], [chain(6)], [50], [0])
    assert float(np.abs(zero.logits(5) - merged.logits(5)).max()) > 1e-3  # row 50 has no adapter
    zero.lora_bind(50, 2)
    zero.step_tree([t], [chain(6)], [50], [0]), merged.step_tree([t], [chain(6)], [50], [0])
    assert float(np.abs(zero.logits(5) - merged.logits(5)).max()) <= 2e-2 * float(merged.logits(5).std())
    zero.close()
    merged.close()


def test_adapters_refuse(checkpoint):
    from gptoss_b200 import model, moe
    m = model.Model(binfmt.config_7m(), max_batch=4, max_seq=16)
    m.load_bin(checkpoint)
    with pytest.raises(moe.GptossError):
        m.lora_bind(0, 0)  # no adapters yet
    with pytest.raises(moe.GptossError):
        m.lora_load(0, 0)
    for n, r in ((0, 8), (1, 0), (1, 12), (1, 136), (8193, 8)):
        with pytest.raises(moe.GptossError):
            m.lora_create(n, r)
    m.lora_create(2, 8)
    with pytest.raises(moe.GptossError) as e:
        m.lora_create(2, 8)
    assert e.value.code == capi.ERR_STATE
    for row, ad in ((-1, 0), (4, 0), (0, 2), (0, -2)):
        with pytest.raises(moe.GptossError):
            m.lora_bind(row, ad)
    with pytest.raises(moe.GptossError):
        m.lora_load(2, 0)
    with pytest.raises(moe.GptossError):
        m.lora_load(0, 99)
    m.close()
