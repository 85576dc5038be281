"""Arguments that the serving operators refuse (checked on the host before anything reaches a GPU), and the host-side
tree masks."""
import ctypes as C

import numpy as np
import pytest

from gptoss_b200 import capi

torch = pytest.importorskip("torch")

A = 4096  # an aligned address that is never read: every case is refused or empty


@pytest.fixture(scope="module")
def lib():
    if capi.needs_build():
        capi.build()
    return capi.load()


def tree_args(**kw):
    d = dict(q=A, k_cache=A, v_cache=A, out=A, offsets=A, ctx_len=A, rows=None, mask=A, depth=A, sinks=None, workspace=None,
             workspace_bytes=0, q_stride=512, out_stride=512, n_tokens=5, n_seqs=2, max_nodes=4, max_ctx=10, mask_words=1,
             cache_rows=3, max_seq=64, n_q_heads=8, n_kv_heads=2, head_dim=64, window=0, scale=0.125)
    d.update(kw)
    return capi.TreeAttentionArgs(*[d[n] for n, _ in capi.TreeAttentionArgs._fields_])


@pytest.mark.parametrize("bad", [
    dict(n_seqs=-1), dict(n_tokens=-1), dict(max_nodes=-1), dict(max_ctx=-1), dict(head_dim=48), dict(head_dim=128),
    dict(n_q_heads=9), dict(n_q_heads=18, n_kv_heads=2), dict(n_kv_heads=0), dict(max_nodes=257), dict(max_nodes=33),
    dict(cache_rows=0), dict(max_seq=0), dict(q=None), dict(k_cache=None), dict(v_cache=None), dict(out=None), dict(offsets=None),
    dict(ctx_len=None), dict(mask=None), dict(window=-1), dict(window=5, depth=None), dict(scale=-1.0), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(workspace=A + 8, max_ctx=64000), dict(max_ctx=64000), dict(workspace=A, workspace_bytes=1000, max_ctx=64000), dict(q=A + 8), dict(k_cache=A + 2),
    dict(v_cache=A + 8), dict(out=A + 4), dict(q_stride=516), dict(out_stride=516), dict(q_stride=504), dict(out_stride=8)])
def test_tree_attention_refuses(lib, bad):
    assert lib.gptoss_tree_attention(C.byref(tree_args(**bad)), None) == capi.ERR_BAD_ARG
    assert lib.gptoss_serving_last_error()


@pytest.mark.parametrize("empty", [dict(n_seqs=0), dict(n_tokens=0), dict(max_nodes=0), dict(n_seqs=0, q=None, out=None)])
def test_tree_attention_of_nothing_is_a_no_op(lib, empty):
    assert lib.gptoss_tree_attention(C.byref(tree_args(**empty)), None) == capi.OK


def test_null_arguments(lib):
    for call in (lib.gptoss_tree_attention, lib.gptoss_lora_apply, lib.gptoss_expert_choice):
        assert call(None, None) == capi.ERR_BAD_ARG
    assert lib.gptoss_tree_attention_workspace(None) == 0 and lib.gptoss_lora_workspace(None) == 0


@pytest.mark.parametrize("bad", [
    (None, A, 1, 2, 2, 16, 64, 1, None, A, A, A, 8, 4), (A, None, 1, 2, 2, 16, 64, 1, None, A, A, A, 8, 4),
    (A, A, -1, 2, 2, 16, 64, 1, None, A, A, A, 8, 4), (A, A, 1, 0, 2, 16, 64, 1, None, A, A, A, 8, 4),
    (A, A, 1, 2, 0, 16, 64, 1, None, A, A, A, 8, 4), (A, A, 1, 2, 2, 0, 64, 1, None, A, A, A, 8, 4),
    (A, A, 1, 2, 2, 16, 48, 1, None, A, A, A, 8, 4), (A, A, 1, 2, 2, 16, 64, -1, None, A, A, A, 8, 4),
    (A, A, 1, 2, 2, 16, 64, 1, None, None, A, A, 8, 4), (A, A, 1, 2, 2, 16, 64, 1, None, A, None, A, 8, 4),
    (A, A, 1, 2, 2, 16, 64, 1, None, A, A, None, 8, 4), (A, A, 1, 2, 2, 16, 64, 1, None, A, A, A, 8, -4),
    (A + 2, A, 1, 2, 2, 16, 64, 1, None, A, A, A, 8, 4), (A, A, 1, 2, 2, 16, 64, 1, None, A, A, A, -8, 4)])
def test_cache_commit_refuses(lib, bad):
    assert lib.gptoss_cache_commit(*bad, None) == capi.ERR_BAD_ARG


@pytest.mark.parametrize("empty", [(None, None, 0, 2, 2, 16, 64, 1, None, None, None, None, 8, 4),
                                   (None, None, 1, 2, 2, 16, 64, 0, None, None, None, None, 8, 4),
                                   (None, None, 1, 2, 2, 16, 64, 1, None, None, None, None, 8, 0),
                                   (None, None, 1, 2, 2, 16, 64, 1, None, None, None, None, 0, 4)])
def test_cache_commit_of_nothing_is_a_no_op(lib, empty):
    assert lib.gptoss_cache_commit(*empty, None) == capi.OK


def lora_args(**kw):
    d = dict(x=A, a=A, b=A, scale=None, ids=A, y=A, out=A, workspace=A, workspace_bytes=1 << 40, x_stride=64, y_stride=32,
             out_stride=32, T=3, K=64, n_out=32, rank=8, n_adapters=2)
    d.update(kw)
    return capi.LoraArgs(*[d[n] for n, _ in capi.LoraArgs._fields_])


@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(K=0), dict(K=60), dict(n_out=0), dict(n_out=30), dict(K=(1 << 30) + 8), dict(n_out=(1 << 30) + 8), dict(rank=0), dict(rank=12), dict(rank=136),
    dict(n_adapters=0), dict(n_adapters=8193), dict(out_stride=36, out=A, y=A), dict(x=None), dict(a=None), dict(b=None), dict(ids=None), dict(y=None), dict(out=None), dict(x=A + 2),
    dict(a=A + 8), dict(b=A + 8), dict(y=A + 4), dict(out=A + 8), dict(x_stride=68), dict(x_stride=56), dict(y_stride=33),
    dict(y_stride=28), dict(out_stride=28), dict(T=513, workspace=None), dict(T=513, workspace=A + 4), dict(T=513, workspace_bytes=4)])
def test_lora_refuses(lib, bad):
    assert lib.gptoss_lora_apply(C.byref(lora_args(**bad)), None) == capi.ERR_BAD_ARG
    assert lib.gptoss_serving_last_error()


def test_lora_of_nothing_is_a_no_op(lib):
    assert lib.gptoss_lora_apply(C.byref(lora_args(T=0, x=None, workspace=None, workspace_bytes=0)), None) == capi.OK


def choice_args(**kw):
    d = dict(logits=A, bias=None, topk_w=A, topk_i=A, stride=64, T=3, E=64, k=4, scoring=0, n_groups=1, topk_groups=1,
             group_top=1, renormalize=1, weight_scale=1.0)
    d.update(kw)
    return capi.ExpertChoiceArgs(*[d[n] for n, _ in capi.ExpertChoiceArgs._fields_])


@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(E=0), dict(E=257, stride=257), dict(scoring=2), dict(n_groups=0), dict(n_groups=3), dict(n_groups=64),
    dict(topk_groups=0), dict(topk_groups=2), dict(group_top=0), dict(group_top=3), dict(k=0), dict(k=9),
    dict(n_groups=32, topk_groups=1, k=3), dict(logits=None), dict(topk_w=None), dict(topk_i=None), dict(stride=63)])
def test_expert_choice_refuses(lib, bad):
    assert lib.gptoss_expert_choice(C.byref(choice_args(**bad)), None) == capi.ERR_BAD_ARG


def test_expert_choice_of_nothing_is_a_no_op(lib):
    assert lib.gptoss_expert_choice(C.byref(choice_args(T=0, logits=None)), None) == capi.OK


def test_python_layer_refuses_host_tensors_and_wrong_types(lib):
    from gptoss_b200 import moe, serving
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    c = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(moe.GptossError) as e:
        serving.tree_attention(q, c, c, i, i[:1], i[:, None], max_nodes=2, max_ctx=1)
    assert e.value.code == capi.ERR_BAD_ARG
    with pytest.raises(moe.GptossError):
        serving.tree_attention(q.float(), c, c, i, i[:1], i[:, None], max_nodes=2, max_ctx=1)
    with pytest.raises(moe.GptossError):
        serving.cache_commit(c, c, i, i, i, max_path=1)
    with pytest.raises(moe.GptossError):
        serving.lora_apply(q[0], c[0], c[0], i, q[0].float())
    with pytest.raises(moe.GptossError):
        serving.route_experts(torch.zeros(2, 8), 2)


def test_tree_masks():
    from gptoss_b200 import moe, serving
    off, mask, depth = serving.tree_masks([[-1, 0, 0, 2], [], [-1] + list(range(39))])
    assert off.tolist() == [0, 4, 4, 44] and mask.shape == (44, 2) and mask.dtype == np.int32
    assert mask[:4, 0].tolist() == [1, 3, 5, 13] and depth[:4].tolist() == [0, 1, 1, 2]
    assert depth[4:].tolist() == list(range(40))
    for i in range(40):
        want = (1 << (i + 1)) - 1
        assert int(np.uint32(mask[4 + i, 0])) | int(np.uint32(mask[4 + i, 1])) << 32 == want
    assert serving.tree_masks([[-1]], max_nodes=256)[1].shape == (1, 8)
    for bad in ([[0]], [[-1, 2, 0]], [[-2]], [[-1] * 257]):
        with pytest.raises(moe.GptossError):
            serving.tree_masks(bad)
