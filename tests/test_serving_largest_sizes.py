"""The largest sizes that the serving operators take, and the first ones that they refuse."""
import ctypes as C

import pytest

import test_serving_refusals as small
from gptoss_b200 import capi

torch = pytest.importorskip("torch")
lib = small.lib


@pytest.mark.parametrize("max_seq", [(1 << 30) + 1, (1 << 31) - 256, (1 << 31) - 1])
def test_tree_attention_refuses_a_cache_whose_slots_do_not_fit_in_an_int(lib, max_seq):
    """Context and drafted tokens together are counted in 32 bits."""
    assert lib.gptoss_tree_attention(C.byref(small.tree_args(max_seq=max_seq)), None) == capi.ERR_BAD_ARG
    assert b"2^30" in lib.gptoss_serving_last_error()


@pytest.mark.gpu
def test_expert_choice_of_as_many_tokens_as_an_int_counts():
    from gptoss_b200 import serving
    T = (1 << 31) - 1
    logits = torch.zeros(T, 1, device="cuda")
    w, i = serving.route_experts(logits, 1, weight_scale=3.0)
    del logits
    assert w.shape == i.shape == (T, 1)
    assert float(w.min()) == 3.0 == float(w.max()) and not i.any()
