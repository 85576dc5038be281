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
