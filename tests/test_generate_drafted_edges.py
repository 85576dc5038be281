"""The loop of ``Model.generate_drafted`` on the host, at its smallest and largest, over a stand-in for the steps on the GPU."""
import ctypes as C

import numpy as np
import pytest

from gptoss_b200 import capi

torch = pytest.importorskip("torch")
VOCAB = 97


def follows(path):
    """The token that the stand-in's greedy decoding puts behind a sequence: depends on all of it."""
    x = 1
    for t in path:
        x = (x * 31 + t + 1) % 1000003
    return x % VOCAB


def make_model(max_batch, max_seq):
    from gptoss_b200 import model, moe

    class Steps(model.Model):
        def __init__(self):
            self._m = C.c_void_p()
            self.max_batch, self.max_seq = max_batch, max_seq
            self.cache = [[] for _ in range(max_batch)]  # cached ids of each row

        def step_tree(self, tokens, parents, rows, ctx, need_next=True):
            if not (0 < len(tokens) <= max_batch and sum(map(len, tokens)) <= max_batch):
                raise moe.GptossError(capi.ERR_BAD_ARG, "size")
            self.drafted, out = {}, []
            for t, p, r, c in zip(tokens, parents, rows, ctx):
                if not 1 <= len(t) <= 256 or c + len(t) > max_seq or any(not -1 <= q < i for i, q in enumerate(p)):
                    raise moe.GptossError(capi.ERR_BAD_ARG, "tree")
                paths = []
                for i in range(len(t)):
                    paths.append((self.cache[r][:c] if p[i] < 0 else paths[p[i]]) + [int(t[i])])
                self.drafted[int(r)] = list(t)
                out.append(np.array([follows(x) for x in paths], np.int32))
            return out

        def accept(self, rows, ctx, paths):
            for r, c, path in zip(rows, ctx, paths):
                assert list(path) == sorted(set(path))
                self.cache[r] = self.cache[r][:c] + [int(self.drafted[int(r)][i]) for i in path]
            return np.asarray(ctx, np.int32) + np.array([len(p) for p in paths], np.int32)

    return Steps()


def greedy(prompt, n):
    h = list(prompt)
    for _ in range(n):
        h.append(follows(h))
    return h[len(prompt):]


def nothing(history):
    return [], []


def mixed(history):
    """A wrong token, then the right ones behind it."""
    right = greedy(history, 3)
    return [(right[0] + 1) % VOCAB] + right, [-1, -1, 1, 2]


@pytest.mark.parametrize("draft", [nothing, mixed])
@pytest.mark.parametrize("prompts", [[], [[1, 2, 3]], [[5], [6, 7]], [[4] * 9, [3], [2, 1]]])
def test_nothing_to_generate(draft, prompts):
    out = make_model(4, 32).generate_drafted(prompts, 0, draft)
    assert out.shape == (len(prompts), 0) and out.dtype == np.int32


@pytest.mark.parametrize("draft", [nothing, mixed])
def test_no_prompts(draft):
    assert make_model(4, 32).generate_drafted([], 5, draft).shape == (0, 5)


@pytest.mark.parametrize("draft", [nothing, mixed])
@pytest.mark.parametrize("n_prompts", [1, 3, 4, 5, 8, 11])
@pytest.mark.parametrize("max_batch", [1, 4, 40])
@pytest.mark.parametrize("n_new", [1, 7])
def test_any_number_of_prompts(draft, n_prompts, max_batch, n_new):
    """Also more than the model has cache rows: they are taken in turn."""
    prompts = [[(7 * i + j) % VOCAB for j in range(1 + 3 * i % 8)] for i in range(n_prompts)]
    out = make_model(max_batch, 32).generate_drafted(prompts, n_new, draft)
    assert out.dtype == np.int32 and out.tolist() == [greedy(p, n_new) for p in prompts]


def test_up_to_the_end_of_the_cache():
    """The last id is never cached: prompt and answer may be one longer than the cache."""
    for draft in (nothing, mixed):
        out = make_model(8, 12).generate_drafted([[1, 2, 3, 4, 5]], 8, draft)
        assert out.tolist() == [greedy([1, 2, 3, 4, 5], 8)]
