"""Rows that lie beyond 2^31 elements from the first: x, y and out of the adapters, queries and outputs of the tree attention."""
import pytest

import serving_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def spread(rows, columns, stride, dtype):
    """[rows, columns] with that row stride, over memory that is mostly not touched."""
    return torch.empty((rows - 1) * stride + columns, dtype=dtype, device="cuda").as_strided((rows, columns), (stride, 1))


@pytest.mark.parametrize("T", [20, 300, 600, 1000])
def test_adapters(T):
    from gptoss_b200 import serving
    g = torch.Generator(device="cuda").manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    K, n_out, rank, n = 200, 264, 16, 3
    stride = (2 ** 31 // (T - 1) // 8 + 64) * 8  # the last row starts behind element 2^31
    assert (T - 1) * stride > 2 ** 31
    x, y, out = (spread(T, c, stride, t) for c, t in ((K, torch.bfloat16), (n_out, torch.float32), (n_out, torch.float32)))
    x.copy_(r(T, K)), y.copy_(r(T, n_out)), out.fill_(float("nan"))
    c = dict(x=x, a=(r(n, rank, K) * K ** -0.5).bfloat16(), b=r(n, n_out, rank).bfloat16(), y=y, scale=r(n),
             ids=(torch.arange(T, device="cuda") % (n + 1) - 1).int())
    want, bound = ref.lora(**{**c, "x": x.contiguous(), "y": y.contiguous()})
    serving.lora_apply(**c, out=out)
    assert float(((out.double() - want).abs() - bound).max()) <= 0
    serving.lora_apply(**c)  # in place
    assert torch.equal(y, out)


@pytest.mark.parametrize("n_seqs", [1, 40])
def test_tree_attention(n_seqs):
    import numpy as np
    from gptoss_b200 import serving
    g = torch.Generator(device="cuda").manual_seed(n_seqs)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    nodes, nq, nkv, hd = 240 if n_seqs == 1 else 6, 8, 2, 64
    T = nodes * n_seqs
    stride = (2 ** 31 // (T - 1) // 8 + 64) * 8
    q, out = (spread(T, nq * hd, stride, torch.bfloat16).unflatten(1, (nq, hd)) for _ in range(2))
    q.copy_(r(T, nq, hd))
    off, mask, depth = serving.tree_masks([list(range(-1, nodes - 1))] * n_seqs)
    i = lambda v: torch.from_numpy(np.ascontiguousarray(v)).int().cuda()  # noqa: E731
    c = dict(q=q, k_cache=r(n_seqs, nkv, 900, hd).bfloat16(), v_cache=r(n_seqs, nkv, 900, hd).bfloat16(), offsets=i(off),
             ctx_len=i([600 + b for b in range(n_seqs)]), mask=i(mask), depth=i(depth), sinks=r(nq))
    serving.tree_attention(**c, max_nodes=nodes, max_ctx=640, out=out)
    want, bound = ref.tree_attention(**{**c, "q": q.contiguous()})
    assert float(((out.double() - want).abs() - bound).max()) <= 0


def test_expert_choice():
    from gptoss_b200 import serving
    g = torch.Generator(device="cuda").manual_seed(3)
    T, E = 600, 64
    stride = 2 ** 31 // (T - 1) + 64
    logits = spread(T, E, stride, torch.float32)
    logits.copy_(torch.randn(T, E, generator=g, device="cuda"))
    w, i = serving.route_experts(logits, 4, n_groups=4, topk_groups=2)
    w2, i2 = serving.route_experts(logits.contiguous(), 4, n_groups=4, topk_groups=2)
    assert torch.equal(i, i2) and torch.equal(w, w2)
    assert torch.equal(i.cpu(), ref.route(logits.contiguous(), 4, n_groups=4, topk_groups=2)[1])
