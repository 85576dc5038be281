"""Calls of the serving operators that run at the same time, on streams of their own and in captured graphs, give the bits that they
give one after the other: nothing of one call's scratch is another's."""
import pytest

import test_gpu_serving as one

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def work():
    """Calls that need scratch (shares through memory, sorted adapters, both adapter kernels), shared memory of clusters, or neither."""
    from gptoss_b200 import serving
    long = one.tree_case(serving, [13, 5], [9000, 7000], 8, 1, seed=1)
    short = one.tree_case(serving, [20] * 30, [700] * 30, 8, 1, seed=2)
    few, some, many = (one.lora_case(T, 520, 1000, 16, 7, seed=T) for T in (40, 600, 2000))
    logits = torch.randn(500, 256, generator=one.gen(4), device="cuda")
    apply = lambda c: lambda: serving.lora_apply(**c, out=torch.empty_like(c["y"]))  # noqa: E731
    return [lambda: serving.tree_attention(**long, max_nodes=13, max_ctx=9000), apply(some),
            lambda: serving.tree_attention(**short, max_nodes=20, max_ctx=700), apply(many), apply(few),
            lambda: serving.route_experts(logits, 8, scoring="sigmoid", n_groups=8, topk_groups=4, group_top=2)[0]]


def test_streams():
    from gptoss_b200 import serving
    calls = work()
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got[i].append(c())
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)
    serving.status()


def test_graphs_replayed_at_the_same_time():
    calls = work()
    want = [c() for c in calls]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in calls]
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([c() for _ in range(4)])
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, os in zip(want, outs):
        assert all(torch.equal(o, w) for o in os)


def test_models_with_drafted_steps(tmp_path):
    """Two models whose steps are under way at the same time, a thread each."""
    import threading

    import numpy as np
    from gptoss_b200 import binfmt, model, synth
    cfg = binfmt.config_7m()
    ckpt = tmp_path / "7m.bin"
    binfmt.write_synthetic(str(ckpt), cfg, 5)
    prompts = [synth.uniform_ids(i, 2, 9 + i, cfg.vocab_size).tolist() for i in range(4)]
    draft = lambda history: ([history[-1], 3, 4], [-1, 0, -1])  # noqa: E731
    models = [model.Model(cfg, max_batch=32, max_seq=64) for _ in range(2)]
    for m in models:
        m.load_bin(ckpt)
    want = models[0].generate_drafted(prompts, 20, draft)
    got = [None, None]

    def run(i):
        got[i] = models[i].generate_drafted(prompts, 20, draft)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert np.array_equal(got[0], want) and np.array_equal(got[1], want)
    for m in models:
        m.close()
