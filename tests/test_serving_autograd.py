"""The serving operators and autograd: what asks for a gradient is refused, what is written in place is known to be written."""
import pytest

from gptoss_b200 import capi

torch = pytest.importorskip("torch")


def calls(device):
    """(name, call, the tensors it takes by name) of each operator, on small inputs."""
    from gptoss_b200 import serving
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    f = lambda *s: torch.linspace(-1, 1, torch.Size(s).numel(), device=device).view(s)  # noqa: E731
    tree = dict(q=f(3, 4, 64).bfloat16(), k_cache=f(2, 2, 16, 64).bfloat16(), v_cache=f(2, 2, 16, 64).bfloat16(), offsets=ints([0, 2, 3]),
                ctx_len=ints([5, 7]), mask=ints([[1], [3], [1]]), sinks=f(4), out=torch.zeros(3, 4, 64, device=device).bfloat16())
    commit = dict(k_cache=f(2, 2, 2, 16, 64).bfloat16(), v_cache=f(2, 2, 2, 16, 64).bfloat16(), ctx_len=ints([5, 7]), offsets=ints([0, 1, 2]),
                  path=ints([1, 2]))
    lora = dict(x=f(3, 16).bfloat16(), a=f(2, 8, 16).bfloat16(), b=f(2, 24, 8).bfloat16(), ids=ints([0, 1, -1]), y=f(3, 24), scale=f(2))
    route = dict(logits=f(3, 16), bias=f(16))
    return [("tree_attention", lambda **t: serving.tree_attention(**t, max_nodes=2, max_ctx=7), tree),
            ("cache_commit", lambda **t: serving.cache_commit(**t, max_path=1), commit),
            ("lora_apply", lambda **t: serving.lora_apply(**t), lora),
            ("route_experts", lambda **t: serving.route_experts(**t, top_k=2), route)]


FLOATING = [("tree_attention", n) for n in ("q", "k_cache", "v_cache", "sinks", "out")] + \
           [("cache_commit", n) for n in ("k_cache", "v_cache")] + \
           [("lora_apply", n) for n in ("x", "a", "b", "y", "scale")] + [("route_experts", n) for n in ("logits", "bias")]


def refuses(device, op, name):
    from gptoss_b200 import moe
    call, tensors = next((c, t) for n, c, t in calls(device) if n == op)
    with pytest.raises(moe.GptossError) as e:
        call(**{**tensors, name: tensors[name].clone().requires_grad_()})
    assert e.value.code == capi.ERR_BAD_ARG and "gradient" in str(e.value)


@pytest.mark.parametrize("op,name", [("tree_attention", "q"), ("cache_commit", "k_cache"), ("lora_apply", "x"), ("route_experts", "logits")])
def test_what_requires_a_gradient_is_refused_before_anything_else(op, name):
    if capi.needs_build():
        capi.build()
    refuses("cpu", op, name)


@pytest.mark.gpu
@pytest.mark.parametrize("op,name", FLOATING)
def test_what_requires_a_gradient_is_refused(op, name):
    refuses("cuda", op, name)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["tree_attention", "cache_commit", "lora_apply", "route_experts"])
def test_without_recording_everything_passes(op):
    call, tensors = next((c, t) for n, c, t in calls("cuda") if n == op)
    plain = call(**{k: t.clone() for k, t in tensors.items()})
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            got = call(**{k: t.clone().requires_grad_() if t.is_floating_point() else t.clone() for k, t in tensors.items()})
        for g, p in zip(*[r if isinstance(r, tuple) else (r,) for r in (got, plain)]):
            assert g is p or torch.equal(g, p)


@pytest.mark.gpu
@pytest.mark.parametrize("op,names", [("tree_attention", ("out",)), ("cache_commit", ("k_cache", "v_cache")), ("lora_apply", ("y",))])
def test_what_a_call_writes_counts_its_version_up(op, names):
    """A graph that saved such a tensor before the call refuses to run backward; the other tensors keep their versions."""
    call, tensors = next((c, t) for n, c, t in calls("cuda") if n == op)
    for name in names:
        w = torch.ones_like(tensors[name], requires_grad=True)
        loss = (w * tensors[name]).sum()  # saves the tensor
        before = {k: t._version for k, t in tensors.items()}
        call(**tensors)
        for k, t in tensors.items():
            assert t._version > before[k] if k in names else t._version == before[k], k
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        call(**{k: t.clone() for k, t in tensors.items()})  # inference tensors have no version


@pytest.mark.gpu
def test_a_refused_call_writes_nothing():
    from gptoss_b200 import moe
    call, tensors = next((c, t) for n, c, t in calls("cuda") if n == "lora_apply")
    before = tensors["y"]._version
    with pytest.raises(moe.GptossError):
        call(**{**tensors, "ids": tensors["ids"].long()})
    assert tensors["y"]._version == before
