"""Groups of experts whose worth is the sum of infinities of both signs."""
import math

import pytest

import serving_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def definition(logits, bias, k, scoring, groups, kept):
    """Ids, token by token: the best `kept` groups by the sum of their two largest choices, NaN counting as -infinity."""
    x = logits.double().cpu()
    choice = (torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)) + bias.double().cpu()
    size, ids = x.shape[1] // groups, []
    for row in choice.tolist():
        worth = []
        for g in range(groups):
            best = sorted(row[g * size:(g + 1) * size], reverse=True)[:2]
            worth.append(-math.inf if math.isnan(sum(best)) else sum(best))
        keep = sorted(range(groups), key=lambda g: (-worth[g], g))[:kept]
        ids.append(sorted((e for e in range(len(row)) if e // size in keep), key=lambda e: (-row[e], e))[:k])
    return torch.tensor(ids, dtype=torch.int32)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("kept", [1, 2, 3, 4])
@pytest.mark.parametrize("groups,size", [(4, 2), (8, 4), (32, 8), (5, 3)])
def test_a_group_with_infinities_of_both_signs_counts_as_the_least(scoring, kept, groups, size):
    """A bias that forces one expert of a group and shuts out the others: the group's worth is inf - inf.  As many groups take part
    as are asked for, never one more."""
    from gptoss_b200 import serving
    E = groups * size
    logits = torch.randn(50, E, generator=torch.Generator(device="cuda").manual_seed(E + kept), device="cuda")
    for forced in range(groups):
        bias = torch.zeros(E, device="cuda")
        bias[forced * size:(forced + 1) * size] = -math.inf
        bias[forced * size] = math.inf
        for also_shut in (False, True):
            if also_shut:
                bias[(forced + 1) % groups * size:((forced + 1) % groups + 1) * size] = -math.inf
            k = min(8, kept * size)
            w, i = serving.route_experts(logits, k, scoring=scoring, bias=bias, n_groups=groups, topk_groups=kept, group_top=2)
            want = definition(logits, bias, k, scoring, groups, kept)
            assert torch.equal(i.cpu(), want)
            assert all(len(set((row // size).tolist())) <= kept for row in i.cpu())
            scores = ref.route(logits, E, scoring=scoring, renormalize=False) if E == 8 else None
            if scores is not None:
                full = torch.zeros(50, E, dtype=torch.float64).scatter_(1, scores[1].long(), scores[0])
                ww = torch.gather(full, 1, want.long())
                torch.testing.assert_close(w.cpu().double(), ww / ww.sum(1, keepdim=True), rtol=2.0 ** -19, atol=0)
