"""What the worst-case bounds of serving_reference.lora are too wide to see: that the adapters' intermediate keeps the bits of fp32,
and how large the error is on the whole."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROUTES = [1, 16, 40, 200, 512, 600, 767, 768, 1500, 4100]  # tokens: a vote, tiles found by the CTAs, sorted, two kernels


@pytest.fixture(scope="module")
def serving():
    from gptoss_b200 import serving
    return serving


def definition(x, a, b, ids, y, scale):
    out = y.double()
    for i in range(a.shape[0]):
        who = (ids == i).nonzero()[:, 0]
        out[who] += float(scale[i]) * ((x[who].double() @ a[i].double().t()) @ b[i].double().t())
    return out


@pytest.mark.parametrize("T", ROUTES)
@pytest.mark.parametrize("rank", [8, 16, 32, 64, 128])
def test_whole_numbers_are_exact(serving, T, rank):
    """Whole numbers whose sums stay below 2^24 have exact results in fp32, in any order; the intermediate needs up to 22 bits, so
    one that is rounded to one or two bf16 terms (8 or 16 bits) would not give them."""
    g = torch.Generator(device="cuda").manual_seed(T * 1000 + rank)
    K, n_out, n = 2880, 264, 3
    whole = lambda top, *s: torch.randint(-top, top + 1, s, generator=g, device="cuda")  # noqa: E731
    x, a = whole(120, T, K), whole(120, n, rank, K)
    b = whole(1, n, n_out, rank) * (torch.rand(n, n_out, rank, generator=g, device="cuda") < 6 / rank)
    ids, y = whole(1, T) + 1, whole(1000, T, n_out)
    scale = torch.tensor([1.0, 2.0, 0.5], device="cuda")
    u = (x.double() @ a.double().view(n * rank, K).t()).abs()
    most = x.double().abs() @ a.double().abs().view(n * rank, K).t()
    assert float(most.max()) < 2 ** 24 and float((u.max() * 2 * b.abs().sum(2).max())) < 2 ** 27  # what is added up, and up to 3 bits more
    assert (u % 32 != 0).any() and float(u.max()) > 2 ** 18
    want = definition(x, a, b, ids, y, scale)
    assert float(want.abs().max()) < 2 ** 23  # halves are exact too
    got = serving.lora_apply(x.bfloat16(), a.bfloat16(), b.bfloat16(), ids.int(), y.float(), scale=scale, out=torch.empty(T, n_out, device="cuda"))
    assert torch.equal(got.double(), want)


# The 2-norm of the error over that of the result.  The tensor core's sums cut off what falls below their last bit: four steps of
# 16 products per sum of 64, at most 2^-23 each, half of it on average and less for the first ones: 1e-7 of the sum.  Adding those
# sums up: each addition is off by up to 2^-24 of a partial sum, 2^-25.8 on average, with either sign; n of them, whose partial sums
# grow like a random walk's: 2^-25.8 sqrt(n / 2).  An adapter's K is cut into two parts at least, so n is up to K / 128: 128 at
# K = 16384, 1.4e-7; 512 at K = 65536, 2.8e-7.  Together 1.7e-7 at 16384, and nearly the same again for the second product's few steps.
def error_of(K):
    return 3e-7 - 1.4e-7 + 1.4e-7 * max(1.0, (K / 16384) ** 0.5)


@pytest.mark.parametrize("T", ROUTES)
@pytest.mark.parametrize("K,rank", [(256, 16), (2880, 64), (4096, 32), (16384, 16), (16384, 128), (65536, 8)])
def test_the_error_on_the_whole(serving, T, K, rank):
    g = torch.Generator(device="cuda").manual_seed(T + K + rank)
    n, n_out = 2, 520
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, a, b = r(T, K).bfloat16(), (r(n, rank, K) * K ** -0.5).bfloat16(), r(n, n_out, rank).bfloat16()
    ids = torch.arange(T, device="cuda").int() % n
    y, scale = torch.zeros(T, n_out, device="cuda"), torch.tensor([1.5, 0.7], device="cuda")
    want = definition(x, a, b, ids, y, scale)
    got = serving.lora_apply(x, a, b, ids, y, scale=scale)
    error = float((got.double() - want).norm() / want.norm())
    print(f"T={T} K={K} rank={rank}: {error:.2e}")
    assert error <= error_of(K)
