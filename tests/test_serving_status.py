"""A bounded wait that gave up on the GPU reaches the caller of the Python layer."""
import pytest

from gptoss_b200 import capi

torch = pytest.importorskip("torch")


class FakeLibrary:
    """The two C functions that ``serving.status`` needs, on a device that reports ``codes`` one after the other."""

    def __init__(self, codes):
        self.codes = list(codes)

    def gptoss_serving_status(self):
        return self.codes.pop(0)

    def gptoss_serving_last_error(self):
        return b"device-side bounded wait gave up"


def test_status_raises_what_the_device_noted(monkeypatch):
    from gptoss_b200 import moe, serving
    lib = FakeLibrary([capi.OK, capi.ERR_TIMEOUT, capi.OK])
    monkeypatch.setattr(capi, "load", lambda: lib)
    serving.status()
    with pytest.raises(moe.GptossError) as e:
        serving.status()
    assert e.value.code == capi.ERR_TIMEOUT and "gave up" in str(e.value)
    serving.status()


@pytest.mark.gpu
def test_status_of_calls_that_ran_well():
    from gptoss_b200 import serving
    w, i = serving.route_experts(torch.randn(3, 16, device="cuda"), 2)
    serving.status()
    serving.status(0)
    serving.status(w.device)
