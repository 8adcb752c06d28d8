"""CPU: what the block-128 wrappers ask of their handle, seen by a handle that records its calls."""
import pytest
import torch


class Recorder:
    def __init__(self, static=True, fail=False):
        self.static_weights, self.fail, self.seen = static, fail, []

    def set_static_weights(self, on):
        self.static_weights = on
        self.seen.append(("static", on))

    def call(self, name, *args):
        self.seen.append((name, self.static_weights))
        if self.fail:
            raise RuntimeError("refused")


@pytest.fixture
def recorded(libb2q, monkeypatch):
    from oxicuda_b200 import _lib, blas
    monkeypatch.setattr(_lib, "require_cuda", lambda *a, **k: None)

    def use(handle):
        monkeypatch.setattr(blas, "default_handle", lambda *a: handle)
        return handle
    return use


def _operands(strided):
    f = torch.float32
    w = torch.zeros(256, 130, dtype=torch.uint8).t() if strided == "transposed" else torch.zeros(130, 512, dtype=torch.uint8)[:, 128:384]
    if not strided:
        w = w.contiguous()
    return torch.zeros(4, 256, dtype=torch.uint8), w, torch.zeros(4, 2, dtype=f), torch.zeros(2, 2, dtype=f)


@pytest.mark.parametrize("strided", ["transposed", "columns"])
def test_copied_weights_are_not_fetched_ahead_of_their_copy(recorded, strided):
    """The copy of a strided weight is the kernel right before the product: the product must not fetch weights before it has ended."""
    from oxicuda_b200 import blas
    h = recorded(Recorder())
    blas.gemm_fp8_block128(*_operands(strided))
    assert h.seen == [("static", False), ("b2q_gemm_fp8_block128", False), ("static", True)]
    h = recorded(Recorder(static=False))                            # off already: stays off
    blas.gemm_fp8_block128(*_operands(strided))
    assert h.seen == [("b2q_gemm_fp8_block128", False)] and not h.static_weights
    h = recorded(Recorder(fail=True))
    with pytest.raises(RuntimeError):
        blas.gemm_fp8_block128(*_operands(strided))
    assert h.static_weights


def test_contiguous_weights_stay_static(recorded):
    from oxicuda_b200 import blas
    h = recorded(Recorder())
    blas.gemm_fp8_block128(*_operands(None))
    assert h.seen == [("b2q_gemm_fp8_block128", True)]
