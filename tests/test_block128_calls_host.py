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


def test_runner_reads_the_blocks_that_a_sequence_fills(libb2q):
    """Block tables come padded: what stands behind the blocks in use is neither refused nor uploaded."""
    from oxicuda_b200 import _lib
    from oxicuda_b200.model_runner import LlamaConfig, QuantizedLlamaRunner
    runner = object.__new__(QuantizedLlamaRunner)
    runner.cfg, runner.dev = LlamaConfig(recipe="block128", block_size=16, num_blocks=64), "cpu"
    lens, tables, starts = runner._cache_batch([(0, 1, 15, [3, -1, -1, -1]), (1, 2, 16, [5, 63, 64, 1 << 40])])
    assert lens.tolist() == [16, 17] and tables.tolist() == [[3, -1], [5, 63]] and starts is None
    lens, tables, starts = runner._cache_batch([(0, 40, 0, (7, 8, 9, -1)), (40, 41, 0, [1])])
    assert lens.tolist() == [40, 1] and tables.tolist() == [[7, 8, 9], [1, -1, -1]] and starts.tolist() == [0, 40, 41]
    with pytest.raises(_lib.InvalidArgument):
        runner._cache_batch([(0, 1, 16, [3, -1])])
    with pytest.raises(_lib.InvalidArgument):
        runner._cache_batch([(0, 1, 16, [3, 64])])
    with pytest.raises(_lib.DimensionMismatch):
        runner._cache_batch([(0, 1, 16, [3])])


def test_a_handle_knows_the_stream_that_was_set_by_its_entry_point(libb2q, monkeypatch):
    """default_handle() sets a handle's stream only where it is another one than the handle launches on: a stream set through call() counts."""
    import ctypes as C
    from oxicuda_b200 import _lib

    class Library:
        def __init__(self):
            self.streams, self.static = [], None

        def b2q_set_stream(self, h, stream):
            self.streams.append(getattr(stream, "value", stream) or 0)
            return 0

        def b2q_set_static_weights(self, h, on):
            self.static = bool(on)
            return 0

    lib = Library()
    h = object.__new__(_lib.Handle)
    h._h, h._stream, h.static_weights, h.device = None, 0, True, 0
    monkeypatch.setattr(_lib, "_lib", lib)
    monkeypatch.setattr(_lib, "_default", {0: h})
    now = [0x10]
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: now[0], raising=False)
    assert _lib.default_handle(0) is h and lib.streams == [0x10]
    _lib.default_handle(0)
    assert lib.streams == [0x10]
    for other in (C.c_void_p(0x20), 0x30, None):
        h.call("b2q_set_stream", other)
        _lib.default_handle(0)
        assert lib.streams[-1] == 0x10
    now[0] = 0
    h.call("b2q_set_stream", None)
    _lib.default_handle(0)
    assert lib.streams[-1] == 0
    h.call("b2q_set_static_weights", 0)
    assert not h.static_weights and lib.static is False


def test_a_width_that_the_cache_does_not_have_is_refused(libb2q):
    from oxicuda_b200 import _lib
    from oxicuda_b200.model_runner import LlamaConfig
    LlamaConfig(kv_bits=4).validate()
    LlamaConfig(recipe="block128", kv_bits=8).validate()
    for bits in (2, 4, 16):
        with pytest.raises(_lib.InvalidConfig):
            LlamaConfig(recipe="block128", kv_bits=bits).validate()
