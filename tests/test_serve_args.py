"""Argument checks of the serving calls that need no GPU: what the binding
refuses before a pointer reaches the library."""
import ctypes

import numpy as np
import pytest

from zynfer_b200 import cuda as zc

torch = pytest.importorskip("torch")

D = 128


class NoGpu(zc.Gpu):
    """A context that is none: its argument checks alone, and a call that gets past them is an error of the test."""

    def __init__(self):
        self.h, self.device = None, 0
        self._rule = zc.DrawRule()
        self._rule_ref = None

    def _enqueue(self, *call):
        raise AssertionError("a call reached the library")


@pytest.fixture
def model():
    m = object.__new__(zc.Model)
    m.gpu = NoGpu()
    m.arch = zc.Arch(vocab=512, hidden=512, inter=512, layers=1, n_q=4, n_kv=2, max_pos=512)
    return m


BROADCAST = [
    # (tensor, sequences, tokens): rows that are one row in memory, or that overlap
    (torch.zeros(1, 4, D).expand(8, -1, -1), 8, None),
    (torch.zeros(1, 1, 4, D).expand(8, 1, -1, -1), 8, 1),
    (torch.zeros(1, 1, 4, D).expand(1, 8, -1, -1), 1, 8),
    (torch.zeros(1, 1, 4, D).expand(3, 8, -1, -1), 3, 8),
    (torch.zeros(16 * D).as_strided((8, 4, D), (D, D, 1)), 8, None),
    (torch.zeros(16 * D).as_strided((1, 8, 4, D), (8 * D, D, D, 1)), 1, 8),
]


@pytest.mark.parametrize("t,n,tokens", BROADCAST)
def test_rows_that_share_memory_are_refused(model, t, n, tokens):
    with pytest.raises(zc.InvalidArgument):
        model._row_stride(t, n, tokens)


def test_strides_of_rows(model):
    q = torch.zeros(8, 7, D)
    assert model._row_stride(q[:, 2:6], 8) == 7 * D
    assert model._row_stride(q[:1, 2:6], 1) == 4 * D                      # one row: its stride says nothing
    assert model._row_stride(torch.zeros(1, 4, D).expand(1, -1, -1), 1) == 4 * D
    assert model._row_stride(torch.zeros(3, 5, 4, D), 3, 5) == 4 * D
    assert model._row_stride(torch.zeros(3, 5, 6, D)[:, :, 1:5], 3, 5) == 6 * D
    assert model._row_stride(torch.zeros(3, 5, 4, D)[:, 2:3], 3, 1) == 20 * D
    for t, n, tokens in ((torch.zeros(3, 5, 4, D)[:, 1:4], 3, 3),         # a gap between the sequences' tokens
                         (torch.zeros(3, 4, D).transpose(1, 2), 3, None), (torch.zeros(3, 4, 64), 3, None)):
        with pytest.raises(zc.InvalidArgument):
            model._row_stride(t, n, tokens)


def test_tensors_off_the_gpu_are_refused(model, monkeypatch):
    """Host tensors, and with every other argument on the GPU each one alone."""
    monkeypatch.setattr(zc, "lib", lambda: type("Lib", (), {"__getattr__": lambda self, name: name})())
    host = torch.zeros

    class Device:
        """A tensor that says it lies on cuda:`index`."""

        def __init__(self, t, index=0):
            self.t, self.index, self.is_cuda, self.device = t, index, True, f"cuda:{index}"

        def get_device(self):
            return self.index

        def __getattr__(self, name):
            return getattr(self.t, name)

    q = lambda: host(2, 4, D)  # noqa: E731
    kv = lambda: host(2, 5, D)  # noqa: E731
    f, i = lambda: host(2), lambda: host(2, dtype=torch.int32)  # noqa: E731
    calls = [
        (lambda a, b: model.attn_shared(0, [0, 1], a, b), [q, q]),
        (lambda a, b: model.attn_window(0, [0, 1], a, b, window=3), [q, q]),
        (lambda a, b: model.kv_write(0, 0, 0, a, b), [kv, kv]),
        (lambda l, u, ids, lp, t, k, p, m: model.gpu.sample_rows(l, u, ids, lp, t, k, p, m), [lambda: host(2, 64), f, i, f, f, i, f, f]),
    ]
    for call, make in calls:
        with pytest.raises(zc.InvalidArgument, match="cuda:0"):
            call(*(x() for x in make))
        for bad in range(len(make)):
            for wrong in (make[bad](), Device(make[bad](), 1)):
                with pytest.raises(zc.InvalidArgument, match="cuda:0"):
                    call(*(wrong if n == bad else Device(x()) for n, x in enumerate(make)))
        with pytest.raises(AssertionError):
            call(*(Device(x()) for x in make))


class Library:
    """The native library as a list of the calls that reach it."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


PATHS = [
    (lambda m, w, s: m.prefill_chunk(0, [1, 2], window=w, sinks=s), 4),
    (lambda m, w, s: m.decode_drawn([0, 1], [1, 2], [0.1, 0.2], window=w, sinks=s), 4),
]


@pytest.mark.parametrize("call,at", PATHS)
def test_windows_of_the_model_path_do_not_wrap(model, monkeypatch, call, at):
    lib = Library()
    monkeypatch.setattr(zc, "lib", lambda: lib)
    for window, sinks in ((-1, 0), (5, -1), (-2 ** 32, 3)):
        with pytest.raises(zc.InvalidArgument):
            call(model, window, sinks)
    assert not lib.calls
    for window, sinks, want in ((0, 0, (0, 0)), (7, 3, (7, 3)), (zc.WINDOW_ALL, 0, (zc.WINDOW_ALL, 0)),
                                (2 ** 32, 2 ** 40, (zc.WINDOW_ALL, zc.WINDOW_ALL)), (2 ** 32 + 10, 1, (zc.WINDOW_ALL, 1))):
        call(model, window, sinks)
        assert lib.calls[-1][1][at:at + 2] == want


def test_indexes_do_not_wrap(model, monkeypatch):
    """2^32 is no slot, layer, position or token, nor is -1: as a Python number or in an array of wider numbers."""
    lib = Library()
    monkeypatch.setattr(zc, "lib", lambda: lib)
    kv, q = torch.zeros(2, 5, D), torch.zeros(1, 4, D)
    for x in (2 ** 32, -1, 2 ** 32 + 3, -2 ** 32):
        wide = np.array([x])
        for call in (lambda: model.kv_write(x, 0, 0, kv, kv), lambda: model.kv_write(0, x, 0, kv, kv), lambda: model.kv_write(0, 0, x, kv, kv),
                     lambda: model.attn_shared(x, [0], q, q), lambda: model.attn_shared(0, [x], q, q), lambda: model.attn_shared(0, wide, q, q),
                     lambda: model.attn_window(x, [0], q, q), lambda: model.attn_window(0, wide, q, q),
                     lambda: model.prefill_chunk(x, [1]), lambda: model.prefill_chunk(0, wide), lambda: model.prefill_chunk(0, [x]),
                     lambda: model.decode_drawn(wide, [1], [0.5]), lambda: model.decode_drawn([0], wide, [0.5]),
                     lambda: model.decode_drawn([0.5], [1], [0.5])):
            with pytest.raises(zc.InvalidArgument, match="index|whole numbers|sequence id"):
                call()
    assert not lib.calls


def test_top_k_beyond_32_bits_keeps_every_token(model, monkeypatch):
    lib = Library()
    seen = []
    lib.zynfer_cu_decode_drawn = lambda *a: seen.append(list((ctypes.c_int32 * 4).from_address(a[7]._obj.top_k))) or 0
    monkeypatch.setattr(zc, "lib", lambda: lib)
    model.decode_drawn([0, 1, 2, 3], [1, 2, 3, 4], [0.5] * 4, top_k=np.array([2 ** 32 + 5, -2 ** 40, 7, 2 ** 31]))
    assert seen == [[2 ** 31 - 1, 0, 7, 2 ** 31 - 1]]
    model.decode_drawn([0, 1, 2, 3], [1, 2, 3, 4], [0.5] * 4, top_k=3)
    assert seen[-1] == [3] * 4
