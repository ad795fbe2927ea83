"""Argument checks of the serving calls that need no GPU: what the binding
refuses before a pointer reaches the library."""
import pytest

from zynfer_b200 import cuda as zc

torch = pytest.importorskip("torch")

D = 128


@pytest.fixture
def model():
    """A model without a context: its argument checks alone."""
    m = object.__new__(zc.Model)
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
