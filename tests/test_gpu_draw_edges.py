"""zynfer_cu_sample_rows (B200 only) at the ends of its parameters: rows whose
exponents span next to nothing. Where every exponential is 1, every weight is
2^33 and the drawn token is exactly the floor(u n)-th of the n kept ones, in
descending order of the logits."""
import numpy as np
import pytest

from test_gpu_draw import check_row, draw
from zynfer_b200 import cuda as zc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

MAX = float(np.finfo(np.float32).max)


@pytest.fixture(scope="module")
def gpu():
    g = zc.Gpu(0)
    yield g
    g.close()


def equal_weights(gpu, logits, t):
    rows, vocab = logits.shape
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices.cpu().numpy()
    for k, p in ((0, 1.0), (min(vocab, 5000), 0.25)):
        kept = vocab if not k else -(-k // 4)
        ids, lp = draw(gpu, logits, u, t=t, k=k, p=p)
        at = (u.astype(np.float64) * kept).astype(np.int64)
        assert np.array_equal(ids, order[np.arange(rows), at]), (t, k)
        assert np.allclose(lp, -np.log(kept), atol=1e-5)


# rows by vocabulary: one CTA a row, clusters of 16, 8, 4 and 2, one CTA that reads its row again
SHAPES = [(3, 700), (2, 151936), (30, 40000), (60, 40000), (130, 20000), (300, 20000)]


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("t", [1e30, 3e36, 1e37, 1e38, MAX])
def test_very_large_temperatures_draw_evenly(gpu, rows, vocab, t):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    equal_weights(gpu, 20.0 * torch.rand(rows, vocab, generator=g, device="cuda"), t)


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("step", [1e-45, 1e-38, -1e-38, 5e-36])
def test_logits_next_to_equal(gpu, rows, vocab, step):
    l = torch.zeros(rows, vocab, device="cuda")
    l[:, vocab // 3] = step
    equal_weights(gpu, l, 1.0)


@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_logits_whole_denormals_apart(gpu, rows, vocab):
    """The bins are a few times the smallest number wide: no token falls between them. The weights are all one."""
    l = -torch.arange(vocab, device="cuda", dtype=torch.float64)[None].repeat(rows, 1) * 2.0 ** -149
    equal_weights(gpu, l.float(), 1e-26)


@pytest.mark.parametrize("t", [4e-39, 1e-42])
def test_very_small_temperatures(gpu, t):
    """Differences of 1e-40 at temperatures near them (1e-42 counts as 2^-128)."""
    vocab, u = 1000, np.linspace(0.02, 0.98, 12).astype(np.float32)
    x = (-1e-40 * torch.arange(vocab, dtype=torch.float64)).float().cuda()[None].repeat(12, 1)
    for k, p in ((0, 1.0), (0, 0.7), (40, 1.0), (40, 0.7)):
        ids, lp = draw(gpu, x, u, t=t, k=k, p=p)
        for r in range(12):
            check_row(x[r], float(u[r]), max(float(np.float32(t)), 1.0 / MAX), k, float(np.float32(p)), 0.0, int(ids[r]), float(lp[r]))
