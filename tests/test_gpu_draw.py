"""zynfer_cu_sample_rows (B200 only) against its definition in 64 bits.

A weight is rint(exp((l - m) / T) 2^33) with the exponent in f32: two
roundings and 1 / T's of an exponent of at most 23 nats, and expf's 2 ulp, are
at most 23 * 3 * 2^-24 + 2^-22 < 5e-6 of a weight, and the rounding to whole
numbers 2^-34. So with running sums C_i in 64 bits, the token drawn at u
satisfies C_before - tol <= u S <= C_with + tol for tol = 5e-6 S + n 2^-34, and
it belongs to the kept run up to the same. Where all weights are equal or
powers of two the token is exact.
"""
import numpy as np
import pytest

from zynfer_b200 import cuda as zc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def gpu():
    g = zc.Gpu(0)
    yield g
    g.close()


def dev(x, dtype=torch.float32):
    return torch.as_tensor(np.asarray(x), dtype=dtype).cuda()


def draw(gpu, logits, u, t=None, k=None, p=None, mp=None):
    rows = logits.shape[0]
    full = lambda x, dt: None if x is None else dev(np.broadcast_to(np.asarray(x), (rows,)).copy(), dt)  # noqa: E731
    ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    lp = torch.full((rows,), float("nan"), device="cuda")
    torch.cuda.synchronize()
    gpu.sample_rows(logits, full(u, torch.float32), ids, logprobs=lp, temperature=full(t, torch.float32),
                    top_k=full(k, torch.int32), top_p=full(p, torch.float32), min_p=full(mp, torch.float32))
    gpu.sync()
    return ids.cpu().numpy(), lp.cpu().numpy()


def check_row(l, u, t, k, p, mp, got, lp):
    l = l.double().cpu().numpy()
    l = np.where(np.isnan(l), -np.inf, l)
    order = np.lexsort((np.arange(l.size), -l))
    if not t > 0:
        assert got == order[0] and lp == 0.0
        return
    with np.errstate(invalid="ignore"):
        x = np.where(l[order] == l[order[0]], 0.0, (l[order] - l[order[0]]) / t)
    e = np.exp(x)
    e = np.where(e >= mp * (1 + 5e-6), e, np.where(e >= mp * (1 - 5e-6), e, 0.0))
    e[np.isneginf(l[order])] = 0.0
    if k > 0:
        e[k:] = 0.0
    c = np.cumsum(e)
    tol = 5e-6 * c[-1] + l.size * 2.0 ** -34
    kept = (c - e < p * c[-1] + tol) & (e > 0)
    sure = (c - e < p * c[-1] - tol) & (e > 0)
    kept[0] = sure[0] = True
    at = int(np.nonzero(order == got)[0][0])
    assert kept[at], (got, at)
    lo, hi = c[sure].max(), c[kept].max()
    assert c[at] - e[at] - tol <= u * hi and u * lo <= c[at] + tol, (u, c[at] - e[at], c[at], lo, hi)
    assert x[at] - np.log(hi) - 2e-5 - 1e-6 * abs(x[at]) <= lp <= x[at] - np.log(lo) + 2e-5 + 1e-6 * abs(x[at])


RULES = [(1.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (1.0, 50, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.3, 0, 0.9, 0.0),
         (0.8, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.1), (0.9, 1000, 0.5, 0.02), (0.0, 5, 0.5, 0.5), (30.0, 0, 0.99, 0.0),
         (0.01, 0, 0.9, 0.0), (1.0, 100000, 1.0, 1.0), (5.0, 0, 0.0, 0.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4099, 32003, 151936, 262144])
def test_draw_follows_the_definition(gpu, vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    rows = 2 * len(RULES)
    wide = torch.full((rows, vocab + 3), float("nan"))
    logits = 3.0 * torch.randn(rows, vocab, generator=g)
    logits[::2, ::5] = float("-inf")
    if vocab > 1:
        logits[1::2, 0] = float("nan")
    logits[:, vocab // 2] = 2.0  # every row keeps something
    wide[:, :vocab] = logits
    x = wide.to(dtype).cuda()[:, :vocab]
    u = torch.rand(rows, generator=g).numpy().astype(np.float32)
    u[0], u[1] = 0.0, np.float32(1 - 2.0 ** -24)
    t, k, p, mp = (np.array([RULES[i % len(RULES)][j] for i in range(rows)]) for j in range(4))
    ids, lp = draw(gpu, x, u, t.astype(np.float32), k.astype(np.int32), p.astype(np.float32), mp.astype(np.float32))
    for r in range(rows):
        check_row(x[r], float(u[r]), float(np.float32(t[r])), int(k[r]), float(np.float32(p[r])), float(np.float32(mp[r])),
                  int(ids[r]), float(lp[r]))
    again, _ = draw(gpu, x, u, t.astype(np.float32), k.astype(np.int32), p.astype(np.float32), mp.astype(np.float32))
    assert np.array_equal(ids, again)


@pytest.mark.parametrize("vocab", [7, 5000, 151936])
@pytest.mark.parametrize("value", [0.0, -3.5, 1e4, float("inf")])
def test_equal_logits_are_drawn_by_index(gpu, vocab, value):
    n = 64
    l = torch.full((n, vocab), value, device="cuda")
    l[:, 1::2] = float("-inf")
    live = np.arange(0, vocab, 2)
    u = (np.arange(n) / n).astype(np.float32)
    ids, lp = draw(gpu, l, u)
    assert np.array_equal(ids, live[(u.astype(np.float64) * live.size).astype(np.int64)])
    assert np.allclose(lp, -np.log(live.size), atol=1e-5)
    ids, _ = draw(gpu, l, u, k=3)  # ties at the cut: the lowest indexes stay
    assert np.array_equal(ids, live[(u.astype(np.float64) * 3).astype(np.int64)])
    ids, _ = draw(gpu, l, u, p=0.5)
    kept = -(-live.size // 2)
    assert np.array_equal(ids, live[(u.astype(np.float64) * kept).astype(np.int64)])


def test_powers_of_two_are_exact(gpu):
    """Logits 0, 0, -inf and a middle token of weight 1/2: the drawn token changes exactly at the sums' edges."""
    l = torch.full((1, 300), float("-inf"), device="cuda")
    l[0, 10] = l[0, 200] = 0.0
    edges = [(0.0, 10), (0.5 - 2.0 ** -25, 10), (0.5, 200), (1 - 2.0 ** -24, 200)]
    for u, want in edges:
        assert draw(gpu, l, [u])[0][0] == want
    # signed zeros are one logit: the lower index first
    l[0, 10] = -0.0
    for u, want in edges:
        assert draw(gpu, l, [u])[0][0] == want
    assert draw(gpu, l, [0.9], k=1)[0][0] == 10


def test_rows_without_weight_and_odd_parameters(gpu):
    l = torch.full((5, 700), float("-inf"), device="cuda")
    l[1] = float("nan")
    l[2, 600] = float("inf")
    l[3, 5], l[3, 6] = -1e30, float("nan")
    l[4, 9], l[4, 8] = 1.0, 0.5
    ids, lp = draw(gpu, l, [0.3] * 5)
    assert ids.tolist()[:4] == [0, 0, 600, 5] and ids[4] in (8, 9)
    assert lp[0] == lp[1] == -np.inf and lp[2] == lp[3] == 0.0
    nan = float("nan")
    # NaN and out-of-range parameters take their documented meaning
    assert draw(gpu, l[4:], [0.99], t=[nan])[0][0] == 9                # the largest
    assert draw(gpu, l[4:], [0.99], t=[-1.0])[0][0] == 9
    assert draw(gpu, l[4:], [0.99], p=[-1.0])[0][0] == 9               # the first
    assert draw(gpu, l[4:], [0.99], mp=[2.0])[0][0] == 9               # at most 1
    assert draw(gpu, l[4:], [0.99], k=[-3], p=[nan], mp=[nan])[0][0] == 8  # off
    assert draw(gpu, l[4:], [7.0])[0][0] == 8 and draw(gpu, l[4:], [-1.0])[0][0] == 9 and draw(gpu, l[4:], [nan])[0][0] == 9
    assert draw(gpu, l[4:], [0.99], t=[1e-42])[0][0] == 9              # 1 / T overflows
    assert draw(gpu, l[4:], [0.99], t=[float("inf")])[0][0] == 8       # all alike, in descending order of the logits


def test_large_sums_and_clustered_logits(gpu):
    """Logits a few f32 steps apart share every leading bit."""
    v = 20000
    base = torch.full((2, v), 17.25)
    base += torch.arange(v)[None] * 2.0 ** -19
    x = base.cuda()
    u = np.array([0.123, 0.77], np.float32)
    ids, lp = draw(gpu, x, u, k=[0, 5000], p=[1.0, 0.6])
    for r, (k, p) in enumerate([(0, 1.0), (5000, 0.6)]):
        check_row(x[r], float(u[r]), 1.0, k, float(np.float32(p)), 0.0, int(ids[r]), float(lp[r]))


def test_refusals(gpu):
    l = torch.zeros(2, 64, device="cuda")
    u, ids = torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (
        lambda: gpu.sample_rows(l, u[:1], ids),
        lambda: gpu.sample_rows(l, u, ids.long()),
        lambda: gpu.sample_rows(l[0], u, ids),
        lambda: gpu.sample_rows(l[:, ::2], u, ids),
        lambda: gpu.sample_rows(l, u, ids, top_k=u),
        lambda: gpu.sample_rows(l[:0], u[:0], ids[:0]),
        lambda: gpu.sample_rows(l[:, :0], u, ids),
    ):
        with pytest.raises(zc.InvalidArgument):
            call()
    with pytest.raises(zc.Unsupported):
        gpu.sample_rows(l.half(), u, ids)
    with pytest.raises(zc.Unsupported):
        gpu.sample_rows(torch.zeros(2, 262145, device="cuda"), u, ids)
    gpu.set_fail_at("launch")
    with pytest.raises(zc.LaunchFailed):
        gpu.sample_rows(l, u, ids)
    gpu.sample_rows(l, u, ids)
    gpu.sync()
    assert ids.tolist() == [0, 0]


def test_one_row_at_any_offset(gpu):
    """Rows that start off every 16-byte boundary."""
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        flat = (2.0 * torch.randn(5 * 4001 + 8, generator=g)).to(dtype).cuda()
        for off in (0, 1, 2, 3, 5, 7):
            x = flat[off:off + 5 * 4001].view(5, 4001)
            u = np.linspace(0.05, 0.95, 5).astype(np.float32)
            ids, lp = draw(gpu, x, u, p=0.9)
            for r in range(5):
                check_row(x[r], float(u[r]), 1.0, 0, float(np.float32(0.9)), 0.0, int(ids[r]), float(lp[r]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [60, 130, 300])
def test_many_rows(gpu, rows, dtype):
    """Fewer CTAs take a row the more rows there are; every split follows the definition."""
    vocab = 50257  # odd: bf16 rows start off 4-byte boundaries in turn
    g = torch.Generator().manual_seed(rows)
    x = (3.0 * torch.randn(rows, vocab, generator=g)).to(dtype)
    x[::4, ::3] = float("-inf")
    x[5, 7] = float("nan")
    x = x.cuda()
    u = torch.rand(rows, generator=g).numpy().astype(np.float32)
    t, k, p, mp = (np.array([RULES[i % len(RULES)][j] for i in range(rows)]) for j in range(4))
    ids, lp = draw(gpu, x, u, t.astype(np.float32), k.astype(np.int32), p.astype(np.float32), mp.astype(np.float32))
    for r in range(rows):
        check_row(x[r], float(u[r]), float(np.float32(t[r])), int(k[r]), float(np.float32(p[r])), float(np.float32(mp[r])),
                  int(ids[r]), float(lp[r]))


@pytest.mark.parametrize("rows", [30, 60, 130, 300])
def test_equal_logits_in_every_split(gpu, rows):
    """One bin holds every token: it is divided down to the index, and its sums pass 32 bits."""
    vocab = 151936
    l = torch.full((rows, vocab), 1.5, device="cuda")
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    ids, _ = draw(gpu, l, u)
    assert np.array_equal(ids, (u.astype(np.float64) * vocab).astype(np.int64))
    ids, _ = draw(gpu, l, u, k=100000, p=0.25)
    assert np.array_equal(ids, (u.astype(np.float64) * 25000).astype(np.int64))
