"""Serving attention over the paged cache (B200 only): zynfer_cu_attn_shared,
zynfer_cu_attn_window and zynfer_cu_kv_write against the formula in 64 bits,
    o = sum_j softmax_j(q . k_j / sqrt(d)) v_j
over the visible positions j, with the cache's exact bf16 K and V.

Tolerances, before any run (|v| <= vmax, scores s = q . k / sqrt(d)):
* f32: a score is a sum of d = 128 products in f32, off by at most
  128 * 2^-24 * |q| |k| / sqrt(d) (about 1.3e-4 at the worst for the norms used
  here, 1e-5 when roundings do not conspire), and o moves by at most vmax
  times twice that; p and the sums add 2^-22. Bound: 1e-4 * vmax.
* bf16: p and o are rounded to 8 significant bits: 2^-9 each of at most vmax,
  besides the f32 part. Bound: 2^-8 * vmax.
One visible position gives its V row itself, bit for bit.
"""
import numpy as np
import pytest

from zynfer_b200 import cuda as zc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

D = 128
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(n_kv=4, max_batch=8, max_seqs=8, max_seq_len=512, layers=1, kv_blocks=0):
    gpu = zc.Gpu(0)
    arch = zc.Arch(vocab=512, hidden=512, inter=512, layers=layers, n_q=2 * n_kv, n_kv=n_kv, max_pos=max_seq_len)
    return zc.Model(gpu, arch, zc.W_BF16, max_batch=max_batch, max_seqs=max_seqs, max_seq_len=max_seq_len,
                    kv_blocks=kv_blocks, max_prefill=16)


def normal(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def reference(q, k, v, seen):
    """q [T, n_q, D], k and v [n_kv, L, D], seen [T, L] -> [T, n_q, D] in 64 bits; rows that see nothing are 0."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for h in range(q.shape[1]):
        s = q[:, h].double() @ k[h // 2].double().T / D ** 0.5
        s = torch.where(seen, s, torch.full_like(s, -float("inf")))
        p = torch.where(seen, torch.exp(s - s.amax(1, keepdim=True)), torch.zeros_like(s))
        total = p.sum(1, keepdim=True)
        vv = torch.where(seen.any(0)[:, None], v[h // 2].double(), torch.zeros_like(v[h // 2].double()))
        out[:, h] = torch.where(total > 0, p @ vv / total, torch.zeros_like(out[:, h]))
    return out


def window_seen(length, tokens, window, sinks):
    i = torch.arange(length - tokens, length, device="cuda")[:, None]
    j = torch.arange(length, device="cuda")[None]
    return (j <= i) & ((j < sinks) | (j > i - window))


def check(got, want, v, dtype):
    tol = (1e-4 if dtype == "f32" else 2.0 ** -8) * float(v.float().abs().max())
    assert got.dtype == DTYPES[dtype]
    if not got.numel():
        return
    off = float((got.double() - want).abs().max())
    assert off <= tol, (off, tol)


def poison(m, seqs, layer=0):
    """Leave NaN in every block of the pool that `seqs` can take, then give the blocks back."""
    n = m.desc.max_seq_len
    nan = torch.full((m.arch.n_kv, n, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    for s in seqs:
        m.kv_write(s, layer, 0, nan, nan)
    m.gpu.sync()
    for s in seqs:
        m.seq_reset(s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_kv_write_reads_back(dtype):
    m = make(n_kv=2, layers=2)
    k, v = normal(1, 2, 45, D, dtype=DTYPES[dtype]), normal(2, 2, 45, D, dtype=DTYPES[dtype])
    for layer in (0, 1):
        m.kv_write(3, layer, 0, k[:, :19].contiguous(), v[:, :19].contiguous())
        m.kv_write(3, layer, 19, k[:, 19:].contiguous(), v[:, 19:].contiguous())
    m.kv_write(3, 1, 7, k[:, 7:9].contiguous(), v[:, 7:9].contiguous())  # within: the length stays
    m.kv_write(3, 1, 45, k[:, :0].contiguous(), v[:, :0].contiguous())   # nothing
    assert m.seq_len(3) == 45
    for layer in (0, 1):
        assert np.array_equal(m.kv(3, layer, False), k.bfloat16().float().cpu().numpy())
        assert np.array_equal(m.kv(3, layer, True), v.bfloat16().float().cpu().numpy())


WINDOW_CASES = [
    # (lengths, tokens, window, sinks)
    ([1], 1, 1, 0),            # one position
    ([1, 2, 17], 1, 5, 3),     # shorter than window and sinks
    ([300, 33, 512, 48], 1, 64, 4),
    ([200, 201], 1, 1, 0),     # only itself
    ([200, 77], 1, 0, 3),      # only the sinks
    ([64, 9], 1, 0, 0),        # nothing
    ([512], 1, zc.WINDOW_ALL, 0),
    ([511, 130], 1, 17, 500),  # sinks past the window's start
    ([512], 512, zc.WINDOW_ALL, 0),
    ([100, 161], 90, 30, 2),
    ([300, 288], 2, 40, 5),
    ([257], 129, 16, 0),
    ([50], 50, 0, 7),          # the first queries are the sinks, the rest see only them
    ([70], 70, 0, 0),          # nothing at all
    ([401, 399, 512], 385, 100, 33),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,tokens,window,sinks", WINDOW_CASES)
def test_attn_window(lens, tokens, window, sinks, dtype):
    m = make(n_kv=2)
    poison(m, range(8))
    seqs = [(3 * i + 1) % 8 for i in range(len(lens))]
    k = [normal(10 + i, 2, n, D, dtype=torch.bfloat16) for i, n in enumerate(lens)]
    v = [normal(30 + i, 2, n, D, dtype=torch.bfloat16) for i, n in enumerate(lens)]
    for s, a, b in zip(seqs, k, v):
        m.kv_write(s, 0, 0, a, b)
    q = normal(50, len(lens), tokens, 4, D, dtype=DTYPES[dtype], scale=1.5)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    m.attn_window(0, seqs, q, out, window=window, sinks=sinks)
    m.gpu.sync()
    for i, n in enumerate(lens):
        seen = window_seen(n, tokens, window, sinks)
        check(out[i], reference(q[i], k[i], v[i], seen), v[i], dtype)
        for t in (~seen.any(1)).nonzero()[:, 0].tolist():
            assert not out[i, t].any()
        for t in (seen.sum(1) == 1).nonzero()[:, 0].tolist():
            j = int(seen[t].nonzero()[0, 0])
            assert torch.equal(out[i, t].float(), v[i][:, j].float().repeat_interleave(2, 0))


def share(m, prompts, plen, own, dtype=torch.bfloat16, seed=100, order=None):
    """Sequences prompt by prompt: K and V of each, filled through kv_write and seq_fork."""
    n_kv, kv, row = m.arch.n_kv, {}, 0
    slots = list(range(sum(len(o) for o in own))) if order is None else order
    for g in range(prompts):
        kp, vp = normal(seed + g, n_kv, plen[g], D, dtype=dtype), normal(seed + 50 + g, n_kv, plen[g], D, dtype=dtype)
        first = slots[row]
        if plen[g]:
            m.kv_write(first, 0, 0, kp, vp)
        for s in slots[row + 1:row + len(own[g])]:
            m.seq_fork(s, first, plen[g])
        for i, n in enumerate(own[g]):
            ks, vs = normal(seed + 200 + row, n_kv, n, D, dtype=dtype), normal(seed + 300 + row, n_kv, n, D, dtype=dtype)
            m.kv_write(slots[row], 0, plen[g], ks, vs)
            kv[slots[row]] = (torch.cat([kp, ks], 1), torch.cat([vp, vs], 1))
            row += 1
    return kv


SHARED_CASES = [
    # (prompt lengths, own positions of each prompt's rows)
    ([0], [[1]]),                                  # a lone position
    ([16], [[0, 1, 0]]),                           # nothing of their own, whole blocks
    ([5], [[3, 1, 2, 0]]),                         # shorter than a block: nothing is shared
    ([64], [[1]]),                                 # one row: a prompt of its own
    ([400], [[1, 40, 17, 100, 16]]),
    ([128, 33, 250], [[5, 1], [20], [3, 3, 60, 9]]),
    ([505], [[7, 1, 3, 2, 5, 6, 4, 7]]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("plen,own", SHARED_CASES)
def test_attn_shared(plen, own, mixed, dtype):
    m = make(n_kv=4)
    poison(m, range(8))
    rows = sum(len(o) for o in own)
    order = [(5 * i + 2) % 8 for i in range(rows)] if mixed else list(range(rows))
    kv = share(m, len(plen), plen, own, order=order)
    seqs = [s for s in (order[::-1] if mixed else order) if m.seq_len(s)]
    big = normal(7, len(seqs), 8 + 5, D, dtype=DTYPES[dtype], scale=1.5)  # q inside a wider row
    q, out = big[:, 3:11], torch.full((len(seqs), 8, D), float("nan"), dtype=DTYPES[dtype], device="cuda")
    torch.cuda.synchronize()
    m.attn_shared(0, seqs, q, out)
    m.gpu.sync()
    for i, s in enumerate(seqs):
        k, v = kv[s]
        seen = torch.ones(1, k.shape[1], dtype=torch.bool, device="cuda")
        check(out[i:i + 1], reference(q[i:i + 1], k, v, seen), v, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [3, 65, 130])
def test_attn_shared_many_rows(rows, dtype):
    """More rows of one prompt than a tile of queries holds, and some rows without a prompt among them."""
    m = make(n_kv=2, max_batch=rows, max_seqs=rows, max_seq_len=1400, kv_blocks=100 + 5 * rows)
    own = [[1 + (13 * i) % 40 for i in range(rows - 1)], [30]]
    kv = share(m, 2, [1300, 0], own)
    q = normal(8, rows, 4, D, dtype=DTYPES[dtype], scale=1.5)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    seqs = list(range(rows))
    seqs[1], seqs[-1] = seqs[-1], seqs[1]
    m.attn_shared(0, seqs, q, out)
    m.gpu.sync()
    for i, s in enumerate(seqs):
        k, v = kv[s]
        seen = torch.ones(1, k.shape[1], dtype=torch.bool, device="cuda")
        check(out[i:i + 1], reference(q[i:i + 1], k, v, seen), v, dtype)


def test_large_scores_stay_finite():
    """Scores in the hundreds: the running maximum carries the softmax."""
    m = make(n_kv=2)
    k, v = normal(1, 2, 300, D, dtype=torch.bfloat16, scale=30.0), normal(2, 2, 300, D, dtype=torch.bfloat16)
    m.kv_write(0, 0, 0, k, v)
    q = normal(3, 1, 4, D, scale=4.0)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    m.attn_shared(0, [0], q, out)
    m.gpu.sync()
    # |q| |k| / sqrt(d) is 120 times the other tests' least: the score's bound grows alike, the result stays a mean of V
    want = reference(q, k, v, torch.ones(1, 300, dtype=torch.bool, device="cuda"))
    assert float((out.double() - want).abs().max()) <= 1e-2 * float(v.float().abs().max())


def test_same_call_gives_the_same_bits_and_streams_are_ordered():
    m = make(n_kv=4, max_seq_len=512)
    kv = share(m, 1, [400], [[9, 30, 1, 12]])
    q = normal(4, 4, 8, D)
    side = torch.cuda.Stream()
    outs = []
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            late = torch.empty_like(q)
            torch.cuda._sleep(20_000_000)
            late.copy_(q)                 # q arrives late on the side stream
            out = torch.zeros_like(q)
            m.attn_shared(0, range(4), late, out, stream=side)
            outs.append(out * 1.0)        # read on the side stream
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    for i in range(4):
        k, v = kv[i]
        check(outs[0][i:i + 1], reference(q[i:i + 1], k, v, torch.ones(1, k.shape[1], dtype=torch.bool, device="cuda")), v, "f32")


def test_calls_between_calls_do_not_mix():
    """Two batches of different shapes in turn, nothing waited for between them."""
    m = make(n_kv=2, max_seq_len=512)
    kv = share(m, 2, [300, 200], [[4, 5, 6], [7, 8]])
    q1, q2 = normal(5, 5, 4, D), normal(6, 2, 100, 4, D)
    a, b = torch.empty_like(q1), torch.empty_like(q2)
    torch.cuda.synchronize()
    for _ in range(3):
        m.attn_shared(0, range(5), q1, a)
        m.attn_window(0, [4, 0], q2, b, window=50, sinks=3)
    m.gpu.sync()
    for i in range(5):
        check(a[i:i + 1], reference(q1[i:i + 1], *kv[i], torch.ones(1, kv[i][0].shape[1], dtype=torch.bool, device="cuda")), kv[i][1], "f32")
    for i, s in enumerate((4, 0)):
        check(b[i], reference(q2[i], *kv[s], window_seen(kv[s][0].shape[1], 100, 50, 3)), kv[s][1], "f32")


def test_refusals():
    m = make(n_kv=2)
    k = normal(1, 2, 40, D)
    m.kv_write(0, 0, 0, k, k)
    m.seq_fork(1, 0, 36)
    q = normal(2, 2, 4, D)
    out = torch.empty_like(q)
    bad = zc.InvalidArgument
    for call in (
        lambda: m.attn_shared(0, [0, 0], q, out),                       # twice
        lambda: m.attn_shared(0, [0, 2], q, out),                       # an empty sequence
        lambda: m.attn_shared(0, [0, 8], q, out),                       # no such slot
        lambda: m.attn_shared(1, [0, 1], q, out),                       # no such layer
        lambda: m.attn_shared(0, [0, 1], q, out.bfloat16()),            # two types
        lambda: m.attn_shared(0, [0, 1], q[:1], out),                   # too few rows
        lambda: m.attn_shared(0, [], q[:0], out[:0]),                   # no rows
        lambda: m.attn_window(0, [0, 1], normal(3, 2, 37, 4, D), torch.empty(2, 37, 4, D, device="cuda")),  # longer than a sequence
        lambda: m.attn_window(0, [0], q[:1].transpose(1, 2), out[:1]),  # heads not dense
        lambda: m.kv_write(0, 0, 41, k, k),                             # a hole
        lambda: m.kv_write(0, 0, 0, k[:, :1].contiguous(), k[:, :1].contiguous()),  # shared with sequence 1
        lambda: m.kv_write(0, 1, 0, k, k),
        lambda: m.kv_write(9, 0, 0, k, k),
        lambda: m.kv_write(2, 0, 0, normal(1, 2, 513, D), normal(1, 2, 513, D)),  # past max_seq_len
        lambda: m.kv_write(2, 0, 0, k, k.bfloat16()),
        lambda: m.kv_write(2, 0, 0, k.transpose(0, 1), k.transpose(0, 1)),
    ):
        with pytest.raises(bad):
            call()
    with pytest.raises(zc.Unsupported):
        m.attn_shared(0, [0, 1], q.double(), out.double())
    with pytest.raises(zc.Unsupported):
        m.kv_write(2, 0, 0, k.half(), k.half())
    odd = torch.empty(2 * 4 * D + 1, device="cuda")[1:].view(2, 4, D)  # 4-byte aligned only
    with pytest.raises(bad):
        m.attn_shared(0, [0, 1], odd, out)
    m.gpu.set_fail_at("launch")
    with pytest.raises(zc.LaunchFailed):
        m.attn_shared(0, [0, 1], q, out)
    m.kv_write(0, 0, 36, k[:, 36:].contiguous(), k[:, 36:].contiguous())  # its own copy of the last block
    m.attn_shared(0, [0, 1], q, out)                                     # and the context still works
    m.gpu.sync()
    assert torch.isfinite(out).all()


def test_pool_exhaustion_is_reported():
    m = make(n_kv=2, kv_blocks=2)
    k = normal(1, 2, 33, D)
    with pytest.raises(zc.OutOfMemory):
        m.kv_write(0, 0, 0, k, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_masked_nan_and_infinity_do_not_spread(value, dtype):
    """A position's NaN or infinity (in V, in K) reaches exactly the queries that see it."""
    m = make(n_kv=2)
    n, tokens, window, sinks = 300, 200, 40, 3
    for which, where in (("v", 171), ("k", 230), ("v", 299), ("v", 1)):
        k, v = normal(11, 2, n, D, dtype=torch.bfloat16), normal(12, 2, n, D, dtype=torch.bfloat16)
        clean_k, clean_v = k.clone(), v.clone()
        (v if which == "v" else k)[1, where, 5:9] = value
        m.seq_reset(0)
        m.kv_write(0, 0, 0, k, v)
        q = normal(13, 1, tokens, 4, D, dtype=DTYPES[dtype])
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        m.attn_window(0, [0], q, out, window=window, sinks=sinks)
        m.gpu.sync()
        seen = window_seen(n, tokens, window, sinks)
        want = reference(q[0], clean_k, clean_v, seen)
        sees = seen[:, where]
        check(out[0, :, :2], want[:, :2], clean_v, dtype)                     # the other kv head
        check(out[0, ~sees][:, 2:], want[~sees][:, 2:], clean_v, dtype)       # queries that do not see it
        hit = out[0, sees][:, 2:]
        if which == "v":
            assert not torch.isfinite(hit[..., 5:9]).any()
            rest = torch.cat([hit[..., :5], hit[..., 9:]], -1)
            w = want[sees][:, 2:]
            check(rest, torch.cat([w[..., :5], w[..., 9:]], -1), clean_v, dtype)
        elif value != value:
            assert torch.isnan(hit).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shared_prompt_nan_stays_in_its_dims(dtype):
    m = make(n_kv=2)
    k, v = normal(21, 2, 400, D, dtype=torch.bfloat16), normal(22, 2, 400, D, dtype=torch.bfloat16)
    clean = v.clone()
    v[0, 37, 64] = float("nan")
    m.kv_write(0, 0, 0, k, v)
    for s in range(1, 6):
        m.seq_fork(s, 0, 400)
    q = normal(23, 6, 4, D, dtype=DTYPES[dtype])
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    m.attn_shared(0, range(6), q, out)
    m.gpu.sync()
    seen = torch.ones(1, 400, dtype=torch.bool, device="cuda")
    for i in range(6):
        want = reference(q[i:i + 1], k, clean, seen)
        assert torch.isnan(out[i, :2, 64]).all()
        keep = torch.tensor([d for d in range(D) if d != 64], device="cuda")
        check(out[i:i + 1][..., keep], want[..., keep], clean, dtype)
        check(out[i:i + 1, 2:], want[:, 2:], clean, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,length,window,sinks", [(70, 2100, zc.WINDOW_ALL, 0), (1, 3000, 1500, 7), (2100, 2100, 900, 20)])
def test_long_loops_over_tiles(tokens, length, window, sinks, dtype):
    """Many tiles of keys per tile of queries: every ring and barrier wraps several times."""
    m = make(n_kv=2, max_seq_len=3008)
    k, v = normal(41, 2, length, D, dtype=torch.bfloat16), normal(42, 2, length, D, dtype=torch.bfloat16)
    m.kv_write(2, 0, 0, k, v)
    q = normal(43, 1, tokens, 4, D, dtype=DTYPES[dtype], scale=1.5)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    for _ in range(3):
        m.attn_window(0, [2], q, out, window=window, sinks=sinks)
    m.gpu.sync()
    check(out[0], reference(q[0], k, v, window_seen(length, tokens, window, sinks)), v, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("plen,rows", [([1000], [60]), ([700, 1000, 16, 333], [40, 30, 5, 7]), ([1015], [64])])
def test_attn_shared_prompts_worth_sharing(plen, rows, dtype):
    """Large groups (their prompts are read once) and small ones in one batch, the rows interleaved."""
    total = sum(rows)
    m = make(n_kv=4, max_batch=total, max_seqs=total, max_seq_len=1100, kv_blocks=sum(p // 16 + 1 for p in plen) + 6 * total)
    own = [[(7 * i) % 50 if g else 1 + (11 * i) % 60 for i in range(n)] for g, n in enumerate(rows)]
    kv = share(m, len(plen), plen, own)
    seqs = [(37 * i + 11) % total for i in range(total)] if total % 37 else list(range(total))
    assert sorted(seqs) == list(range(total))
    q = normal(9, total, 8, D, dtype=DTYPES[dtype], scale=1.5)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    for _ in range(2):
        m.attn_shared(0, seqs, q, out)
    m.gpu.sync()
    for i, s in enumerate(seqs):
        k, v = kv[s]
        check(out[i:i + 1], reference(q[i:i + 1], k, v, torch.ones(1, k.shape[1], dtype=torch.bool, device="cuda")), v, dtype)


def test_attn_shared_forks_of_forks():
    """A common start, two longer prompts on top of it, and their samples: each run at its own depth."""
    m = make(n_kv=4, max_batch=80, max_seqs=80, max_seq_len=1400, kv_blocks=700)
    k, v = normal(51, 4, 1300, D, dtype=torch.bfloat16), normal(52, 4, 1300, D, dtype=torch.bfloat16)
    k2, v2 = normal(53, 4, 1300, D, dtype=torch.bfloat16), normal(54, 4, 1300, D, dtype=torch.bfloat16)
    kv = {}
    m.kv_write(0, 0, 0, k[:, :400].contiguous(), v[:, :400].contiguous())
    for first, kk, vv in ((1, k, v), (40, k2, v2)):
        m.seq_fork(first, 0, 400)
        m.kv_write(first, 0, 400, kk[:, 400:1290].contiguous(), vv[:, 400:1290].contiguous())
        full = (torch.cat([k[:, :400], kk[:, 400:1290]], 1), torch.cat([v[:, :400], vv[:, 400:1290]], 1))
        kv[first] = full
        for s in range(first + 1, first + 39):
            m.seq_fork(s, first, 1290)
            e = normal(100 + s, 4, s % 5, D, dtype=torch.bfloat16)
            m.kv_write(s, 0, 1290, e, e)
            kv[s] = (torch.cat([full[0], e], 1), torch.cat([full[1], e], 1))
    kv[0] = (k[:, :400], v[:, :400])
    seqs = sorted(kv)
    q = normal(9, len(seqs), 8, D, scale=1.5)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    m.attn_shared(0, seqs, q, out)
    m.gpu.sync()
    for i, s in enumerate(seqs):
        kk, vv = kv[s]
        check(out[i:i + 1], reference(q[i:i + 1], kk, vv, torch.ones(1, kk.shape[1], dtype=torch.bool, device="cuda")), vv, "f32")


def test_shared_tiles_keep_nan_in_its_dims():
    m = make(n_kv=4, max_batch=64, max_seqs=64, max_seq_len=1100, kv_blocks=300)
    k, v = normal(61, 4, 1000, D, dtype=torch.bfloat16), normal(62, 4, 1000, D, dtype=torch.bfloat16)
    clean = v.clone()
    v[1, 500, 7] = float("nan")
    m.kv_write(0, 0, 0, k, v)
    for s in range(1, 64):
        m.seq_fork(s, 0, 1000)
    q = normal(63, 64, 8, D)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    m.attn_shared(0, range(64), q, out)
    m.gpu.sync()
    want = torch.cat([reference(q[i:i + 1], k, clean, torch.ones(1, 1000, dtype=torch.bool, device="cuda")) for i in range(64)])
    assert torch.isnan(out[:, 2:4, 7]).all()
    keep = torch.tensor([d for d in range(D) if d != 7], device="cuda")
    check(out[..., keep], want[..., keep], clean, "f32")
    assert torch.isfinite(out[:, [0, 1, 4, 5, 6, 7]]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,tokens,window,sinks", [([2900], 2, zc.WINDOW_ALL, 0), ([2900, 700], 33, 2000, 5), ([3000, 64, 1500], 64, 1024, 70)])
def test_few_queries_with_many_keys(lens, tokens, window, sinks, dtype):
    """A tile's keys shared by several CTAs, rows of one batch with very different ranges."""
    m = make(n_kv=2, max_seq_len=3008)
    k = [normal(70 + i, 2, n, D, dtype=torch.bfloat16) for i, n in enumerate(lens)]
    v = [normal(80 + i, 2, n, D, dtype=torch.bfloat16) for i, n in enumerate(lens)]
    for s, (a, b) in enumerate(zip(k, v)):
        m.kv_write(s, 0, 0, a, b)
    q = normal(90, len(lens), tokens, 4, D, dtype=DTYPES[dtype], scale=1.5)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    for _ in range(2):
        m.attn_window(0, range(len(lens)), q, out, window=window, sinks=sinks)
    m.gpu.sync()
    for i, n in enumerate(lens):
        check(out[i], reference(q[i], k[i], v[i], window_seen(n, tokens, window, sinks)), v[i], dtype)


@pytest.mark.parametrize("plen,grows", [(30000, 0), (40000, 1)])
def test_workspace_stays_and_grows(plen, grows):
    """Calls allocate nothing until one needs more partial results than model_init left room for: two rows
    that share a very long prompt, split over many CTAs, in a batch of many rows. (The shorter prompt saves
    too few block reads to be shared.)"""
    rows = 300
    m = make(n_kv=4, max_batch=rows, max_seqs=rows, max_seq_len=plen + 16, kv_blocks=plen // 16 + 2 * rows + 4)
    kv = share(m, 2, [plen, 0], [[3, 9], [1 + i % 16 for i in range(rows - 2)]])
    q = normal(21, rows, 8, D)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()

    def call(seqs):
        m.attn_shared(0, seqs, q[:len(seqs)], out[:len(seqs)])
        m.gpu.sync()
        for i, s in list(enumerate(seqs))[:12]:
            k, v = kv[s]
            check(out[i:i + 1], reference(q[i:i + 1], k, v, torch.ones(1, k.shape[1], dtype=torch.bool, device="cuda")), v, "f32")

    before = m.gpu.alloc_events()[0]
    call([0, 1])
    call(list(range(2, 40)))
    assert m.gpu.alloc_events()[0] == before
    call(list(range(rows)))
    assert m.gpu.alloc_events()[0] == before + grows
    call(list(range(rows)))
    call([1, 0, 5])
    assert m.gpu.alloc_events()[0] == before + grows


@pytest.mark.parametrize("tokens,length,window", [(64, 8192, zc.WINDOW_ALL), (200, 6000, zc.WINDOW_ALL), (1500, 3100, 2900)])
def test_long_f32_sums_keep_their_precision(tokens, length, window):
    """f32 queries over thousands of keys. The matrix units round each of the 64 additions that 1024 keys take
    toward 0, half of 2^-23 on average of a sum that is half its final size on average: 64 * 2^-25 = 1.9e-6 of
    the result's norm; products, exponentials and the sums in shared memory add well below 1e-6. Bound: 4e-6."""
    m = make(n_kv=2, max_seq_len=8192)
    k, v = normal(31, 2, length, D, dtype=torch.bfloat16), normal(32, 2, length, D, dtype=torch.bfloat16)
    m.kv_write(0, 0, 0, k, v)
    q = normal(33, 1, tokens, 4, D, scale=1.5)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    m.attn_window(0, [0], q, out, window=window, sinks=3)
    m.gpu.sync()
    want = reference(q[0], k, v, window_seen(length, tokens, window, 3))
    assert float((out[0].double() - want).norm() / want.norm()) <= 4e-6


def test_long_f32_sums_follow_a_growing_maximum():
    """Scores that grow along the cache: the sums kept so far are scaled down each time the maximum grows."""
    length, tokens = 4000, 100
    m = make(n_kv=2, max_seq_len=4096)
    k, v = normal(34, 2, length, D, dtype=torch.float32), normal(35, 2, length, D, dtype=torch.bfloat16)
    k = (k * torch.linspace(0.1, 6.0, length, device="cuda")[None, :, None]).bfloat16()
    m.kv_write(0, 0, 0, k, v)
    q = normal(36, 1, tokens, 4, D, scale=1.5)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    m.attn_window(0, [0], q, out)
    m.gpu.sync()
    check(out[0], reference(q[0], k, v, window_seen(length, tokens, zc.WINDOW_ALL, 0)), v, "f32")


@pytest.mark.parametrize("dims", ["same", "growing"])
def test_long_single_tokens_keep_their_precision(dims):
    """One query over 16384 positions in each of 16 rows: a warp takes about 900 positions, 55 additions of 16
    products each where they are not added up apart, rounded toward 0. Apart after every 512 positions: 32
    additions, half of 2^-23 on average of a sum that is half its final size on average: 1e-6 of the result's
    norm; the joins and exponentials add below 1e-6. Bound: 2e-6. Where the
    maximum keeps growing, the sums are scaled down with it: the bound of the other tests."""
    rows, length = 16, 16384
    m = make(n_kv=4, max_batch=rows, max_seqs=rows, max_seq_len=length, kv_blocks=rows * length // 16)
    kv = {}
    for i in range(rows):
        k, v = normal(40 + i, 4, length, D, dtype=torch.bfloat16), normal(80 + i, 4, length, D, dtype=torch.bfloat16)
        if dims == "growing":
            k = (k.float() * torch.linspace(0.1, 4.0, length, device="cuda")[None, :, None]).bfloat16()
        m.kv_write(i, 0, 0, k, v)
        m.gpu.sync()
        if i in (0, 9):
            kv[i] = (k, v)
    q = normal(39, rows, 8, D, scale=1.5)
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    m.attn_window(0, range(rows), q, out)
    m.gpu.sync()
    for i, (k, v) in kv.items():
        want = reference(q[i:i + 1], k, v, torch.ones(1, length, dtype=torch.bool, device="cuda"))
        if dims == "same":
            assert float((out[i:i + 1].double() - want).norm() / want.norm()) <= 2e-6
        check(out[i:i + 1], want, v, "f32")
