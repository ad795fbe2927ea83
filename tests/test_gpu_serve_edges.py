"""Serving attention where it is easily wrong (B200 only), against the formula
in 64 bits: the precision of bf16 results, infinities and NaN that cross
splits, and plans of batches whose prompts are nested."""
import time

import pytest

from test_gpu_serve_attn import DTYPES, D, check, make, normal, reference, window_seen
from zynfer_b200 import cuda as zc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def all_seen(n):
    return torch.ones(1, n, dtype=torch.bool, device="cuda")


def forked(rows, length, n_kv=4, own=0):
    """`rows` sequences over the same `length` positions: the model, K and V."""
    m = make(n_kv=n_kv, max_batch=rows, max_seqs=rows, max_seq_len=length + own + 16, kv_blocks=length // 16 + 2 + rows * (2 + own // 16))
    k, v = normal(201, n_kv, length, D, dtype=torch.bfloat16), normal(202, n_kv, length, D, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    m.kv_write(0, 0, 0, k, v)
    for s in range(1, rows):
        m.seq_fork(s, 0, length)
    return m, k, v


@pytest.mark.parametrize("case", ["chunk", "few queries", "prompt", "one token"])
def test_bf16_results_are_rounded_once(case):
    """The probabilities' two bf16 terms are off by 2^-17 of each, a result by at most 2^-17 sum p |v|: about 100 keys
    share most of the weight here, of random sign, so that is at most 2^-17 sqrt(100) of the result's norm, 8e-5.
    Sums in f32 add 1e-5 at most. What is left is the rounding of the result itself."""
    if case == "prompt":
        m, k, v = forked(64, 1000)
        q = normal(203, 64, 8, D, dtype=torch.bfloat16, scale=1.5)
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        m.attn_shared(0, range(64), q, out)
        m.gpu.sync()
        want = torch.cat([reference(q[i:i + 1], k, v, all_seen(1000)) for i in range(64)])
    else:
        length, tokens = {"chunk": (1500, 1200), "few queries": (3000, 40), "one token": (3000, 1)}[case]
        m, k, v = forked(1, length)
        q = normal(203, 1, tokens, 8, D, dtype=torch.bfloat16, scale=1.5)
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        m.attn_window(0, [0], q, out, sinks=2)
        m.gpu.sync()
        want = reference(q[0], k, v, window_seen(length, tokens, zc.WINDOW_ALL, 2))[None]
    norm = want.norm()
    once = float((want.bfloat16().double() - want).norm() / norm)
    assert float((out.double() - want).norm() / norm) <= once + 1e-4


# ways a row is split: (sequences, cached positions, queries of each, own positions of forked rows)
SPLITS = {"one token": (3, 3000, 1), "short": (8, 40, 1), "few queries": (2, 3000, 40), "chunk": (1, 900, 700), "prompt": (64, 992, 0)}


def split_case(how, dtype, edit):
    """K and V [rows, n_kv, L, D], q [rows, T, n_q, D] and the model that has them in its cache, after edit(q, k, v) (the
    rows of "prompt" share every position but their last 3)."""
    rows, length, tokens = SPLITS[how]
    own = 3 if how == "prompt" else 0
    m = make(n_kv=4, max_batch=rows, max_seqs=rows, max_seq_len=length + own + 16, kv_blocks=rows * (length // 16 + 3) if not own else length // 16 + 4 * rows)
    k, v = (normal(seed, 1 if own else rows, 4, length, D, dtype=torch.bfloat16) for seed in (211, 212))
    if own:
        k, v = (torch.cat([x.expand(rows, -1, -1, -1), normal(seed, rows, 4, own, D, dtype=torch.bfloat16)], 2) for x, seed in ((k, 213), (v, 214)))
    q = normal(215, rows, max(1, tokens), 8, D, dtype=DTYPES[dtype], scale=1.5)
    edit(q, k, v)
    torch.cuda.synchronize()
    for i in range(rows):
        if own and i:
            m.seq_fork(i, 0, length)
        first = length if own and i else 0
        a, b = k[i, :, first:].contiguous(), v[i, :, first:].contiguous()
        if own and not i:  # the prompt is forked before the first row's own positions
            torch.cuda.synchronize()
            m.kv_write(0, 0, 0, a[:, :length].contiguous(), b[:, :length].contiguous())
            m.gpu.sync()
            continue
        torch.cuda.synchronize()
        m.kv_write(i, 0, first, a, b)
        m.gpu.sync()
    if own:
        a, b = k[0, :, length:].contiguous(), v[0, :, length:].contiguous()
        torch.cuda.synchronize()
        m.kv_write(0, 0, length, a, b)
        m.gpu.sync()
    out = torch.full_like(q, 7.0)
    torch.cuda.synchronize()
    if own:
        m.attn_shared(0, range(rows), q[:, 0], out[:, 0])
    else:
        m.attn_window(0, range(rows), q, out)
    m.gpu.sync()
    return q, k, v, out


def expect(q, k, v, out, dtype, nan):
    """nan [rows, T, n_q]: query heads that are NaN in every dim; the others follow the formula."""
    tokens, length = q.shape[1], k.shape[2]
    seen = window_seen(length, tokens, zc.WINDOW_ALL, 0)
    for i in range(q.shape[0]):
        assert torch.isnan(out[i][nan[i]]).all()
        want = reference(torch.nan_to_num(q[i]), torch.nan_to_num(k[i]), torch.nan_to_num(v[i]), seen)
        check(out[i][~nan[i]], want[~nan[i]], torch.nan_to_num(v[i]), dtype)


def none(q):
    return torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how", list(SPLITS))
def test_a_nan_query_gives_nan_however_its_row_is_split(how, dtype):
    def edit(q, k, v):
        q[-1, -1, 5, 17] = float("nan")
    q, k, v, out = split_case(how, dtype, edit)
    nan = none(q)
    nan[-1, -1, 5] = True
    expect(q, k, v, out, dtype, nan)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how,where", [("one token", slice(512, 1536)), ("one token", slice(2999, 3000)), ("short", slice(39, 40)),
                                       ("few queries", slice(512, 1536)), ("prompt", slice(994, 995)), ("prompt", slice(992, 995))])
def test_nan_scores_that_fill_a_piece_reach_the_result(how, where, dtype):
    """Every key of a piece of the last row is NaN in one kv head: the piece has no maximum, its sum is NaN."""
    def edit(q, k, v):
        k[-1, 2, where] = float("nan")
    q, k, v, out = split_case(how, dtype, edit)
    nan = none(q)
    seen = window_seen(k.shape[2], q.shape[1], zc.WINDOW_ALL, 0)[:, where].any(1)
    nan[-1, seen, 4:6] = True
    expect(q, k, v, out, dtype, nan)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how", ["one token", "few queries", "prompt"])
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_behind_a_weight_of_zero_reaches_the_result(how, which, dtype):
    """A NaN key or value among keys whose weights are too small for f32 beside the first positions'."""
    def edit(q, k, v):
        k[:, :, :64] *= 30.0
        at = 500 if how == "prompt" else k.shape[2] - 100
        (k if which == "k" else v)[-1 if how != "prompt" else slice(None), 1, at] = float("nan")
    q, k, v, out = split_case(how, dtype, edit)
    rows = slice(None) if how == "prompt" else slice(-1, None)
    nan = none(q)
    nan[rows, -1, 2:4] = True
    hit = out[rows, -1, 2:4]
    assert torch.isnan(hit).all()
    clean = torch.isfinite(out[:, -1])
    assert clean[~nan[:, -1]].all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how", list(SPLITS))
def test_an_infinite_value_that_is_seen_is_infinite(how, dtype):
    """sum p v with p > 0: infinity of its sign in its dims, NaN where two of both signs meet, the formula elsewhere."""
    own = SPLITS[how][1] + 1 if how == "prompt" else SPLITS[how][1] - 1  # the last row alone sees it, and its last query

    def edit(q, k, v):
        v[-1, 2, 3, 5:9] = float("inf") if how != "prompt" else v[-1, 2, 3, 5:9]
        v[-1, 2, own, 8] = v[-1, 2, own, 90] = -float("inf")
    q, k, v, out = split_case(how, dtype, edit)
    hit = out[-1, -1, 4:6]
    if how != "prompt":
        assert (hit[:, 5:8] == float("inf")).all() and torch.isnan(hit[:, 8]).all()
    else:
        assert (hit[:, 8] == -float("inf")).all()
    assert (hit[:, 90] == -float("inf")).all()
    odd = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    odd[-1, :, 4:6, 5:9] = odd[-1, -1, 4:6, 90] = True
    seen = window_seen(k.shape[2], q.shape[1], zc.WINDOW_ALL, 0)
    clean = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    for i in range(q.shape[0]):
        want = reference(q[i], k[i], clean[i], seen)
        check(out[i][~odd[i]], want[~odd[i]], clean[i], dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how", list(SPLITS))
def test_an_infinite_key_weighs_nothing_or_everything(how, dtype):
    """A score of -infinity is a weight of 0, one of +infinity has no softmax."""
    at = SPLITS[how][1] + 2 if how == "prompt" else 1

    def edit(q, k, v):
        k[-1, 1, at, 77] = float("inf")
    q, k, v, out = split_case(how, dtype, edit)
    seen = window_seen(k.shape[2], q.shape[1], zc.WINDOW_ALL, 0)
    nan = none(q)
    nan[-1, :, 2:4] = q[-1, :, 2:4, 77] > 0
    assert not nan.all() and (q[..., 77] != 0).all()
    for i in range(q.shape[0]):
        assert torch.isnan(out[i][nan[i]]).all()
        kk = torch.where(torch.isfinite(k[i]), k[i], torch.zeros_like(k[i]))
        want = reference(q[i], kk, v[i], seen)
        if i == q.shape[0] - 1:
            without = seen.clone()
            without[:, at] = False
            want[:, 2:4] = reference(q[i], kk, v[i], without)[:, 2:4]
        check(out[i][~nan[i]], want[~nan[i]], v[i], dtype)


def test_a_chain_of_forks_is_planned_in_linear_time():
    """Each of 1024 sequences forked from the one before, one block longer: every depth is a run of its own. The host's
    part of a call is well below a millisecond where it is linear (it was 0.2 s)."""
    rows, n_kv = 1024, 2
    m = make(n_kv=n_kv, max_batch=rows, max_seqs=rows, max_seq_len=16 * rows, kv_blocks=rows + 2)
    k, v = normal(221, n_kv, 16 * rows, D, dtype=torch.bfloat16), normal(222, n_kv, 16 * rows, D, dtype=torch.bfloat16)
    for i in range(rows):
        if i:
            m.seq_fork(i, i - 1, 16 * i)
        m.kv_write(i, 0, 16 * i, k[:, 16 * i:16 * i + 16].contiguous(), v[:, 16 * i:16 * i + 16].contiguous())
    q = normal(223, rows, 2 * n_kv, D, scale=1.5)
    out = torch.empty_like(q)
    took = []
    for _ in range(4):
        torch.cuda.synchronize()
        began = time.perf_counter()
        m.attn_shared(0, range(rows), q, out)
        took.append(time.perf_counter() - began)
        m.gpu.sync()
    assert min(took) < 0.02
    for i in (0, 1, 2, 63, 64, 511, 1000, 1023):
        n = 16 * (i + 1)
        check(out[i:i + 1], reference(q[i:i + 1], k[:, :n], v[:, :n], all_seen(n)), v, "f32")


def nested(layers=1):
    """64 sequences: a start of 16 positions, two questions of 960 behind it, 32 samples of each with 0 to 2 positions of
    their own; slots 0 .. 31 the first question's, 32 .. 63 the second's. The model, K and V of every sequence."""
    arch = zc.Arch(vocab=512, hidden=512, inter=512, layers=layers, n_q=8, n_kv=4, max_pos=1040)
    m = zc.Model(zc.Gpu(0), arch, zc.W_BF16, max_batch=64, max_seqs=65, max_seq_len=1040, kv_blocks=400, max_prefill=16)
    m.fill_synthetic(1, 0.05, 0.1)
    start = [normal(s, 4, 16, D, dtype=torch.bfloat16) for s in (231, 232)]
    kv = {}

    def write(seq, pos, k, v):
        for layer in range(layers):
            m.kv_write(seq, layer, pos, k, v)
    write(64, 0, *start)
    for first, seed in ((0, 233), (32, 235)):
        m.seq_fork(first, 64, 16)
        question = [normal(s, 4, 960, D, dtype=torch.bfloat16) for s in (seed, seed + 1)]
        write(first, 16, *question)
        for s in range(first + 1, first + 32):
            m.seq_fork(s, first, 976)
        for s in range(first, first + 32):
            own = [normal(300 + 2 * s + e, 4, s % 3, D, dtype=torch.bfloat16) for e in (0, 1)]
            write(s, 976, *own)
            kv[s] = [torch.cat(x, 1) for x in zip(start, question, own)]
    return m, kv


ORDERS = {"in order": list(range(64)), "in turn": [32 * (i % 2) + i // 2 for i in range(64)], "mixed": [(37 * i + 11) % 64 for i in range(64)]}


@pytest.mark.parametrize("order", list(ORDERS))
def test_nested_prompts_in_any_order(order):
    m, kv = nested()
    q = normal(240, 64, 8, D, scale=1.5)
    out = torch.full_like(q, float("nan"))
    m.attn_shared(0, ORDERS[order], q, out)
    m.gpu.sync()
    for i, s in enumerate(ORDERS[order]):
        k, v = kv[s]
        check(out[i:i + 1], reference(q[i:i + 1], k, v, all_seen(k.shape[1])), v, "f32")


def test_nested_prompts_are_shared_in_any_order():
    """Both questions are read once, whatever the order of the batch: the step has the launches of shared prompts (tiles,
    own blocks, join) in each layer. In turn, neighbours have no more than the start in common."""
    launches = {}
    for order, seqs in ORDERS.items():
        m, _ = nested(layers=2)
        m.decode_drawn(seqs, [5] * 64, [0.5] * 64, temperature=0.0)
        launches[order] = m.gpu.step_launches
    assert len(set(launches.values())) == 1, launches
