"""Serving attention where it is easily wrong (B200 only), against the formula
in 64 bits: the precision of bf16 results, infinities and NaN that cross
splits, and plans of batches whose prompts are nested."""
import numpy as np
import pytest

from test_gpu_serve_attn import DTYPES, D, make, normal, reference, window_seen
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
