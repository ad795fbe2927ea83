"""zynfer_cu_sample_rows (B200 only) over a hundred calls of the range that
serving has: 1 to 32 rows, vocabularies of 1000 to 151936, rules alike or
mixed, f32 and bf16. Every row is held to the definition (the tolerances of
test_gpu_draw.py), and the same seed gives the same inputs, ids and
log-probabilities, bit for bit."""
from contextlib import closing

import numpy as np
import pytest

from test_gpu_draw import check_row
from zynfer_b200 import cuda as zc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

CASES = 100


def prepare(seed):
    rng = np.random.default_rng(seed)
    rows, vocab = int(round(32 ** rng.random())), int(round(1000 * 151.936 ** rng.random()))
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = 2.5 * torch.randn(rows, vocab, generator=g, device="cuda")
    # a few tokens well above the rest, several of them at one place: the largest stays, whatever the order
    at = torch.randint(min(vocab, 400), (rows, 24), generator=g, device="cuda")
    logits.scatter_reduce_(1, at, 6.0 + 2.5 * torch.randn((rows, 24), generator=g, device="cuda"), "amax")
    if seed % 3 == 0:
        logits[::3, ::7] = float("-inf")
    logits = logits.to(torch.bfloat16 if seed % 2 else torch.float32)
    pick = lambda values: rng.choice(values, rows) if seed % 4 else np.full(rows, rng.choice(values))  # noqa: E731
    rule = {"temperature": pick([0.8, 1.0, 0.6, 1.3, 0.0]).astype(np.float32), "top_k": pick([50, 0, 20, 1, 1000]).astype(np.int32),
            "top_p": pick([0.95, 1.0, 0.9, 0.8, 0.5]).astype(np.float32), "min_p": pick([0.02, 0.0, 0.05, 0.1]).astype(np.float32)}
    return logits, rng.random(rows, dtype=np.float32), rule


def draw(gpu, logits, u, rule):
    ids = torch.full((len(u),), -1, dtype=torch.int32, device="cuda")
    lp = torch.full((len(u),), float("nan"), device="cuda")
    given = {k: torch.from_numpy(v).cuda() for k, v in rule.items()}
    u = torch.from_numpy(u).cuda()
    torch.cuda.synchronize()
    gpu.sample_rows(logits, u, ids, logprobs=lp, **given)
    gpu.sync()
    return ids, lp


@pytest.mark.parametrize("part", range(4))
def test_draws_over_the_range(part):
    with closing(zc.Gpu(0)) as gpu, closing(zc.Gpu(0)) as other:
        for seed in range(part, CASES, 4):
            logits, u, rule = prepare(seed)
            again, u2, rule2 = prepare(seed)
            assert torch.equal(logits, again) and np.array_equal(u, u2)
            ids, lp = draw(gpu, logits, u, rule)
            ids2, lp2 = draw(other, again, u2, rule2)
            assert torch.equal(ids, ids2) and torch.equal(lp, lp2)
            for r, (i, p) in enumerate(zip(ids.tolist(), lp.tolist())):
                check_row(logits[r], float(u[r]), float(rule["temperature"][r]), int(rule["top_k"][r]), float(rule["top_p"][r]),
                          float(rule["min_p"][r]), i, p)
