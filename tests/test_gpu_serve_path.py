"""The serving operators in the model's own path (B200 only):
zynfer_cu_prefill_chunk and zynfer_cu_decode_drawn against zynfer_cu_prefill,
zynfer_cu_decode_step and the draw's definition.

Logits tolerance: both sides run the same linears on bf16 K/V; the attention
differs in the order of f32 sums (1e-6 of its output), which two layers and the
LM head (hidden 512, weights 0.05) carry to at most about 1e-4; bound: the
f32 path's 2e-3 (tolerances.F32_PATH).
"""
import numpy as np
import pytest

from oracle import oracle as O
from zynfer_b200 import cuda as zc

pytestmark = pytest.mark.gpu

ARCH = dict(vocab=4096, hidden=512, inter=1024, layers=2, n_q=4, n_kv=2, head_dim=128, max_pos=4096)
TOL = 2e-3


def make(max_batch=8, weights=zc.W_Q8):
    m = zc.Model(zc.Gpu(0), zc.Arch(**ARCH), weights, max_batch=max_batch, max_seqs=max_batch, max_seq_len=512, max_prefill=300)
    m.fill_synthetic(1, 0.05, 0.1)
    return m


def prompt(n):
    return O.synth_tokens(n, 1, 3, ARCH["vocab"])


@pytest.mark.parametrize("weights", [zc.W_Q8, zc.W_BF16])
@pytest.mark.parametrize("cuts", [(200,), (1, 199), (137, 16, 47), (64, 135, 1)])
def test_prefill_chunks_match_prefill(weights, cuts):
    m = make(weights=weights)
    ids = prompt(200)
    want, am = m.prefill(0, ids)
    at = 0
    for n in cuts:
        got, first = m.prefill_chunk(1, ids[at:at + n])
        at += n
    assert m.seq_len(1) == 200 and first == am
    assert float(np.abs(got - want).max()) <= TOL
    # the cache they leave is one decode goes on with
    a, la = m.decode_step([0], [am], want_logits=True)
    b, lb = m.decode_step([1], [am], want_logits=True)
    assert float(np.abs(la - lb).max()) <= TOL and a[0] == b[0]


@pytest.mark.parametrize("window,sinks", [(32, 4), (1, 0), (64, 0)])
def test_windowed_chunk_is_windowed_decode(window, sinks):
    m = make()
    ids = prompt(120)
    m.prefill_chunk(0, ids[:70], window=window, sinks=sinks)
    m.prefill_chunk(1, ids[:70], window=window, sinks=sinks)
    got, am = m.prefill_chunk(0, ids[70:], window=window, sinks=sinks)
    for t in ids[70:]:
        drawn, lp = m.decode_drawn([1], [t], [0.5], temperature=0.0, window=window, sinks=sinks)
    assert drawn[0] == am and lp[0] == 0.0
    full, _ = m.prefill(2, ids)
    assert float(np.abs(got - full).max()) > 10 * TOL  # the window matters here
    for layer in range(2):
        for which in (False, True):
            a, b = m.kv(0, layer, which), m.kv(1, layer, which)
            assert float(np.abs(a - b).max()) <= 0.05  # a bf16 step of values up to about 4


def test_many_answers_from_one_prompt():
    """Fork, then decode together: the tokens each sequence would draw alone."""
    m, alone = make(), make()
    ids = prompt(203)
    am = m.prefill(0, ids, want_logits=False)
    for s in range(1, 6):
        m.seq_fork(s, 0, 203)
    for s in range(6):
        alone.prefill(s, ids, want_logits=False)
    tok, tok1 = [am] * 6, [am] * 6
    rng = np.random.default_rng(5)
    for step in range(20):
        u = rng.random(6, dtype=np.float32)
        tok, lp = m.decode_drawn(range(6), tok, u, temperature=0.9, top_k=[0, 20, 50, 0, 5, 1], top_p=0.95, min_p=0.01)
        assert np.all(lp <= 0.0) and lp[5] == 0.0
        for s in range(6):
            d, _ = alone.decode_drawn([s], [tok1[s]], u[s:s + 1], temperature=0.9, top_k=[0, 20, 50, 0, 5, 1][s], top_p=0.95, min_p=0.01)
            tok1[s] = d[0]
        assert list(tok) == list(tok1), step
    assert len(set(map(int, tok[:5]))) > 1


def test_greedy_draws_are_decode_step():
    m, ref = make(), make()
    ids = prompt(60)
    a, b = m.prefill(0, ids, False), ref.prefill(0, ids, False)
    for _ in range(12):
        got, lp = m.decode_drawn([0], [a], [0.9], temperature=0.0)
        want = ref.decode_step([0], [b])
        assert got[0] == want[0] and lp[0] == 0.0
        a, b = int(got[0]), int(want[0])
    assert m.seq_len(0) == 72
    # and the two kinds of step mix
    assert m.decode_step([0], [a])[0] == ref.decode_drawn([0], [b], [0.1], temperature=0.0)[0][0]


def test_refusals():
    m = make(max_batch=2)
    ids = prompt(10)
    m.prefill(0, ids, False)
    for call in (
        lambda: m.prefill_chunk(0, []),
        lambda: m.prefill_chunk(0, [4096]),
        lambda: m.prefill_chunk(2, ids),
        lambda: m.prefill_chunk(1, prompt(301)),
        lambda: m.decode_drawn([0, 0], [1, 2], [0.1, 0.2]),
        lambda: m.decode_drawn([0, 1, 1], [1, 2, 3], [0.1, 0.2, 0.3]),
        lambda: m.decode_drawn([0], [4096], [0.1]),
        lambda: m.decode_drawn([0], [1], [0.1, 0.2]),
    ):
        with pytest.raises(zc.InvalidArgument):
            call()
    m.prefill_chunk(1, prompt(300), want_logits=False)
    with pytest.raises(zc.InvalidArgument):
        m.prefill_chunk(1, prompt(213))
    m.gpu.set_fail_at("launch")
    with pytest.raises(zc.LaunchFailed):
        m.decode_drawn([0], [1], [0.1])
    assert m.seq_len(0) == 10
    m.decode_drawn([0], [1], [0.1])
    assert m.seq_len(0) == 11


def test_cli_sample(capsys):
    import json

    from zynfer_b200 import cli
    base = ["sample", "--backend", "cuda", "--prompt-tokens", "1100", "--samples", "3", "--new-tokens", "4", "--seed", "7"]

    def run(*flags):
        assert cli.main([*base, *flags]) == 0
        return json.loads(capsys.readouterr().out)

    a, b = run("--temperature", "0.9", "--top-p", "0.95"), run("--temperature", "0.9", "--top-p", "0.95")
    assert a["ids"] == b["ids"] and a["logprobs"] == b["logprobs"]       # the seed decides
    assert np.array(a["ids"]).shape == (3, 4) and all(x < 0 for x in a["logprobs"])
    greedy = run("--temperature", "0")
    assert greedy["ids"][0] == greedy["ids"][1] == greedy["ids"][2] and greedy["logprobs"] == [0.0] * 3
    windowed = run("--temperature", "0", "--window", "128", "--sinks", "4")
    assert np.array(windowed["ids"]).shape == (3, 4)
