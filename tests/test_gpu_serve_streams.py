"""The serving calls in the order of the caller's stream (B200 only): their
tensors are written late on torch's current stream, their results are read
there, and nothing else waits."""
import numpy as np
import pytest

from test_gpu_serve_attn import D, make, normal
from zynfer_b200 import cuda as zc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

LATE = 40_000_000  # clock cycles, about 20 ms


def late(*given):
    """Tensors of zeros that take their values only after a while on the current stream."""
    empty = [torch.zeros_like(x) for x in given]
    torch.cuda._sleep(LATE)
    for e, x in zip(empty, given):
        e.copy_(x)
    return empty


@pytest.fixture(params=["default", "side"])
def stream(request):
    s = torch.cuda.Stream() if request.param == "side" else torch.cuda.default_stream()
    with torch.cuda.stream(s):
        yield s


@pytest.mark.parametrize("tokens", [None, 1, 70])
def test_attention_follows_the_current_stream(stream, tokens):
    m = make(n_kv=4)
    k, v = normal(1, 4, 300, D, dtype=torch.bfloat16), normal(2, 4, 300, D, dtype=torch.bfloat16)
    for s in range(4):
        m.kv_write(s, 0, 0, k, v)
    q = normal(3, 4, *([] if tokens is None else [tokens]), 8, D)

    def call(q, out):
        if tokens is None:
            m.attn_shared(0, range(4), q, out)
        else:
            m.attn_window(0, range(4), q, out, window=100, sinks=2)
    torch.cuda.synchronize()
    want = torch.zeros_like(q)
    call(q, want)
    torch.cuda.synchronize()
    assert want.any()
    x, = late(q)
    out = torch.zeros_like(q)
    call(x, out)
    got = out.clone()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_cache_writes_follow_the_current_stream(stream):
    m = make(n_kv=2)
    k, v = normal(1, 2, 100, D, dtype=torch.bfloat16), normal(2, 2, 100, D, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    a, b = late(k, v)
    m.kv_write(0, 0, 0, a, b)
    a.zero_()  # after the call, on the same stream
    b.zero_()
    torch.cuda.synchronize()
    m.gpu.sync()
    assert np.array_equal(m.kv(0, 0, False), k.float().cpu().numpy())
    assert np.array_equal(m.kv(0, 0, True), v.float().cpu().numpy())


def test_draws_follow_the_current_stream(stream):
    gpu = zc.Gpu(0)
    logits, u = 3.0 * normal(5, 6, 5000), torch.rand(6, generator=torch.Generator().manual_seed(6)).cuda()
    torch.cuda.synchronize()

    def call(l, u):
        ids, lp = torch.full((6,), -1, dtype=torch.int32, device="cuda"), torch.zeros(6, device="cuda")
        gpu.sample_rows(l, u, ids, lp)
        return ids.clone(), lp.clone()
    want = call(logits, u)
    torch.cuda.synchronize()
    got = call(*late(logits, u))
    torch.cuda.synchronize()
    assert (want[0] >= 0).all() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    gpu.close()


def test_a_contexts_calls_keep_their_order_across_streams():
    """Calls on different streams, and the context's own work between them, see what the call before wrote."""
    m = make(n_kv=2)
    k, v = normal(1, 2, 100, D, dtype=torch.bfloat16), normal(2, 2, 100, D, dtype=torch.bfloat16)
    k2, v2 = normal(3, 2, 100, D, dtype=torch.bfloat16), normal(4, 2, 100, D, dtype=torch.bfloat16)
    q = normal(5, 2, 4, D)
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.default_stream()]
    want = []
    for a, b in ((k, v), (k2, v2)):
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        m.kv_write(0, 0, 0, a, b)
        m.kv_write(1, 0, 0, a, b)
        m.attn_shared(0, [0, 1], q, out)
        torch.cuda.synchronize()
        want.append(out)
    assert not torch.equal(*want)
    m.seq_reset(0)
    m.seq_reset(1)
    outs = []
    for i in range(6):
        a, b = ((k, v), (k2, v2))[i % 2]
        with torch.cuda.stream(streams[i % 3]):
            torch.cuda._sleep(LATE // 8)
        m.seq_reset(1)                                               # (it may hold blocks of sequence 0)
        m.kv_write(0, 0, 0, a, b, stream=streams[i % 3])             # behind the sleep
        if i % 2:
            m.seq_fork(1, 0, 100)                                    # on the context's own stream
        else:
            m.kv_write(1, 0, 0, a, b, stream=streams[(i + 2) % 3])
        with torch.cuda.stream(streams[(i + 1) % 3]):
            out = torch.zeros_like(q)
            m.attn_shared(0, [0, 1], q, out)
        outs.append(out)
    m.gpu.sync()
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, want[i % 2])


def test_the_library_keeps_to_its_own_stream_until_one_is_named():
    """zynfer_cu_use_stream by itself: named, changed, and given back."""
    m = make(n_kv=2)
    lib, own = zc.lib(), (1 << 64) - 1
    k = normal(1, 2, 40, D, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for seq, handle in enumerate((own, side.cuda_stream, 0, own)):
        assert lib.zynfer_cu_use_stream(m.gpu.h, handle) == zc.OK
        x = k
        if handle not in (own, 0):
            with torch.cuda.stream(side):
                x, = late(k)
        assert lib.zynfer_cu_kv_write(m.gpu.h, seq, 0, 0, 40, x.data_ptr(), x.data_ptr(), zc.DT_BF16) == zc.OK
    m.gpu.sync()
    for seq in range(4):
        assert np.array_equal(m.kv(seq, 0, False), k.float().cpu().numpy())
