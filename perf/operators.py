"""The serving operators of this backend as measured cases: decode attention
that reads a batch's common prompt once (`attn_shared`), sliding-window
attention whose first positions stay visible (`attn_window`, single tokens and
chunks), and the draw of next tokens from given random numbers
(`sample_rows`). `own` False computes them in elementary torch operations in
32 bits; True calls zynfer_b200."""
import torch

own = False

D = 128  # head dimension of the cache; two query heads per kv head
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
WEIGHT_ONE = 2.0 ** 33  # the draw's integer weight of the largest logit


def listed():
    return [
        # four answers to one short prompt: the latency of a small call
        {"name": "shared 4 x 512", "op": "shared", "prompts": 1, "samples": 4, "prefix": 512, "suffix": 16, "kv_heads": 8, "dtype": "f32"},
        # 64 answers to one prompt of ordinary length, part of the way through their own tokens
        {"name": "shared 64 x 4096", "op": "shared", "prompts": 1, "samples": 64, "prefix": 4096, "suffix": 200, "kv_heads": 8, "dtype": "f32"},
        # several prompts at once, none of whose lengths ends a cache block
        {"name": "shared 3 x 11 x 1531", "op": "shared", "prompts": 3, "samples": 11, "prefix": 1531, "suffix": 77, "kv_heads": 8, "dtype": "f32"},
        # many samples of one long document, 16-bit activations
        {"name": "shared 128 x 16384 bf16", "op": "shared", "prompts": 1, "samples": 128, "prefix": 16384, "suffix": 256, "kv_heads": 8, "dtype": "bf16"},
        # one conversation, token by token
        {"name": "window decode 1", "op": "window", "batch": 1, "tokens": 1, "length": 4096, "window": 1024, "sinks": 4, "kv_heads": 8, "dtype": "f32"},
        # a full serving batch of uneven lengths
        {"name": "window decode 64", "op": "window", "batch": 64, "tokens": 1, "length": 4096, "window": 1024, "sinks": 4, "kv_heads": 8, "dtype": "f32"},
        # the next chunk of a prompt after 1200 cached positions, odd sizes
        {"name": "window chunk 301", "op": "window", "batch": 2, "tokens": 301, "length": 1501, "window": 250, "sinks": 5, "kv_heads": 4, "dtype": "f32"},
        # a long prompt as one chunk, 16-bit activations
        {"name": "window chunk 8192 bf16", "op": "window", "batch": 1, "tokens": 8192, "length": 8192, "window": 1024, "sinks": 16, "kv_heads": 8, "dtype": "bf16"},
        # one sequence's next token, the usual mix of rules
        {"name": "sample 1", "op": "sample", "rows": 1, "vocab": 151936, "rule": "top", "dtype": "f32"},
        # a serving batch, each request with its own rule
        {"name": "sample 64 mixed", "op": "sample", "rows": 64, "vocab": 151936, "rule": "mixed", "dtype": "f32"},
        # a small odd vocabulary
        {"name": "sample 5 x 4099", "op": "sample", "rows": 5, "vocab": 4099, "rule": "mixed", "dtype": "bf16"},
        # many rows of the whole softmax, 16-bit logits with their many ties
        {"name": "sample 256 bf16", "op": "sample", "rows": 256, "vocab": 151936, "rule": "whole", "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["shared", "window", "window", "sample"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "shared":
        prompts = rng.choice([1, 1, 2, 3, 4])
        samples = _spread(rng, 1, 128 // prompts)
        return {"op": op, "prompts": prompts, "samples": samples, "prefix": _spread(rng, 16, 16384 // prompts),
                "suffix": _spread(rng, 1, 256), "kv_heads": rng.choice([2, 4, 8]), "dtype": dtype}
    if op == "window":
        kv_heads, window, sinks = rng.choice([2, 4, 8]), _spread(rng, 16, 1024), rng.choice([0, 1, 4, 16, 33])
        if rng.random() < 0.5:
            return {"op": op, "batch": _spread(rng, 1, 64), "tokens": 1, "length": _spread(rng, 2, 4096),
                    "window": window, "sinks": sinks, "kv_heads": kv_heads, "dtype": dtype}
        batch, tokens = rng.choice([1, 1, 2, 3]), _spread(rng, 2, 4096)
        length = tokens + rng.choice([0, _spread(rng, 1, 4096)])
        if batch > 1:
            tokens, length = (tokens + 1) // 2, (length + 1) // 2
        return {"op": op, "batch": batch, "tokens": tokens, "length": length, "window": window, "sinks": sinks,
                "kv_heads": kv_heads, "dtype": dtype}
    return {"op": op, "rows": _spread(rng, 1, 256), "vocab": _spread(rng, 1000, 151936),
            "rule": rng.choice(["top", "mixed", "whole"]), "dtype": dtype}


# ---- sizes that follow from a case alone

def _shared_lens(case):
    """Prompt lengths, and each row's own positions after its prompt (at least its current token)."""
    p = case["prefix"]
    prefix = [max(1, p - g * p // 5) for g in range(case["prompts"])]
    rows = case["prompts"] * case["samples"]
    return prefix, [1 + (7919 * i + 13) % case["suffix"] for i in range(rows)]


def _window_lens(case):
    """Cached positions of each sequence, the chunk's own among them."""
    least = max(case["tokens"], (case["length"] + 1) // 2)
    return [case["length"] - (7919 * i) % (case["length"] - least + 1) for i in range(case["batch"])]


def _visible(length, tokens, window, sinks):
    """(query, key) pairs inside the mask and positions that any of the queries sees."""
    pairs, first = 0, length - tokens
    for pos in range(first, length):
        low = max(0, pos - window + 1)
        pairs += pos + 1 - low + min(sinks, low)
    low = max(0, first - window + 1)
    return pairs, length - low + min(sinks, low)


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * DTYPES[case["dtype"]].itemsize + 28 * case["rows"], "flops": 4 * n}
    heads, size = 2 * case["kv_heads"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "shared":
        prefix, own_len = _shared_lens(case)
        rows = len(own_len)
        keys = sum(prefix) + sum(own_len)
        pairs = sum(prefix[i // case["samples"]] + n for i, n in enumerate(own_len))
    else:
        rows, pairs, keys = case["batch"] * case["tokens"], 0, 0
        for n in _window_lens(case):
            p, k = _visible(n, case["tokens"], case["window"], case["sinks"])
            pairs, keys = pairs + p, keys + k
    return {"bytes": keys * case["kv_heads"] * D * 2 * 2 + 2 * rows * heads * D * size, "flops": 4 * D * heads * pairs}


# ---- inputs

def _model(case, layers, max_batch, max_seqs, max_len, blocks):
    """A context with the cache that the attention reads (the weights are not used)."""
    from zynfer_b200 import cuda as zc
    gpu = zc.Gpu(0)
    arch = zc.Arch(vocab=1024, hidden=512, inter=512, layers=layers, n_q=2 * case["kv_heads"], n_kv=case["kv_heads"],
                   head_dim=D, max_pos=max_len)
    return zc.Model(gpu, arch, zc.W_BF16, max_batch=max_batch, max_seqs=max_seqs, max_seq_len=max_len,
                    kv_blocks=blocks, max_prefill=16)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)

    dtype = DTYPES[case["dtype"]]
    if case["op"] == "sample":
        return _prepare_sample(case, g, normal, dtype)
    h = case["kv_heads"]
    if case["op"] == "shared":
        prefix, own_len = _shared_lens(case)
        rows = len(own_len)
        kp, vp = (normal(len(prefix), h, max(prefix), D, dtype=torch.bfloat16) for _ in range(2))
        ks, vs = (normal(rows, h, max(own_len), D, dtype=torch.bfloat16) for _ in range(2))
        q = normal(rows, 2 * h, D, dtype=dtype, scale=1.5)
        state = {"case": case, "q": q}
        if not own:
            state.update(kp=kp, vp=vp, ks=ks, vs=vs, prefix=torch.tensor(prefix, device="cuda"),
                         own_len=torch.tensor(own_len, device="cuda"))
            return state
        longest = max(prefix) + max(own_len)
        blocks = sum(n // 16 + 1 for n in prefix) + sum(n // 16 + 2 for n in own_len)
        torch.cuda.synchronize()
        m = state["model"] = _model(case, 1, rows, rows, longest, blocks)
        for i, n in enumerate(own_len):
            p, first = prefix[i // case["samples"]], i - i % case["samples"]
            if i == first:  # the prompt once, shared by its samples
                m.kv_write(i, 0, 0, kp[i // case["samples"], :, :p].contiguous(), vp[i // case["samples"], :, :p].contiguous())
                m.gpu.sync()
                for j in range(i + 1, i + case["samples"]):
                    m.seq_fork(j, i, p)
            m.kv_write(i, 0, p, ks[i, :, :n].contiguous(), vs[i, :, :n].contiguous())
            m.gpu.sync()
        state.update(seqs=list(range(rows)), out=torch.empty_like(q))
        return state
    lens = _window_lens(case)
    k, v = (normal(len(lens), h, max(lens), D, dtype=torch.bfloat16) for _ in range(2))
    q = normal(len(lens), case["tokens"], 2 * h, D, dtype=dtype, scale=1.5)
    state = {"case": case, "q": q}
    if not own:
        state.update(k=k, v=v, lens=torch.tensor(lens, device="cuda"))
        return state
    torch.cuda.synchronize()
    m = state["model"] = _model(case, 1, len(lens), len(lens), max(lens), sum(n // 16 + 1 for n in lens))
    for i, n in enumerate(lens):
        m.kv_write(i, 0, 0, k[i, :, :n].contiguous(), v[i, :, :n].contiguous())
        m.gpu.sync()
    state.update(seqs=list(range(len(lens))), out=torch.empty_like(q))
    return state


def _prepare_sample(case, g, normal, dtype):
    rows, vocab, rule = case["rows"], case["vocab"], case["rule"]
    logits = normal(rows, vocab, scale=2.5)
    # a model's logits: a broad body and a few tokens well above it (the larger where two meet: a plain scatter would
    # take either, and the inputs would not follow from the seed)
    at = torch.randint(vocab, (rows, 24), generator=g, device="cuda")
    logits.scatter_reduce_(1, at, 6.0 + 2.5 * torch.randn((rows, 24), generator=g, device="cuda"), "amax")
    logits = logits.to(dtype)
    if rule == "mixed":  # some vocabulary entries are ruled out, as by a grammar
        logits[::3, ::7] = float("-inf")

    def per_row(values, kind):
        values = torch.tensor(values, dtype=kind, device="cuda")
        pick = torch.randint(len(values), (rows,), generator=g, device="cuda")
        return values[pick] if rule == "mixed" else values[:1].repeat(rows)

    whole = rule == "whole"
    state = {
        "case": case, "logits": logits,
        "temperature": per_row([1.0] if whole else [0.8, 1.0, 0.6, 1.3, 0.0], torch.float32),
        "top_k": per_row([0] if whole else [50, 0, 20, 1, 1000], torch.int32),
        "top_p": per_row([1.0] if whole else [0.95, 1.0, 0.9, 0.8, 0.5], torch.float32),
        "min_p": per_row([0.0] if whole else [0.02, 0.0, 0.05, 0.1], torch.float32),
        "uniforms": torch.rand(rows, generator=g, device="cuda"),
    }
    if own:
        from zynfer_b200 import cuda as zc
        state.update(gpu=zc.Gpu(0), ids=torch.empty(rows, dtype=torch.int32, device="cuda"),
                     logprobs=torch.empty(rows, dtype=torch.float32, device="cuda"))
    return state


# ---- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        if op == "shared":
            state["model"].attn_shared(0, state["seqs"], state["q"], state["out"])
            return state["out"]
        if op == "window":
            state["model"].attn_window(0, state["seqs"], state["q"], state["out"], window=state["case"]["window"],
                                       sinks=state["case"]["sinks"])
            return state["out"]
        state["gpu"].sample_rows(state["logits"], state["uniforms"], state["ids"], logprobs=state["logprobs"],
                                 temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                                 min_p=state["min_p"])
        return {"ids": state["ids"], "logprobs": state["logprobs"]}
    return {"shared": _shared, "window": _window, "sample": _sample}[op](state)


def _shared(state):
    """softmax over a row's prompt and own positions: the products with a prompt are taken for all its rows together."""
    case, q, kp, vp, ks, vs = (state[n] for n in ("case", "q", "kp", "vp", "ks", "vs"))
    b, h, prompts = q.shape[0], case["kv_heads"], case["prompts"]
    r, p, s = b // prompts, kp.shape[2], ks.shape[2]
    x = q.float().view(b, h, 2, D) * D ** -0.5
    xp = x.view(prompts, r, h, 2, D).transpose(1, 2).reshape(prompts, h, 2 * r, D)
    over = torch.arange(p, device="cuda") >= state["prefix"][:, None]
    sp = (xp @ kp.float().transpose(2, 3)).masked_fill(over[:, None, None], float("-inf"))
    sp = sp.reshape(prompts, h, r, 2, p).transpose(1, 2).reshape(b, h, 2, p)
    over = torch.arange(s, device="cuda") >= state["own_len"][:, None]
    ss = (x @ ks.float().transpose(2, 3)).masked_fill(over[:, None, None], float("-inf"))
    top = torch.maximum(sp.amax(3, keepdim=True), ss.amax(3, keepdim=True))
    ep, es = torch.exp(sp - top), torch.exp(ss - top)
    total = ep.sum(3, keepdim=True) + es.sum(3, keepdim=True)
    ep = ep.reshape(prompts, r, h, 2, p).transpose(1, 2).reshape(prompts, h, 2 * r, p)
    op = (ep @ vp.float()).reshape(prompts, h, r, 2, D).transpose(1, 2).reshape(b, h, 2, D)
    return ((op + es @ vs.float()) / total).reshape(b, 2 * h, D).to(q.dtype)


def _window(state):
    """softmax over the positions j <= i with j < sinks or j > i - window, for the last `tokens` positions i."""
    case, q, k, v = (state[n] for n in ("case", "q", "k", "v"))
    b, t, h, length = q.shape[0], q.shape[1], case["kv_heads"], k.shape[2]
    x = (q.float() * D ** -0.5).view(b, t, h, 2, D).permute(0, 2, 3, 1, 4).reshape(b, h, 2 * t, D)
    i = (state["lens"][:, None] - t + torch.arange(t, device="cuda"))[:, :, None]
    j = torch.arange(length, device="cuda")
    seen = (j <= i) & ((j < case["sinks"]) | (j > i - case["window"]))
    scores = (x @ k.float().transpose(2, 3)).view(b, h, 2, t, length).masked_fill(~seen[:, None, None], float("-inf"))
    e = torch.exp(scores - scores.amax(4, keepdim=True))
    e = (e / e.sum(4, keepdim=True)).view(b, h, 2 * t, length)
    return (e @ v.float()).view(b, h, 2, t, D).permute(0, 3, 1, 2, 4).reshape(b, t, 2 * h, D).to(q.dtype)


def _sample(state):
    """Weights exp((l - max) / T) as whole numbers of 2^-33, those of at least min_p; in descending order (the lower
    index first among equals) the first top_k, of these the shortest run whose sum reaches top_p of theirs, and the
    first whose running sum exceeds u of that run's. Temperature 0 takes the largest."""
    l = state["logits"].float()
    greedy = (state["temperature"] <= 0)[:, None]
    inv_t = torch.where(greedy, 1.0, 1.0 / state["temperature"][:, None])
    top_k = torch.where(greedy, 1, torch.where(state["top_k"][:, None] > 0, state["top_k"][:, None], l.shape[1]))
    top = l.amax(1, keepdim=True)
    x = torch.where(l == top, 0.0, (l - top) * inv_t)
    e = torch.exp(x)
    w = torch.where(e >= state["min_p"][:, None], torch.round(e * WEIGHT_ONE), 0.0).long()
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    w = w.gather(1, order)
    rank = torch.arange(l.shape[1], device="cuda")
    w = w.masked_fill(rank >= top_k, 0)
    run_sum = w.cumsum(1)
    reach = run_sum[:, -1:].double() * state["top_p"][:, None].double()
    w = w.masked_fill(((run_sum - w).double() >= reach) & (rank > 0), 0)
    run_sum = w.cumsum(1)
    total = run_sum[:, -1:]
    target = torch.minimum((state["uniforms"][:, None].double() * total.double()).long(), total - 1)
    at = (run_sum <= target).sum(1, keepdim=True)
    token = order.gather(1, at)
    logprob = x.gather(1, token) - torch.log(total.double() / WEIGHT_ONE).float()
    return {"ids": token[:, 0].int(), "logprobs": logprob[:, 0]}


# ---- the same from the definitions in 64 bits

def _attend64(q, k, v, seen=None):
    """q [n, D] over k, v [m, D]: sum_j exp(q k_j / sqrt D) v_j / sum_j exp(q k_j / sqrt D)."""
    s = q.double() @ k.double().T / D ** 0.5
    if seen is not None:
        s = torch.where(seen, s, torch.full_like(s, float("-inf")))
    p = torch.softmax(s, 1)
    return p @ v.double()


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "sample":
        return _exact_sample(s)
    q = s["q"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    if case["op"] == "shared":
        prefix, own_len = _shared_lens(case)
        for i, n in enumerate(own_len):
            g = i // case["samples"]
            for h in range(case["kv_heads"]):
                k = torch.cat([s["kp"][g, h, :prefix[g]], s["ks"][i, h, :n]])
                v = torch.cat([s["vp"][g, h, :prefix[g]], s["vs"][i, h, :n]])
                out[i, 2 * h:2 * h + 2] = _attend64(q[i, 2 * h:2 * h + 2], k, v)
        return out
    for b, n in enumerate(_window_lens(case)):
        i = torch.arange(n - case["tokens"], n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        seen = (j <= i) & ((i - j < case["window"]) | (j < case["sinks"]))
        for h in range(2 * case["kv_heads"]):
            out[b, :, h] = _attend64(q[b, :, h], s["k"][b, h // 2, :n], s["v"][b, h // 2, :n], seen)
    return out


def _exact_sample(s):
    """The drawn ids are whole numbers; what a drawn token's log-probability is follows from the sets in 64 bits."""
    ids = _sample(s)["ids"]
    got = []
    for r in range(len(ids)):
        l = s["logits"][r].double()
        t, k, p, least = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            got.append(0.0)
            continue
        v, order = torch.sort(l, descending=True, stable=True)
        e = torch.exp((v - v[0]) / t)
        e = e[e >= least]
        e = e[:int(k)] if k > 0 else e
        c = torch.cumsum(e, 0)
        e = e[:int((c < p * c[-1] * (1 - 1e-12)).sum()) + 1]
        got.append(float((l[int(ids[r])] - v[0]) / t - torch.log(e.sum())))
    return {"ids": None, "logprobs": torch.tensor(got, dtype=torch.float64)}
