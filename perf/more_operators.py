"""What each request of a batch brings of its own, case by case: a low-rank adapter beside the projections that all requests share, and its own
way of choosing tokens. Inputs, one pass through an operator in plain torch operations or through this package's entry points, the bytes and
operations a pass cannot do without, and what the same pass gives in 64 bits.

Kinds of case, and what each stands for in real use:

``linear``   a projection of a step's tokens beside the adapters of their requests: y_t = W x_t + c_s B_s (A_s x_t), s the adapter of token t's
             request (-1: none). A stacked projection (q|k|v) has an A for each of its parts and a B for the part's rows
``glu``      the stacked gate|up projection beside the adapters, with silu(gate) * up behind it
``sample``   a token per row from its logits and a random number in [0, 1) given for it: temperature, the top_k likeliest, of those the likeliest
             whose mass before them is below top_p, of those the ones at least min_p times as likely as the likeliest; then the first token, in
             the order of the vocabulary, up to which there is more mass than the random number's share. Temperature 0: the likeliest token"""

import math

import torch

own = False

DEV = "cuda:0"


def listed():
    return [
        # one user with an adapter of theirs: the q|k|v product of the 1.7b preset, all latency
        {"name": "qkv_one_token", "kind": "linear", "k": 2048, "parts": "2048,1024,1024", "rank": 16, "slots": 8, "rows": "1@5", "dtype": "bf16"},
        # eight users, some on the same adapter, one without: the down projection of the 8b preset
        {"name": "down_8_tokens", "kind": "linear", "k": 12288, "parts": "4096", "rank": 16, "slots": 8, "rows": "1@0,1@3,1@3,1@7,1@-1,1@0,1@5,1@1", "dtype": "bf16"},
        # a full house on sixteen adapters: q|k|v of the 8b preset
        {"name": "qkv_64_tokens", "kind": "linear", "k": 4096, "parts": "4096,1024,1024", "rank": 32, "slots": 16,
         "rows": ",".join("1@%d" % ((7 * i) % 17 - 1) for i in range(64)), "dtype": "bf16"},
        # a mixed step: 24 decoding requests in front of a prompt of odd length, the attention's output projection
        {"name": "o_mixed_925", "kind": "linear", "k": 4096, "parts": "4096", "rank": 16, "slots": 8, "rows": ",".join(["1@%d" % (i % 8) for i in range(24)] + ["901@2"]), "dtype": "bf16"},
        # a full portion of prompts: two requests, two adapters
        {"name": "qkv_prompt_2048", "kind": "linear", "k": 4096, "parts": "4096,1024,1024", "rank": 16, "slots": 8, "rows": "1531@4,517@1", "dtype": "bf16"},
        # the 32-bit mode (what numerics are checked with)
        {"name": "qkv_float32_300", "kind": "linear", "k": 1024, "parts": "2048,1024,1024", "rank": 8, "slots": 4, "rows": "171@3,1@0,128@-1", "dtype": "f32"},
        # eight users again, the gated feed-forward of the 8b preset
        {"name": "glu_8_tokens", "kind": "glu", "k": 4096, "parts": "12288,12288", "rank": 16, "slots": 8, "rows": "1@0,1@3,1@3,1@7,1@-1,1@0,1@5,1@1", "dtype": "bf16"},
        # prompts of five requests through it, wide adapters
        {"name": "glu_prompt_2048", "kind": "glu", "k": 4096, "parts": "12288,12288", "rank": 64, "slots": 8, "rows": "700@2,33@6,1@-1,801@0,513@2", "dtype": "bf16"},
        # one conversation, the usual settings of a chat
        {"name": "sample_one_row", "kind": "sample", "rows": 1, "vocab": 151936, "temperature": 0.7, "top_k": 20, "top_p": 0.8, "min_p": 0.0, "mixed": False},
        # eight rows, the nucleus alone
        {"name": "sample_8_nucleus", "kind": "sample", "rows": 8, "vocab": 151936, "temperature": 1.0, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "mixed": False},
        # a full house, every request with settings of its own (greedy ones among them)
        {"name": "sample_64_mixed", "kind": "sample", "rows": 64, "vocab": 151936, "temperature": 0.9, "top_k": 50, "top_p": 0.9, "min_p": 0.05, "mixed": True},
        # a small vocabulary of odd size
        {"name": "sample_17_of_32001", "kind": "sample", "rows": 17, "vocab": 32001, "temperature": 1.3, "top_k": 0, "top_p": 1.0, "min_p": 0.02, "mixed": False},
    ]


def draw(rng):
    """One more case of the same ranges; sizes spread over their logarithm."""

    def about(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["linear", "linear", "linear", "glu", "glu", "sample", "sample"])
    if kind == "sample":
        vocab = rng.choice([151936, 151936, about(1000, 151936)])
        return {"kind": kind, "rows": about(1, 64), "vocab": vocab, "temperature": round(rng.uniform(0.2, 1.5), 2), "top_k": rng.choice([0, 0, about(1, 1000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 2)]), "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.3), 2)]),
                "mixed": rng.random() < 0.4}
    dtype = rng.choice(["bf16"] * 5 + ["f32"])
    most = 400 if dtype == "f32" else 2048
    slots = rng.choice([1, 2, 4, 8, 16])
    count = about(1, 64)
    if rng.random() < 0.5:
        lens = [1] * count
    else:
        lens = [1] * (count // 2) + [about(1, max(1, most // 4)) for _ in range(rng.choice([1, 1, 2, 3, 4]))]
    rows = ",".join("%d@%d" % (n, rng.randint(-1, slots - 1)) for n in lens)
    k = 8 * about(32, 128 if dtype == "f32" else 512)
    if kind == "glu":
        width = 8 * about(32, 128 if dtype == "f32" else 1536)
        parts = "%d,%d" % (width, width)
    elif rng.random() < 0.5:
        kv = 128 * rng.choice([1, 2, 4, 8])
        parts = "%d,%d,%d" % (kv * rng.choice([1, 2, 4]), kv, kv)
    else:
        parts = "%d" % (8 * about(32, 512))
    return {"kind": kind, "k": k, "parts": parts, "rank": 8 * about(1, 8), "slots": slots, "rows": rows, "dtype": dtype}


def _rows(case):
    """(tokens, adapter) of every request of the step."""
    return [tuple(int(x) for x in r.split("@")) for r in case["rows"].split(",")]


def _parts(case):
    return [int(x) for x in case["parts"].split(",")]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = {"case": case}
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a few likely tokens above a broad rest, as behind a trained head
        logits = torch.randn((rows, vocab), generator=gen, device=DEV) * 2.0
        peaks = torch.randint(0, vocab, (rows, 32), generator=gen, device=DEV)
        logits.scatter_add_(1, peaks, 4 + 8 * torch.rand((rows, 32), generator=gen, device=DEV))
        st["logits"] = logits
        st["uniform"] = torch.rand((rows,), generator=gen, device=DEV, dtype=torch.float64)
        t, k, p, m = (torch.full((rows,), float(case[n]), device=DEV) for n in ("temperature", "top_k", "top_p", "min_p"))
        if case["mixed"]:  # every row has settings of its own; some leave one out
            pick = torch.rand((4, rows), generator=gen, device=DEV)
            t = torch.where(pick[0] < 0.1, 0.0, t * (0.5 + pick[0]))
            k = torch.where(pick[1] < 0.4, 0.0, torch.floor(k * (0.1 + 2 * pick[1])))
            p = torch.where(pick[2] < 0.3, 1.0, (p * (0.6 + 0.5 * pick[2])).clamp(max=1.0))
            m = torch.where(pick[3] < 0.5, 0.0, m * 2 * pick[3])
        st.update(temperature=t, top_k=k.to(torch.int32), top_p=p, min_p=m, tokens=torch.empty((rows,), dtype=torch.int32, device=DEV))
        return st
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    rows, parts, k, r, slots = _rows(case), _parts(case), case["k"], case["rank"], case["slots"]
    n, tokens = sum(parts), sum(c for c, _ in rows)

    def made(*shape, std):
        return (torch.randn(shape, generator=gen, device=DEV) * std).to(dt)

    st["x"] = made(tokens, k, std=1.0)
    st["w"] = made(n, k, std=0.7 * k ** -0.5)
    # an adapter's part of the output is a fraction of the projection's; c = alpha / rank
    st["a"] = made(slots, len(parts) * r, k, std=k ** -0.5)
    st["b"] = made(slots, n, r, std=0.25 * r ** -0.5)
    st["scale"] = 0.5 + 1.5 * torch.rand((slots,), generator=gen, device=DEV)
    st["slot_of_row"] = torch.tensor([s for _, s in rows], dtype=torch.int32, device=DEV)
    st["row_of_token"] = torch.repeat_interleave(torch.arange(len(rows), device=DEV), torch.tensor([c for c, _ in rows], device=DEV)).to(torch.int32)
    st["out"] = torch.empty((tokens, n // 2 if case["kind"] == "glu" else n), dtype=dt, device=DEV)
    return st


# ------------------------------------------------------------------ one pass
def _plain_linear(st):
    """float32 [tokens, n]: the shared projection and the adapters'."""
    case = st["case"]
    parts, r = _parts(case), case["rank"]
    x = st["x"].float()
    y = torch.matmul(x, st["w"].float().T)
    slot = st["slot_of_row"][st["row_of_token"].long()]
    for s in range(case["slots"]):
        mine = (slot == s).float()[:, None]
        v = torch.matmul(x * mine, st["a"][s].float().T) * st["scale"][s]
        at = 0
        for p, width in enumerate(parts):
            y[:, at:at + width] += torch.matmul(v[:, p * r:(p + 1) * r], st["b"][s, at:at + width].float().T)
            at += width
    return y


def _plain_sample(st):
    """In 64 bits: which tokens a border leaves out hangs on sums of 150,000 terms."""
    z = st["logits"].double()
    rows, vocab = z.shape
    t = st["temperature"].double()[:, None]
    greedy = t <= 0
    z = z / torch.where(greedy, torch.ones_like(t), t)
    z, order = torch.sort(z, dim=1, descending=True, stable=True)
    w = torch.exp(z - z[:, :1])
    place = torch.arange(vocab, device=DEV).expand(rows, vocab)
    k = st["top_k"].long()[:, None]
    w = torch.where((k > 0) & (place >= k), 0.0, w)
    before = torch.cumsum(w, 1) - w
    p = st["top_p"].double()[:, None]
    cut = torch.where((p < 1) & (before >= p * w.sum(1, keepdim=True)), 0.0, w)
    cut[:, :1] = w[:, :1]
    cut = torch.where(cut < st["min_p"].double()[:, None], 0.0, cut)
    kept = torch.zeros_like(cut).scatter_(1, order, cut)
    total = torch.cumsum(kept, 1)
    token = (total <= st["uniform"][:, None] * total[:, -1:]).sum(1)
    st["tokens"].copy_(torch.where(greedy[:, 0], order[:, 0], token))
    return st["tokens"]


def run(state):
    st, case = state, state["case"]
    if own:
        from miniserve_b200 import ops

        if case["kind"] == "sample":
            ops.sample_filtered(st["tokens"], st["logits"], st["temperature"], st["uniform"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
            return st["tokens"]
        if "low_rank" not in st:  # the weights as the engine holds them
            ends = [sum(_parts(case)[:i + 1]) for i in range(len(_parts(case)))]
            st["low_rank"] = ops.LowRank(st["a"], st["b"], st["scale"], tuple(ends))
        # a step's, made in the pass with all that products make of it (a model's layers share one)
        rows = ops.AdapterRows(st["slot_of_row"], st["row_of_token"])
        product = ops.linear_silu_mul if case["kind"] == "glu" else ops.linear
        product(st["x"], st["w"], out=st["out"], low_rank=st["low_rank"], adapter_rows=rows)
        return st["out"]
    if case["kind"] == "sample":
        return _plain_sample(st)
    y = _plain_linear(st)
    if case["kind"] == "glu":
        half = y.shape[1] // 2
        gate = y[:, :half]
        y = gate / (1 + torch.exp(-gate)) * y[:, half:]
    st["out"].copy_(y)
    return st["out"]


# ------------------------------------------------------------------ what a pass needs, and its result in 64 bits
def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 28), "flops": case["rows"] * case["vocab"] * 8}
    rows, parts, k, r = _rows(case), _parts(case), case["k"], case["rank"]
    item, n, tokens = (2 if case["dtype"] == "bf16" else 4), sum(parts), sum(c for c, _ in rows)
    adapted, used = sum(c for c, s in rows if s >= 0), len({s for _, s in rows if s >= 0})
    outputs = n // 2 if case["kind"] == "glu" else n
    return {"bytes": item * (tokens * k + n * k + used * r * (len(parts) * k + n) + tokens * outputs) + 4 * tokens,
            "flops": 2 * tokens * k * n + 2 * adapted * r * (len(parts) * k + n)}


def _exact_row(logits, t, k, p, m, u):
    """The token of one row, by sums over sorted and unsorted lists of its own."""
    z = logits.double()
    if t <= 0:
        return int((z == z.max()).nonzero()[0, 0])
    w = torch.exp(z / t - z.max() / t)
    by_size = torch.argsort(z, descending=True, stable=True)
    if 0 < k < z.numel():
        by_size = by_size[:k]
    if p < 1:
        sums = torch.cumsum(w[by_size], 0)
        target = p * float(sums[-1])
        by_size = by_size[:max(1, int((torch.cat([sums.new_zeros(1), sums[:-1]]) < target).sum()))]
    by_size = by_size[w[by_size] >= m]
    kept = torch.sort(by_size).values
    sums = torch.cumsum(w[kept], 0)
    at = int(torch.searchsorted(sums, torch.tensor(u * float(sums[-1]), dtype=torch.float64, device=DEV), right=True))
    return int(kept[min(at, kept.numel() - 1)])


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "sample":
        settings = [st[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p", "uniform")]
        return torch.tensor([_exact_row(st["logits"][i], *(s[i] for s in settings)) for i in range(case["rows"])], dtype=torch.int32, device=DEV)
    parts, r = _parts(case), case["rank"]
    x = st["x"].double()
    out, at = [], 0
    y = x @ st["w"].double().T
    for tokens, slot in _rows(case):
        mine, at = slice(at, at + tokens), at + tokens
        if slot < 0:
            out.append(y[mine])
            continue
        a, b = st["a"][slot].double(), st["b"][slot].double()
        # the adapter as a matrix of the projection's own size, a part after the other
        whole = torch.cat([bp @ a[i * r:(i + 1) * r] for i, bp in enumerate(torch.split(b, parts))])
        out.append(y[mine] + float(st["scale"][slot]) * (x[mine] @ whole.T))
    y = torch.cat(out)
    if case["kind"] == "glu":
        gate, up = y.chunk(2, 1)
        y = gate * torch.sigmoid(gate) * up
    return y
