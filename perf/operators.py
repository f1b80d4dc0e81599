"""The paged cache of keys and values in 8 bits, case by case: inputs, one pass through an operator in plain torch operations or through
this package's entry points, the bytes and operations a pass cannot do without, and what the same pass gives in 64 bits.

A head's vector of d numbers is held as d codes of 8 bits (4 of exponent, 3 of mantissa: ``torch.float8_e4m3fn``) and one byte b: it
stands for code * 2^(b - 127). The exponent e = b - 127 is the smallest with max |x| <= 448 * 2^e, kept within [-60, 7]; numbers
beyond 448 * 2^7 become that; a vector with a number that is not finite has b = 255 and stands for NaN. Codes lie in pages
[pages, kv heads, page size, d], their exponents in [pages, kv heads, page size].

Kinds of case, and what each stands for in real use:

``write``    a step's q|k|v projection: norm per head, rotation, queries out, keys and values quantised into their pages; what the pages
             then hold of the step's tokens is read back (as a copy of them for elsewhere would be)
``read``     the keys and values of whole requests as dense bfloat16 rows, for leaving this cache
``decode``   attention of one new token per request over the pages
``chunk``    attention of several new tokens per request: drafted tokens, whole prompts, portions of prompts behind a long prefix"""

import math

import torch

own = False

DEV = "cuda:0"
EPS, THETA = 1e-6, 1e6
EXP_MIN, EXP_MAX, BIAS, TOP = -60, 7, 127, 448.0


def listed():
    return [
        # the step that eight users wait for, again and again: eight tokens' projections (sizes of the two smaller presets)
        {"name": "write_decode_b8", "kind": "write", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "rows": "2047:1,1799:1,2299:1,2110:1,1932:1,2047:1,2204:1,1998:1"},
        # a full portion of prompts (the scheduler's budget of tokens), heads of the 8b preset
        {"name": "write_prompt_2048", "kind": "write", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "rows": "0:1531,4096:517"},
        # a prompt of odd length in a model of narrow heads
        {"name": "write_d64_777", "kind": "write", "heads": 32, "kv_heads": 4, "dim": 64, "page": 16, "rows": "33:777"},
        # one conversation moves to another place
        {"name": "read_1999", "kind": "read", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "rows": "0:1999"},
        # long ones, ragged
        {"name": "read_long", "kind": "read", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "rows": "0:32768,0:20011,0:7777"},
        # one user, the beginning of a conversation: all latency
        {"name": "decode_b1_300", "kind": "decode", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "rows": "299:1"},
        # eight users reading their answers
        {"name": "decode_b8", "kind": "decode", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "rows": "2047:1,1799:1,2299:1,2110:1,1932:1,2047:1,2204:1,1998:1"},
        # a full house: 64 requests, contexts of all lengths
        {"name": "decode_b64", "kind": "decode", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "rows": ",".join("%d:1" % (1024 + 47 * i) for i in range(64))},
        # one request over a book
        {"name": "decode_b1_131072", "kind": "decode", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "rows": "131071:1"},
        # sixteen requests of narrow heads check five drafted tokens each
        {"name": "chunk_drafts_d64", "kind": "chunk", "heads": 32, "kv_heads": 4, "dim": 64, "page": 16, "rows": ",".join("%d:5" % (1500 + 61 * i) for i in range(16))},
        # a mixed step's prompts: two new ones and a portion behind a cached prefix
        {"name": "chunk_prompts", "kind": "chunk", "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "rows": "0:1531,1024:517,4096:900"},
        # the last portion of a long prompt
        {"name": "chunk_2048_behind_30720", "kind": "chunk", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "rows": "30720:2048"},
    ]


def draw(rng):
    """One more case of the same ranges; sizes spread over their logarithm."""

    def about(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk", "chunk"])
    dim = rng.choice([128, 128, 128, 128, 64, 64, 80, 256])
    kv_heads = rng.choice([2, 4, 8])
    case = {"kind": kind, "heads": kv_heads * rng.choice([1, 2, 4, 5, 8]), "kv_heads": kv_heads, "dim": dim, "page": rng.choice([8, 16, 16, 16, 32, 64])}
    if kind == "write":
        count = about(1, 64)
        rows = [(rng.choice([0, about(1, 30000)]), about(1, max(1, 2048 // count))) for _ in range(count)]
    elif kind == "read":
        count = about(1, 16)
        rows = [(0, about(1, 32768 // count)) for _ in range(count)]
    elif kind == "decode":
        count = about(1, 64)
        longest = about(16, min(131072, 262144 // count))
        rows = [(about(1, longest) - 1, 1) for _ in range(count)]
    elif rng.random() < 0.4:  # drafted tokens
        count = about(1, 32)
        longest = about(16, 65536 // count)
        rows = [(about(1, longest), rng.randint(1, 8)) for _ in range(count)]
    else:
        count = rng.choice([1, 1, 2, 3, 4])
        rows = [(rng.choice([0, about(1, 16384 // count)]), about(17, 2048 // count)) for _ in range(count)]
    case["rows"] = ",".join("%d:%d" % r for r in rows)
    if kind in ("decode", "chunk"):
        case["window"] = rng.choice([0, 0, 0, about(16, 4096)])
        case["sink"] = rng.choice([False, False, True])
    return case


def _rows(case):
    return [tuple(int(x) for x in r.split(":")) for r in case["rows"].split(",")]


# ------------------------------------------------------------------ inputs
def _power(field):
    """2^(field - 127), float32, of fields in 1..254."""
    return (field.to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """The codes (as the numbers they are, float32) and the exponents' bytes of x [..., d] float32."""
    amax = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    m, ex = torch.frexp(torch.where(fine, amax, torch.zeros_like(amax)))
    e = (ex - 9 + (m > 0.875).to(ex.dtype)).clamp(EXP_MIN, EXP_MAX)
    codes = (x * _power(BIAS - e)[..., None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return codes, torch.where(fine, e + BIAS, torch.full_like(e, 255)).to(torch.uint8)


def _dequantise(codes, exps):
    """float32 [..., d] of codes (uint8 [..., d]) and exponents (uint8 [...])."""
    factor = torch.where(exps == 255, math.nan, _power(exps))
    return codes.view(torch.float8_e4m3fn).float() * factor[..., None]


def prepare(case, seed):
    rows = _rows(case)
    heads, kvh, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=DEV)
    bf = dict(dtype=torch.bfloat16, device=DEV)
    tokens = sum(n for _, n in rows)
    need = [-(-(s + n) // page) for s, n in rows]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    cu = [0]
    indptr = [0]
    for (_, n), p in zip(rows, need):
        cu.append(cu[-1] + n)
        indptr.append(indptr[-1] + p)
    lens = torch.tensor([n for _, n in rows], device=DEV)
    starts = torch.tensor([s for s, _ in rows], device=DEV)
    row_of = torch.repeat_interleave(torch.arange(len(rows), device=DEV), lens)
    positions = torch.arange(tokens, device=DEV) - torch.tensor(cu[:-1], device=DEV)[row_of] + starts[row_of]
    st = {"case": case, "rows": rows, "scale": d ** -0.5, "window": case.get("window") or None, "sink": bool(case.get("sink")),
          "cu_q": torch.tensor(cu, **i32), "q_start": starts.to(torch.int32), "kv_len": (starts + lens).to(torch.int32), "row_of_token": row_of.to(torch.int32),
          "positions": positions.to(torch.int32), "page_indptr": torch.tensor(indptr, **i32), "page_indices": order[:indptr[-1]].contiguous()}
    if case["kind"] in ("write", "read"):
        st["k_out"], st["v_out"] = torch.empty((tokens, kvh, d), **bf), torch.empty((tokens, kvh, d), **bf)
    if case["kind"] == "write":
        st["qkv"] = torch.randn((tokens, (heads + 2 * kvh) * d), generator=gen, **bf) * 1.3
        st["q_norm"] = 1 + 0.3 * torch.randn((d,), generator=gen, **bf)
        st["k_norm"] = 1 + 0.3 * torch.randn((d,), generator=gen, **bf)
        freq = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
        angle = positions.double()[:, None] * freq
        st["inv_freq"] = freq.float()
        st["cos_sin"] = torch.cat([angle.cos(), angle.sin()], -1).float().contiguous()
        st["q_out"] = torch.empty((tokens, heads, d), **bf)
        for w in "kv":
            st[w + "_codes"] = torch.zeros((pages, kvh, page, d), dtype=torch.uint8, device=DEV)
            st[w + "_exps"] = torch.zeros((pages, kvh, page), dtype=torch.uint8, device=DEV)
        return st
    # keys have channels that stand out, as behind a rotation of slow pairs; values differ in size from token to token
    channel = torch.exp(0.5 * torch.randn((kvh, 1, d), generator=gen, device=DEV))
    k = torch.randn((pages, kvh, page, d), generator=gen, device=DEV) * channel
    codes, st["k_exps"] = _quantise(k)
    st["k_codes"] = codes.view(torch.uint8)
    del k
    v = torch.randn((pages, kvh, page, d), generator=gen, device=DEV) * torch.exp(0.5 * torch.randn((pages, kvh, page, 1), generator=gen, device=DEV))
    codes, st["v_exps"] = _quantise(v)
    st["v_codes"] = codes.view(torch.uint8)
    del v
    if case["kind"] in ("decode", "chunk"):
        st["q"] = torch.randn((tokens, heads, d), generator=gen, **bf)
        st["out"] = torch.empty((tokens, heads, d), **bf)
    return st


# ------------------------------------------------------------------ one pass
def _slots(st, row, pos):
    """Flat index of the cache rows of positions `pos` of requests `row` in [pages * page]: (page, slot)."""
    page = st["case"]["page"]
    entry = (st["page_indptr"][row] + torch.div(pos, page, rounding_mode="floor")).long()
    return st["page_indices"][entry.clamp(max=st["page_indices"].numel() - 1)].long(), pos % page


def _plain_write(st):
    case, d = st["case"], st["case"]["dim"]
    heads, kvh = case["heads"], case["kv_heads"]
    x = st["qkv"].float().view(-1, heads + 2 * kvh, d)
    q, k, v = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]

    def turned(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        cos, sin = st["cos_sin"][:, None, :d // 2], st["cos_sin"][:, None, d // 2:]
        lo, hi = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)

    st["q_out"].copy_(turned(q, st["q_norm"]))
    page, slot = _slots(st, st["row_of_token"], st["positions"])

    def stored(x, codes, exps):
        c, e = _quantise(x)
        codes[page, :, slot] = c.view(torch.uint8)
        exps[page, :, slot] = e
        return _dequantise(codes[page, :, slot], exps[page, :, slot]).bfloat16()

    return {"q": st["q_out"], "k": stored(turned(k, st["k_norm"]), st["k_codes"], st["k_exps"]), "v": stored(v, st["v_codes"], st["v_exps"])}


def _plain_read(st):
    page, slot = _slots(st, st["row_of_token"], st["positions"])
    return {w: _dequantise(st[w + "_codes"][page, :, slot], st[w + "_exps"][page, :, slot]).bfloat16() for w in "kv"}


def _plain_attention(st):
    case = st["case"]
    heads, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    rows, most, longest = len(st["rows"]), max(n for _, n in st["rows"]), max(s + n for s, n in st["rows"])
    pos = torch.arange(longest, device=DEV).expand(rows, longest)
    page, slot = _slots(st, torch.arange(rows, device=DEV)[:, None].expand(rows, longest), torch.minimum(pos, st["kv_len"][:, None] - 1))
    k = _dequantise(st["k_codes"][page, :, slot], st["k_exps"][page, :, slot])  # [rows, keys, kv heads, d]
    v = _dequantise(st["v_codes"][page, :, slot], st["v_exps"][page, :, slot])
    at = (st["row_of_token"].long(), (st["positions"] - st["q_start"][st["row_of_token"].long()]).long())
    q = torch.zeros((rows, most, heads, d), device=DEV)
    q[at] = st["q"].float()
    q = q.view(rows, most, kvh, heads // kvh, d).permute(0, 2, 3, 1, 4).reshape(rows, kvh, -1, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)).view(rows, heads, most, longest).mul_(st["scale"])
    q_pos = st["q_start"][:, None] + torch.arange(most, device=DEV)  # [rows, most]
    hidden = pos[:, None, :] > q_pos[:, :, None]
    if st["window"]:
        hidden = hidden | (pos[:, None, :] <= q_pos[:, :, None] - st["window"])
    s.masked_fill_(hidden[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))  # rows behind a request's last token
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True) + (torch.exp(-m) if st["sink"] else 0.0)
    o = torch.matmul(p.view(rows, kvh, -1, longest), v.permute(0, 2, 1, 3)).view(rows, heads, most, d) / total
    st["out"].copy_(o.permute(0, 2, 1, 3)[at])
    return st["out"]


def _step(st):
    """What the engine has of a step before its layers run: the batch's geometry, and the pools."""
    from miniserve_b200 import ops
    from miniserve_b200.engine.context import StepContext

    rows = st["rows"]
    st["k8"], st["v8"] = ops.Pool8(st["k_codes"], st["k_exps"]), ops.Pool8(st["v_codes"], st["v_exps"])
    st["status"] = ops.device_status(DEV)
    return StepContext(
        num_tokens=st["positions"].numel(), num_rows=len(rows), num_logit_rows=0, stream=torch.cuda.current_stream().cuda_stream, token_ids=None,
        positions=st["positions"], row_of_token=st["row_of_token"], cu_q=st["cu_q"], q_start=st["q_start"], kv_len=st["kv_len"], state_slot=None,
        logit_rows=None, page_indptr=[st["page_indptr"]], page_indices=[st["page_indices"]], status=st["status"], host_q_start=[s for s, _ in rows],
        host_q_len=[n for _, n in rows], host_state_slot=[-1] * len(rows), max_q_len=max(n for _, n in rows), max_kv_len=max(s + n for s, n in rows),
        decode_only=all(n == 1 for _, n in rows), leading_single_rows=next((i for i, (_, n) in enumerate(rows) if n != 1), len(rows)),
        sm_count=torch.cuda.get_device_properties(0).multi_processor_count)


def run(state):
    st, kind = state, state["case"]["kind"]
    if own:
        from miniserve_b200 import ops

        ctx = st.get("step")
        if ctx is None:
            ctx = st["step"] = _step(st)
        if kind in ("decode", "chunk"):
            ops.attention(st["out"], st["q"], st["k8"], st["v8"], ctx, 0, st["scale"], st["window"], st["sink"])
            return st["out"]
        if kind == "write":
            ops.qk_norm_rope_kv(st["q_out"], st["k8"], st["v8"], st["qkv"], st["q_norm"], st["k_norm"], st["inv_freq"], st["case"]["dim"], EPS, st["positions"],
                                st["row_of_token"], st["page_indptr"], st["page_indices"], st["case"]["page"], st["status"], stream=ctx.stream, cos_sin=st["cos_sin"])
        ops.read_cache(st["k_out"], st["v_out"], st["k8"], st["v8"], st["positions"], st["row_of_token"], st["page_indptr"], st["page_indices"], st["status"], stream=ctx.stream)
        read = {"k": st["k_out"], "v": st["v_out"]}
        return {"q": st["q_out"], **read} if kind == "write" else read
    if kind == "write":
        return _plain_write(st)
    if kind == "read":
        return _plain_read(st)
    return _plain_attention(st)


# ------------------------------------------------------------------ what a pass needs, and its result in 64 bits
def work(case):
    rows, d, heads, kvh, window = _rows(case), case["dim"], case["heads"], case["kv_heads"], case.get("window") or 0
    tokens = sum(n for _, n in rows)
    vector = d + 1  # a head's vector in the cache: its codes and its exponent
    if case["kind"] == "read":
        return {"bytes": tokens * kvh * 2 * (vector + 2 * d), "flops": tokens * kvh * 2 * d}
    if case["kind"] == "write":  # in: the projection, a table row, positions; out: queries, the cache, what is read back
        return {"bytes": tokens * ((heads + 2 * kvh) * d * 2 + d * 4 + 8 + heads * d * 2 + kvh * 2 * (vector + 2 * d)) + 4 * d, "flops": tokens * (heads + 2 * kvh) * d * 10}
    keys = pairs = 0
    for s, n in rows:
        keys += min(s + n, window + n - 1) if window else s + n
        if window:
            pairs += sum(min(p + 1, window) for p in range(s, s + n))
        else:
            pairs += n * s + n * (n + 1) // 2
    return {"bytes": keys * kvh * 2 * vector + tokens * heads * d * 4, "flops": 4 * d * heads * pairs}


def _values64(codes, exps):
    """What codes and exponents stand for, from their bits."""
    c = codes.long()
    field, mantissa = (c >> 3) & 15, c & 7
    size = torch.where(field > 0, torch.ldexp((8 + mantissa).double(), field - 10), torch.ldexp(mantissa.double(), torch.full_like(field, -9)))
    size = torch.where((c & 127) == 127, math.nan, size)
    out = torch.where(c >= 128, -size, size) * torch.ldexp(torch.ones_like(exps, dtype=torch.float64), exps.long() - 127)[..., None]
    return torch.where((exps == 255)[..., None], math.nan, out)


def _through8(x):
    """x [..., d] in 64 bits as the cache gives it back: the nearest number of the format, ties to the even mantissa."""
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, float(EXP_MIN))
    for n in range(EXP_MIN, EXP_MAX):
        e = torch.where(amax > TOP * 2.0 ** n, float(n + 1), e)
    y = x / torch.exp2(e)
    lead = torch.floor(torch.log2(y.abs().clamp_min(1e-300)))
    lead = torch.where(torch.exp2(lead) > y.abs(), lead - 1, lead).clamp_min(-6)
    step = torch.exp2(lead - 3)
    return (torch.round(y / step) * step).clamp(-TOP, TOP) * torch.exp2(e)


def exact(case, seed):
    st = prepare(case, seed)
    rows, page, d, heads, kvh = st["rows"], case["page"], case["dim"], case["heads"], case["kv_heads"]
    group = heads // kvh
    if case["kind"] == "write":
        x = st["qkv"].double().view(-1, heads + 2 * kvh, d)
        cos, sin = (st["cos_sin"].double()[:, :d // 2], st["cos_sin"].double()[:, d // 2:])

        def turned(x, w):
            y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * w.double()
            z = torch.complex(y[..., :d // 2], y[..., d // 2:]) * torch.complex(cos, sin)[:, None]
            return torch.cat([z.real, z.imag], -1)

        return {"q": turned(x[:, :heads], st["q_norm"]), "k": _through8(turned(x[:, heads:heads + kvh], st["k_norm"])), "v": _through8(x[:, heads + kvh:])}
    table, at = st["page_indices"].long(), st["page_indptr"].tolist()
    out = {"k": [], "v": []} if case["kind"] == "read" else []
    for r, (s, n) in enumerate(rows):
        mine = table[at[r]:at[r + 1]]
        k, v = (_values64(st[w + "_codes"][mine], st[w + "_exps"][mine]).permute(1, 0, 2, 3).reshape(kvh, -1, d)[:, :s + n] for w in "kv")
        if case["kind"] == "read":
            out["k"].append(k.transpose(0, 1)[s:])
            out["v"].append(v.transpose(0, 1)[s:])
            continue
        q = st["q"][st["cu_q"][r]:st["cu_q"][r + 1]].double()  # [n, heads, d]
        key, pos = torch.arange(s + n, device=DEV), torch.arange(s, s + n, device=DEV)[:, None]
        seen = (key <= pos) & ((key > pos - st["window"]) if st["window"] else torch.ones_like(key, dtype=torch.bool))
        o = torch.empty((n, heads, d), dtype=torch.float64, device=DEV)
        for h in range(heads):
            w = (q[:, h] @ k[h // group].T) * st["scale"]
            w = torch.where(seen, w, -math.inf)
            if st["sink"]:
                w = torch.softmax(torch.cat([w, torch.zeros_like(w[:, :1])], 1), 1)[:, :-1]
            else:
                w = torch.softmax(w, 1)
            o[:, h] = w @ v[h // group]
        out.append(o)
    return {w: torch.cat(x) for w, x in out.items()} if case["kind"] == "read" else torch.cat(out)
