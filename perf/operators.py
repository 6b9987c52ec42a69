"""Cases, plain forms and 64-bit forms of the encoder-layer operators in ``ops``: rotary positions,
attention with score caps, distance biases and document / prefix masks, and the matrix product in 8-bit
integers. ``run`` computes a case by elementary torch operations, or, with ``own`` set, by the framework's
calls on the same tensors.

Head layouts and lengths are those of the text tower (4 query heads over 2 K/V heads of 256 on sliding
layers, over 1 of 512 on global ones; documents of 2,208 tokens, queries of 17), of the vision tower
(12 heads of 64, 2,304 patches) and generic ones.
"""
import importlib
import math

import torch

own = False

PKG = "embeddinggemma2-rust_b200"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GOLDEN = 0.6180339887498949


# ---- cases ------------------------------------------------------------------------------------------
def rotary_case(name, kind, rows, nh, nkv, hd, rot, layout, scaling="none", factor=1.0, inverse=False, first=0):
    """`rot` of the `hd` channels of each head are rotated; documents start at position `first`."""
    return {"name": name, "op": "rotary", "kind": kind, "rows": rows, "nh": nh, "nkv": nkv, "hd": hd, "rot": rot,
            "layout": layout, "scaling": scaling, "factor": factor, "inverse": inverse, "first": first}


def attention_case(name, kind, seqs, longest, queries, nh, nkv, hd, softcap=0.0, window=-1, causal=False,
                   prefix=False, doc=0, bias="none", radius=0, empty=False):
    """`seqs` sequences of up to `longest` keys; `queries` query tokens each (0: one per key); `doc`: the
    longest document inside a sequence (0: no document mask); `empty`: the last sequence has no rows."""
    return {"name": name, "op": "attention", "kind": kind, "seqs": seqs, "longest": longest, "queries": queries,
            "nh": nh, "nkv": nkv, "hd": hd, "softcap": softcap, "window": window, "causal": causal, "prefix": prefix,
            "doc": doc, "bias": bias, "radius": radius, "empty": empty}


def linear_case(name, kind, m, n, k, out, bias=False):
    """x [m, k] in `kind`, 8-bit weights [n, k]; the result in `out`."""
    return {"name": name, "op": "linear", "kind": kind, "m": m, "n": n, "k": k, "out": out, "bias": bias}


def listed():
    return [
        # One 17-token search query on a sliding layer: the smallest call, latency only.
        rotary_case("rotary query", "bf16", 17, 4, 2, 256, 256, "half"),
        # A pass of 16 documents of 2,208 tokens on a global layer, q and k inside the fused projection's rows.
        rotary_case("rotary pass", "bf16", 35328, 4, 1, 512, 512, "half", "linear", 4.0),
        # A long document in f32: half of each head rotated in the interleaved layout, positions stretched.
        rotary_case("rotary long", "f32", 131071, 12, 12, 64, 32, "interleaved", "yarn", 8.0),
        # One new query token for each of 8 cached documents of up to 11,774 tokens: bound by reading K and V.
        attention_case("attention one token", "bf16", 8, 11774, 1, 4, 2, 256, softcap=50.0),
        # Documents of 1 to 2,208 tokens packed into one buffer on a sliding layer, scores capped.
        attention_case("attention documents", "bf16", 1, 16384, 0, 4, 2, 256, softcap=30.0, window=512, doc=2208),
        # Images of 2,304 patches and fewer, a learned bias per clipped distance for each of 12 heads.
        attention_case("attention patches", "bf16", 8, 2304, 0, 12, 12, 64, bias="table", radius=127),
        # One long text with a prefix that every token sees, linear distance penalties, scores capped: the largest.
        attention_case("attention prefix", "bf16", 1, 12001, 0, 8, 2, 128, softcap=50.0, causal=True, prefix=True,
                       bias="slopes"),
        # Full precision: ragged sequences of at most 777 tokens, one of them empty.
        attention_case("attention f32", "f32", 6, 777, 0, 4, 1, 128, softcap=20.0, window=300, doc=150, empty=True),
        # The fused q | k | v projection of one 17-token query.
        linear_case("int8 query", "bf16", 17, 2048, 512, "bf16"),
        # Odd sizes throughout, f32 on both sides, a bias.
        linear_case("int8 odd", "f32", 1111, 1001, 777, "f32", bias=True),
        # gate | up of a pass of 16 documents of 2,208 tokens.
        linear_case("int8 pass", "bf16", 35328, 4096, 512, "bf16"),
        # A wide layer, bound by the 8-bit tensor rate: the largest.
        linear_case("int8 wide", "bf16", 16384, 8192, 8192, "bf16", bias=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rotary", "attention", "attention", "linear"])
    if op == "rotary":
        hd = rng.choice([64, 80, 96, 128, 256, 512])
        nkv = rng.choice([1, 2, 4])
        nh = nkv * rng.choice([1, 2, 3, 4])
        kind = rng.choice(["bf16", "f32"])
        most = 1_600_000_000 // ((nh + nkv) * hd * (4 if kind == "bf16" else 8))
        rows = min(log_int(1, 131072), most)
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        c = rotary_case("", kind, rows, nh, nkv, hd, rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]),
                        rng.choice(["half", "interleaved"]), scaling, rng.choice([2.0, 4.0, 8.0, 16.0]),
                        rng.random() < 0.25, rng.choice([0, 0, log_int(1, 1_000_000)]))
    elif op == "attention":
        kind = rng.choice(["bf16", "bf16", "bf16", "f32"])
        hd = rng.choice([64, 128, 256, 512] if kind == "bf16" else [64, 80, 128, 256])
        nkv = rng.choice([1, 2, 4])
        nh = nkv * rng.choice([1, 2, 3, 4])
        queries = rng.choice([0, 0, 0, 1, log_int(1, 64)])
        seqs = log_int(1, 32)
        # At most 1.1e9 scores in bf16 and 2e7 in f32 (the listed cases' largest), padded lengths counted.
        most = (1_100_000_000 if kind == "bf16" else 20_000_000) // (nh * seqs)
        longest = log_int(1, min(32768, most // queries) if queries else int(math.sqrt(most)))
        causal = rng.random() < 0.4
        doc = rng.choice([0, 0, log_int(1, max(1, longest))])
        bias = rng.choice(["none", "none", "slopes", "table"])
        c = attention_case("", kind, seqs, longest, min(queries, longest), nh, nkv, hd,
                           rng.choice([0.0, 0.0, 20.0, 30.0, 50.0]), rng.choice([-1, -1, log_int(1, 1024)]), causal,
                           causal and rng.random() < 0.5, doc, bias, rng.choice([7, 64, 127, 500]) if bias == "table" else 0,
                           seqs > 1 and rng.random() < 0.25)
    else:
        n, k = log_int(16, 8192), log_int(16, 8192)
        m = min(log_int(1, 65536), 1_000_000_000_000 // (n * k), 300_000_000 // max(n, k))
        c = linear_case("", rng.choice(["bf16", "bf16", "f32"]), max(1, m), n, k, rng.choice(["bf16", "bf16", "f32"]),
                        rng.random() < 0.5)
    del c["name"]
    return c


# ---- lengths, positions and masks that go by the case alone -------------------------------------------
def spread(count, most):
    """`count` lengths of 1 .. most, the first of them `most`, spread evenly in no order."""
    return [max(1, math.ceil(most * (1.0 - (i * GOLDEN) % 1.0))) for i in range(count)]


def key_lens(c):
    lens = spread(c["seqs"], c["longest"])
    if c["empty"]:
        lens[-1] = 0
    return lens


def query_lens(c):
    return [min(n, c["queries"]) if c["queries"] else n for n in key_lens(c)]


def doc_lens(c, total):
    """Lengths of the documents that fill `total` rows."""
    lens, i = [], 0
    while total > 0:
        n = min(total, max(1, math.ceil(c["doc"] * (1.0 - (i * GOLDEN) % 1.0))))
        lens.append(n)
        total -= n
        i += 1
    return lens


def visible_pairs(c):
    """(query, key) pairs that the masks leave, for one head."""
    total = 0
    for nk, nq in zip(key_lens(c), query_lens(c)):
        if nk == 0 or nq == 0:
            continue
        i = torch.arange(nk - nq, nk)
        lo, hi = torch.zeros_like(i), torch.full_like(i, nk)
        if c["window"] >= 0:
            lo, hi = torch.maximum(lo, i - c["window"]), torch.minimum(hi, i + c["window"] + 1)
        if c["causal"]:
            hi = torch.minimum(hi, torch.clamp(i + 1, min=nk // 4) if c["prefix"] else i + 1)
        if c["doc"]:
            lens = torch.tensor(doc_lens(c, nk))
            end = torch.cumsum(lens, 0)
            d = torch.searchsorted(end, i, right=True)
            lo, hi = torch.maximum(lo, (end - lens)[d]), torch.minimum(hi, end[d])
        total += int(torch.clamp(hi - lo, min=0).sum())
    return total


def work(c):
    size = 4 if c["kind"] == "f32" else 2
    if c["op"] == "rotary":
        per_row = (c["nh"] + c["nkv"]) * c["hd"]
        return {"bytes": c["rows"] * (2 * per_row * size + 4), "flops": 3 * c["rows"] * (c["nh"] + c["nkv"]) * c["rot"]}
    if c["op"] == "attention":
        nq, nk = sum(query_lens(c)), sum(key_lens(c))
        return {"bytes": (2 * nq * c["nh"] + 2 * nk * c["nkv"]) * c["hd"] * size + 4 * nq * c["nh"],
                "flops": 4 * c["hd"] * c["nh"] * visible_pairs(c)}
    out = 4 if c["out"] == "f32" else 2
    return {"bytes": c["m"] * c["k"] * size + c["n"] * c["k"] + c["m"] * c["n"] * out + 4 * c["n"] * (2 if c["bias"] else 1),
            "flops": 2 * c["m"] * c["n"] * c["k"]}


# ---- inputs -------------------------------------------------------------------------------------------
def frequencies(rot, theta, scaling, factor, original):
    """Angle per position of each rotated pair, in turns, and the factor on cos and sin."""
    if scaling == "ntk":
        theta *= factor ** (rot / max(1, rot - 2))
    freq = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    magnitude = 1.0
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "yarn":
        # Pairs that turn more than 32 times over the original length keep their frequency, those that turn
        # less than once are stretched, a linear ramp over the pair's number between them.
        def pair(turns):
            return rot * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

        low, high = max(0, math.floor(pair(32.0))), min(rot - 1, math.ceil(pair(1.0)))
        ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(rot // 2)]
        freq = [f * (1.0 - r) + f / factor * r for f, r in zip(freq, ramp)]
        magnitude = 0.1 * math.log(factor) + 1.0
    return [f / (2.0 * math.pi) for f in freq], magnitude


def fixed_point(turns):
    """Turns per position in units of 2^-64 turn, as the signed 64-bit integer of the same bits."""
    v = int(math.ldexp(turns, 64)) & (2**64 - 1)
    return v - 2**64 if v >= 2**63 else v


def offsets(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()


def prepare(c, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[c["kind"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    s = {"case": c}
    if c["op"] == "rotary":
        nh, nkv, hd, rows = c["nh"], c["nkv"], c["hd"], c["rows"]
        qkv = normal(rows, (nh + 2 * nkv) * hd) if rows * (nh + 2 * nkv) * hd < 1 << 28 else normal(rows, (nh + nkv) * hd)
        s["q"] = qkv[:, : nh * hd].unflatten(1, (nh, hd))
        s["k"] = qkv[:, nh * hd : (nh + nkv) * hd].unflatten(1, (nkv, hd))
        # Documents of 2,208 tokens back to back; a longer input than 100,000 rows is one document.
        pos = torch.arange(rows, device="cuda", dtype=torch.int32)
        s["pos"] = c["first"] + (pos if rows > 100_000 else pos % 2208)
        turns, s["magnitude"] = frequencies(c["rot"], 10000.0, c["scaling"], c["factor"], 4096)
        s["steps"] = torch.tensor([fixed_point(t) for t in turns], dtype=torch.int64).cuda()
    elif c["op"] == "attention":
        nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
        ql, kl = query_lens(c), key_lens(c)
        # Scores of deviation 2: weights from smooth to peaked.
        s["q"] = normal(sum(ql), nh, hd, scale=2.0)
        s["k"] = normal(sum(kl), nkv, hd)
        s["v"] = normal(sum(kl), nkv, hd)
        s["q_off"], s["k_off"], s["max_q"], s["max_k"] = offsets(ql), offsets(kl), max(ql), max(kl)
        s["scale"] = hd ** -0.5
        for key in ("prefix_len", "q_doc", "k_doc", "slopes", "table"):
            s[key] = None
        if c["prefix"]:
            s["prefix_len"] = torch.tensor([n // 4 for n in kl], dtype=torch.int32).cuda()
        if c["doc"]:
            per = [torch.repeat_interleave(torch.arange(len(d)), torch.tensor(d)) if (d := doc_lens(c, n)) else
                   torch.zeros(0, dtype=torch.int64) for n in kl]
            s["k_doc"] = torch.cat(per).to(torch.int32).cuda()
            s["q_doc"] = torch.cat([p[n - m :] for p, n, m in zip(per, kl, ql)]).to(torch.int32).cuda()
        if c["bias"] == "slopes":
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)]).cuda()
        if c["bias"] == "table":
            s["table"] = normal(nh, 2 * c["radius"] + 1, dtype=torch.float32)
    else:
        m, n, k = c["m"], c["n"], c["k"]
        s["x"] = normal(m, k)
        # Weights as a user's program keeps them: whole numbers of -127 .. 127 in rows padded to 16 bytes, and
        # one scale per output channel.
        w = normal(n, k, scale=k ** -0.5, dtype=torch.float32)
        s["w_scale"] = w.abs().amax(1).clamp(min=1e-30) / 127.0
        s["w"] = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :k]
        s["w"].copy_(torch.round(w / s["w_scale"][:, None]))
        s["bias"] = normal(n, dtype=torch.float32) if c["bias"] else None
    return s


# ---- plain forms, in 32 bits ----------------------------------------------------------------------------
def rotary_plain(s):
    c = s["case"]
    # The angle in whole 2^-64 turns: the product wraps at full turns, so positions of any size lose nothing.
    phase = s["pos"].to(torch.int64)[:, None] * s["steps"]
    angle = (phase >> 32).to(torch.float32) * (2.0 * math.pi / 2.0**32)
    cos = (torch.cos(angle) * s["magnitude"])[:, None]
    sin = (torch.sin(angle) * (-s["magnitude"] if c["inverse"] else s["magnitude"]))[:, None]
    rot = c["rot"]

    def turn(x):
        y = x.to(torch.float32)
        a, b = (y[..., : rot // 2], y[..., rot // 2 : rot]) if c["layout"] == "half" else (y[..., 0:rot:2], y[..., 1:rot:2])
        u, v = a * cos - b * sin, b * cos + a * sin
        r = torch.cat([u, v], -1) if c["layout"] == "half" else torch.stack([u, v], -1).flatten(-2)
        return torch.cat([r, y[..., rot:]], -1).to(x.dtype)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def attention_plain(s):
    c = s["case"]
    q, k, v, nkv = s["q"], s["k"], s["v"], c["nkv"]
    G, hd, nh = c["nh"] // nkv, c["hd"], c["nh"]
    q0, k0 = s["q_off"].to(torch.int64), s["k_off"].to(torch.int64)
    ql, kl = q0.diff(), k0.diff()
    B, Lq, Lk = len(ql), s["max_q"], s["max_k"]
    i, j = torch.arange(Lq, device="cuda"), torch.arange(Lk, device="cuda")
    at_q = torch.clamp(q0[:-1, None] + i, max=max(len(q) - 1, 0))
    at_k = torch.clamp(k0[:-1, None] + j, max=max(len(k) - 1, 0))
    qp = q[at_q].to(torch.float32).view(B, Lq, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, G * Lq, hd)
    kp = k[at_k].to(torch.float32).permute(0, 2, 3, 1)
    vp = v[at_k].to(torch.float32).permute(0, 2, 1, 3)
    x = torch.matmul(qp, kp).view(B, nkv, G, Lq, Lk)
    x *= s["scale"]
    if c["softcap"]:
        x /= c["softcap"]
        x.tanh_()
        x *= c["softcap"]
    place = (kl - ql)[:, None] + i  # of each query among its sequence's keys
    apart = j - place[:, :, None]  # [B, Lq, Lk]
    if s["slopes"] is not None:
        x -= s["slopes"].view(1, nkv, G, 1, 1) * apart.abs()[:, None, None]
    if s["table"] is not None:
        R = c["radius"]
        x += s["table"][:, apart.clamp(-R, R) + R].permute(1, 0, 2, 3).reshape(B, nkv, G, Lq, Lk)
    seen = (j < kl[:, None])[:, None].expand(B, Lq, Lk)
    if c["window"] >= 0:
        seen = seen & (apart.abs() <= c["window"])
    if c["causal"]:
        before = apart <= 0
        if s["prefix_len"] is not None:
            before = before | (j < s["prefix_len"][:, None])[:, None]
        seen = seen & before
    if s["k_doc"] is not None:
        seen = seen & (s["q_doc"][at_q][:, :, None] == s["k_doc"][at_k][:, None])
    del apart
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    x -= top
    x.exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, nkv, G * Lq, Lk), vp).view(B, nkv, G, Lq, hd) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Lq, nh, hd)
    lse = (torch.log(total) + top)[..., 0].permute(0, 3, 1, 2).reshape(B, Lq, nh)
    row = torch.arange(len(q), device="cuda")
    seq = torch.searchsorted(q0[1:], row, right=True)
    return {"out": o[seq, row - q0[seq]].to(q.dtype), "lse": lse[seq, row - q0[seq]]}


def linear_plain(s):
    x = s["x"].to(torch.float32)
    top = x.abs().amax(1)
    whole = torch.round(x * torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top))[:, None])
    y = torch.matmul(whole, s["w"].to(torch.float32).t())  # whole numbers: exact below 2^24
    y *= (top / torch.full_like(top, 127.0))[:, None]
    y *= s["w_scale"]
    if s["bias"] is not None:
        y += s["bias"]
    return y.to(DTYPES[s["case"]["out"]])


# ---- the framework's calls --------------------------------------------------------------------------------
def run_own(s):
    c = s["case"]
    ops = importlib.import_module(PKG + ".ops")
    if c["op"] == "rotary":
        q, k = ops.rotary(s["q"], s["k"], s["pos"], s["steps"], layout=c["layout"], rot_dim=c["rot"],
                          magnitude=s["magnitude"], inverse=c["inverse"])
        return {"q": q, "k": k}
    if c["op"] == "attention":
        out, lse = ops.attention_masked(s["q"], s["k"], s["v"], s["q_off"], s["k_off"], s["max_q"], s["max_k"],
                                        scale=s["scale"], softcap=c["softcap"], window=c["window"], causal=c["causal"],
                                        prefix_len=s["prefix_len"], q_doc=s["q_doc"], k_doc=s["k_doc"],
                                        slopes=s["slopes"], dist_bias=s["table"], return_lse=True)
        return {"out": out, "lse": lse}
    x, x_scale = ops.quantize_rows(s["x"])
    return ops.gemm_i8(x, x_scale, s["w"], s["w_scale"], bias=s["bias"], out_dtype=DTYPES[c["out"]])


def run(s):
    if own:
        return run_own(s)
    return {"rotary": rotary_plain, "attention": attention_plain, "linear": linear_plain}[s["case"]["op"]](s)


# ---- 64 bits, from the definitions --------------------------------------------------------------------------
def rotary_exact(c, s):
    turns, magnitude = frequencies(c["rot"], 10000.0, c["scaling"], c["factor"], 4096)
    whole = s["pos"].to(torch.float64)[:, None] * torch.tensor(turns, dtype=torch.float64, device="cuda")
    angle = 2.0 * math.pi * (whole - torch.round(whole))
    z = torch.polar(torch.full_like(angle, magnitude), -angle if c["inverse"] else angle)[:, None]
    half = c["rot"] // 2

    def turn(x):
        y = x.to(torch.float64).clone()
        first = slice(0, half) if c["layout"] == "half" else slice(0, c["rot"], 2)
        second = slice(half, c["rot"]) if c["layout"] == "half" else slice(1, c["rot"], 2)
        w = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z
        y[..., first], y[..., second] = w.real, w.imag
        return y

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def attention_exact(c, s):
    G = c["nh"] // c["nkv"]
    ql, kl = query_lens(c), key_lens(c)
    out = torch.zeros(sum(ql), c["nh"], c["hd"], dtype=torch.float64, device="cuda")
    lse = torch.full((sum(ql), c["nh"]), -math.inf, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for b, (nq, nk) in enumerate(zip(ql, kl)):
        for start in range(0, nq, 2048):
            n = min(2048, nq - start)
            rows = slice(q0 + start, q0 + start + n)
            i = torch.arange(nk - nq + start, nk - nq + start + n, device="cuda")[:, None]
            j = torch.arange(nk, device="cuda")[None]
            bad = torch.zeros(n, nk, dtype=torch.bool, device="cuda")
            if c["window"] >= 0:
                bad |= (i - j > c["window"]) | (j - i > c["window"])
            if c["causal"]:
                bad |= (j > i) & (j >= (nk // 4 if c["prefix"] else 0))
            if c["doc"]:
                bad |= s["q_doc"][rows][:, None] != s["k_doc"][k0 : k0 + nk][None]
            for h in range(c["nh"]):
                kk, vv = (s[x][k0 : k0 + nk, h // G].double() for x in "kv")
                t = s["q"][rows, h].double() @ kk.T * s["scale"]
                if c["softcap"]:
                    t = c["softcap"] * torch.tanh(t / c["softcap"])
                if c["bias"] == "slopes":
                    t = t - s["slopes"][h].double() * (i - j).abs()
                if c["bias"] == "table":
                    t = t + s["table"][h].double()[torch.clamp(j - i, -c["radius"], c["radius"]) + c["radius"]]
                t[bad] = -math.inf
                z = torch.logsumexp(t, 1)
                lse[rows, h] = z
                out[rows, h] = torch.nan_to_num(torch.exp(t - z[:, None]), nan=0.0) @ vv
        q0, k0 = q0 + nq, k0 + nk
    return {"out": out, "lse": lse}


def linear_exact(c, s):
    w, w_scale = s["w"].double().T.contiguous(), s["w_scale"].double()
    y = torch.empty(c["m"], c["n"], dtype=torch.float64, device="cuda")
    for a in range(0, c["m"], 8192):
        x = s["x"][a : a + 8192].double()
        step = x.abs().amax(1, keepdim=True) / 127.0
        y[a : a + 8192] = torch.round(x / torch.where(step > 0, step, torch.ones_like(step))) @ w * step * w_scale
    return y if s["bias"] is None else y + s["bias"].double()


def exact(c, seed):
    s = prepare(c, seed)
    return {"rotary": rotary_exact, "attention": attention_exact, "linear": linear_exact}[c["op"]](c, s)
