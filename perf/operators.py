"""Three operators of a decoding round, measured next to their plain forms:

  matmul   y = act(W x + bias) + residual for several tokens, W in Q4_K, Q6_K, Q8_0 or fp16
  route    experts and weights from router logits: softmax or sigmoid scores, selection bias, groups
  verify   drafted tokens against the target's probabilities, by given uniform numbers

Shapes are the ones of the repository's benchmark and tests (hidden 2048, experts of 512, 256 experts, top-8,
vocabulary 248,320) and powers of two around them.  Weights are random superblocks whose dequantised values have the
spread of a trained model's (about 0.03); logits have a flat body and a few tokens that stand out.
"""
import math

import torch

own = False

Q8, Q4, Q6, F16 = 8, 12, 14, 1
BLOCK = {Q4: (256, 144), Q6: (256, 210), Q8: (32, 34), F16: (1, 2)}
VOCAB = 248320


def listed():
    return [
        # one token's expert-sized projection: the smallest product, launch latency counts
        {"name": "matmul_1_512x2048_q4k", "op": "matmul", "tokens": 1, "rows": 512, "cols": 2048, "qtype": Q4,
         "bias": True, "act": "silu", "residual": False, "y": "f16"},
        # a speculative round of 9 tokens through a wide projection, into the fp32 residual stream's type
        {"name": "matmul_9_8192x2048_q4k", "op": "matmul", "tokens": 9, "rows": 8192, "cols": 2048, "qtype": Q4,
         "bias": False, "act": "none", "residual": False, "y": "f32"},
        # that round's logits from a six-bit output matrix: the largest single read of weights
        {"name": "matmul_9_head_q6k", "op": "matmul", "tokens": 9, "rows": VOCAB, "cols": 2048, "qtype": Q6,
         "bias": False, "act": "none", "residual": False, "y": "f16"},
        # a batch of 67 requests through an eight-bit output projection, added to the residual stream
        {"name": "matmul_67_2048x4096_q8", "op": "matmul", "tokens": 67, "rows": 2048, "cols": 4096, "qtype": Q8,
         "bias": False, "act": "none", "residual": True, "y": "f32"},
        # a prefill chunk of odd length through a dense down projection
        {"name": "matmul_509_2048x4096_q6k", "op": "matmul", "tokens": 509, "rows": 2048, "cols": 4096, "qtype": Q6,
         "bias": True, "act": "none", "residual": True, "y": "f16"},
        # a long prefill chunk through a wide projection with its activation: the most arithmetic
        {"name": "matmul_2048_8192x2048_q4k", "op": "matmul", "tokens": 2048, "rows": 8192, "cols": 2048, "qtype": Q4,
         "bias": True, "act": "gelu", "residual": False, "y": "f16"},
        # one decode token's experts by softmax scores: the smallest call
        {"name": "route_1_softmax", "op": "route", "tokens": 1, "experts": 256, "top_k": 8, "score": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "group_top": 1, "renorm": True, "scale": 1.0},
        # a batch of requests, sigmoid scores with a balance bias, half of eight groups kept
        {"name": "route_100_groups", "op": "route", "tokens": 100, "experts": 256, "top_k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "group_top": 2, "renorm": True, "scale": 2.5},
        # the same router over a long prefill
        {"name": "route_16384_groups", "op": "route", "tokens": 16384, "experts": 256, "top_k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "group_top": 2, "renorm": True, "scale": 2.5},
        # one request, four drafts looked up in the text (no draft probabilities)
        {"name": "verify_1x4_lookup", "op": "verify", "requests": 1, "drafts": 4, "ragged": False, "vocab": VOCAB,
         "logits": "f16", "probs": False},
        # nine requests with 0 to 6 drafts of a small draft model, fp32 logits, an odd vocabulary
        {"name": "verify_9_ragged_odd", "op": "verify", "requests": 9, "drafts": 6, "ragged": True, "vocab": 32003,
         "logits": "f32", "probs": True},
        # many requests with eight drafts each: the most bytes
        {"name": "verify_64x8", "op": "verify", "requests": 64, "drafts": 8, "ragged": False, "vocab": VOCAB,
         "logits": "f16", "probs": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["matmul", "matmul", "matmul", "route", "verify"])
    if op == "matmul":
        qtype = rng.choice([Q4, Q4, Q6, Q6, Q8, F16])
        tokens = rng.choice([1, _log(rng, 2, 32), _log(rng, 33, 400), _log(rng, 400, 2048)])
        cols = 256 * rng.choice([1, 2, 3, 4, 7, 8, 8, 16])
        if qtype in (Q8, F16) and rng.random() < 0.5:
            cols += 32 * rng.randint(1, 7)
        per, size = BLOCK[qtype]
        most = min(8192 * 2048 * 2048 // (tokens * cols), VOCAB, 400_000_000 * per // (cols * size))
        rows = _log(rng, 200, min(most, 16384) if rng.random() < 0.8 else most)
        return {"op": "matmul", "tokens": tokens, "rows": rows, "cols": cols, "qtype": qtype, "bias": rng.random() < 0.5,
                "act": rng.choice(["none", "none", "silu", "gelu", "gelu_tanh", "relu"]),
                "residual": rng.random() < 0.5, "y": rng.choice(["f16", "f32"])}
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _log(rng, 6, 512 // groups)
        experts = groups * per
        top_groups = rng.randint(1, groups)
        return {"op": "route", "tokens": _log(rng, 1, 16384), "experts": experts,
                "top_k": rng.randint(1, min(16, top_groups * per)), "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.6, "groups": groups, "top_groups": top_groups, "group_top": rng.choice([1, 2]),
                "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5])}
    requests = _log(rng, 1, 64)
    drafts = rng.randint(1, 8)
    return {"op": "verify", "requests": requests, "drafts": drafts, "ragged": rng.random() < 0.5,
            "vocab": _log(rng, 1000, VOCAB), "logits": rng.choice(["f16", "f16", "f32"]) if requests <= 32 else "f16",
            "probs": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 17)
    return g


def _weights(qtype, elems, gen):
    """Random blocks of `elems` weights as bytes; dequantised values of about 0.03 around zero."""
    if qtype == F16:
        return (0.03 * torch.randn(elems, device="cuda", generator=gen)).half().view(torch.uint8)
    per, size = BLOCK[qtype]
    n = elems // per
    words = torch.empty((n * size + 3) // 4, dtype=torch.int32, device="cuda")
    words.random_(-(2**31), 2**31, generator=gen)
    b = words.view(torch.uint8)[:n * size].view(n, size)

    def scale(mean):
        return (mean * (0.5 + torch.rand(n, device="cuda", generator=gen))).half().view(torch.uint8).view(n, 2)

    if qtype == Q4:  # d, dmin, 12 scale bytes, 128 nibble pairs
        b[:, 0:2] = scale(1.5e-4)
        b[:, 2:4] = scale(1.1e-3)
    elif qtype == Q6:  # ql, qh, 16 int8 scales, d
        b[:, 208:210] = scale(2.2e-5)
    else:  # d, 32 int8
        b[:, 0:2] = scale(4e-4)
    return b.view(-1)


def _peaked(rows, vocab, gen):
    """Logits with a flat body and sixteen tokens a row that stand out."""
    z = 2.0 * torch.randn(rows, vocab, device="cuda", generator=gen)
    at = torch.randint(0, vocab, (rows, 16), device="cuda", generator=gen)
    z.scatter_add_(1, at, 4.0 + 10.0 * torch.rand(rows, 16, device="cuda", generator=gen))
    return z


def _rows(case):
    """Rows of each request in some order: one more than its drafts."""
    k = case["drafts"]
    return [1 + (5 * b + 2) % (k + 1) if case["ragged"] else k + 1 for b in range(case["requests"])]


def _inputs(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "matmul":
        n, rows, cols = case["tokens"], case["rows"], case["cols"]
        kind = torch.float32 if case["y"] == "f32" else torch.float16
        d = {"w": _weights(case["qtype"], rows * cols, g),
             "x": torch.randn(n, cols, device="cuda", generator=g).half(), "bias": None, "residual": None,
             "y": torch.empty(n, rows, dtype=kind, device="cuda")}
        if case["bias"]:
            d["bias"] = 0.5 * torch.randn(rows, device="cuda", generator=g)
        if case["residual"]:
            d["residual"] = (2.0 * torch.randn(n, rows, device="cuda", generator=g)).to(kind)
        return d
    if op == "route":
        e = case["experts"]
        d = {"logits": torch.randn(case["tokens"], e, device="cuda", generator=g), "bias": None}
        if case["bias"]:
            d["bias"] = 0.1 * torch.randn(e, device="cuda", generator=g)
        return d
    b, k, v = case["requests"], case["drafts"], case["vocab"]
    n = torch.tensor(_rows(case), dtype=torch.int64, device="cuda")[torch.randperm(b, device="cuda", generator=g)]
    offsets = torch.cat([n.new_zeros(1), n.cumsum(0)]).int()
    rows = sum(_rows(case))
    z = _peaked(rows, v, g)
    first = torch.zeros(rows, dtype=torch.bool, device="cuda")
    first[offsets[:-1].long()] = True
    tokens = torch.randint(0, v, (rows,), device="cuda", generator=g)
    judged = torch.nonzero(~first).view(-1) - 1  # the row whose distribution each draft is held against
    q = None
    if case["probs"]:  # a draft model: the target's logits with errors, and tokens drawn from it
        q = 0.9 * z[judged] + 0.6 * torch.randn(judged.numel(), v, device="cuda", generator=g)
        drafted = torch.empty(judged.numel(), dtype=torch.int64, device="cuda")
        for part in torch.arange(judged.numel(), device="cuda").split(64):
            noise = -torch.log(torch.rand(part.numel(), v, device="cuda", generator=g).clamp_min(1e-20))
            drafted[part] = (q[part] - torch.log(noise)).argmax(1)
        q = torch.softmax(q, 1)
    else:  # looked up: most often the likeliest token
        drafted = z[judged].argmax(1)
        other = torch.rand(judged.numel(), device="cuda", generator=g) < 0.2
        drafted = torch.where(other, torch.randint(0, v, drafted.shape, device="cuda", generator=g), drafted)
    tokens[~first] = drafted
    temperature = 0.6 + 0.5 * torch.rand(b, device="cuda", generator=g)
    temperature[3::5] = 0.0  # some requests decode greedily
    return {"logits": z if case["logits"] == "f32" else z.half(), "probs": q, "tokens": tokens.int(), "offsets": offsets,
            "u": torch.rand(rows, device="cuda", generator=g), "temperature": temperature, "eos": 2}


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = dict(case)
    if own:
        import breadv2_amd as B

        if case["op"] == "route":
            d["rule"] = B.RouteRule(score=case["score"], bias=d["bias"], n_groups=case["groups"],
                                    top_groups=case["top_groups"], group_top=case["group_top"], renorm=case["renorm"],
                                    scale=case["scale"])
        elif case["op"] == "verify":
            d["ctx"] = B.MoeContext(B.shape(), max_tokens=d["logits"].shape[0])
    return d


# ------------------------------------------------------------------ one pass


def run(state):
    c = state["case"]
    if own:
        import breadv2_amd as B

        if c["op"] == "matmul":
            B.bread_matmul(state["w"], state["x"], state["y"], c["rows"], c["cols"], c["qtype"], bias=state["bias"],
                           act=c["act"], residual=state["residual"])
            return {"y": state["y"]}
        if c["op"] == "route":
            idx, w = B.route_select(state["logits"], c["top_k"], state["rule"])
            return {"idx": idx, "w": w}
        n, nxt, logp = state["ctx"].spec_verify(state["logits"], state["tokens"], state["offsets"], state["u"],
                                                draft_probs=state["probs"], temperature=state["temperature"],
                                                eos=state["eos"])
        return {"accepted": n, "next": nxt, "logprob": logp}
    return {"matmul": _matmul, "route": _route, "verify": _verify}[c["op"]](state, c)


def _f16(b, at):
    return b[:, at:at + 2].contiguous().view(torch.float16).float()


def _dequant(w, qtype, rows, cols):
    if qtype == F16:
        return w.view(torch.float16).view(rows, cols).float()
    per, size = BLOCK[qtype]
    b = w.view(-1, size)
    n = b.shape[0]
    if qtype == Q8:
        v = _f16(b, 0) * b[:, 2:].contiguous().view(torch.int8).float()
    elif qtype == Q4:
        s = b[:, 4:16]
        sc = torch.cat([s[:, 0:4] & 63, (s[:, 8:12] & 15) | ((s[:, 0:4] >> 6) << 4)], 1).float()
        m = torch.cat([s[:, 4:8] & 63, (s[:, 8:12] >> 4) | ((s[:, 4:8] >> 6) << 4)], 1).float()
        q = b[:, 16:].view(n, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], 2).view(n, 8, 32).float()
        v = (_f16(b, 0) * sc)[:, :, None] * q - (_f16(b, 2) * m)[:, :, None]
    else:
        ql, qh = b[:, 0:128].view(n, 2, 64), b[:, 128:192].view(n, 2, 32)
        lo, hi = ql & 15, ql >> 4
        parts = [lo[:, :, :32] | ((qh & 3) << 4), lo[:, :, 32:] | (((qh >> 2) & 3) << 4),
                 hi[:, :, :32] | (((qh >> 4) & 3) << 4), hi[:, :, 32:] | ((qh >> 6) << 4)]
        q = torch.stack(parts, 2).view(n, 16, 16).float() - 32.0
        sc = b[:, 192:208].contiguous().view(torch.int8).float()
        v = (_f16(b, 208) * sc)[:, :, None] * q
    return v.reshape(rows, cols)


def _activate(v, act):
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return torch.maximum(v, v.new_zeros(())) if act == "relu" else v


def _matmul(state, c):
    y = state["x"].float() @ _dequant(state["w"], c["qtype"], c["rows"], c["cols"]).T
    if state["bias"] is not None:
        y = y + state["bias"]
    y = _activate(y, c["act"])
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return {"y": y.to(state["y"].dtype)}


def _ranked(v, k):
    """The k largest of each row, the lower index first among equals."""
    return torch.sort(v, dim=1, descending=True, stable=True).indices[:, :k]


def _route(state, c):
    x = state["logits"].double()  # 64 bits: which of two close scores is larger decides
    e, groups = c["experts"], c["groups"]
    if c["score"] == "softmax":
        s = torch.exp(x - x.amax(1, keepdim=True))
        s = s / s.sum(1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-x))
    choice = s if state["bias"] is None else s + state["bias"].double()
    if groups > 1:
        g = choice.view(-1, groups, e // groups)
        score = torch.sort(g, dim=2, descending=True).values[:, :, :c["group_top"]].sum(2)
        kept = torch.zeros_like(score, dtype=torch.bool).scatter_(1, _ranked(score, c["top_groups"]), True)
        choice = torch.where(kept[:, :, None], g, g.new_full((), -math.inf)).view(-1, e)
    idx = _ranked(choice, c["top_k"])
    w = s.gather(1, idx)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return {"idx": idx.int(), "w": (w * c["scale"]).float()}


def _verify(state, c):
    off, v = state["offsets"].long(), c["vocab"]
    b, rows = off.numel() - 1, state["logits"].shape[0]
    row = torch.arange(rows, device=off.device)
    req = torch.searchsorted(off, row, right=True) - 1
    last = row + 1 == off[req + 1]
    # the target's probabilities, in 64 bits: sums of a whole vocabulary decide borders between tokens
    t = state["temperature"].double()[req][:, None]
    z = state["logits"].double()
    top = z.amax(1, keepdim=True)
    column = torch.arange(v, device=off.device)
    z = (z - top) / torch.where(t > 0, t, torch.ones_like(t))
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    p = p / total
    logp = z - torch.log(total)  # a greedy request's at temperature 1
    best = torch.where(z == 0, column, v).amin(1)
    p = torch.where(t > 0, p, (column == best[:, None]).double())
    # each draft against the row before it
    draft = torch.cat([state["tokens"][1:].long(), off.new_zeros(1)])
    pd = p.gather(1, draft[:, None])[:, 0]
    at = (row - req).clamp_max(rows - b - 1)
    qd = pd.new_ones(rows)
    if state["probs"] is not None and rows > b:
        qd = state["probs"][at, draft].double()
    u = state["u"].double()
    passed = (u * qd < pd) & ~last
    stop = torch.where(passed & (draft != state["eos"]), rows, row)
    stop = off.new_full((b,), rows).scatter_reduce(0, req, stop, "amin")
    ends = passed[stop]  # an accepted end token closes the request and is its next token
    # the token after the last accepted one: from what the draft left over, or from the target's own
    w = p[stop]
    if state["probs"] is None or rows == b:
        one = (column == draft[stop][:, None]).double()
    else:
        one = state["probs"][at[stop]].double()
    left = torch.clamp_min(w - torch.where(last[stop][:, None], torch.zeros_like(one), one), 0.0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, w)
    cum = left.cumsum(1)
    nxt = (cum > u[off[1:] - 1][:, None] * cum[:, -1:]).int().argmax(1)
    nxt = torch.where(ends, draft[stop], nxt)
    # log-probabilities of the drafts, and in each request's last row of its next token
    logp_next = logp[stop, nxt]
    logp = logp.gather(1, draft[:, None])[:, 0].scatter(0, off[1:] - 1, logp_next)
    return {"accepted": (stop - off[:-1]).int(), "next": nxt.int(), "logprob": logp.float()}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "matmul":
        n, rows, cols = case["tokens"], case["rows"], case["cols"]
        per, size = BLOCK[case["qtype"]]
        y = 4 if case["y"] == "f32" else 2
        return {"bytes": rows * cols // per * size + 2 * n * cols + n * rows * y * (2 if case["residual"] else 1)
                + (4 * rows if case["bias"] else 0), "flops": 2 * n * rows * cols}
    if op == "route":
        n, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": n * (4 * e + 8 * k) + (4 * e if case["bias"] else 0), "flops": 4 * n * e}
    # every row of logits, and of the draft's probabilities the row that each request stops at
    b, v = case["requests"], case["vocab"]
    rows = sum(_rows(case))
    z = 4 if case["logits"] == "f32" else 2
    return {"bytes": rows * v * z + (4 * b * v if case["probs"] else 0) + 16 * rows + 16 * b, "flops": 3 * rows * v}


# ------------------------------------------------------------------ from the definitions, in 64 bits


def _blocks64(w, qtype, rows, cols):
    """Dequantised rows in 64 bits, element by element from the formats' bit positions."""
    dev = w.device
    if qtype == F16:
        return w.view(torch.float16).view(rows, cols).double()
    per, size = BLOCK[qtype]
    b = w.view(-1, size).to(torch.int64)

    def half(lo):
        bits = b[:, lo] | (b[:, lo + 1] << 8)
        return bits.to(torch.int32).to(torch.int16).view(torch.float16).double()[:, None]

    def signed(x):
        return x - 256 * (x > 127)

    i = torch.arange(per, device=dev)
    if qtype == Q8:
        v = half(0) * signed(b[:, 2:]).double()
    elif qtype == Q4:
        sub = i // 32
        low = sub < 4
        at = torch.where(low, 4 + sub, 8 + sub)
        sc = torch.where(low, b[:, at] & 63, (b[:, at] & 15) + 16 * (b[:, torch.where(low, 0, sub)] >> 6))
        am = torch.where(low, 8 + sub, 8 + sub)
        m = torch.where(low, b[:, am] & 63, (b[:, am] >> 4) + 16 * (b[:, torch.where(low, 0, 4 + sub)] >> 6))
        byte = b[:, 16 + 32 * (i // 64) + i % 32]
        q = torch.where(i % 64 < 32, byte & 15, byte >> 4)
        v = half(0) * (sc * q).double() - half(2) * m.double()
    else:
        h, j = i // 128, i % 128
        quarter, l = j // 32, j % 32
        byte = b[:, 64 * h + l + 32 * (quarter % 2)]
        nib = torch.where(quarter < 2, byte & 15, byte >> 4)
        q = nib + 16 * ((b[:, 128 + 32 * h + l] >> (2 * quarter)) & 3) - 32
        v = half(208) * (signed(b[:, 192 + i // 16]) * q).double()
    return v.reshape(rows, cols)


def _exact_matmul(d, c):
    x, out = d["x"].double(), []
    w = d["w"].view(c["rows"], -1)
    for at in range(0, c["rows"], 8192):
        part = w[at:at + 8192]
        y = torch.mm(x, _blocks64(part.reshape(-1), c["qtype"], part.shape[0], c["cols"]).t().contiguous())
        if d["bias"] is not None:
            y += d["bias"][at:at + 8192].double()
        if c["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["act"] in ("gelu", "gelu_tanh"):
            y = torch.nn.functional.gelu(y, approximate="tanh" if c["act"] == "gelu_tanh" else "none")
        elif c["act"] == "relu":
            y = torch.relu(y)
        if d["residual"] is not None:
            y += d["residual"][:, at:at + 8192].double()
        out.append(y)
    return {"y": torch.cat(out, 1)}


def _exact_route(d, c):
    z = d["logits"].double().cpu()
    s = torch.softmax(z, 1) if c["score"] == "softmax" else torch.sigmoid(z)
    choice = s + (d["bias"].double().cpu() if d["bias"] is not None else 0.0)
    n, per = z.shape[0], c["experts"] // c["groups"]
    every = torch.arange(n)
    if c["groups"] > 1:
        rest, score = choice.reshape(n, c["groups"], per).clone(), 0.0
        for _ in range(min(c["group_top"], per)):
            m, at = rest.max(2)
            score = score + m
            rest.scatter_(2, at[:, :, None], -math.inf)
        allowed = torch.zeros(n, c["groups"], dtype=torch.bool)
        for _ in range(c["top_groups"]):
            m = score.max(1, keepdim=True).values
            at = (score == m).int().argmax(1)
            allowed[every, at] = True
            score[every, at] = -math.inf
        choice = choice.masked_fill(~allowed.repeat_interleave(per, 1), -math.inf)
    idx = torch.empty(n, c["top_k"], dtype=torch.int64)
    for k in range(c["top_k"]):
        m = choice.max(1, keepdim=True).values
        idx[:, k] = (choice == m).int().argmax(1)
        choice[every, idx[:, k]] = -math.inf
    w = s.gather(1, idx)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return {"idx": idx.int(), "w": w * c["scale"]}


def _exact_verify(d, c):
    off, tokens = d["offsets"].tolist(), d["tokens"].tolist()
    u, temperature = d["u"].double().tolist(), d["temperature"].double().tolist()
    accepted, nxt, logp = [], [], torch.empty(off[-1], dtype=torch.float64)
    for b in range(len(off) - 1):
        n, done = 0, None

        def p_of(row):
            z = d["logits"][row].double()
            if temperature[b] > 0:
                return torch.softmax(z / temperature[b], 0)
            p = torch.zeros_like(z)
            p[int(torch.nonzero(z == z.max())[0])] = 1.0
            return p

        def logp_of(row, t):
            z = d["logits"][row].double() / (temperature[b] if temperature[b] > 0 else 1.0)
            return float(z[t] - torch.logsumexp(z, 0))

        for r in range(off[b], off[b + 1] - 1):
            logp[r] = logp_of(r, tokens[r + 1])
        p = p_of(off[b])
        for r in range(off[b], off[b + 1] - 1):
            t = tokens[r + 1]
            q = None if d["probs"] is None else d["probs"][r - b].double()
            if not u[r] * (1.0 if q is None else float(q[t])) < float(p[t]):
                if q is None:
                    q = torch.zeros_like(p)
                    q[t] = 1.0
                rest = (p - q).clamp_min(0.0)
                p = rest if float(rest.sum()) > 0 else p
                break
            if t == d["eos"]:
                done = t
                break
            n += 1
            p = p_of(r + 1)
        if done is None:
            cum = torch.cumsum(p, 0)
            done = int(torch.nonzero(cum > u[off[b + 1] - 1] * cum[-1])[0])
        logp[off[b + 1] - 1] = logp_of(off[b] + n, done)
        accepted.append(n)
        nxt.append(done)
    dev = d["logits"].device
    return {"accepted": torch.tensor(accepted, dtype=torch.int32, device=dev),
            "next": torch.tensor(nxt, dtype=torch.int32, device=dev), "logprob": logp.to(dev)}


def exact(case, seed):
    d = _inputs(case, seed)
    return {"matmul": _exact_matmul, "route": _exact_route, "verify": _exact_verify}[case["op"]](d, case)
