"""Four operators of a feed-forward layer in 8-bit floating point (e4m3 codes, an fp32 scale for each block of 128),
measured next to their plain forms:

  norm     h = x + residual, RMSNorm of h, quantised: codes and a scale for every 128 columns of a token
  matmul   act(W x + bias) + residual, W with a scale for each 128 x 128 block; a second matrix for gated units;
           results in 16 or 32 bits, or quantised again
  grouped  the same products by expert: ragged groups of rows, gathered from tokens or scattered to pairs
  block    the routed experts of a layer with the caller's routing, added to the residual stream

Sizes are the ones of the repository's benchmark and tests (hidden 2048, experts of 512, 256 experts, top-8), powers of two
around them and odd ones.  Activations have a few channels that stand out, weights a spread of about 0.03.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
F8 = torch.float8_e4m3fn
KINDS = {"f16": torch.float16, "f32": torch.float32, "bf16": torch.bfloat16, "e4m3": F8}
BYTES = {"f16": 2, "f32": 4, "bf16": 2, "e4m3": 1}


def listed():
    return [
        # one decode token on the fp32 residual stream, with the plain norm for the router: the smallest call
        {"name": "norm_1_2048_f32", "op": "norm", "tokens": 1, "cols": 2048, "x": "f32", "residual": False,
         "normed": "f32"},
        # an odd batch of a bf16 model, the last layer's result added
        {"name": "norm_509_4096_bf16", "op": "norm", "tokens": 509, "cols": 4096, "x": "bf16", "residual": True,
         "normed": "none"},
        # a long prefill on the fp16 stream, with the plain norm: the most bytes
        {"name": "norm_16384_2048_f16", "op": "norm", "tokens": 16384, "cols": 2048, "x": "f16", "residual": True,
         "normed": "f16"},
        # one token's shared expert, gate and up with SwiGLU, quantised for the down product
        {"name": "matmul_1_512x2048_glu", "op": "matmul", "tokens": 1, "rows": 512, "cols": 2048, "glu": True,
         "bias": False, "act": "silu", "residual": False, "y": "e4m3"},
        # a speculative round of 9 tokens through a wide projection
        {"name": "matmul_9_8192x2048", "op": "matmul", "tokens": 9, "rows": 8192, "cols": 2048, "glu": False,
         "bias": True, "act": "none", "residual": False, "y": "bf16"},
        # a batch of 131 requests through an output projection, added to the fp32 residual stream
        {"name": "matmul_131_2048x4096_res", "op": "matmul", "tokens": 131, "rows": 2048, "cols": 4096, "glu": False,
         "bias": False, "act": "none", "residual": True, "y": "f32"},
        # a long prefill chunk through a wide projection: the most arithmetic of a single matrix
        {"name": "matmul_4096_8192x2048", "op": "matmul", "tokens": 4096, "rows": 8192, "cols": 2048, "glu": False,
         "bias": False, "act": "none", "residual": False, "y": "bf16"},
        # nine tokens' gate and up products: 72 pairs over 256 experts, one or two rows an expert
        {"name": "grouped_72_glu_gather", "op": "grouped", "tokens": 9, "top_k": 8, "groups": 256, "rows": 512,
         "cols": 2048, "glu": True, "index": "gather", "y": "e4m3", "spare": 0},
        # 200 tokens' down products written back by pair, a ragged tail of the buffer unused
        {"name": "grouped_1600_down_scatter", "op": "grouped", "tokens": 200, "top_k": 8, "groups": 256, "rows": 2048,
         "cols": 512, "glu": False, "index": "scatter", "y": "f32", "spare": 37},
        # a prefill's gate and up products: the largest grouped one
        {"name": "grouped_32768_glu_gather", "op": "grouped", "tokens": 4096, "top_k": 8, "groups": 256, "rows": 512,
         "cols": 2048, "glu": True, "index": "gather", "y": "e4m3", "spare": 0},
        # the experts of one decode token
        {"name": "block_1", "op": "block", "tokens": 1, "top_k": 8, "groups": 256, "hidden": 2048, "inter": 512,
         "y": "f16"},
        # the experts of a long prefill
        {"name": "block_4096", "op": "block", "tokens": 4096, "top_k": 8, "groups": 256, "hidden": 2048, "inter": 512,
         "y": "f16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "matmul", "matmul", "grouped", "grouped", "block"])
    if op == "norm":
        cols = 16 * _log(rng, 16, 512)
        return {"op": op, "tokens": _log(rng, 1, min(16384, (1 << 25) // cols)), "cols": cols,
                "x": rng.choice(["f16", "bf16", "f32"]), "residual": rng.random() < 0.6,
                "normed": rng.choice(["none", "f16", "bf16", "f32"])}
    if op == "matmul":
        tokens = rng.choice([1, _log(rng, 2, 32), _log(rng, 33, 400), _log(rng, 400, 4096)])
        cols = 128 * rng.choice([1, 2, 3, 4, 8, 16, 16, 32, 56]) + (16 * rng.randint(1, 7) if rng.random() < 0.2 else 0)
        most = min(16384, 4096 * 8192 * 2048 // (tokens * cols))
        y = rng.choice(["f16", "bf16", "f32", "e4m3"])
        glu = rng.random() < 0.3
        rows = _log(rng, 64, most // (2 if glu else 1))
        if y == "e4m3":
            rows = 16 * max(1, rows // 16)
        return {"op": op, "tokens": tokens, "rows": rows, "cols": cols, "glu": glu,
                "bias": not glu and rng.random() < 0.4, "act": rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]),
                "residual": y != "e4m3" and rng.random() < 0.4, "y": y}
    if op == "grouped":
        groups = _log(rng, 4, 256)
        top_k = rng.randint(1, min(8, groups))
        rows, cols = 64 * rng.choice([2, 3, 4, 8, 16, 32]), 128 * rng.choice([2, 4, 8, 16, 16])
        glu = rng.random() < 0.5
        most = 32768 * 1024 * 2048 // (rows * cols * (2 if glu else 1))
        return {"op": op, "tokens": _log(rng, 1, min(4096, most // top_k)), "top_k": top_k, "groups": groups,
                "rows": rows, "cols": cols, "glu": glu, "index": rng.choice(["gather", "scatter", "none"]),
                "y": rng.choice(["f16", "bf16", "f32", "e4m3"]), "spare": rng.choice([0, 0, rng.randint(1, 100)])}
    groups = _log(rng, 8, 256)
    return {"op": "block", "tokens": _log(rng, 1, 4096), "top_k": rng.randint(1, 8), "groups": groups,
            "hidden": 256 * rng.choice([2, 4, 8, 8]), "inter": rng.choice([256, 512, 512]),
            "y": rng.choice(["f16", "bf16"])}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 29)
    return g


def _blocks(n):
    return -(-n // BLOCK)


def _stream(tokens, cols, gen):
    """Activations of a residual stream: rows of different size, a few channels that stand out."""
    size = 0.3 + 2.0 * torch.rand(tokens, 1, device="cuda", generator=gen)
    channel = 1.0 + 9.0 * (torch.rand(cols, device="cuda", generator=gen) < 0.01).float()
    return size * channel * torch.randn(tokens, cols, device="cuda", generator=gen)


def _activations(tokens, cols, gen):
    return _quantise(_stream(tokens, cols, gen))


def _weights(groups, rows, cols, gen):
    """Codes and scales as blocks of normally distributed weights have them: the largest of 16384 is about four
    deviations out."""
    codes = (108.0 * torch.randn(groups, rows, cols, device="cuda", generator=gen)).clamp_(-448.0, 448.0).to(F8)
    scale = 2.8e-4 * (0.5 + torch.rand(groups, _blocks(rows), _blocks(cols), device="cuda", generator=gen))
    return codes, scale


def _routing(case):
    """Experts [tokens][top_k] of a router that prefers some experts, the same for every seed up to names."""
    t, k, g = case["tokens"], case["top_k"], case["groups"]
    rng = np.random.default_rng([t, k, g])
    logits = -0.7 * np.log1p(np.arange(g)) + rng.gumbel(size=(t, g))
    return np.argsort(-logits, axis=1, kind="stable")[:, :k]


def _named(case, gen):
    """The same with experts and tokens in an order of the seed."""
    idx = torch.from_numpy(_routing(case)).cuda()
    idx = torch.randperm(case["groups"], device="cuda", generator=gen)[idx]
    return idx[torch.randperm(case["tokens"], device="cuda", generator=gen)]


def _used(case):
    return len(np.unique(_routing(case)))


def _inputs(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "norm":
        t, n, kind = case["tokens"], case["cols"], KINDS[case["x"]]
        return {"x": _stream(t, n, g).to(kind), "w": 1.0 + 0.2 * torch.randn(n, device="cuda", generator=g),
                "residual": _stream(t, n, g).to(kind) if case["residual"] else None, "eps": 1e-6}
    if op == "matmul":
        n, rows, cols = case["tokens"], case["rows"], case["cols"]
        d = {"up": None, "up_scale": None, "bias": None, "residual": None}
        d["x"], d["x_scale"] = _activations(n, cols, g)
        w, s = _weights(1, rows, cols, g)
        d["w"], d["w_scale"] = w[0], s[0]
        if case["glu"]:
            w, s = _weights(1, rows, cols, g)
            d["up"], d["up_scale"] = w[0], s[0]
        if case["bias"]:
            d["bias"] = 0.5 * torch.randn(rows, device="cuda", generator=g)
        if case["residual"]:
            d["residual"] = (2.0 * torch.randn(n, rows, device="cuda", generator=g)).to(KINDS[case["y"]])
        return d
    idx = _named(case, g)
    t, k, e = case["tokens"], case["top_k"], case["groups"]
    if op == "grouped":
        rows, cols, spare = case["rows"], case["cols"], case["spare"]
        order = torch.argsort(idx.reshape(-1), stable=True).int()  # pairs by expert
        sizes = torch.zeros(e, dtype=torch.int64, device="cuda").scatter_add_(0, idx.reshape(-1), torch.ones_like(idx).reshape(-1))
        d = {"offsets": torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).int(), "x_rows": None, "y_rows": None,
             "up": None, "up_scale": None}
        last = torch.arange(t * k, t * k + spare, dtype=torch.int32, device="cuda")  # rows of no group
        if case["index"] == "gather":
            d["x_rows"] = torch.cat([order // k, torch.zeros_like(last)])
        elif case["index"] == "scatter":
            d["y_rows"] = torch.cat([order, last])
        d["x"], d["x_scale"] = _activations(t if case["index"] == "gather" else t * k + spare, cols, g)
        d["w"], d["w_scale"] = _weights(e, rows, cols, g)
        if case["glu"]:
            d["up"], d["up_scale"] = _weights(e, rows, cols, g)
        return d
    h, i = case["hidden"], case["inter"]
    d = {"idx": idx.int(), "hidden": torch.randn(t, h, device="cuda", generator=g).to(KINDS[case["y"]])}
    w = torch.rand(t, k, device="cuda", generator=g) + 0.1
    d["weight"] = w / w.sum(1, keepdim=True)
    d["x"], d["x_scale"] = _activations(t, h, g)
    d["gate"], d["gate_scale"] = _weights(e, i, h, g)
    d["up"], d["up_scale"] = _weights(e, i, h, g)
    d["down"], d["down_scale"] = _weights(e, h, i, g)
    return d


def _results(case):
    """Buffers that a program writes a product's results into."""
    rows = case["rows"]
    n = case["tokens"] if case["op"] == "matmul" else case["tokens"] * case["top_k"] + case["spare"]
    y = torch.zeros(n, rows, dtype=torch.uint8 if case["y"] == "e4m3" else KINDS[case["y"]], device="cuda")
    if case["y"] != "e4m3":
        return y, None
    return y.view(F8), torch.zeros(n, _blocks(rows), device="cuda")


def prepare(case, seed):
    d = _inputs(case, seed)
    d["case"] = dict(case)
    if case["op"] == "norm":
        t, n = case["tokens"], case["cols"]
        d["codes"] = torch.empty(t, n, dtype=F8, device="cuda")
        d["scales"] = torch.empty(t, _blocks(n), device="cuda")
        d["sum"] = torch.empty_like(d["x"]) if case["residual"] else None
        d["normed"] = None if case["normed"] == "none" else torch.empty(t, n, dtype=KINDS[case["normed"]], device="cuda")
    elif case["op"] in ("matmul", "grouped"):
        d["y"], d["y_scale"] = _results(case)
    else:
        d["out"] = torch.empty_like(d["hidden"])
    if own and case["op"] == "block":
        import breadv2_amd as B

        d["ctx"] = B.MoeContext(B.shape(hidden=case["hidden"], expert_inter=case["inter"], shared_inter=case["inter"],
                                        n_experts=case["groups"], top_k=case["top_k"]), max_tokens=case["tokens"])
        d["experts"] = B.Fp8Experts(d["gate"], d["gate_scale"], d["up"], d["up_scale"], d["down"], d["down_scale"])
    return d


# ------------------------------------------------------------------ one pass


def run(state):
    c = state["case"]
    if own:
        import breadv2_amd as B

        if c["op"] == "norm":
            B.bread_rmsnorm_fp8(state["x"], state["w"], state["codes"], state["scales"], state["eps"],
                                residual=state["residual"], hidden=state["sum"], normed=state["normed"])
            return {"codes": state["codes"], "scales": state["scales"], "sum": state["sum"], "normed": state["normed"]}
        if c["op"] == "matmul":
            B.bread_matmul_fp8(state["w"], state["w_scale"], state["x"], state["x_scale"], state["y"],
                               y_scale=state["y_scale"], up=state["up"], up_scale=state["up_scale"],
                               bias=state["bias"], act=c["act"], residual=state["residual"])
            return {"y": state["y"], "y_scale": state["y_scale"]}
        if c["op"] == "grouped":
            B.bread_matmul_fp8_grouped(state["w"], state["w_scale"], state["x"], state["x_scale"], state["offsets"],
                                       state["y"], y_scale=state["y_scale"], up=state["up"],
                                       up_scale=state["up_scale"], act="silu" if c["glu"] else None,
                                       x_rows=state["x_rows"], y_rows=state["y_rows"])
            return {"y": state["y"], "y_scale": state["y_scale"]}
        state["ctx"].expert_block_fp8(state["experts"], state["x"], state["x_scale"], state["out"], state["idx"],
                                      state["weight"], residual=state["hidden"])
        return {"hidden": state["out"]}
    return {"norm": _norm, "matmul": _matmul, "grouped": _grouped, "block": _block}[c["op"]](state, c)


def _quantise(v):
    """Codes and scales of fp32 rows."""
    t, n = v.shape
    wide = torch.zeros(t, _blocks(n) * BLOCK, device=v.device)
    wide[:, :n] = v
    wide = wide.view(t, -1, BLOCK)
    s = torch.clamp_min(wide.abs().amax(2) / 448.0, 2.0**-126)
    return (wide / s[:, :, None]).view(t, -1)[:, :n].to(F8).contiguous(), s


def _values(codes, scale):
    """fp32 values of codes [..., rows, cols] with a scale a block (of weights) or a row's block (of activations)."""
    rows, cols = codes.shape[-2:]
    if scale.shape[-2] != rows:
        scale = scale.repeat_interleave(BLOCK, -2)[..., :rows, :]
    return codes.float() * scale.repeat_interleave(BLOCK, -1)[..., :cols]


def _activate(v, act):
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return torch.maximum(v, v.new_zeros(())) if act == "relu" else v


def _norm(state, c):
    h = state["x"] if state["residual"] is None else (state["x"].float() + state["residual"].float()).to(state["x"].dtype)
    f = h.float()
    v = f * torch.rsqrt((f * f).mean(1, keepdim=True) + state["eps"]) * state["w"]
    codes, scales = _quantise(v)
    return {"codes": codes, "scales": scales, "sum": None if state["residual"] is None else h,
            "normed": None if state["normed"] is None else v.to(state["normed"].dtype)}


def _matmul(state, c):
    x = _values(state["x"], state["x_scale"])
    y = x @ _values(state["w"], state["w_scale"]).T
    if state["bias"] is not None:
        y = y + state["bias"]
    y = _activate(y, c["act"])
    if c["glu"]:
        y = y * (x @ _values(state["up"], state["up_scale"]).T)
    if c["y"] == "e4m3":
        codes, scales = _quantise(y)
        return {"y": codes, "y_scale": scales}
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return {"y": y.to(KINDS[c["y"]]), "y_scale": None}


def _padded(x, offsets):
    """Rows [n][cols] of the groups that have any, as [groups][most][cols] with zeros behind: those, the groups' numbers
    and the place of every row."""
    off = offsets.long()
    sizes = off[1:] - off[:-1]
    used = torch.nonzero(sizes).view(-1)
    row = torch.arange(int(off[-1]), device=x.device)
    group = torch.searchsorted(off, row, right=True) - 1
    slot = torch.searchsorted(used, group)
    out = torch.zeros(used.numel(), int(sizes.max()), x.shape[1], device=x.device)
    at = (slot, row - off[group])
    out[at] = x[: row.numel()]
    return out, used, at


def _product(padded, used, codes, scale):
    """padded [groups][most][cols] times the used groups' weights."""
    w = _values(codes.view(torch.uint8)[used].view(F8), scale[used])
    return torch.bmm(padded, w.transpose(1, 2).contiguous())


def _grouped(state, c):
    x = _values(state["x"], state["x_scale"])
    if state["x_rows"] is not None:
        x = x[state["x_rows"].long()]
    padded, used, at = _padded(x, state["offsets"])
    y = _product(padded, used, state["w"], state["w_scale"])
    if c["glu"]:
        y = _activate(y, "silu") * _product(padded, used, state["up"], state["up_scale"])
    y = y[at]
    n = c["tokens"] * c["top_k"]
    place = torch.arange(n, device=y.device) if state["y_rows"] is None else state["y_rows"][:n].long()
    out, scales = _results(c)
    if c["y"] == "e4m3":
        codes, s = _quantise(y)
        out.view(torch.uint8)[place] = codes.view(torch.uint8)
        scales[place] = s
    else:
        out[place] = y.to(out.dtype)
    return {"y": out, "y_scale": scales}


def _block(state, c):
    t, k, e = c["tokens"], c["top_k"], c["groups"]
    flat = state["idx"].reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    sizes = torch.zeros(e, dtype=torch.int64, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    offsets = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)])
    x = _values(state["x"], state["x_scale"])[order // k]
    padded, used, at = _padded(x, offsets)
    a = _activate(_product(padded, used, state["gate"], state["gate_scale"]), "silu")
    a = a * _product(padded, used, state["up"], state["up_scale"])
    a, _, _ = _padded(_values(*_quantise(a[at])), offsets)
    y = _product(a, used, state["down"], state["down_scale"])[at]
    pairs = torch.zeros_like(y)
    pairs[order] = y
    out = (pairs.view(t, k, -1) * state["weight"][:, :, None]).sum(1)
    return {"hidden": (state["hidden"].float() + out).to(state["hidden"].dtype)}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "norm":
        t, n, size = case["tokens"], case["cols"], BYTES[case["x"]]
        normed = 0 if case["normed"] == "none" else BYTES[case["normed"]]
        return {"bytes": t * n * (size * (3 if case["residual"] else 1) + normed + 1) + 4 * t * _blocks(n) + 4 * n,
                "flops": 6 * t * n}
    mats = 2 if case.get("glu") else 1
    if op == "block":
        p, h, i = case["tokens"] * case["top_k"], case["hidden"], case["inter"]
        weights = 3 * (h * i + 4 * _blocks(h) * _blocks(i)) * _used(case)
        return {"bytes": weights + case["tokens"] * (h + 4 * _blocks(h) + 2 * BYTES[case["y"]] * h) + 8 * p,
                "flops": 6 * p * h * i}
    rows, cols, size = case["rows"], case["cols"], BYTES[case["y"]]
    out = size * rows + (4 * _blocks(rows) if case["y"] == "e4m3" else 0)
    one = mats * (rows * cols + 4 * _blocks(rows) * _blocks(cols))
    token = cols + 4 * _blocks(cols)
    if op == "matmul":
        n = case["tokens"]
        return {"bytes": one + n * (token + out + (size * rows if case["residual"] else 0))
                + (4 * rows if case["bias"] else 0), "flops": 2 * mats * n * rows * cols}
    p = case["tokens"] * case["top_k"]
    x = case["tokens"] if case["index"] == "gather" else p
    return {"bytes": one * _used(case) + x * token + p * (out + (0 if case["index"] == "none" else 4))
            + 4 * case["groups"], "flops": 2 * mats * p * rows * cols}


# ------------------------------------------------------------------ from the definitions, in 64 bits


def _table(dev):
    """The values of the 256 e4m3 codes: sign, 4 bits of exponent with bias 7, 3 of mantissa, no infinities."""
    v = []
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        size = m * 2.0**-9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        if e == 15 and m == 7:
            size = math.nan
        v.append(-size if code & 128 else size)
    return torch.tensor(v, dtype=torch.float64, device=dev)


def _codes64(v):
    """The nearest e4m3 value of each v, ties to the even one."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp_min(e - 1, -6) - 3)
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def _quantise64(v):
    """(codes' values, scales): a loop over the blocks."""
    codes, scales = torch.empty_like(v), []
    for at in range(0, v.shape[1], BLOCK):
        part = v[:, at:at + BLOCK]
        s = torch.clamp_min(part.abs().amax(1) / 448.0, 2.0**-126)
        codes[:, at:at + BLOCK] = _codes64(part / s[:, None])
        scales.append(s)
    return codes, torch.stack(scales, 1)


def _scaled64(codes, scale, down):
    """codes' values times scales; `down`: rows that share a scale."""
    rows, cols = codes.shape
    r = torch.arange(rows, device=codes.device) // down
    c = torch.arange(cols, device=codes.device) // BLOCK
    return codes * scale.double()[r][:, c]


def _bits64(codes, scale, down):
    return _scaled64(_table(codes.device)[codes.view(torch.uint8).long()], scale, down)


def _act64(v, act):
    f = torch.nn.functional
    return {"none": lambda: v, "silu": lambda: f.silu(v), "relu": lambda: torch.relu(v), "gelu": lambda: f.gelu(v),
            "gelu_tanh": lambda: f.gelu(v, approximate="tanh")}[act]()


def _exact_norm(d, c):
    h = d["x"].double()
    if d["residual"] is not None:
        h = (h + d["residual"].double()).to(d["x"].dtype).double()
    v = h / torch.sqrt(torch.mean(h * h, 1, keepdim=True) + d["eps"]) * d["w"].double()
    codes, scales = _quantise64(v)
    return {"codes": codes, "scales": scales, "sum": None if d["residual"] is None else h,
            "normed": None if c["normed"] == "none" else v}


def _times64(x, codes, scale):
    return torch.mm(x, _bits64(codes, scale, BLOCK).t().contiguous())


def _exact_matmul(d, c):
    x = _bits64(d["x"], d["x_scale"], 1)
    y = _times64(x, d["w"], d["w_scale"])
    if d["bias"] is not None:
        y += d["bias"].double()
    y = _act64(y, c["act"])
    if c["glu"]:
        y *= _times64(x, d["up"], d["up_scale"])
    if c["y"] == "e4m3":
        codes, scales = _quantise64(y)
        return {"y": codes, "y_scale": scales}
    if d["residual"] is not None:
        y += d["residual"].double()
    return {"y": y, "y_scale": None}


def _exact_grouped(d, c):
    off = d["offsets"].tolist()
    n = c["tokens"] * c["top_k"] + c["spare"]
    y = torch.zeros(n, c["rows"], dtype=torch.float64, device="cuda")
    scales = torch.zeros(n, _blocks(c["rows"]), dtype=torch.float64, device="cuda") if c["y"] == "e4m3" else None
    for e in range(c["groups"]):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        at = torch.arange(lo, hi, device="cuda")
        src = at if d["x_rows"] is None else d["x_rows"][lo:hi].long()
        dst = at if d["y_rows"] is None else d["y_rows"][lo:hi].long()
        x = _bits64(d["x"].view(torch.uint8)[src], d["x_scale"][src], 1)
        v = _times64(x, d["w"][e], d["w_scale"][e])
        if c["glu"]:
            v = torch.nn.functional.silu(v) * _times64(x, d["up"][e], d["up_scale"][e])
        if scales is None:
            y[dst] = v
        else:
            y[dst], scales[dst] = _quantise64(v)
    return {"y": y, "y_scale": scales}


def _exact_block(d, c):
    out = d["hidden"].double()
    for e in range(c["groups"]):
        t, k = torch.nonzero(d["idx"] == e, as_tuple=True)
        if t.numel() == 0:
            continue
        x = _bits64(d["x"].view(torch.uint8)[t], d["x_scale"][t], 1)
        a = torch.nn.functional.silu(_times64(x, d["gate"][e], d["gate_scale"][e]))
        a = a * _times64(x, d["up"][e], d["up_scale"][e])
        y = _times64(_scaled64(*_quantise64(a), 1), d["down"][e], d["down_scale"][e])
        out.index_add_(0, t, y * d["weight"].double()[t, k][:, None])
    return {"hidden": out}


def exact(case, seed):
    d = _inputs(case, seed)
    return {"norm": _exact_norm, "matmul": _exact_matmul, "grouped": _exact_grouped, "block": _exact_block}[case["op"]](d, case)
