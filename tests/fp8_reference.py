"""Plain forms of the 8-bit floating point operators in 64 bits, from their definitions, and the bounds that their tests
hold results to.  No part of the library is used.

Half a step of a rounding, relative: fp32 2^-24, fp16 2^-11, bf16 2^-8, e4m3 2^-4."""
import math

import torch

BLOCK = 128
F8 = torch.float8_e4m3fn
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}


def blocks(n):
    return -(-n // BLOCK)


def table():
    v = []
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        size = m * 2.0**-9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        if e == 15 and m == 7:
            size = math.nan
        v.append(-size if code & 128 else size)
    return torch.tensor(v, dtype=torch.float64)


def decode(codes):
    """The codes' values, in 64 bits on the CPU."""
    return table()[codes.cpu().contiguous().view(torch.uint8).long()]


def expand(scale, rows, cols, down):
    """A scale for every value: `down` rows share one."""
    s = scale.cpu().double()
    return s[torch.arange(rows) // down][:, torch.arange(cols) // BLOCK]


def activations(codes, scale):
    v = decode(codes)
    return v * expand(scale, *v.shape, 1)


def weights(codes, scale):
    v = decode(codes)
    return v * expand(scale, *v.shape, BLOCK)


def act64(v, act):
    f = torch.nn.functional
    return {None: lambda: v, "none": lambda: v, "silu": lambda: f.silu(v), "relu": lambda: torch.relu(v),
            "gelu": lambda: f.gelu(v), "gelu_tanh": lambda: f.gelu(v, approximate="tanh")}[act]()


def product(x, xs, w, ws):
    """(sums, bound of a kernel's error) of x [T][cols] through w [rows][cols]: exact products summed in fp32.  The 128
    products of a block: no more than 16 roundings each on a partial sum that the magnitudes' sum bounds (four matrix
    instructions, each a tree over 32 products and the sum so far); the blocks' sums: one a block; scales: two."""
    a, b = activations(x, xs), weights(w, ws)
    mag = a.abs() @ b.abs().T
    return a @ b.T, (16 + blocks(x.shape[1]) + 2) * 2.0**-24 * mag


def product_cut(x, xs, w, ws):
    """The same for the 8-bit matrix instructions: besides, of eight neighbouring products each loses less than 2^-13 of
    the largest one."""
    y, tol = product(x, xs, w, ws)
    a, b = activations(x, xs).abs(), weights(w, ws).abs()
    n = a.shape[1] // 8
    cut = torch.zeros_like(y)
    for t in range(a.shape[0]):
        cut[t] = (a[t].view(1, n, 8) * b.view(-1, n, 8)).amax(2).sum(1)
    return y, tol + 8 * 2.0**-13 * cut


def epilogue(v, tol, act=None, bias=None, up=None, up_tol=None, residual=None):
    """act(v + bias) [* up] + residual, and the bound: the activations' slopes are below 1.13, their own error is a
    few 2^-24 of v and 1.5e-7 of it (GELU); each other operation rounds once."""
    if bias is not None:
        v = v + bias.cpu().double()
        tol = tol + 2.0**-24 * v.abs()
    y = act64(v, act)
    if act not in (None, "none"):
        tol = 1.13 * tol + (8 * 2.0**-24 + 1.5e-7) * v.abs()
    if up is not None:
        tol = tol * up.abs() + up_tol * y.abs() + tol * up_tol + 2.0**-24 * (y * up).abs()
        y = y * up
    if residual is not None:
        y = y + residual.cpu().double()
        tol = tol + 2.0**-24 * y.abs()
    return y, tol


def check_wide(got, want, tol):
    """got within tol of want and half a step of its type."""
    g = got.cpu().double()
    lim = tol + HALF_STEP[got.dtype] * (want.abs() + tol) + TINY[got.dtype]
    off = (g - want).abs() - lim
    assert torch.isfinite(g).all()
    assert off.max() <= 0, f"{int((off > 0).sum())} of {off.numel()} beyond their bound, worst by {off.max():.3g}"


def quantise(v):
    """(codes' values, scales) of rows, in 64 bits."""
    codes, scales = torch.empty_like(v), []
    for at in range(0, v.shape[1], BLOCK):
        part = v[:, at:at + BLOCK]
        s = torch.clamp_min(part.abs().amax(1) / 448.0, 2.0**-126)
        q = part / s[:, None]
        _, e = torch.frexp(q)
        step = torch.ldexp(torch.ones_like(q), torch.clamp_min(e - 1, -6) - 3)
        codes[:, at:at + BLOCK] = torch.clamp(torch.round(q / step) * step, -448.0, 448.0)
        scales.append(s)
    return codes, torch.stack(scales, 1)


def check_quantised(codes, scale, want, tol):
    """Scales within tol / 448 of a block's largest magnitude (and two roundings), codes within half a step of the
    value over the scale that was given, tol besides."""
    s, v = scale.cpu().double(), decode(codes)
    T, n = want.shape
    for at in range(0, n, BLOCK):
        part, t = want[:, at:at + BLOCK], tol[:, at:at + BLOCK]
        b = s[:, at // BLOCK]
        top = torch.clamp_min(part.abs().amax(1) / 448.0, 2.0**-126)
        assert ((b - top).abs() <= t.amax(1) / 448.0 + 3 * 2.0**-24 * top).all(), "scale"
        q = part / b[:, None]
        _, e = torch.frexp(q)
        step = torch.ldexp(torch.ones_like(q), torch.clamp_min(e - 1, -6) - 3)
        lim = 0.5 * step * (1 + 2.0**-20) + t / b[:, None] + 4 * 2.0**-24 * q.abs()
        off = (v[:, at:at + BLOCK] - q).abs() - lim
        assert off.max() <= 0, f"codes of block {at // BLOCK}: worst by {off.max():.3g}"


def random_codes(*shape, gen, spread=108.0):
    """Codes of normally distributed values, zeros, the largest and the smallest among them."""
    v = spread * torch.randn(*shape, generator=gen)
    v = torch.where(torch.rand(*shape, generator=gen) < 0.02, torch.zeros(()), v)
    v = torch.where(torch.rand(*shape, generator=gen) < 0.02, 2.0**-9 * torch.sign(v), v)
    v = torch.where(torch.rand(*shape, generator=gen) < 0.02, 448.0 * torch.sign(v), v)
    return v.clamp(-448.0, 448.0).to(F8)


def random_weights(rows, cols, gen, groups=None):
    lead = () if groups is None else (groups,)
    s = 3e-4 * torch.exp2(4 * torch.rand(*lead, blocks(rows), blocks(cols), generator=gen) - 2)
    return random_codes(*lead, rows, cols, gen=gen), s


def random_activations(T, cols, gen):
    s = 0.01 * torch.exp2(6 * torch.rand(T, blocks(cols), generator=gen) - 3)
    return random_codes(T, cols, gen=gen), s
