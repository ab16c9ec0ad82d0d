"""bread_matmul against 64-bit products of the oracle's dequantised weights.

Bound, derived before the first run.  Products of the kernels' operands are
exact, so a result's error is that of its fp32 sums: at most n roundings, each
of 2^-23 (the matrix cores may cut where IEEE rounds) of the sum S of the
magnitudes added, with S = sum |x| (|d sc q| + |dmin m|) and, of one path
through the sums, n <= 256 products of a chunk + 4 to apply its scales + a
rescaling and an addition for each of the cols / 256 chunks + 8 waves + bias and
residual = 270 + 2 cols / 256.  The oracle's fp32 weights are off by 2^-24 of the
same magnitudes.  fp16 results from Q6_K: weights rounded to 11 bits, 2^-11 S / 2.
Activations have slopes below 1.13 and are computed to 8 steps of 2^-24 of
their argument.  fp16 results: half a step, 2^-11 |y| (2^-25 among subnormals).
"""
import numpy as np
import pytest
import torch

import breadv2_amd as B
from breadv2_amd import api, synth
from oracle import oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
Q4, Q6, Q8, F16 = 12, 14, 8, 1
NAMES = {Q4: "q4k", Q6: "q6k", Q8: "q80", F16: "f16"}


def weights(qtype, rows, cols, seed, scale=1.0 / 64):
    """Bytes of random blocks; scales of about 0.0055 times `scale`."""
    rng = np.random.default_rng(seed)
    if qtype == F16:
        return (rng.standard_normal(rows * cols) * 0.03).astype(np.float16).view(np.uint8)
    if qtype == Q8:
        b = rng.integers(0, 256, size=(rows * cols // 32, 34), dtype=np.uint8)
        b[:, 0:2] = (rng.uniform(1e-3, 1e-2, len(b)) * scale).astype(np.float16).reshape(-1, 1).view(np.uint8)
        return b.reshape(-1)
    w = synth.synth_q4k(rows * cols // 256, seed) if qtype == Q4 else synth.synth_q6k(rows * cols // 256, seed)
    b = w.reshape(-1, 144 if qtype == Q4 else 210).copy()
    at = slice(0, 4) if qtype == Q4 else slice(208, 210)
    b[:, at] = (b[:, at].copy().view(np.float16) * np.float16(scale)).view(np.uint8)
    if qtype == Q6:  # the whole range of int8 scales, not only [-32, 31]
        b[:, 192:208] = rng.integers(0, 256, size=(len(b), 16), dtype=np.uint8)
    return b.reshape(-1)


def dense(w, qtype, rows, cols):
    """(weights, magnitudes of their parts) in 64 bits."""
    if qtype == F16:
        v = w.view(np.float16).astype(np.float64).reshape(rows, cols)
        return v, np.abs(v)
    v = O.dequant_rows(w, qtype, rows, cols).astype(np.float64).reshape(rows, cols)
    if qtype != Q4:
        return v, np.abs(v)
    z = w.reshape(-1, 144).copy()
    z[:, 16:] = 0
    m = O.dequant_rows(z.reshape(-1), qtype, rows, cols).astype(np.float64).reshape(rows, cols)
    return v, np.abs(v - m) + np.abs(m)


def erf(v):
    return torch.erf(torch.from_numpy(v)).numpy()


ACTS = {
    None: lambda v: v,
    "silu": lambda v: v / (1 + np.exp(-v)),
    "gelu": lambda v: 0.5 * v * (1 + erf(v / np.sqrt(2.0))),
    "gelu_tanh": lambda v: 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3))),
    "relu": lambda v: np.maximum(v, 0),
}


def expected(w, qtype, rows, cols, x, bias, act, res, half):
    wd, wm = dense(w, qtype, rows, cols)
    xd = x.astype(np.float64)
    v = xd @ wd.T
    s = np.abs(xd) @ wm.T
    tol = ((270 + 2 * cols / 256) * 2.0 ** -23 + (2.0 ** -12 if half and qtype == Q6 else 0.0)) * s
    if bias is not None:
        v = v + bias
        tol = tol + 2.0 ** -23 * np.abs(v)
    y = ACTS[act](v)
    if act is not None:
        tol = 1.13 * tol + 8 * 2.0 ** -24 * np.abs(v)
    if res is not None:
        y = y + res.astype(np.float64)
        tol = tol + 2.0 ** -24 * np.abs(y)
    if half:
        tol = tol + 2.0 ** -11 * (np.abs(y) + tol) + 2.0 ** -25
    return y, tol + 1e-30


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def case(qtype, T, rows, cols, seed, bias=True, act=None, res=True, half=True):
    rng = np.random.default_rng(seed)
    w = weights(qtype, rows, cols, seed)
    x = rng.standard_normal((T, cols)).astype(np.float16)
    b = rng.standard_normal(rows).astype(np.float32) if bias else None
    kind = np.float16 if half else np.float32
    r = rng.standard_normal((T, rows)).astype(kind) if res else None
    y = torch.full((T, rows), 7.0, dtype=torch.float16 if half else torch.float32, device=DEV)
    B.bread_matmul(dev(w), dev(x), y, rows, cols, qtype, bias=None if b is None else dev(b), act=act,
                   residual=None if r is None else dev(r))
    want, tol = expected(w, qtype, rows, cols, x, b, act, r, half)
    got = y.cpu().numpy().astype(np.float64)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (f"{NAMES[qtype]} T={T} rows={rows} cols={cols} half={half} act={act}: {bad.sum()} off, "
                           f"first {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]} +- {tol[bad][0]}")


COLS = {Q4: [256, 512, 2048, 2304], Q6: [256, 512, 2048, 2304], Q8: [32, 96, 256, 2080], F16: [8, 72, 256, 2056]}


@pytest.mark.parametrize("half", [True, False], ids=["y16", "y32"])
@pytest.mark.parametrize("qtype", [Q4, Q6, Q8, F16], ids=lambda q: NAMES[q])
@pytest.mark.parametrize("T", [1, 2, 9, 16, 17, 33, 64, 65])
def test_few_tokens(qtype, T, half):
    for i, cols in enumerate(COLS[qtype]):
        for rows in (1, 16, 50):
            case(qtype, T, rows, cols, seed=100 * T + 10 * i + rows, bias=i % 2 == 0, act=None, res=i % 2 == 1,
                 half=half)


@pytest.mark.parametrize("half", [True, False], ids=["y16", "y32"])
@pytest.mark.parametrize("qtype", [Q4, Q6, Q8, F16], ids=lambda q: NAMES[q])
@pytest.mark.parametrize("T", [66, 127, 128, 129, 200, 256, 300, 513])
def test_many_tokens(qtype, T, half):
    for i, cols in enumerate(COLS[qtype][1:]):
        for rows in (33, 128, 300):
            case(qtype, T, rows, cols, seed=100 * T + 10 * i + rows, bias=i % 2 == 1, act=None, res=i % 2 == 0,
                 half=half)


@pytest.mark.parametrize("qtype", [Q4, Q6, Q8, F16], ids=lambda q: NAMES[q])
def test_large(qtype):
    """Enough rows for every workgroup to take several tiles, and enough tokens for the largest tiles."""
    case(qtype, 3, 20000, 512, seed=5, half=True)
    case(qtype, 21, 9000, 4096 if qtype in (Q4, Q6) else 4128, seed=6, half=False)
    case(qtype, 1100, 2100, 512, seed=7, half=True)
    case(qtype, 1030, 2048, 768, seed=8, half=False)


@pytest.mark.parametrize("half", [True, False], ids=["y16", "y32"])
@pytest.mark.parametrize("qtype", [Q4, Q6, Q8, F16], ids=lambda q: NAMES[q])
@pytest.mark.parametrize("T", [33, 70, 97])
def test_long_rows_for_a_few_dozen_tokens(qtype, T, half):
    """Superblocks over eight groups of waves: fewer than groups, some more, the last one cut short."""
    short = {Q4: 0, Q6: 0, Q8: 32, F16: 8}[qtype]
    for i, cols in enumerate((1280, 2048, 2304 + short, 4352 - short)):
        for rows in (31, 96):
            case(qtype, T, rows, cols, seed=T + 10 * i + rows, bias=i % 2 == 0, act=None, res=i % 2 == 1, half=half)


@pytest.mark.parametrize("half", [True, False], ids=["y16", "y32"])
@pytest.mark.parametrize("qtype", [Q4, Q6, Q8, F16], ids=lambda q: NAMES[q])
def test_many_rows_of_two_chunks_a_wave(qtype, half):
    """Rows enough for every workgroup to take several tiles, with 9 to 16 superblocks, the last one cut short."""
    short = {Q4: 0, Q6: 0, Q8: 32, F16: 8}[qtype]
    case(qtype, 7, 16403, 2304, seed=21, bias=True, act=None, res=False, half=half)
    case(qtype, 16, 24601, 2304 + short, seed=22, bias=False, act=None, res=True, half=half)
    case(qtype, 1, 20000, 4096 - short, seed=23, half=half)


@pytest.mark.parametrize("qtype", [Q4, Q6, Q8, F16], ids=lambda q: NAMES[q])
def test_tokens_far_apart(qtype):
    """Tokens 2^22 elements from each other: beyond the tiles' 32-bit offsets."""
    rows, cols = 50, 512
    wide = torch.zeros(70, 1 << 22, dtype=torch.float16, device=DEV)
    w = weights(qtype, rows, cols, 8)
    for T in (33, 64, 70):
        x = np.random.default_rng(T).standard_normal((T, cols)).astype(np.float16)
        wide[:T, 64:64 + cols] = dev(x)
        y = torch.empty(T, rows, device=DEV)
        B.bread_matmul(dev(w), wide[:T, 64:64 + cols], y, rows, cols, qtype)
        want, tol = expected(w, qtype, rows, cols, x, None, None, None, False)
        assert np.all(np.abs(y.cpu().numpy() - want) <= tol), (NAMES[qtype], T)


@pytest.mark.parametrize("act", [a for a in ACTS if a])
@pytest.mark.parametrize("T", [3, 150])
def test_activations(act, T):
    for qtype in (Q4, Q8):
        case(qtype, T, 70, 512, seed=T, act=act, half=True)
        case(qtype, T, 70, 512, seed=T + 1, act=act, half=False, res=False)


def test_activations_far_out():
    """Arguments of +-40 (a bias): the gates are 0 and 1 there, nothing overflows."""
    w = np.zeros(16 * 256 // 32 * 34, np.uint8)
    x = torch.zeros(2, 256, dtype=torch.float16, device=DEV)
    b = torch.tensor([-1e4, -100.0, -40.0, -10.0, -6.0, -3.0, -1.0, -1e-3, 0.0, 1e-3, 1.0, 3.0, 6.0, 10.0, 40.0, 1e4],
                     device=DEV)
    for act in ACTS:
        y = torch.empty(2, 16, device=DEV)
        B.bread_matmul(dev(w), x, y, 16, 256, Q8, bias=b, act=act)
        v = b.cpu().numpy().astype(np.float64)
        with np.errstate(over="ignore"):
            want = ACTS[act](v)
        assert np.all(np.abs(y.cpu().numpy() - want) <= 8 * 2.0 ** -24 * np.abs(v) + 1e-30), act


@pytest.mark.parametrize("qtype", [Q4, Q6, Q8, F16], ids=lambda q: NAMES[q])
@pytest.mark.parametrize("T", [5, 150])
def test_strided_rows_and_what_lies_between(qtype, T):
    """x and y as column slices of wider buffers; everything outside y's slice stays."""
    rows, cols = 37, 512
    rng = np.random.default_rng(T)
    w = weights(qtype, rows, cols, 3)
    wide = dev(rng.standard_normal((T, cols + 40)).astype(np.float16))
    x = wide[:, 16:16 + cols]
    out = torch.full((T, rows + 11), -3.0, device=DEV)
    res = dev(rng.standard_normal((T, rows + 11)).astype(np.float32))
    y = out[:, 5:5 + rows]
    B.bread_matmul(dev(w), x, y, rows, cols, qtype, residual=res[:, 5:5 + rows])
    want, tol = expected(w, qtype, rows, cols, x.cpu().numpy(), None, None, res[:, 5:5 + rows].cpu().numpy(), False)
    assert np.all(np.abs(y.cpu().numpy() - want) <= tol)
    assert torch.all(out[:, :5] == -3.0) and torch.all(out[:, 5 + rows:] == -3.0)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("T", [4, 140])
def test_residual_in_place(T, half):
    rows, cols = 100, 768
    rng = np.random.default_rng(9)
    w = weights(Q4, rows, cols, 4)
    x = rng.standard_normal((T, cols)).astype(np.float16)
    h = rng.standard_normal((T, rows)).astype(np.float16 if half else np.float32)
    y = dev(h)
    B.bread_matmul(dev(w), dev(x), y, rows, cols, Q4, residual=y)
    want, tol = expected(w, Q4, rows, cols, x, None, None, h, half)
    assert np.all(np.abs(y.cpu().numpy().astype(np.float64) - want) <= tol)


@pytest.mark.parametrize("qtype", [Q4, Q6, Q8, F16], ids=lambda q: NAMES[q])
@pytest.mark.parametrize("T", [6, 150])
def test_a_tokens_infinities_stay_with_it(qtype, T):
    """Inf and NaN in one token's row or one weight row's scale leave the others as they were."""
    rows, cols = 40, 512
    rng = np.random.default_rng(T)
    w = weights(qtype, rows, cols, 8)
    x = rng.standard_normal((T, cols)).astype(np.float16)
    y0 = torch.empty(T, rows, device=DEV)
    B.bread_matmul(dev(w), dev(x), y0, rows, cols, qtype)
    xb = x.copy()
    xb[2, 17], xb[4, 300] = np.nan, np.inf
    wb = w.reshape(rows, -1).copy()
    at = {Q4: 0, Q6: 208, Q8: 0, F16: 0}[qtype]
    wb[11, at:at + 2] = np.array([np.nan], np.float16).view(np.uint8)
    y1 = torch.empty(T, rows, device=DEV)
    B.bread_matmul(dev(wb.reshape(-1)), dev(xb), y1, rows, cols, qtype)
    t = np.setdiff1d(np.arange(T), [2, 4])
    r = np.setdiff1d(np.arange(rows), [11])
    a, b = y0.cpu().numpy(), y1.cpu().numpy()
    assert np.array_equal(a[np.ix_(t, r)], b[np.ix_(t, r)])
    assert np.isnan(b[2]).all() and not np.isfinite(b[4][r]).any() and np.isnan(b[:, 11]).all()


@pytest.mark.parametrize("T", [2, 150])
def test_scales_of_all_sizes(T):
    """Superblocks whose scale is zero, subnormal, large or negative next to ordinary ones, min terms without a scale,
    scales that jump by 2^20 from one superblock to the next."""
    rows, cols = 48, 2048
    rng = np.random.default_rng(1)
    x = rng.standard_normal((T, cols)).astype(np.float16)
    kinds = np.array([0.0, 6e-8, 1e-6, 1e-3, -1e-3, 0.5, 8.0, -0.0], np.float16)
    for qtype in (Q4, Q6, Q8):
        per, size = {Q4: (256, 144), Q6: (256, 210), Q8: (32, 34)}[qtype]
        b = weights(qtype, rows, cols, 12).reshape(-1, size).copy()
        at = 208 if qtype == Q6 else 0
        b[:, at:at + 2] = kinds[rng.integers(0, len(kinds), len(b))].reshape(-1, 1).view(np.uint8)
        if qtype == Q4:
            b[:, 2:4] = kinds[rng.integers(0, len(kinds), len(b))].reshape(-1, 1).view(np.uint8)
        b = b.reshape(rows, -1)
        b[3] = 0  # a row of nothing
        w = b.reshape(-1)
        y = torch.empty(T, rows, device=DEV)
        B.bread_matmul(dev(w), dev(x), y, rows, cols, qtype)
        want, tol = expected(w, qtype, rows, cols, x, None, None, None, False)
        got = y.cpu().numpy()
        assert np.all(np.abs(got - want) <= tol), NAMES[qtype]
        assert np.all(got[:, 3] == 0)


def test_one_token_alone_and_among_others():
    """A token's result through the same kernel does not depend on its neighbours."""
    rows, cols = 64, 1024
    for qtype in (Q4, Q6, Q8, F16):
        w = dev(weights(qtype, rows, cols, 2))
        x = dev(np.random.default_rng(0).standard_normal((16, cols)).astype(np.float16))
        y = torch.empty(16, rows, device=DEV)
        B.bread_matmul(w, x, y, rows, cols, qtype)
        for t in (0, 7, 15):
            one = torch.empty(1, rows, device=DEV)
            B.bread_matmul(w, x[t:t + 1], one, rows, cols, qtype)
            assert torch.equal(one[0], y[t])


def test_nothing_to_do():
    w = dev(weights(Q4, 4, 256, 1))
    y = torch.full((3, 4), 5.0, device=DEV)
    B.bread_matmul(w, torch.empty(0, 256, dtype=torch.float16, device=DEV), y[:0], 4, 256, Q4)
    B.bread_matmul(w, torch.ones(3, 256, dtype=torch.float16, device=DEV), y[:, :0], 0, 256, Q4)
    torch.cuda.synchronize()
    assert torch.all(y == 5.0)


def test_stream_and_graph():
    """On another stream than the current one, and captured and replayed with new inputs in the same buffers."""
    rows, cols = 96, 512
    for T in (7, 150):
        w = dev(weights(Q6, rows, cols, 2))
        x = torch.randn(T, cols, device=DEV).half()
        y = torch.empty(T, rows, device=DEV)
        ref = torch.empty(T, rows, device=DEV)
        B.bread_matmul(w, x, ref, rows, cols, Q6)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        B.bread_matmul(w, x, y, rows, cols, Q6, stream=s)
        s.synchronize()
        assert torch.equal(y, ref)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            B.bread_matmul(w, x, y, rows, cols, Q6)
        for _ in range(3):
            x.copy_(torch.randn(T, cols, device=DEV).half())
            y.zero_()
            g.replay()
            B.bread_matmul(w, x, ref, rows, cols, Q6)
            torch.cuda.synchronize()
            assert torch.equal(y, ref)
