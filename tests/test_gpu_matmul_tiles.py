"""bread_matmul's large tiles, each with the fewest tokens and rows that choose it, odd sizes and ends.

The bound is test_gpu_matmul.py's.  The sizes are checked against the rule that chooses the tile: the largest one
with at least 200 workgroups (256 x 256: Q4_K and fp16 only).
"""
import numpy as np
import pytest
import torch

import breadv2_amd as B

from test_gpu_matmul import DEV, F16, NAMES, Q4, Q6, Q8, case, dev, expected, weights

pytestmark = pytest.mark.gpu

TILES = [(256, 256), (128, 256), (128, 128), (64, 64)]
SIZES = {(128, 128): (1537, 2100), (128, 256): (2049, 3300), (256, 256): (3585, 3400)}
CASES = [(q, m, n) for m, n in SIZES for q in (Q4, Q6, Q8, F16) if (m, n) != (256, 256) or q in (Q4, F16)]


def tile_of(qtype, T, rows):
    for m, n in TILES:
        if (m, n) == (256, 256) and qtype in (Q6, Q8):
            continue
        if -(-T // m) * -(-rows // n) >= 200:
            return m, n


@pytest.mark.parametrize("half", [True, False], ids=["y16", "y32"])
@pytest.mark.parametrize("qtype,m,n", CASES, ids=[f"{NAMES[q]}-{m}x{n}" for q, m, n in CASES])
def test_large_tiles(qtype, m, n, half):
    T, rows = SIZES[m, n]
    assert tile_of(qtype, T, rows) == (m, n)
    short = {Q4: 0, Q6: 0, Q8: 32, F16: 8}[qtype]
    case(qtype, T, rows, 512, seed=m + n, bias=True, act="gelu" if half else "silu", res=False, half=half)
    case(qtype, T, rows, 768 - short, seed=m + n + 1, bias=False, act=None, res=True, half=half)
    case(qtype, T, rows, 256 + short, seed=m + n + 2, bias=True, act=None, res=True, half=half)


@pytest.mark.parametrize("qtype,m,n", [c for c in CASES if c[0] != F16],
                         ids=[f"{NAMES[q]}-{m}x{n}" for q, m, n in CASES if q != F16])
def test_large_tiles_with_scales_of_all_sizes(qtype, m, n):
    """Scales of zero, subnormal, negative and large ones side by side; a row of nothing; strided tokens and results."""
    T, rows = SIZES[m, n]
    cols = 1024
    rng = np.random.default_rng(m + n)
    kinds = np.array([0.0, 6e-8, 1e-6, 1e-3, -1e-3, 0.5, 8.0, -0.0], np.float16)
    size = {Q4: 144, Q6: 210, Q8: 34}[qtype]
    b = weights(qtype, rows, cols, 12).reshape(-1, size).copy()
    at = 208 if qtype == Q6 else 0
    b[:, at:at + 2] = kinds[rng.integers(0, len(kinds), len(b))].reshape(-1, 1).view(np.uint8)
    if qtype == Q4:
        b[:, 2:4] = kinds[rng.integers(0, len(kinds), len(b))].reshape(-1, 1).view(np.uint8)
    b = b.reshape(rows, -1)
    b[3] = 0
    w = b.reshape(-1)
    x = rng.standard_normal((T, cols)).astype(np.float16)
    wide = torch.zeros(T, cols + 24, dtype=torch.float16, device=DEV)
    wide[:, 8:8 + cols] = dev(x)
    out = torch.full((T, rows + 9), -3.0, device=DEV)
    B.bread_matmul(dev(w), wide[:, 8:8 + cols], out[:, 5:5 + rows], rows, cols, qtype)
    want, tol = expected(w, qtype, rows, cols, x, None, None, None, False)
    got = out[:, 5:5 + rows].cpu().numpy()
    assert np.all(np.abs(got - want) <= tol)
    assert np.all(got[:, 3] == 0)
    assert torch.all(out[:, :5] == -3.0) and torch.all(out[:, 5 + rows:] == -3.0)


@pytest.mark.parametrize("qtype,m,n", CASES, ids=[f"{NAMES[q]}-{m}x{n}" for q, m, n in CASES])
def test_large_tiles_in_place_and_captured(qtype, m, n):
    """The residual is y; a graph's replays with new inputs equal eager calls, and tokens' NaN stay with them."""
    T, rows = SIZES[m, n]
    cols = 512
    w = dev(weights(qtype, rows, cols, 2))
    x = torch.randn(T, cols, device=DEV).half()
    h = torch.randn(T, rows, device=DEV)
    y, ref = h.clone(), h.clone()
    B.bread_matmul(w, x, ref, rows, cols, qtype, residual=ref)
    plain = torch.empty_like(h)
    B.bread_matmul(w, x, plain, rows, cols, qtype)
    assert torch.equal(plain + h, ref)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        B.bread_matmul(w, x, y, rows, cols, qtype, residual=y)
    for k in range(3):
        x.copy_(torch.randn(T, cols, device=DEV).half())
        x[k::500, 7] = float("nan")
        y.copy_(h)
        g.replay()
        torch.cuda.synchronize()
        ref.copy_(h)
        B.bread_matmul(w, x, ref, rows, cols, qtype, residual=ref)
        assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y.nan_to_num(), ref.nan_to_num())
        bad = torch.zeros(T, dtype=torch.bool, device=DEV)
        bad[k::500] = True
        assert y[bad].isnan().all() and not y[~bad].isnan().any()
