"""8-bit products at the ends of what the header allows of scales: products of two scales just below 2^128, below 2^-126
(where fp32 holds them to 2^-150, which is what a block's sum is multiplied by), infinite and NaN scales."""
import pytest
import torch

import breadv2_amd as B
import fp8_reference as R

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
KINDS = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": F8}
W = (8e7, 1e-9)     # scales of the weights' first two blocks of columns, times 0.25 to 4
UP = (1e-34, 1e30)  # of a second matrix


def tokens(T, cols, g):
    """Of four tokens: one that is ordinary; one with a scale of 1e30 and zeros under it; one with the smallest code
    under it; one with codes under a scale of 1e-33 alone."""
    x, xs = R.random_activations(T, cols, g)
    v = x.float()
    v[:, :256] = 0
    xs[:, :2] = 1.0
    xs[1::4, 0] = 1e30
    xs[2::4, 0] = 1e30
    v[2::4] = 0
    v[2::4, 5] = 2.0**-9
    v[3::4] = 0
    v[3::4, 128:256] = x.float()[3::4, 128:256]
    xs[3::4, 1] = 1e-33
    return v.to(F8), xs


def matrix(rows, cols, g, first, groups=None):
    w, ws = R.random_weights(rows, cols, g, groups)
    v = w.float()
    v[..., 5] = 2.0**-9
    for b, s in enumerate(first):
        ws[..., b] *= s / 3e-4
    return v.to(F8), ws


def product(y, x, xs, w, ws):
    v, tol = (R.product_cut if y == "bf16" else R.product)(x, xs, w, ws)
    return v, tol + 2.0**-150 * (R.decode(x).abs() @ R.decode(w).abs().T)


def check(y, out, scale, x, xs, w, ws, up, us):
    v, tol = product(y, x, xs, w, ws)
    u, ut = product(y, x, xs, up, us) if up is not None else (None, None)
    want, tol = R.epilogue(v, tol, None, None, u, ut)
    if y == "e4m3":
        R.check_quantised(out, scale, want, tol)
    else:
        R.check_wide(out, want, tol)


def results(n, rows, y):
    s = torch.zeros(n, R.blocks(rows), device="cuda") if y == "e4m3" else None
    return torch.zeros(n, rows, device="cuda").to(KINDS[y]), s


@pytest.mark.parametrize("y,glu", [("f32", False), ("bf16", False), ("e4m3", False), ("f32", True), ("bf16", True), ("e4m3", True)])
@pytest.mark.parametrize("T,rows", [(4, 64), (40, 4112), (100, 4080), (131, 2064), (300, 2064), (700, 800), (1300, 2608)])
def test_one_matrix(T, rows, y, glu):
    g = torch.Generator().manual_seed(T)
    x, xs = tokens(T, 400, g)
    w, ws = matrix(rows, 400, g, W)
    up, us = matrix(rows, 400, g, UP) if glu else (None, None)
    out, scale = results(T, rows, y)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), out, y_scale=scale, up=dev(up), up_scale=dev(us))
    check(y, out, scale, x, xs, w, ws, up, us)


@pytest.mark.parametrize("y,glu", [("f32", False), ("bf16", False), ("e4m3", False), ("f32", True), ("bf16", True), ("e4m3", True)])
@pytest.mark.parametrize("G,n,rows", [(3, 12, 144), (8, 540, 512), (24, 1500, 528), (6, 1500, 256)])
def test_groups(G, n, rows, y, glu):
    g = torch.Generator().manual_seed(n + G)
    x, xs = tokens(n, 400, g)
    w, ws = matrix(rows, 400, g, W, G)
    up, us = matrix(rows, 400, g, UP, G) if glu else (None, None)
    off = torch.arange(G + 1) * n // G
    out, scale = results(n, rows, y)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    B.bread_matmul_fp8_grouped(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), off.int().cuda(), out, y_scale=scale, up=dev(up),
                               up_scale=dev(us))
    for e in range(G):
        at = slice(int(off[e]), int(off[e + 1]))
        check(y, out.view(torch.uint8)[at].view(F8) if y == "e4m3" else out[at], None if scale is None else scale[at],
              x.view(torch.uint8)[at].view(F8), xs[at], w[e], ws[e], None if up is None else up[e], None if us is None else us[e])


@pytest.mark.parametrize("T", [0, 5, 150])
def test_rows_of_zeros_beside_others(T):
    """A row of zeros has the smallest scale, whose product with a weight's is below fp32's normal numbers."""
    n = 300
    x, xs = R.random_activations(n, 512, torch.Generator().manual_seed(1))
    w, ws = R.random_weights(272, 512, torch.Generator().manual_seed(2))
    x.view(torch.uint8)[T:] = 0
    xs[T:] = 2.0**-126
    for y in ("f32", "bf16", "e4m3"):
        out, scale = results(n, 272, y)
        B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), out, y_scale=scale)
        check(y, out, scale, x, xs, w, ws, None, None)
        assert (out.float()[T:] == 0).all()


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan"), 0.0])
def test_scales_that_are_no_numbers_or_zero(bad):
    """They are what the definition makes of them: an infinity times a sum of zero is NaN, times another an infinity."""
    T, rows = 150, 144
    g = torch.Generator().manual_seed(3)
    x, xs = R.random_activations(T, 256, g)
    w, ws = R.random_weights(rows, 256, g)
    xs[4, 1] = bad
    xs[9, 0] = bad
    x.view(torch.uint8)[9, :128] = 0
    a, b = R.activations(x, xs.double().nan_to_num(1.0, 1.0, 1.0).float()), R.weights(w, ws)
    out = torch.zeros(T, rows, device="cuda")
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), out)
    got = out.cpu().double()
    rest = [t for t in range(T) if t not in (4, 9)]
    R.check_wide(out[rest], *[v[rest] for v in R.product(x, xs.double().nan_to_num(1.0, 1.0, 1.0).float(), w, ws)])
    z = R.decode(x)[4, 128:] @ R.decode(w)[:, 128:].T
    if bad == 0:
        assert (got[9] - (a[9, 128:] @ b[:, 128:].T)).abs().max() <= 1e-5 * (a[9].abs() @ b.abs().T).max()
        assert (got[4] - (a[4, :128] @ b[:, :128].T)).abs().max() <= 1e-5 * (a[4].abs() @ b.abs().T).max()
    else:
        assert torch.isnan(got[9]).all()
        want = bad * z
        assert torch.equal(torch.isnan(got[4]), torch.isnan(want))
        keep = ~torch.isnan(want)
        assert torch.equal(got[4][keep], want[keep])


def test_products_of_scales_beyond_fp32():
    """Infinite from 2^128 on: so is the result, or NaN where the block's sum is zero."""
    g = torch.Generator().manual_seed(4)
    x, xs = R.random_activations(20, 128, g)
    w, ws = R.random_weights(64, 128, g)
    x.view(torch.uint8)[7] = 0
    xs[:], ws[:] = 2.0**64, 2.0**64
    out = torch.zeros(20, 64, device="cuda")
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), out)
    z = R.decode(x) @ R.decode(w).T
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), z == 0) and torch.isnan(got[7]).all()
    assert torch.equal(got[z != 0], (z * float("inf"))[z != 0])
