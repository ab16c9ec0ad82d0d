"""8-bit operators in buffers whose rows and matrices lie further than 32 bits reach."""
import pytest
import torch

import breadv2_amd as B
import fp8_reference as R

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
DEV = dict(device="cuda")


@pytest.fixture(autouse=True)
def release():
    """Some tens of GB go back before the next test."""
    yield
    torch.cuda.empty_cache()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def strided(t, step):
    """A copy of t on the GPU whose rows lie `step` elements apart."""
    one = torch.uint8 if t.dtype == F8 else t.dtype
    buf = torch.empty(t.shape[0], step, dtype=one, **DEV)
    buf[:, :t.shape[1]].copy_(t.view(one) if t.dtype == F8 else t)
    rows = buf[:, :t.shape[1]]
    return rows.view(F8) if t.dtype == F8 else rows


@pytest.mark.parametrize("glu,y", [(False, torch.float32), (True, torch.bfloat16), (True, F8)])
def test_strides_of_a_product(glu, y):
    T, rows, cols = 1100, 272, 400
    g = gen(1)
    x, xs = R.random_activations(T, cols, g)
    w, ws = R.random_weights(rows, cols, g)
    up, us = R.random_weights(rows, cols, g) if glu else (None, None)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    near = torch.zeros(T, rows, **DEV).to(y)
    far = strided(torch.zeros(T, rows).to(y), 1 << 22)  # 4.6 to 18 GB
    scales = [torch.zeros(T, 3, **DEV), strided(torch.zeros(T, 3), 1 << 20)] if y == F8 else [None, None]
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), near, y_scale=scales[0], up=dev(up), up_scale=dev(us))
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), strided(x, 1 << 22), strided(xs, 1 << 20), far, y_scale=scales[1], up=dev(up),
                       up_scale=dev(us))
    bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(bits(near), bits(far))
    assert y != F8 or torch.equal(*scales)
    v, tol = (R.product_cut if y == torch.bfloat16 else R.product)(x, xs, w, ws)
    u, ut = R.product(x, xs, up, us) if glu else (None, None)
    want, tol = R.epilogue(v, tol, None, None, u, ut)
    if y == F8:
        R.check_quantised(near, scales[0], want, tol)
    else:
        R.check_wide(near, want, tol)


def test_strides_of_a_norm():
    T, n = 1100, 512
    g = gen(2)
    x, r = torch.randn(T, n, generator=g), torch.randn(T, n, generator=g)
    step = 1 << 21
    out = []
    for far in (False, True):
        place = (lambda t: strided(t, step)) if far else (lambda t: t.cuda())
        codes, scales = place(torch.zeros(T, n).to(F8)), place(torch.zeros(T, 4))
        hidden, normed = place(torch.zeros(T, n)), place(torch.zeros(T, n))
        B.bread_rmsnorm_fp8(place(x), None, codes, scales, 1e-6, residual=place(r), hidden=hidden, normed=normed)
        out.append([t.contiguous().view(torch.uint8) for t in (codes, scales, hidden, normed)])
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [30, 700])
def test_matrices_of_groups(n):
    """The last of seventy matrices of 64 MB, two of them, and rows of x and y behind the first 2^32 bytes."""
    G, rows, cols = 70, 8192, 8192
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    w = torch.empty(G, rows, cols, dtype=torch.uint8, **DEV)
    for e in range(G):
        w[e] = (60 * torch.randn(rows, cols, generator=g, **DEV)).to(F8).view(torch.uint8)
    w = w.view(F8)
    ws = 3e-4 * (0.5 + torch.rand(G, rows // 128, cols // 128, generator=g, **DEV))
    x, xs = R.random_activations(n, cols, gen(n))
    off = torch.zeros(G + 1, dtype=torch.int32)
    off[34:], off[G - 1:], off[G] = n // 3, n // 2, n  # rows of matrices 33, 68 and 69
    y = strided(torch.zeros(n, rows), 1 << 21)
    B.bread_matmul_fp8_grouped(w, ws, x.cuda(), xs.cuda(), off.cuda(), y)
    for e in (33, G - 2, G - 1):
        at = torch.arange(int(off[e]), int(off[e + 1]))[:5]
        want, tol = R.product(x.view(torch.uint8)[at].view(F8), xs[at], w[e], ws[e])
        R.check_wide(y[at.cuda()], want, tol)


def test_gathered_activations_up_to_the_limit():
    """x of 2^31 bytes, whose last rows are named."""
    n_x, cols, step, n = 1 << 13, 272, 1 << 18, 300
    buf = torch.empty(n_x, step, dtype=torch.uint8, **DEV)
    x, xs = R.random_activations(n, cols, gen(4))
    at = torch.randperm(n_x, generator=gen(5))[:n]
    at[0], at[1] = n_x - 1, 0
    buf[at.cuda(), :cols] = x.view(torch.uint8).cuda()
    sbuf = torch.zeros(n_x, R.blocks(cols), **DEV)
    sbuf[at.cuda()] = xs.cuda()
    w, ws = R.random_weights(144, cols, gen(6), groups=3)
    off = torch.tensor([0, 100, 101, n], dtype=torch.int32)
    y = torch.empty(n, 144, **DEV)
    B.bread_matmul_fp8_grouped(w.cuda(), ws.cuda(), buf[:, :cols].view(F8), sbuf, off.cuda(), y, x_rows=at.int().cuda())
    for e in range(3):
        s = slice(int(off[e]), int(off[e + 1]))
        R.check_wide(y[s], *R.product(x.view(torch.uint8)[s].view(F8), xs[s], w[e], ws[e]))
