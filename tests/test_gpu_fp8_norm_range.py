"""bread_rmsnorm_fp8 of rows whose squares leave fp32's range although their norm does not."""
import pytest
import torch

import breadv2_amd as B
import fp8_reference as R

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def norm(x, eps, w=None, residual=None):
    T, n = x.shape
    codes, scales = torch.empty(T, n, dtype=F8, device="cuda"), torch.empty(T, R.blocks(n), device="cuda")
    normed, hidden = torch.empty(T, n, device="cuda"), torch.empty(T, n, dtype=x.dtype, device="cuda")
    B.bread_rmsnorm_fp8(x.cuda(), None if w is None else w.cuda(), codes, scales, eps, normed=normed, hidden=hidden,
                        residual=None if residual is None else residual.cuda())
    return codes, scales, normed, hidden


def check(x, eps, w=None, residual=None):
    codes, scales, normed, hidden = norm(x, eps, w, residual)
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    assert torch.equal(hidden.cpu(), h)
    f = h.double()
    n = x.shape[1]
    eps = torch.tensor(eps).double().item()  # as the call takes it: a float32
    # (in 64 bits the squares of all fp32 numbers are normal)
    v = f / torch.sqrt((f * f).mean(1, keepdim=True) + eps) * (1.0 if w is None else w.double())
    tol = (0.5 * (n / 64 + 12) + 5) * 2.0**-24 * v.abs()
    R.check_quantised(codes, scales, v, tol)
    R.check_wide(normed, v, tol)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [16, 512, 2048, 4096, 16400])
@pytest.mark.parametrize("size", [1e18, 3e19, 1e25, 1e37])
def test_large_values(n, size, kind):
    g = torch.Generator().manual_seed(n)
    x = torch.randn(5, n, generator=g)
    x[1, ::7] *= 1e-20  # beside others
    x[3] *= 1e-10
    x[4, 3] = 3.0
    w = 1 + 0.3 * torch.randn(n, generator=g)
    check((x * size).to(kind), 1e-6, w)
    check((x * size).to(kind), 1e30)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [16, 512, 4096, 16400])
@pytest.mark.parametrize("size", [1e-18, 1e-22, 1e-30, 1e-37])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-35])
def test_small_values(n, size, eps, kind):
    """Without an eps that holds the root up the norm is that of any size."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(5, n, generator=g)
    x[3] *= 1e5
    check((x * size).to(kind), eps, 1 + 0.3 * torch.randn(n, generator=g))


def test_the_smallest_and_the_largest_numbers():
    for n in (256, 4096):
        x = torch.full((3, n), 2.0**-149)
        x[1] = torch.finfo(torch.float32).max
        x[2, ::2] = 2.0**-140
        check(x, 0.0)


def test_beside_ordinary_rows():
    """A row's way is its own: the others' results are bit for bit those without it."""
    g = torch.Generator().manual_seed(7)
    for n in (512, 4096):
        x = torch.randn(9, n, generator=g)
        alone = norm(x, 1e-6)
        y = x.clone()
        y[4] *= 1e30
        with_it = norm(y, 1e-6)
        keep = [0, 1, 2, 3, 5, 6, 7, 8]
        for a, b in zip(alone, with_it):
            assert torch.equal(a.cpu().view(torch.uint8)[keep], b.cpu().view(torch.uint8)[keep])
        check(y, 1e-6, residual=torch.randn(9, n, generator=g))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_what_is_not_finite_among_large_values(bad):
    x = 1e30 * torch.randn(2, 512, generator=torch.Generator().manual_seed(8))
    x[0, 200] = bad
    codes, scales, normed, _ = norm(x, 1e-6)
    assert torch.isnan(scales[0, 1]) and torch.isnan(codes.float()[0, 128:256]).all() and torch.isnan(normed[0, 200])
    if bad != bad:
        assert torch.isnan(scales[0]).all()
    check(x[1:], 1e-6)
    assert torch.isfinite(scales[1]).all()
