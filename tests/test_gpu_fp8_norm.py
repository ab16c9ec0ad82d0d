"""bread_rmsnorm_fp8 against its definition in 64 bits."""
import pytest
import torch

import breadv2_amd as B
import fp8_reference as R

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
KINDS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def norm(T, n, kind, residual=True, hidden=True, normed="f32", weight=True, seed=0, pad=0, alias=None, eps=1e-6):
    g = torch.Generator().manual_seed(seed)
    x = (2.0 * torch.randn(T, n, generator=g)).to(kind)
    x[:, 1::97] *= 30
    r = torch.randn(T, n, generator=g).to(kind) if residual else None
    w = 1 + 0.3 * torch.randn(n, generator=g) if weight else None

    def wide(t, value, step):
        buf = torch.full((t.shape[0], t.shape[1] + pad * step), value, device="cuda").to(t.dtype)
        buf[:, :t.shape[1]].copy_(t)
        return buf, buf[:, :t.shape[1]]

    _, xd = wide(x, 9.0, 3)
    rd = wide(r, 9.0, 5)[1] if residual else None
    cb, codes = wide(torch.zeros(T, n).to(F8), 7.0, 16)
    sb, scales = wide(torch.zeros(T, R.blocks(n)), 7.0, 1)
    hb, hd = wide(torch.zeros(T, n).to(kind), 7.0, 7) if hidden else (None, None)
    if alias:
        hb, hd = None, xd if alias == "x" else rd
    ob, od = wide(torch.zeros(T, n).to(KINDS[normed]), 7.0, 1) if normed else (None, None)
    B.bread_rmsnorm_fp8(xd, None if w is None else w.cuda(), codes, scales, eps, residual=rd, hidden=hd, normed=od)
    torch.cuda.synchronize()
    h = x if r is None else (x.float() + r.float()).to(kind)  # rounded to x's type, as the operator does
    f = h.double()
    v = f / torch.sqrt((f * f).mean(1, keepdim=True) + eps) * (1.0 if w is None else w.double())
    # the sum of n squares: no rounding but on sums of positive terms, (n / 64 + 12) of them, half of it through the
    # root; root, division, two products: four more
    tol = (0.5 * (n / 64 + 12) + 5) * 2.0**-24 * v.abs()
    if hd is not None:
        assert torch.equal(hd.cpu(), h)
    R.check_quantised(codes, scales, v, tol)
    if od is not None:
        R.check_wide(od, v, tol)
    for buf, m in ((cb, n), (sb, R.blocks(n)), (hb, n), (ob, n)):
        if buf is not None:
            assert (buf[:, m:].float() == 7.0).all(), "behind a row"


@pytest.mark.parametrize("n", [16, 128, 144, 1040, 2048, 2064, 4096, 8192, 8208, 32768])
@pytest.mark.parametrize("T", [1, 3, 50])
@pytest.mark.parametrize("kind", list(KINDS))
def test_sizes(T, n, kind):
    norm(T, n, KINDS[kind], seed=n + T)


@pytest.mark.parametrize("T", [700, 3000])
def test_many_tokens(T):
    norm(T, 512, torch.float16, seed=T)
    norm(T, 2048, torch.bfloat16, residual=False, hidden=False, normed=None, seed=T)


@pytest.mark.parametrize("normed", ["f16", "bf16", "f32", None])
@pytest.mark.parametrize("residual,hidden,weight", [(True, True, True), (False, False, False), (True, False, False),
                                                    (False, True, True)])
def test_forms(normed, residual, hidden, weight):
    norm(7, 1040, torch.bfloat16, residual, hidden, normed, weight, seed=4, pad=1)
    norm(7, 272, torch.float32, residual, hidden, normed, weight, seed=5, pad=2)


@pytest.mark.parametrize("alias", ["x", "residual"])
@pytest.mark.parametrize("n", [512, 4096])
def test_hidden_in_place(alias, n):
    norm(9, n, torch.float16, alias=alias, seed=6)


def call(x, **kw):
    T, n = x.shape
    codes = torch.ones(T, n, device="cuda").to(F8)
    scales = torch.ones(T, R.blocks(n), device="cuda")
    B.bread_rmsnorm_fp8(x.cuda(), None, codes, scales, 1e-6, **kw)
    return codes.float().cpu(), scales.cpu()


def test_zeros_and_small_values():
    c, s = call(torch.zeros(2, 256))
    assert (c == 0).all() and (s == 2.0**-126).all()
    codes, scales = torch.ones(2, 256, device="cuda").to(F8), torch.ones(2, 2, device="cuda")
    x = torch.full((2, 256), 2.0**-130)  # eps holds the root up: values far below 448 * 2^-126
    x[:, 7] = -2.0**-127
    B.bread_rmsnorm_fp8(x.cuda(), None, codes, scales, 1.0)
    assert (scales == 2.0**-126).all()
    want = torch.round(x.double() * 2.0**126 / 2.0**-9) * 2.0**-9
    assert torch.equal(codes.double().cpu(), want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_stays_in_its_token(bad):
    x = torch.randn(5, 384, generator=torch.Generator().manual_seed(1))
    x[2, 130] = bad
    good = x.clone()
    good[2] = 0
    c, s = call(x)
    cg, sg = call(good)
    assert torch.isnan(s[2, 1]) and torch.isnan(c[2, 128:256]).all()
    keep = [0, 1, 3, 4]
    assert torch.equal(c[keep], cg[keep]) and torch.equal(s[keep], sg[keep])
    if bad != bad:
        assert torch.isnan(s[2]).all() and torch.isnan(c[2]).all()


def test_every_code_is_reached_and_ties_go_to_even():
    """One block whose values over the scale are every code's and the midpoints between neighbours."""
    t = R.table()[:127]  # 0 .. 448
    mid = (t[1:] + t[:-1]) / 2
    v = torch.cat([t, mid, -t, -mid])
    n = -(-v.numel() // 127) * 128
    x = torch.zeros(n, dtype=torch.float64)
    src = v.clone()
    for b in range(n // 128):  # 448 first in every block: the scale is the root's inverse
        x[128 * b] = 448.0
        part = src[127 * b:127 * b + 127]
        x[128 * b + 1:128 * b + 1 + part.numel()] = part
    x = x.float().view(1, -1)
    rms = torch.sqrt((x.double() ** 2).mean())
    pow2 = 2.0 ** torch.round(torch.log2(rms))
    # eps makes the root a power of two, so that nothing but the quantising rounds
    big = 4 * pow2
    eps = float((big * big - rms * rms))
    codes, scales = torch.ones(1, n, device="cuda").to(F8), torch.ones(1, n // 128, device="cuda")
    B.bread_rmsnorm_fp8(x.cuda(), None, codes, scales, eps)
    ratio = (scales.double().cpu() * big - 1).abs().max()
    assert ratio < 2.0**-20
    want, _ = R.quantise(x.double())
    got = codes.double().cpu()
    exact = torch.isin(x.double().abs(), t)
    assert torch.equal(got[exact], want[exact])
    if ratio == 0:  # the midpoints are ties
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", list(KINDS))
def test_codes_are_those_of_exact_numbers(kind):
    """A block's codes are of h w 448 / max|h w|, where the row's factor is not: each is the nearest one, but where the
    exact number lies on a tie (to 1e-14 of it, of three roundings of 2^-53)."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(400, 4096, generator=g).to(KINDS[kind])
    w = 1 + 0.3 * torch.randn(4096, generator=g)
    codes = torch.empty(400, 4096, dtype=F8, device="cuda")
    scales = torch.empty(400, 32, device="cuda")
    B.bread_rmsnorm_fp8(x.cuda(), w.cuda(), codes, scales, 1e-6)
    u = (x.double() * w.double()).view(400, 32, 128)
    ratio = (u * (448.0 / u.abs().amax(2, keepdim=True))).view(400, 4096)
    values = R.decode(torch.arange(127, dtype=torch.uint8).view(F8)).double()
    middle = (values[1:] + values[:-1]) / 2
    at = torch.searchsorted(middle, ratio.abs())
    near = middle[torch.clamp(torch.stack([at - 1, at]), 0, 125)]
    tie = ((near - ratio.abs()).abs() <= 1e-14 * near).any(0)
    got = R.decode(codes.cpu()).double()
    assert tie.sum() < 1000
    assert torch.equal(got[~tie], (values[at] * ratio.sign())[~tie])
