"""Which 16-bit results of 8-bit products are exact products' and how far the others are off; residuals of many tokens; a
block without a residual; groups in order before others that are not."""
import ctypes

import pytest
import torch

import breadv2_amd as B
import fp8_reference as R
from breadv2_amd._lib import check, lib
from test_gpu_fp8_block import experts, reference
from test_gpu_fp8_matmul import dense

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
HALVES = [torch.float16, torch.bfloat16]
DEV = dict(device="cuda")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ordinary(*shape, gen):
    """Codes of normally distributed values."""
    return (108.0 * torch.randn(*shape, generator=gen)).clamp(-448.0, 448.0).to(F8)


def operands(T, rows, cols, g, groups=None):
    lead = () if groups is None else (groups,)
    x, xs = ordinary(T, cols, gen=g), 0.01 * (0.5 + torch.rand(T, R.blocks(cols), generator=g))
    w = ordinary(*lead, rows, cols, gen=g)
    return x, xs, w, 3e-4 * (0.5 + torch.rand(*lead, R.blocks(rows), R.blocks(cols), generator=g))


@pytest.mark.parametrize("kind", HALVES)
@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("T,rows,cols", [(1, 200, 2048), (9, 4096, 512), (19, 200, 384), (40, 1000, 2048), (130, 200, 2064)])
def test_a_few_tokens_are_exact_products(T, rows, cols, glu, kind):
    """The fp32 results of the same call, rounded; and those are within exact products' bound."""
    g = gen(T + cols)
    x, xs = R.random_activations(T, cols, g)
    w, ws = R.random_weights(rows, cols, g)
    up, us = R.random_weights(rows, cols, g) if glu else (None, None)
    wide, half = torch.empty(T, rows, **DEV), torch.empty(T, rows, dtype=kind, **DEV)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    for y in (wide, half):
        B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), y, up=dev(up), up_scale=dev(us))
    assert torch.equal(half, wide.to(kind))
    v, tol = R.product(x, xs, w, ws)
    u, ut = R.product(x, xs, up, us) if glu else (None, None)
    R.check_wide(wide, *R.epilogue(v, tol, None, None, u, ut))


@pytest.mark.parametrize("kind", HALVES)
@pytest.mark.parametrize("index", ["none", "gather"])
@pytest.mark.parametrize("G,n,rows,cols,glu", [(8, 3, 144, 512, False), (40, 150, 144, 272, True), (256, 1600, 512, 512, False)])
def test_small_groups_are_exact_products(G, n, rows, cols, glu, index, kind):
    g = gen(G + n)
    x, xs, w, ws = (t.cuda() for t in operands(n, rows, cols, g, G))
    up = ordinary(G, rows, cols, gen=g).cuda() if glu else None
    off = torch.sort(torch.randint(0, n + 1, (G + 1,), generator=g))[0].int()
    off[0], off[G] = 0, n
    x_rows = torch.randint(0, n, (n,), generator=g).int().cuda() if index == "gather" else None
    wide, half = torch.empty(n, rows, **DEV), torch.empty(n, rows, dtype=kind, **DEV)
    for y in (wide, half):
        B.bread_matmul_fp8_grouped(w, ws, x, xs, off.cuda(), y, up=up, up_scale=ws if glu else None, x_rows=x_rows)
    assert torch.equal(half, wide.to(kind))


@pytest.mark.parametrize("kind", HALVES)
@pytest.mark.parametrize("T,rows,cols", [(1300, 2600, 2048), (700, 3000, 512)])
def test_many_tokens_are_off_by_what_the_header_says(T, rows, cols, kind):
    """A residual that is minus the fp32 result, rounded, leaves the difference: it shows the sum before its rounding, to
    half a step of 2^-8 or less of half a step.  Off by 5e-5 of the results' size at most, and not exact (these are the
    8-bit instructions); each within what they cut of its eights."""
    g = gen(T)
    x, xs, w, ws = operands(T, rows, cols, g)
    wide = torch.empty(T, rows, **DEV)
    d = [t.cuda() for t in (w, ws, x, xs)]
    B.bread_matmul_fp8(*d, wide)
    r = (-wide).to(kind)
    y = torch.empty_like(r)
    B.bread_matmul_fp8(*d, y, residual=r)
    sums = y.cpu().double() - r.cpu().double()
    want, exact_tol = R.product(x, xs, w, ws)
    off = (sums - want).square().mean().sqrt() / want.square().mean().sqrt()
    # the difference's own rounding: half a step of one half step, 2^-22 or 2^-16 of the results
    own = R.HALF_STEP[kind] ** 2
    assert 1e-6 < off < 5e-5 + own, off
    assert (wide.cpu().double() - want).square().mean().sqrt() / want.square().mean().sqrt() < 1e-6
    rest = torch.arange(0, T, 97)
    _, tol = R.product_cut(x.view(torch.uint8)[rest].view(F8), xs[rest], w, ws)
    assert ((sums[rest] - want[rest]).abs() <= tol + 4 * own * want[rest].abs() + own * want[rest].abs().max()).all()


@pytest.mark.parametrize("glu", [False, True])
def test_many_rows_a_group_are_off_by_what_the_header_says(glu):
    """An error of 5e-5 of the results' size (two of them in a gated product) is a tenth (a fifth, a seventh together) of
    fp16's step, 2^-11 of it or more, in results of that size and larger: it moves so many of them to the next number.  No
    result is off by more than twenty such errors besides its own rounding."""
    G, n, rows, cols = 4, 3000, 1024, 512
    g = gen(3)
    x, xs, w, ws = (t.cuda() for t in operands(n, rows, cols, g, G))
    up = ordinary(G, rows, cols, gen=g).cuda() if glu else None
    off = torch.tensor([0, 700, 1500, 1501, n], dtype=torch.int32).cuda()
    wide, half = torch.empty(n, rows, **DEV), torch.empty(n, rows, dtype=torch.float16, **DEV)
    for y in (wide, half):
        B.bread_matmul_fp8_grouped(w, ws, x, xs, off, y, up=up, up_scale=ws if glu else None)
    size = wide.square().mean().sqrt()
    large = wide.abs() >= size
    moved = (half != wide.half())[large].float().mean()
    assert 0 < moved < (0.2 if glu else 0.1)
    assert ((half.float() - wide).abs() <= 2.0**-11 * wide.abs() + 20 * 5e-5 * size).all()


@pytest.mark.parametrize("y,glu", [("f32", False), ("bf16", False), ("f16", False), ("f32", True), ("bf16", True)])
@pytest.mark.parametrize("T,rows", [(1300, 2600), (700, 803), (260, 2050)])
def test_residuals_of_many_tokens(T, rows, y, glu):
    dense(T, rows, 272, y, "silu" if glu else None, glu, bias=not glu, residual=True, pad=1, seed=T)


@pytest.mark.parametrize("T,rows", [(1300, 2600), (300, 1000)])
def test_residuals_of_many_tokens_in_place(T, rows):
    g = gen(T)
    x, xs = R.random_activations(T, 256, g)
    w, ws = R.random_weights(rows, 256, g)
    y = torch.randn(T, rows, generator=g)
    out = y.cuda()
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), out, residual=out)
    v, tol = R.product(x, xs, w, ws)
    R.check_wide(out, *R.epilogue(v, tol, residual=y))


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 3, 400])
def test_a_block_without_a_residual(T, kind):
    """At the C entry a residual of NULL is zeros: what hidden holds before the call has no part in it."""
    E, I, H, K = 8, 256, 512, 2
    g = gen(T)
    t = experts(E, I, H, g)
    x, xs = R.random_activations(T, H, g)
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).int()
    w = torch.rand(T, K, generator=g)
    ctx = B.MoeContext(B.shape(H, I, I, E, K), max_tokens=T)
    ex = B.Fp8Experts(*[v.cuda() for v in t])
    hidden = torch.full((T, H), float("nan"), dtype=kind, **DEV)
    d = [v.cuda() for v in (x, xs, idx, w)]
    types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
    check(lib.bread_moe_expert_block_fp8(ctx._h, ctypes.byref(ex.desc), d[0].data_ptr(), d[1].data_ptr(), None,
                                         hidden.data_ptr(), types[kind], T, d[2].data_ptr(), d[3].data_ptr(),
                                         torch.cuda.current_stream().cuda_stream), "bread_moe_expert_block_fp8")
    assert ctx.check_device() == 0
    want, tol = reference(t, x, xs, idx, w, torch.zeros(T, H))
    R.check_wide(hidden, want, tol)


@pytest.mark.parametrize("y,glu", [("f32", False), ("bf16", False), ("f32", True)])
@pytest.mark.parametrize("n,rows,good", [(300, 144, 50), (2000, 528, 20)])
def test_groups_in_order_before_others_that_are_not(n, rows, good, y, glu):
    """The first groups ascend and hold rows that no other does; those behind fall, overlap and leave the rows."""
    G, cols = 120, 128
    g = gen(n)
    x, xs = R.random_activations(n, cols, g)
    w, ws = R.random_weights(rows, cols, g, groups=G)
    off = torch.randint(n // 2, 2**31 - 1, (G + 1,), generator=g)
    off[2::3] = torch.randint(n // 2, n, off[2::3].shape, generator=g)
    off[:good + 1] = torch.sort(torch.randint(0, n // 2, (good + 1,), generator=g))[0]
    kind = {"f32": torch.float32, "bf16": torch.bfloat16}[y]
    out = torch.full((n, rows), 3.0, **DEV).to(kind)
    B.bread_matmul_fp8_grouped(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), off.int().cuda(), out, up=w.cuda() if glu else None,
                               up_scale=ws.cuda() if glu else None)
    assert (out[:off[0]].float() == 3.0).all()
    for e in range(good):
        at = slice(int(off[e]), int(off[e + 1]))
        if at.start == at.stop:
            continue
        v, tol = (R.product_cut if y == "bf16" else R.product)(x.view(torch.uint8)[at].view(F8), xs[at], w[e], ws[e])
        R.check_wide(out[at], *(R.epilogue(v, tol, None, None, v, tol) if glu else (v, tol)))
