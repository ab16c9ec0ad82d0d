"""bread_matmul_fp8 and bread_matmul_fp8_grouped against 64-bit products of the decoded values."""
import pytest
import torch

import breadv2_amd as B
import fp8_reference as R

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
KINDS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": F8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cut(y):
    """Whether results of this type may come from the 8-bit matrix instructions."""
    return y in ("f16", "bf16")


def dense(T, rows, cols, y="f32", act=None, glu=False, bias=False, residual=False, seed=0, pad=0):
    g = gen(seed)
    x, xs = R.random_activations(T, cols, g)
    w, ws = R.random_weights(rows, cols, g)
    up, us = R.random_weights(rows, cols, g) if glu else (None, None)
    b = torch.randn(rows, generator=g) if bias else None
    kind = KINDS[y]
    r = torch.randn(T, rows, generator=g).to(kind) if residual else None

    def wide(t, value):
        """A copy in a wider buffer, `value` behind every row."""
        step = 16 if t.dtype == F8 else 3
        buf = torch.full((t.shape[0], t.shape[1] + pad * step), value, device="cuda").to(t.dtype)
        buf[:, :t.shape[1]].copy_(t)
        return buf, buf[:, :t.shape[1]]

    out_buf, out = wide(torch.zeros(T, rows).to(kind), 7.0)
    scale_buf, scale = wide(torch.zeros(T, R.blocks(rows)), 7.0) if y == "e4m3" else (None, None)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    res = wide(r, 5.0)[1] if residual else None
    B.bread_matmul_fp8(dev(w), dev(ws), wide(x, 448.0)[1], wide(xs, 1e30)[1], out, y_scale=scale, up=dev(up),
                       up_scale=dev(us), bias=dev(b), act=act, residual=res)
    torch.cuda.synchronize()
    product = R.product_cut if cut(y) else R.product
    v, tol = product(x, xs, w, ws)
    u, ut = product(x, xs, up, us) if glu else (None, None)
    want, tol = R.epilogue(v, tol, act, b, u, ut, r)
    if y == "e4m3":
        R.check_quantised(out, scale, want, tol)
    else:
        R.check_wide(out, want, tol)
    for buf, n in ((out_buf, rows), (scale_buf, R.blocks(rows))):
        if buf is not None:
            assert (buf[:, n:].float() == 7.0).all(), "behind a row"


@pytest.mark.parametrize("cols", [16, 112, 128, 144, 256, 512, 2064])
@pytest.mark.parametrize("T,rows", [(1, 1), (1, 130), (3, 64), (16, 16), (17, 257), (33, 128), (65, 48), (130, 300)])
def test_shapes(T, rows, cols):
    dense(T, rows, cols, seed=T * rows + cols)


@pytest.mark.parametrize("y", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T", [1, 19, 130])
def test_types(T, y):
    dense(T, 200, 384, y=y, act="silu", bias=True, residual=True, seed=T, pad=1)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("T", [2, 40, 129])
def test_activations(T, glu, act):
    dense(T, 129, 256, act=act, glu=glu, bias=not glu, residual=True, seed=3 * T)


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("T,rows,cols", [(1, 16, 128), (1, 512, 2048), (5, 112, 272), (16, 256, 128), (40, 400, 512), (131, 272, 256)])
def test_quantised(T, rows, cols, glu):
    dense(T, rows, cols, y="e4m3", act="silu", glu=glu, seed=T + rows, pad=1)


@pytest.mark.parametrize("y", ["f32", "bf16"])
@pytest.mark.parametrize("T,rows,cols", [(300, 1000, 256), (1030, 520, 384), (260, 2050, 144)])
def test_many_tokens(T, rows, cols, y):
    dense(T, rows, cols, y=y, seed=T)


@pytest.mark.parametrize("y,glu", [("f32", False), ("bf16", False), ("e4m3", False), ("f32", True), ("f16", True), ("e4m3", True)])
def test_the_largest_tiles(y, glu):
    dense(1300, 2600 if y != "e4m3" else 2608, 272, y, "silu" if glu else None, glu, pad=1, seed=31)


@pytest.mark.parametrize("T,rows", [(24, 8200), (40, 4112), (100, 4080), (130, 1504), (131, 2064), (300, 2064), (700, 800)])
@pytest.mark.parametrize("y,glu", [("f32", False), ("e4m3", False), ("bf16", True), ("e4m3", True)])
def test_tiles_between(T, rows, y, glu):
    """More tiles than run at a time, or just as many, of each size."""
    dense(T, rows if y != "e4m3" else rows // 16 * 16, 400, y, None, glu, seed=T)


def test_residual_in_place():
    g = gen(5)
    x, xs = R.random_activations(9, 256, g)
    w, ws = R.random_weights(40, 256, g)
    y = torch.randn(9, 40, generator=g)
    out = y.cuda()
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), out, residual=out)
    v, tol = R.product(x, xs, w, ws)
    R.check_wide(out, *R.epilogue(v, tol, residual=y))


def test_residual_of_one_token_out_of_a_wider_buffer():
    """One row has no stride: the residual's and y's may differ."""
    g = gen(6)
    x, xs = R.random_activations(1, 256, g)
    w, ws = R.random_weights(40, 256, g)
    y = torch.randn(1, 64, generator=g)
    out = torch.zeros(1, 40, device="cuda")
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), out, residual=y.cuda()[:, :40])
    v, tol = R.product(x, xs, w, ws)
    R.check_wide(out, *R.epilogue(v, tol, residual=y[:, :40]))


@pytest.mark.parametrize("T", [1, 20, 140])
def test_nan_stays_in_its_token(T):
    """NaN codes, scales and infinite scales of one token reach that token's results and no other's."""
    g = gen(6)
    x, xs = R.random_activations(T, 384, g)
    w, ws = R.random_weights(144, 384, g)
    x, bad = x.view(torch.uint8), sorted({0, T // 2})
    x[bad[0], 200] = 0x7F
    if len(bad) > 1:
        xs[bad[1], 1] = float("nan")
    x = x.view(F8)
    for kind in (torch.float32, torch.float16):
        y = torch.zeros(T, 144, dtype=kind, device="cuda")
        B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), y)
        nan = torch.isnan(y).cpu()
        assert nan[bad].all() and int(nan.sum()) == 144 * len(bad)
    q, s = torch.zeros(T, 144, dtype=torch.uint8, device="cuda").view(F8), torch.zeros(T, 2, device="cuda")
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), q, y_scale=s)
    nan = torch.isnan(s).cpu()
    assert nan[bad].all() and int(nan.sum()) == 2 * len(bad)
    assert torch.isnan(q.float()).cpu().all(1).nonzero().view(-1).tolist() == bad


def test_zero_results_have_the_smallest_scale():
    x, xs = torch.zeros(3, 128).to(F8), torch.ones(3, 1)
    w, ws = R.random_weights(32, 128, gen(7))
    q, s = torch.ones(3, 32, device="cuda").to(F8), torch.ones(3, 1, device="cuda")
    B.bread_matmul_fp8(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), q, y_scale=s)
    assert (q.float() == 0).all() and (s == 2.0**-126).all()


# ------------------------------------------------------------------ groups


def sizes_of(G, n, g, empty=0.3):
    """Group sizes that add up to n, some of them zero, one large."""
    p = torch.rand(G, generator=g) * (torch.rand(G, generator=g) > empty)
    p[G // 2] += 1.0
    return torch.bincount(torch.multinomial(p, n, replacement=True, generator=g), minlength=G)


def grouped(G, n, rows, cols, y="f32", glu=False, index="none", spare=0, first=0, seed=0):
    g = gen(seed)
    sizes = sizes_of(G, n, g)
    off = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]) + first
    total = n + first + spare
    n_x = total if index != "gather" else max(1, n // 3)
    x, xs = R.random_activations(n_x, cols, g)
    w, ws = R.random_weights(rows, cols, g, groups=G)
    up, us = R.random_weights(rows, cols, g, groups=G) if glu else (None, None)
    x_rows = torch.randint(0, n_x, (total,), generator=g) if index == "gather" else None
    n_y = total if index != "scatter" else total + 5
    y_rows = torch.randperm(n_y, generator=g)[:total] if index == "scatter" else None
    kind = KINDS[y]
    out = torch.full((n_y, rows), 3.0, device="cuda").to(kind)
    scale = torch.full((n_y, R.blocks(rows)), 3.0, device="cuda") if y == "e4m3" else None
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    i32 = lambda t: None if t is None else t.int().cuda()  # noqa: E731
    B.bread_matmul_fp8_grouped(dev(w), dev(ws), dev(x), dev(xs), i32(off), out, y_scale=scale, up=dev(up),
                               up_scale=dev(us), act="silu" if glu else None, x_rows=i32(x_rows), y_rows=i32(y_rows))
    torch.cuda.synchronize()
    left = torch.ones(n_y, dtype=torch.bool)
    product = R.product_cut if cut(y) else R.product
    for e in range(G):
        at = torch.arange(int(off[e]), int(off[e + 1]))
        if not at.numel():
            continue
        src = at if x_rows is None else x_rows[at]
        dst = at if y_rows is None else y_rows[at]
        left[dst] = False
        xe, se = x.view(torch.uint8)[src].view(F8), xs[src]
        v, tol = product(xe, se, w[e], ws[e])
        u, ut = product(xe, se, up[e], us[e]) if glu else (None, None)
        want, tol = R.epilogue(v, tol, "silu" if glu else None, None, u, ut)
        if y == "e4m3":
            R.check_quantised(out.view(torch.uint8)[dst.cuda()].view(F8), scale[dst.cuda()], want, tol)
        else:
            R.check_wide(out[dst.cuda()], want, tol)
    rest = left.nonzero().view(-1).cuda()
    if rest.numel():
        assert (out.view(torch.uint8)[rest].view(kind).float() == 3.0).all(), "rows of no group"
        assert scale is None or (scale[rest] == 3.0).all()


@pytest.mark.parametrize("index", ["none", "gather", "scatter"])
@pytest.mark.parametrize("y,glu", [("f32", False), ("bf16", True), ("e4m3", True), ("e4m3", False), ("f16", False)])
@pytest.mark.parametrize("G,n", [(1, 1), (8, 3), (5, 40), (40, 150), (300, 500)])
def test_groups(G, n, y, glu, index):
    grouped(G, n, 144, 272, y=y, glu=glu, index=index, spare=3, first=2, seed=G + n)


@pytest.mark.parametrize("y", ["f32", "f16", "e4m3"])
def test_groups_of_many_rows(y):
    grouped(6, 1500, 256, 256, y=y, glu=y == "e4m3", index="gather", seed=11)


def test_groups_at_the_expert_shape():
    grouped(12, 40, 512, 2048, y="e4m3", glu=True, index="gather", seed=12)
    grouped(12, 40, 2048, 512, y="f32", index="scatter", seed=13)


@pytest.mark.parametrize("y,glu", [("f32", False), ("e4m3", True), ("bf16", True), ("f16", False)])
@pytest.mark.parametrize("n", [700, 2100, 9000])
def test_groups_of_more_tiles_than_run_at_a_time(n, y, glu):
    """Workgroups that take several tiles, full ones and rests of every size, over groups of 0 to some hundred rows."""
    grouped(70, n, 528, 272, y=y, glu=glu, index="gather", spare=2, first=1, seed=n)


@pytest.mark.parametrize("y,glu", [("f32", False), ("f32", True), ("e4m3", False), ("e4m3", True)])
@pytest.mark.parametrize("G,n,rows", [(20, 300, 272), (24, 1500, 528), (40, 900, 1040), (8, 540, 512), (54, 1500, 192)])
def test_groups_of_every_tile(G, n, rows, y, glu):
    grouped(G, n, rows, 400, y=y, glu=glu, index="scatter", seed=G)


def test_offsets_that_fall():
    """Groups that overlap, end before they begin or leave the rows: nothing behind the rows is written, and groups in
    order before them are right."""
    g = gen(21)
    n, rows, cols, G = 300, 144, 128, 200
    x, xs = R.random_activations(n, cols, g)
    w, ws = R.random_weights(rows, cols, g, groups=G)
    off = torch.randint(-2**31, 2**31 - 1, (G + 1,), generator=g)
    off[2::3] = torch.randint(0, n, off[2::3].shape, generator=g)
    for up in (None, w.cuda()):
        for y_type in (torch.float32, torch.bfloat16, F8):
            y = torch.full((n + 64, rows), 3.0, device="cuda").to(y_type)
            s = torch.full((n + 64, 2), 3.0, device="cuda") if y_type == F8 else None
            B.bread_matmul_fp8_grouped(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), off.int().cuda(), y[:n],
                                       y_scale=None if s is None else s[:n], up=up, up_scale=None if up is None else ws.cuda())
            torch.cuda.synchronize()
            assert (y[n:].float() == 3.0).all() and (s is None or (s[n:] == 3.0).all())


def test_products_on_two_streams_at_once():
    """Calls keep no workspace: products that overlap give what they give alone."""
    g = gen(22)
    x, xs = (t.cuda() for t in R.random_activations(600, 512, g))
    w, ws = (t.cuda() for t in R.random_weights(1024, 512, g, groups=8))
    off = torch.tensor([0, 50, 50, 130, 300, 301, 420, 600, 600], dtype=torch.int32, device="cuda")
    one, two = [torch.empty(600, 1024, device="cuda") for _ in range(2)]
    codes, scale = torch.empty(600, 1024, dtype=F8, device="cuda"), torch.empty(600, 8, device="cuda")

    def dense_call():
        B.bread_matmul_fp8(w[0], ws[0], x, xs, codes, y_scale=scale, up=w[1], up_scale=ws[1], act="silu")

    B.bread_matmul_fp8_grouped(w, ws, x, xs, off, one)
    dense_call()
    torch.cuda.synchronize()
    alone = one.clone(), codes.view(torch.uint8).clone(), scale.clone()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        one.fill_(0), two.fill_(0), scale.fill_(0)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            B.bread_matmul_fp8_grouped(w, ws, x, xs, off, one)
            B.bread_matmul_fp8_grouped(w, ws, x, xs, off, two)
        with torch.cuda.stream(b):
            dense_call()
        torch.cuda.synchronize()
        assert torch.equal(one, alone[0]) and torch.equal(two, alone[0])
        assert torch.equal(codes.view(torch.uint8), alone[1]) and torch.equal(scale, alone[2])


@pytest.mark.parametrize("n", [3, 200])
def test_rows_out_of_range(n):
    """x rows outside x count as zeros, y rows outside y are not written, offsets are held to the rows."""
    g = gen(14)
    x, xs = R.random_activations(4, 128, g)
    w, ws = R.random_weights(64, 128, g, groups=3)
    x_rows = torch.randint(0, 4, (n,), generator=g)
    x_rows[0], x_rows[n - 1] = -1, 4
    y_rows = torch.arange(n)
    y_rows[1] = -5
    y_rows[n - 1] = n
    y = torch.full((n, 64), 3.0, device="cuda")
    off = torch.tensor([-7, n // 2, n // 2 - 1, n + 100], dtype=torch.int32)
    off[2] = n // 2
    B.bread_matmul_fp8_grouped(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), off.cuda(), y, x_rows=x_rows.int().cuda(),
                               y_rows=y_rows.int().cuda())
    y = y.cpu()
    assert (y[1] == 3.0).all() and (y[n - 1] == 3.0).all()
    if n > 1 and 0 != 1:
        assert (y[0] == 0.0).all()
    for i in range(2, n - 1):
        e = 0 if i < n // 2 else 2
        r = int(x_rows[i])
        want, tol = R.product(x.view(torch.uint8)[r:r + 1].view(F8), xs[r:r + 1], w[e], ws[e])
        R.check_wide(y[i:i + 1], want, tol)


def test_no_groups_and_empty_groups():
    w, ws = R.random_weights(16, 128, gen(1), groups=4)
    x, xs = R.random_activations(5, 128, gen(2))
    y = torch.full((5, 16), 3.0, device="cuda")
    B.bread_matmul_fp8_grouped(w.cuda(), ws.cuda(), x.cuda(), xs.cuda(), torch.full((5,), 2, dtype=torch.int32).cuda(), y)
    B.bread_matmul_fp8_grouped(w[:0].cuda(), ws[:0].cuda(), x.cuda(), xs.cuda(), torch.zeros(1, dtype=torch.int32).cuda(), y)
    assert (y == 3.0).all()
