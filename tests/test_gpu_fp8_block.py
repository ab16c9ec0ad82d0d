"""bread_moe_expert_block_fp8 against 64-bit experts, and an 8-bit layer run together as a program runs it."""
import pytest
import torch

import breadv2_amd as B
import fp8_reference as R
from breadv2_amd import _lib

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def experts(E, I, H, g):
    t = []
    for rows, cols in ((I, H), (I, H), (H, I)):
        t += R.random_weights(rows, cols, g, groups=E)
    return t


def reference(t, x, xs, idx, w, residual):
    """hidden and a bound of the kernel's error.  The codes of the experts' inner values may fall to the other side
    of a border: a value's error there is up to a step of e4m3, 2^-3 of it (or 2^-9 scales), for those within their
    bound of a border."""
    gate, gs, up, us, down, ds = t
    out, tol = residual.double().clone(), torch.zeros(residual.shape, dtype=torch.float64)
    size = residual.double().abs()
    for e in range(gate.shape[0]):
        tok, k = torch.nonzero(idx == e, as_tuple=True)
        if not tok.numel():
            continue
        xe, se = x.view(torch.uint8)[tok].view(F8), xs[tok]
        v, vt = R.product(xe, se, gate[e], gs[e])
        u, ut = R.product(xe, se, up[e], us[e])
        a, at = R.epilogue(v, vt, "silu", None, u, ut)
        codes, scales = R.quantise(a)
        full = R.expand(scales, *a.shape, 1)
        top = torch.stack([at[:, b:b + 128].amax(1) for b in range(0, a.shape[1], 128)], 1)
        rel = R.expand(top / 448.0 / scales + 3 * 2.0**-24, *a.shape, 1)  # of the scale
        q = a / full
        _, ex = torch.frexp(q)
        step = torch.ldexp(torch.ones_like(q), torch.clamp_min(ex - 1, -6) - 3)
        slack = at / full + q.abs() * (rel + 4 * 2.0**-24)
        border = (0.5 * step - (q - codes).abs()).abs() <= slack
        inner = torch.where(border, step, torch.zeros_like(q)) * full + rel * (codes * full).abs()
        wd = R.weights(down[e], ds[e])
        y = (codes * full) @ wd.T
        mag = (codes * full).abs() @ wd.abs().T
        yt = inner @ wd.abs().T + (16 + R.blocks(a.shape[1]) + 2) * 2.0**-24 * mag
        wk = w[tok, k].double()[:, None]
        out.index_add_(0, tok, wk * y)
        tol.index_add_(0, tok, wk.abs() * (yt + 2.0**-24 * y.abs()))
        size.index_add_(0, tok, (wk * y).abs())
    return out, tol + idx.shape[1] * 2.0**-24 * size


def block(T, E, I, H, K, kind=torch.float32, route="random", residual="in place", seed=0, ctx=None):
    g = torch.Generator().manual_seed(seed)
    t = experts(E, I, H, g)
    x, xs = R.random_activations(T, H, g)
    if route == "random":
        idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).int()
    elif route == "same":
        idx = torch.randperm(E, generator=g)[:K].int().repeat(T, 1)
    else:  # the same expert at every rank
        idx = torch.randint(0, E, (T, 1), generator=g).int().repeat(1, K)
    w = torch.rand(T, K, generator=g)
    r = torch.randn(T, H, generator=g).to(kind)
    ctx = ctx or B.MoeContext(B.shape(H, I, I, E, K), max_tokens=T)
    ex = B.Fp8Experts(*[v.cuda() for v in t])
    hidden = r.cuda()
    if residual != "in place":
        hidden = torch.full((T, H), 9.0, dtype=kind, device="cuda")
    ctx.expert_block_fp8(ex, x.cuda(), xs.cuda(), hidden, idx.cuda(), w.cuda(),
                         residual=None if residual == "in place" else r.cuda())
    assert ctx.check_device() == 0
    want, tol = reference(t, x, xs, idx, w, r)
    R.check_wide(hidden, want, tol)
    return hidden


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 2, 5, 33, 150])
def test_tokens(T, kind):
    block(T, 16, 256, 512, 4, kind, seed=T)


@pytest.mark.parametrize("E,K,I,H", [(1, 1, 256, 256), (8, 8, 256, 256), (300, 3, 256, 256), (4, 2, 512, 1024),
                                     (6, 1, 768, 256)])
@pytest.mark.parametrize("T", [1, 20])
def test_shapes(T, E, K, I, H):
    block(T, E, I, H, K, seed=E + T, residual="apart")


@pytest.mark.parametrize("route", ["same", "repeated"])
@pytest.mark.parametrize("T", [1, 3, 90])
def test_routing(T, route):
    block(T, 9, 256, 256, 4, torch.float32, route, seed=T)


@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("E,K,I,H", [(5, 3, 1024, 512), (33, 32, 256, 256), (12, 9, 512, 768)])
def test_a_few_tokens(T, E, K, I, H):
    """Lanes a pair by the inner size, and more pairs than go at a time."""
    block(T, E, I, H, K, torch.float16, seed=T + K)


@pytest.mark.parametrize("E,K,I,H", [(1, 1, 256, 256), (8, 8, 256, 256), (300, 3, 256, 256), (4, 2, 512, 1024), (6, 2, 768, 256)])
def test_many_pairs(E, K, I, H):
    """Pairs sorted by expert."""
    block(400, E, I, H, K, torch.bfloat16, seed=E + K, residual="apart")


def test_repeated_experts_and_ones_that_are_none_among_many_pairs():
    block(300, 9, 256, 512, 4, torch.float32, "repeated", seed=7)
    g = torch.Generator().manual_seed(5)
    t = experts(8, 256, 256, g)
    x, xs = R.random_activations(600, 256, g)
    idx = torch.stack([torch.randperm(8, generator=g)[:2] for _ in range(600)]).int()
    idx[::7, 0], idx[3::50, 1] = -1, 8
    w, r = torch.rand(600, 2, generator=g), torch.randn(600, 256, generator=g)
    ctx = B.MoeContext(B.shape(256, 256, 256, 8, 2), max_tokens=600)
    hidden = r.cuda()
    ctx.expert_block_fp8(B.Fp8Experts(*[v.cuda() for v in t]), x.cuda(), xs.cuda(), hidden, idx.cuda(), w.cuda())
    with pytest.raises(B.BreadError) as e:
        ctx.check_device()
    assert e.value.device_error == 32
    want, tol = reference(t, x, xs, idx, w, r)
    R.check_wide(hidden, want, tol)


def test_at_the_decode_shape():
    block(1, 16, 512, 2048, 8, torch.float16, seed=1)
    block(9, 16, 512, 2048, 8, torch.float32, seed=2)


def test_an_expert_that_is_none_sets_its_bit_and_is_left_out():
    for bad in (-1, 8):
        for T in (1, 40):
            g = torch.Generator().manual_seed(3)
            t = experts(8, 256, 256, g)
            x, xs = R.random_activations(T, 256, g)
            idx = torch.stack([torch.randperm(8, generator=g)[:2] for _ in range(T)]).int()
            idx[T - 1, 1] = bad
            w, r = torch.rand(T, 2, generator=g), torch.randn(T, 256, generator=g)
            ctx = B.MoeContext(B.shape(256, 256, 256, 8, 2), max_tokens=T)
            hidden = r.cuda()
            ctx.expert_block_fp8(B.Fp8Experts(*[v.cuda() for v in t]), x.cuda(), xs.cuda(), hidden, idx.cuda(), w.cuda())
            with pytest.raises(B.BreadError) as e:
                ctx.check_device()
            assert e.value.device_error == 32
            want, tol = reference(t, x, xs, idx, w, r)  # (no expert has that index)
            R.check_wide(hidden, want, tol)


def test_nothing_to_do():
    ctx = B.MoeContext(B.shape(256, 256, 256, 4, 2), max_tokens=2)
    t = experts(4, 256, 256, torch.Generator().manual_seed(4))
    e = B.Fp8Experts(*[v.cuda() for v in t])
    z = lambda n, d: torch.zeros(0, n, dtype=d, device="cuda")  # noqa: E731
    ctx.expert_block_fp8(e, z(256, torch.uint8).view(F8), z(2, torch.float32), z(256, torch.float32), z(2, torch.int32),
                         z(2, torch.float32))
    with pytest.raises(B.BreadError) as err:
        o = lambda n, d: torch.zeros(3, n, dtype=d, device="cuda")  # noqa: E731
        ctx.expert_block_fp8(e, o(256, torch.uint8).view(F8), o(2, torch.float32), o(256, torch.float32),
                             o(2, torch.int32), o(2, torch.float32))
    assert err.value.status == _lib.ERR_CAPACITY


class Layer:
    """One layer with a shared expert on the fp32 residual stream, as a serving program keeps it."""

    def __init__(self, T, seed, E=16, I=256, H=512, K=4):
        g = torch.Generator().manual_seed(seed)
        self.T, self.E, self.I, self.H, self.K = T, E, I, H, K
        self.host = experts(E, I, H, g)
        self.shared = [*R.random_weights(I, H, g), *R.random_weights(I, H, g), *R.random_weights(H, I, g)]
        self.norm_w = 1 + 0.2 * torch.randn(H, generator=g)
        self.router = 0.05 * torch.randn(E, H, generator=g)
        self.ex = B.Fp8Experts(*[v.cuda() for v in self.host])
        self.sh = [v.cuda() for v in self.shared]
        self.nw, self.rw = self.norm_w.cuda(), self.router.cuda()
        self.rule = B.RouteRule(score="sigmoid", renorm=True, scale=2.5)
        self.ctx = B.MoeContext(B.shape(H, I, I, E, K), max_tokens=T)
        f = dict(device="cuda")
        self.codes, self.scales = torch.empty(T, H, dtype=torch.uint8, **f).view(F8), torch.empty(T, H // 128, **f)
        self.normed, self.hidden = torch.empty(T, H, **f), torch.empty(T, H, **f)
        self.mid, self.mids = torch.empty(T, I, dtype=torch.uint8, **f).view(F8), torch.empty(T, I // 128, **f)
        self.out = torch.empty(T, H, **f)
        self.logits = torch.empty(T, E, **f)

    def __call__(self, x, residual):
        B.bread_rmsnorm_fp8(x, self.nw, self.codes, self.scales, 1e-6, residual=residual, hidden=self.hidden,
                            normed=self.normed)
        torch.mm(self.normed, self.rw.T, out=self.logits)
        idx, w = B.route_select(self.logits, self.K, self.rule)
        g, gs, u, us, d, ds = self.sh
        B.bread_matmul_fp8(g, gs, self.codes, self.scales, self.mid, y_scale=self.mids, up=u, up_scale=us, act="silu")
        B.bread_matmul_fp8(d, ds, self.mid, self.mids, self.out, residual=self.hidden)
        self.ctx.expert_block_fp8(self.ex, self.codes, self.scales, self.out, idx, w)
        return self.out, idx, w


@pytest.mark.parametrize("T", [1, 7, 200])
def test_a_layer(T):
    layer = Layer(T, seed=T)
    g = torch.Generator().manual_seed(50 + T)
    x, r = torch.randn(T, layer.H, generator=g), torch.randn(T, layer.H, generator=g)
    out, idx, w = layer(x.cuda(), r.cuda())
    torch.cuda.synchronize()
    h = x + r
    assert torch.equal(layer.hidden.cpu(), h)
    f = h.double()
    v = f / torch.sqrt((f * f).mean(1, keepdim=True) + 1e-6) * layer.norm_w.double()
    tol = (0.5 * (layer.H / 64 + 12) + 5) * 2.0**-24 * v.abs()
    R.check_quantised(layer.codes, layer.scales, v, tol)
    R.check_wide(layer.normed, v, tol)
    # from the layer's own codes on
    codes, scales = layer.codes.cpu(), layer.scales.cpu()
    one = [layer.shared[i][None] for i in range(6)]
    zero = torch.zeros(T, 1, dtype=torch.int32)
    want, tol = reference(one, codes, scales, zero, torch.ones(T, 1), h)
    more, tol2 = reference(layer.host, codes, scales, idx.cpu(), w.cpu(), torch.zeros(T, layer.H))
    R.check_wide(out, want + more, tol + tol2 + 4 * 2.0**-24 * (want.abs() + more.abs()))


@pytest.mark.parametrize("T", [1, 70])
def test_a_layer_captured_and_on_another_stream(T):
    """A graph of the layer's own calls, replayed with new inputs and eager work between, and the same on a side
    stream: bit for bit the eager results."""
    layer, other = Layer(T, seed=8), Layer(T, seed=9)
    g = torch.Generator().manual_seed(60)
    data = [(torch.randn(T, layer.H, generator=g).cuda(), torch.randn(T, layer.H, generator=g).cuda()) for _ in range(4)]
    eager = [layer(*d)[0].clone() for d in data]
    idx, w = layer(*data[0])[1:]
    x, r = data[0][0].clone(), data[0][1].clone()
    sh = layer.sh

    def body():
        B.bread_rmsnorm_fp8(x, layer.nw, layer.codes, layer.scales, 1e-6, residual=r, hidden=layer.hidden, normed=layer.normed)
        B.bread_matmul_fp8(sh[0], sh[1], layer.codes, layer.scales, layer.mid, y_scale=layer.mids, up=sh[2], up_scale=sh[3], act="silu")
        B.bread_matmul_fp8(sh[4], sh[5], layer.mid, layer.mids, layer.out, residual=layer.hidden)
        layer.ctx.expert_block_fp8(layer.ex, layer.codes, layer.scales, layer.out, idx, w)

    routes = []
    for d in data:
        routes.append([t.clone() for t in layer(*d)[1:]])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for rep in range(3):
        for d, e, (i2, w2) in zip(data, eager, routes):
            x.copy_(d[0]), r.copy_(d[1]), idx.copy_(i2), w.copy_(w2)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(layer.out, e), rep
            other(*d)  # eager work between
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        for d, e in zip(data, eager):
            out = layer(*d)[0]
            side.synchronize()
            assert torch.equal(out, e)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_a_context_of_another_device_is_refused():
    with torch.cuda.device(1):
        t = experts(4, 256, 256, torch.Generator().manual_seed(4))
        e = B.Fp8Experts(*[v.cuda() for v in t])
    with torch.cuda.device(0):
        ctx = B.MoeContext(B.shape(256, 256, 256, 4, 2), max_tokens=2)
    with torch.cuda.device(1):
        o = lambda n, d: torch.zeros(1, n, dtype=d, device="cuda")  # noqa: E731
        with pytest.raises(B.BreadError) as err:
            ctx.expert_block_fp8(e, o(256, torch.uint8).view(F8), o(2, torch.float32), o(256, torch.float32),
                                 o(2, torch.int32), o(2, torch.float32))
    assert err.value.status == _lib.ERR_ARG
