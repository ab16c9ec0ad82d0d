"""Routing by a rule against a plain 64-bit selection, expert by expert.

Indices are compared exactly: both sides hold scores in 64 bits, where random
choices are equal or apart by far more than a rounding.
Weights are computed in 64 bits and rounded once: within 2^-24 of themselves,
plus 1e-12 for the 64-bit functions' own errors.
"""
import numpy as np
import pytest
import torch

import breadv2_amd as B
from breadv2_amd import api
from oracle import oracle as O

from helpers import assert_moe_close, host_layer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def scores(z, score):
    z = np.where(np.isnan(z), -np.inf, z).astype(np.float64)
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return 1.0 / (1.0 + np.exp(-z))
    out = np.zeros_like(z)
    for t, row in enumerate(z):
        m = row.max()
        if m == -np.inf:
            continue
        with np.errstate(invalid="ignore"):
            e = np.where(row == m, 1.0, np.exp(row - m))
        out[t] = e / e.sum()
    return out


def plain(z, K, score="softmax", bias=None, n_groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0):
    s = scores(z, score)
    T, E = s.shape
    c = s + (0.0 if bias is None else bias.astype(np.float64))
    per = E // n_groups
    idx = np.zeros((T, K), np.int32)
    w = np.zeros((T, K))
    for t in range(T):
        order = range(E)
        if top_groups < n_groups:
            gs = [sum(sorted(c[t, g * per:(g + 1) * per], reverse=True)[:group_top]) for g in range(n_groups)]
            kept = sorted(range(n_groups), key=lambda g: (-gs[g], g))[:top_groups]
            order = [e for e in range(E) if e // per in kept]
        best = sorted(order, key=lambda e: (-c[t, e], e))[:K]
        idx[t] = best
        w[t] = s[t, best]
        if renorm:
            w[t] = w[t] / w[t].sum() if w[t].sum() > 0 else 0.0
    return idx, w * np.float64(np.float32(scale))


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def compare(z, K, **rule):
    bias = rule.pop("bias", None)
    idx, w = B.route_select(dev(z), K, B.RouteRule(bias=None if bias is None else dev(bias), **rule))
    ri, rw = plain(z, K, bias=bias, **rule)
    assert np.array_equal(idx.cpu().numpy(), ri), (z.shape, K, rule)
    got = w.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - rw) <= (2.0 ** -24 + 1e-12) * np.abs(rw) + 2.0 ** -150), (z.shape, K, rule)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [1, 2, 7, 60, 64, 65, 128, 256, 257, 512, 1000, 1024])
def test_plain_rules(score, E):
    rng = np.random.default_rng(E)
    for T in (1, 2, 5, 67):
        z = rng.standard_normal((T, E)).astype(np.float32)
        bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
        for K in sorted({1, min(E, 6), min(E, 8), min(E, 32)}):
            compare(z, K, score=score)
            compare(z, K, score=score, bias=bias, renorm=False, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,n_groups,top_groups,K", [
    (256, 8, 4, 8), (256, 8, 1, 8), (256, 8, 7, 8), (64, 2, 1, 6), (64, 64, 8, 8), (160, 8, 3, 6), (72, 12, 5, 7),
    (1024, 8, 4, 8), (1024, 1024, 32, 32), (1020, 4, 2, 16), (300, 100, 40, 9), (256, 4, 4, 8), (512, 2, 1, 32),
    (96, 3, 2, 8), (200, 5, 2, 8), (128, 16, 4, 4)])
def test_groups(score, E, n_groups, top_groups, K):
    rng = np.random.default_rng(E + n_groups)
    z = rng.standard_normal((33, E)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    for group_top in (1, 2):
        for b in (None, bias):
            compare(z, K, score=score, bias=b, n_groups=n_groups, top_groups=top_groups, group_top=group_top,
                    scale=1.5)


def test_ties_go_to_the_lower_index():
    z = np.zeros((4, 256), np.float32)
    z[1, 100:] = 1.0
    z[2, ::3] = 2.0
    z[3] = np.random.default_rng(0).integers(0, 3, 256)
    for score in ("softmax", "sigmoid"):
        compare(z, 8, score=score)
        compare(z, 8, score=score, n_groups=8, top_groups=4, group_top=2)
        compare(z, 8, score=score, n_groups=8, top_groups=4, group_top=1, bias=np.zeros(256, np.float32))


def test_scores_that_fp32_cannot_tell_apart():
    """Sigmoids of logits around 20 differ by less than a step of fp32 (all round to 1), and are ordered all the same."""
    rng = np.random.default_rng(5)
    z = (20.0 + 0.01 * rng.permutation(256).reshape(1, 256)).astype(np.float32)
    assert np.unique((1.0 / (1.0 + np.exp(-z.astype(np.float64)))).astype(np.float32)).size == 1
    compare(z, 8, score="sigmoid")
    compare(z, 8, score="sigmoid", n_groups=8, top_groups=3)


def test_masked_and_infinite_logits():
    inf = np.inf
    z = np.random.default_rng(2).standard_normal((8, 64)).astype(np.float32)
    z[0] = -inf                       # nothing is left
    z[1, 3:] = -inf                   # fewer experts than top_k
    z[2, 10] = np.nan
    z[3, 5] = inf
    z[4, [7, 9]] = inf
    z[5] = np.nan
    z[6] = np.finfo(np.float32).min   # a mask of the type's lowest value
    z[6, 60] = 0.5
    z[7, :32] = -inf
    for score in ("softmax", "sigmoid"):
        compare(z, 8, score=score)
        compare(z, 8, score=score, n_groups=8, top_groups=2, group_top=2, bias=np.linspace(0, 1, 64, dtype=np.float32))
        compare(z, 8, score=score, renorm=False)


def test_extreme_bias():
    """Biases of +-inf force and forbid experts; their weights stay the scores."""
    z = np.random.default_rng(3).standard_normal((5, 64)).astype(np.float32)
    b = np.zeros(64, np.float32)
    b[[50, 20]] = np.inf
    b[:16] = -np.inf
    compare(z, 8, score="sigmoid", bias=b)
    compare(z, 8, score="softmax", bias=b, n_groups=4, top_groups=3, group_top=1)


def test_strided_logits_and_many_tokens():
    rng = np.random.default_rng(4)
    wide = dev(rng.standard_normal((3000, 100)).astype(np.float32))
    rule = B.RouteRule(score="sigmoid", n_groups=4, top_groups=2, group_top=2)
    idx, w = B.route_select(wide[:, 10:74], 4, rule)
    ri, rw = plain(wide[:, 10:74].cpu().numpy(), 4, score="sigmoid", n_groups=4, top_groups=2, group_top=2)
    assert np.array_equal(idx.cpu().numpy(), ri)
    assert np.all(np.abs(w.cpu().numpy() - rw) <= (2.0 ** -24 + 1e-12) * rw)
    idx, w = B.route_select(wide[:0, :64], 4, rule)
    assert idx.shape == (0, 4)


def test_stream_and_graph():
    z = torch.randn(50, 256, device=DEV)
    rule = B.RouteRule(score="sigmoid", bias=0.1 * torch.randn(256, device=DEV), n_groups=8, top_groups=4, group_top=2)
    ref = B.route_select(z, 8, rule)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = B.route_select(z, 8, rule, stream=s)
    s.synchronize()
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = B.route_select(z, 8, rule)
    for _ in range(3):
        z.copy_(torch.randn(50, 256, device=DEV))
        g.replay()
        ref = B.route_select(z, 8, rule)
        torch.cuda.synchronize()
        assert torch.equal(ref[0], out[0]) and torch.equal(ref[1], out[1])


# ------------------------------------------------------------------ the MoE block by a rule


@pytest.fixture(scope="module")
def layer():
    s = api.shape(hidden=2048, expert_inter=512, shared_inter=512, n_experts=64, top_k=8)
    t = api.synth_layer_tensors(s, seed=77, layer=0)
    torch.cuda.synchronize()
    return s, t, host_layer(t)


def block(hl, x, hidden, idx, w, gsh):
    """The oracle's routed experts with given routing, and its shared expert."""
    out = hidden.copy()
    O.expert_block(hl, x, out, idx, w)
    both = hidden.copy()
    O.moe_forward(hl, x, both, x.shape[0], nthreads=8)
    ri, rw, _ = O.route_batch(hl, x)
    own = hidden.copy()
    O.expert_block(hl, x, own, ri, rw)
    return out.astype(np.float64) + (both.astype(np.float64) - own)


@pytest.mark.parametrize("T", [1, 3, 16, 17, 40])
def test_layer_by_rule(layer, T):
    """Logits are the reference's bit for bit; the block is the oracle's with the rule's experts and weights."""
    s, t, hl = layer
    rng = np.random.default_rng(T)
    x = rng.standard_normal((T, s.hidden)).astype(np.float32)
    hidden = rng.standard_normal((T, s.hidden)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(64)).astype(np.float32)
    kw = dict(score="sigmoid", n_groups=8, top_groups=4, group_top=2, renorm=True, scale=2.5)
    rule = B.RouteRule(bias=dev(bias), **kw)
    logits = O.route_batch(hl, x, want_logits=True)[-1]
    ri, rw = plain(np.asarray(logits), 8, bias=bias, **kw)
    ctx = B.MoeContext(s, max_tokens=T)
    idx, w, g = ctx.route_by_rule(t.desc(), rule, dev(x), T)
    assert np.array_equal(idx.cpu().numpy(), ri)
    assert np.all(np.abs(w.cpu().numpy() - rw) <= (2.0 ** -24 + 1e-12) * rw)
    want = block(hl, x, hidden, ri, rw.astype(np.float32), g.cpu().numpy())
    for path in (B.api.PATH_AUTO, B.api.PATH_PER_TOKEN, B.api.PATH_GROUPED) + ((B.api.PATH_SMALL,) if T <= 32 else ()):
        ctx.set_path(path)
        h = dev(hidden)
        i2, w2, _ = ctx.forward_by_rule(t.desc(), rule, dev(x), h, T, want_routing=True)
        torch.cuda.synchronize()
        assert ctx.check_device() == 0
        assert torch.equal(i2, idx) and torch.equal(w2, w)
        assert_moe_close(h.cpu().numpy(), want, base=hidden)


@pytest.mark.parametrize("dims,types", [
    ((512, 256, 256, 12, 4), (12, 12, 12, 12, 12, 12)),
    ((512, 256, 256, 12, 4), (12, 12, 14, 12, 12, 14)),
    ((1024, 512, 256, 60, 6), (14, 12, 14, 14, 12, 12)),
    ((256, 768, 512, 10, 3), (12, 12, 14, 12, 12, 14)),
])
def test_other_layers_by_rule(dims, types):
    """Shapes and weight types of the per-token and the grouped paths, one token to a chunk."""
    s = api.shape(*dims)
    t = api.synth_layer_tensors(s, seed=5, layer=0, types=types)
    torch.cuda.synchronize()
    hl = host_layer(t)
    E, K = s.n_experts, s.top_k
    kw = dict(score="sigmoid", n_groups=2, top_groups=1, group_top=2, renorm=False, scale=0.5)
    rng = np.random.default_rng(E)
    bias = (0.2 * rng.standard_normal(E)).astype(np.float32)
    rule = B.RouteRule(bias=dev(bias), **kw)
    ctx = B.MoeContext(s, max_tokens=150)
    for T in (1, 5, 40, 150):
        x = rng.standard_normal((T, s.hidden)).astype(np.float32)
        hidden = rng.standard_normal((T, s.hidden)).astype(np.float32)
        logits = O.route_batch(hl, x, want_logits=True)[-1]
        ri, rw = plain(np.asarray(logits), K, bias=bias, **kw)
        h = dev(hidden)
        idx, w, g = ctx.forward_by_rule(t.desc(), rule, dev(x), h, T, want_routing=True)
        torch.cuda.synchronize()
        assert ctx.check_device() == 0
        assert np.array_equal(idx.cpu().numpy(), ri)
        assert np.all(np.abs(w.cpu().numpy() - rw) <= (2.0 ** -24 + 1e-12) * rw)
        assert_moe_close(h.cpu().numpy(), block(hl, x, hidden, ri, rw.astype(np.float32), g.cpu().numpy()), base=hidden)


def test_route_layers_own_rule_is_the_default(layer):
    """RouteRule() chooses route_layer's experts in its order, with its weights to fp32 roundings."""
    s, t, hl = layer
    x = np.random.default_rng(1).standard_normal((33, s.hidden)).astype(np.float32)
    ctx = B.MoeContext(s, max_tokens=33)
    a = ctx.route(t.desc(), dev(x), 33)
    b = ctx.route_by_rule(t.desc(), B.RouteRule(), dev(x), 33)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    # fp32 softmax, sum of eight and a division: below 2^-20 of the weight
    assert torch.all((a[1] - b[1]).abs() <= 2.0 ** -20 * b[1])


def test_decode_path_refuses_a_rule(layer):
    s, t, _ = layer
    ctx = B.MoeContext(s, max_tokens=1)
    ctx.set_path(api.PATH_DECODE)
    x = torch.randn(1, s.hidden, device=DEV)
    h = torch.zeros(1, s.hidden, device=DEV)
    with pytest.raises(B.BreadError) as e:
        ctx.forward_by_rule(t.desc(), B.RouteRule(), x, h, 1)
    assert e.value.status == api._lib.ERR_SHAPE
    torch.cuda.synchronize()
    assert torch.all(h == 0)
