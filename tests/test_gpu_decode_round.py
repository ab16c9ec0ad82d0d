"""A verifying round as a program runs it: output projection onto the residual
stream, norm, MoE block by a rule, norm, output matrix, verification by
sampling.  Every stage is compared with its plain form on the inputs that it
had on the device, within that stage's own bound; the same round captured into
a graph and on another stream gives the same bits.
"""
import numpy as np
import pytest
import torch

import breadv2_amd as B
from breadv2_amd import api
from oracle import oracle as O

from helpers import assert_moe_close, host_layer, scale_layer_d
from test_gpu_matmul import Q6, Q8, dev, expected, weights
from test_gpu_route_rule import block, plain as plain_route
from test_gpu_spec_verify import plain as plain_verify

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, ATTN, VOCAB, E, K = 2048, 1056, 5003, 64, 8
RULE = dict(score="sigmoid", n_groups=8, top_groups=4, group_top=2, renorm=True, scale=2.5)


class Model:
    def __init__(self):
        self.s = api.shape(hidden=H, expert_inter=512, shared_inter=512, n_experts=E, top_k=K)
        self.t = api.synth_layer_tensors(self.s, seed=21, layer=0)
        scale_layer_d(self.t, 8)
        torch.cuda.synchronize()
        rng = np.random.default_rng(4)
        self.wo = weights(Q8, H, ATTN, 5)
        self.head = weights(Q6, VOCAB, H, 6, scale=1.0 / 256)
        self.bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
        self.rule = B.RouteRule(bias=dev(self.bias), **RULE)
        self.d_wo, self.d_head = dev(self.wo), dev(self.head)
        self.norm = dev((1 + 0.1 * rng.standard_normal(H)).astype(np.float32))
        self.desc = self.t.desc()


class Round:
    """The round's buffers; run() leaves every stage's outputs in them."""

    def __init__(self, model, T):
        self.m, self.T = model, T
        self.ctx = B.MoeContext(model.s, max_tokens=max(T, 64))
        self.ctx_v = B.MoeContext(model.s, max_tokens=max(T, 64))
        f = lambda *shape, t=torch.float32: torch.zeros(*shape, dtype=t, device=DEV)
        self.attn, self.h0 = f(T, ATTN, t=torch.float16), f(T, H)
        self.h1, self.h2, self.x1, self.x2 = f(T, H), f(T, H), f(T, H), f(T, H)
        self.logits = f(T, VOCAB, t=torch.float16)

    def fill(self, seed):
        rng = np.random.default_rng(seed)
        self.attn.copy_(dev(rng.standard_normal((self.T, ATTN)).astype(np.float16)))
        self.h0.copy_(dev(rng.standard_normal((self.T, H)).astype(np.float32)))

    def run(self, tokens, off, u, temp, stream=None):
        m, T = self.m, self.T
        with torch.cuda.stream(stream or torch.cuda.current_stream()):
            self.h1.copy_(self.h0)
            B.bread_matmul(m.d_wo, self.attn, self.h1, H, ATTN, Q8, residual=self.h1)
            api.bread_rmsnorm_f32(self.h1, m.norm, self.x1, H, T, 1e-6)
            self.h2.copy_(self.h1)
            self.routing = self.ctx.forward_by_rule(m.desc, m.rule, self.x1, self.h2, T, want_routing=True)
            api.bread_rmsnorm_f32(self.h2, m.norm, self.x2, H, T, 1e-6)
            self.x16 = self.x2.half()
            B.bread_matmul(m.d_head, self.x16, self.logits, VOCAB, H, Q6)
            self.out = self.ctx_v.spec_verify(self.logits, tokens, off, u, temperature=temp)
        return (self.h1, *self.routing, self.h2, self.logits, *self.out)


@pytest.fixture(scope="module")
def model():
    return Model()


def request(counts, seed):
    rng = np.random.default_rng(seed)
    off = np.concatenate([[0], np.cumsum(np.asarray(counts) + 1)]).astype(np.int32)
    R = int(off[-1])
    return (rng.integers(0, VOCAB, R).astype(np.int32), off, rng.random(R).astype(np.float32),
            np.array([0.7, 0.0, 1.3, 0.9] * len(counts), np.float32)[: len(counts)])


@pytest.mark.parametrize("counts", [[0], [4], [4, 0, 2], [3] * 10])
def test_every_stage(model, counts):
    tokens, off, u, temp = request(counts, len(counts))
    r = Round(model, len(tokens))
    r.fill(3)
    # drafts that are likely to stand: the first run's own most likely tokens
    d = [dev(v) for v in (tokens, off, u, temp)]
    r.run(*d)
    likely = r.logits.float().argmax(1).cpu().numpy()
    for b in range(len(counts)):
        for i in range(off[b], off[b + 1] - 1):
            if i % 3 != 2:
                tokens[i + 1] = likely[i]
    d[0].copy_(dev(tokens))
    r.run(*d)
    torch.cuda.synchronize()
    assert r.ctx.check_device() == 0 and r.ctx_v.check_device() == 0
    # projection
    want, tol = expected(model.wo, Q8, H, ATTN, r.attn.cpu().numpy(), None, None, r.h0.cpu().numpy(), False)
    h1 = r.h1.cpu().numpy()
    assert np.all(np.abs(h1 - want) <= tol)
    # block
    x1, hl = r.x1.cpu().numpy(), host_layer(model.t)
    ri, rw = plain_route(np.asarray(O.route_batch(hl, x1, want_logits=True)[-1]), K, bias=model.bias, **RULE)
    idx, w, g = r.routing
    assert np.array_equal(idx.cpu().numpy(), ri)
    assert np.all(np.abs(w.cpu().numpy() - rw) <= (2.0 ** -24 + 1e-12) * rw)
    assert_moe_close(r.h2.cpu().numpy(), block(hl, x1, h1, ri, rw.astype(np.float32), g.cpu().numpy()), base=h1)
    # logits
    want, tol = expected(model.head, Q6, VOCAB, H, r.x16.cpu().numpy(), None, None, None, True)
    assert np.all(np.abs(r.logits.cpu().numpy() - want) <= tol)
    # verification
    acc, nxt, lp = (v.cpu().numpy() for v in r.out)
    ra, rn, rl = plain_verify(r.logits.cpu().numpy(), tokens, off, u, None, temp, -1)
    assert np.array_equal(acc, ra) and np.array_equal(nxt, rn)
    assert np.all(np.abs(lp - rl) <= 2.0 ** -24 * np.abs(rl) + 1e-12)
    if len(counts) == 10:
        assert 0 < acc.sum() < sum(counts)


def test_a_captured_round_and_one_on_another_stream(model):
    tokens, off, u, temp = (dev(v) for v in request([4, 0, 2], 9))
    r = Round(model, len(tokens))
    r.fill(5)
    r.run(tokens, off, u, temp)  # (first calls load code)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = r.run(tokens, off, u, temp)
    eager = Round(model, r.T)
    side = torch.cuda.Stream()
    for seed in range(4):
        r.fill(seed)
        eager.fill(seed)
        u.copy_(torch.rand(len(u), generator=torch.Generator().manual_seed(seed)))
        torch.cuda.synchronize()
        g.replay()
        want = eager.run(tokens, off, u, temp, stream=side if seed % 2 else None)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        assert torch.isfinite(out[-1]).all()


def test_two_rounds_at_once(model):
    """Contexts of their own on two streams: neither round sees the other's."""
    req = [request([4, 1], 1), request([2, 2, 5], 2)]
    rounds = [Round(model, len(q[0])) for q in req]
    d = [[dev(v) for v in q] for q in req]
    alone = []
    for i, r in enumerate(rounds):
        r.fill(i)
        alone.append([v.clone() for v in r.run(*d[i])])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in rounds]
    both = []
    for _ in range(5):
        both = [r.run(*d[i], stream=streams[i]) for i, r in enumerate(rounds)]
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
