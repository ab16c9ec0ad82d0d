"""Outputs of calls on another stream than the current one: what the current stream still has to do to memory that
was freed there does not reach them."""
import numpy as np
import pytest
import torch

import breadv2_amd as B
from breadv2_amd import api

from test_gpu_spec_verify import dev, round_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def calls():
    s = api.shape(1024, 512, 256, 64, 6)
    t = api.synth_layer_tensors(s, seed=3, layer=0)
    T = 24
    x, h = torch.randn(T, s.hidden, device=DEV), torch.zeros(T, s.hidden, device=DEV)
    ctx = B.MoeContext(s, max_tokens=64)
    rule = B.RouteRule(score="sigmoid", n_groups=8, top_groups=4, group_top=2)
    z = torch.randn(T, 64, device=DEV)
    lz, tokens, off, u, q = round_of([3, 0, 5], 700, 4)
    args = [dev(lz), dev(tokens.astype(np.int32)), dev(off.astype(np.int32)), dev(u)]
    dq, d = dev(q), t.desc()
    return (t, ctx), {
        "route_select": lambda st: B.route_select(z, 6, rule, stream=st),
        "route_by_rule": lambda st: ctx.route_by_rule(d, rule, x, T, stream=st),
        "forward_by_rule": lambda st: ctx.forward_by_rule(d, rule, x, h, T, True, stream=st),
        "spec_verify": lambda st: ctx.spec_verify(*args, draft_probs=dq, stream=st),
        "route": lambda st: ctx.route(d, x, T, stream=st),
        "forward": lambda st: ctx.forward(d, x, h, T, True, stream=st),
        "argmax_f16": lambda st: (B.argmax_f16(args[0], stream=st),),
    }


@pytest.fixture(scope="module")
def busy():
    """(work that keeps the current stream busy, a stream that does not wait for it: streams share a few queues)."""
    big = torch.randn(8192, 8192, device=DEV).half()

    def work():
        for _ in range(20):
            torch.mm(big, big)

    one = torch.zeros(1, device=DEV)
    work()
    for _ in range(8):
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        work()
        done = torch.cuda.Event()
        done.record()
        with torch.cuda.stream(side):
            one.add(1)
        side.synchronize()
        if not done.query():
            return work, side
    pytest.skip("no stream runs beside the current one")


@pytest.mark.parametrize("name", ["route_select", "route_by_rule", "forward_by_rule", "spec_verify", "route", "forward",
                                  "argmax_f16"])
def test_work_queued_on_freed_memory_does_not_reach_outputs(name, busy):
    work, side = busy
    keep, fs = calls()
    f = fs[name]
    want = [v.clone() for v in f(None)]
    f(side)
    for _ in range(3):
        torch.cuda.synchronize()
        work()
        old = [torch.full_like(v, 77) for v in want]  # not yet written
        del old
        got = f(side)
        side.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["route_select", "route_by_rule", "spec_verify", "argmax_f16"])
def test_a_side_stream_in_a_graph(name):
    """A call on a stream that branches off a capture and joins it again."""
    keep, fs = calls()
    f = fs[name]
    side = torch.cuda.Stream()
    want = f(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        got = f(side)
        main.wait_stream(side)
    for _ in range(3):
        for v in got:
            v.fill_(9)
        g.replay()
        again = f(None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, want, again))
