"""The block by a rule uses and returns the shared gate's scores of bread_route_by_rule, bit for bit, on every path."""
import pytest
import torch

import breadv2_amd as B
from breadv2_amd import api

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
RULE = dict(score="sigmoid", n_groups=8, top_groups=4, group_top=2, renorm=True, scale=2.5)


# the decode shape, and one that the small path takes by other kernels
@pytest.mark.parametrize("dims", [(2048, 512, 512, 64, 8), (1024, 512, 256, 64, 6)], ids=["decode", "other"])
@pytest.mark.parametrize("T", [1, 2, 4, 5, 9, 16, 17, 32, 40])
def test_the_same_gate_on_every_path(dims, T):
    s = api.shape(*dims)
    t = api.synth_layer_tensors(s, seed=31, layer=0)
    g = torch.Generator(device=DEV).manual_seed(T)
    rule = B.RouteRule(bias=0.1 * torch.randn(s.n_experts, device=DEV, generator=g), **RULE)
    x = torch.randn(T, s.hidden, device=DEV, generator=g)
    h0 = torch.randn(T, s.hidden, device=DEV, generator=g)
    ctx = B.MoeContext(s, max_tokens=T)
    idx, w, gate = ctx.route_by_rule(t.desc(), rule, x, T)
    for path in (api.PATH_AUTO, api.PATH_PER_TOKEN, api.PATH_GROUPED) + ((api.PATH_SMALL,) if T <= 32 else ()):
        ctx.set_path(path)
        i2, w2, g2 = ctx.forward_by_rule(t.desc(), rule, x, h0.clone(), T, want_routing=True)
        torch.cuda.synchronize()
        assert ctx.check_device() == 0
        assert torch.equal(i2, idx) and torch.equal(w2, w) and torch.equal(g2, gate), path


def test_large_activations_keep_their_tokens(T=3):
    """Tokens of very different sizes side by side: each token's fixed-point scales are its own."""
    s = api.shape(2048, 512, 512, 64, 8)
    t = api.synth_layer_tensors(s, seed=32, layer=0)
    rule = B.RouteRule(**RULE)
    x = torch.randn(T, s.hidden, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    x *= torch.tensor([[1e-4], [1.0], [1e3]], device=DEV)
    ctx = B.MoeContext(s, max_tokens=T)
    ctx.set_path(api.PATH_SMALL)
    h = torch.zeros(T, s.hidden, device=DEV)
    ctx.forward_by_rule(t.desc(), rule, x, h, T)
    for i in range(T):
        one = torch.zeros(1, s.hidden, device=DEV)
        ctx.forward_by_rule(t.desc(), rule, x[i:i + 1], one, 1)
        # the same weights in another order of sums: 2^-20 of the row's size
        assert torch.all((one[0] - h[i]).abs() <= 2.0 ** -20 * s.hidden ** 0.5 * h[i].abs().max())
