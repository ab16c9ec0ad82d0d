"""NaN in routing by a rule: a signalling NaN logit counts as -inf as a quiet one does, a NaN bias as -inf."""
import numpy as np
import pytest
import torch

import breadv2_amd as B

from test_gpu_route_rule import compare, dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [60, 128, 256, 300])
def test_signalling_nan_logits(score, E):
    rng = np.random.default_rng(E)
    z = rng.standard_normal((9, E)).astype(np.float32)
    bits = z.view(np.uint32)
    for t in range(9):
        at = rng.integers(0, E, 12)
        at = at[at != np.argmax(z[t])]
        bits[t, at] = np.array([0x7F800001, 0x7FBFFFFF, 0xFF800001, 0x7FC00000], np.uint32)[rng.integers(0, 4, len(at))]
        bits[t, (np.argmax(np.nan_to_num(z[t], nan=-9.0)) + 1) % E] = 0x7FA00000
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    compare(z, 6, score=score)
    compare(z, 6, score=score, n_groups=4, top_groups=2, group_top=2, bias=bias)
    compare(z, 6, score=score, n_groups=2, top_groups=1, group_top=1, bias=bias, renorm=False)


@pytest.mark.parametrize("E,n_groups", [(256, 1), (256, 8), (60, 5), (300, 100)])
def test_nan_bias_is_minus_infinity(E, n_groups):
    rng = np.random.default_rng(E)
    z = dev(rng.standard_normal((33, E)).astype(np.float32))
    off = rng.permutation(E)[: E // 5]
    a = (0.1 * rng.standard_normal(E)).astype(np.float32)
    b = a.copy()
    a[off], b[off] = np.nan, -np.inf
    a.view(np.uint32)[off[::2]] = 0x7FA00000
    for score in ("softmax", "sigmoid"):
        for group_top in (1, 2):
            kw = dict(score=score, n_groups=n_groups, top_groups=-(-n_groups // 2), group_top=group_top)
            got = B.route_select(z, 8, B.RouteRule(bias=dev(a), **kw))
            want = B.route_select(z, 8, B.RouteRule(bias=dev(b), **kw))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
