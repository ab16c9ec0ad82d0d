"""The block's errors name the entry point that was called."""
import pytest
import torch

import breadv2_amd as B
from breadv2_amd import api

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_errors_name_the_entry_point():
    for dims, types, cases in (((2048, 512, 512, 64, 8), (12, 12, 14, 12, 12, 14), [(api.PATH_DECODE, 2), (api.PATH_SMALL, 33)]),
                               ((512, 256, 256, 12, 4), (12, 12, 12, 12, 12, 12), [(api.PATH_GROUPED, 2), (api.PATH_DECODE, 1)])):
        s = api.shape(*dims)
        t = api.synth_layer_tensors(s, seed=1, layer=0, types=types)
        x, h = torch.zeros(40, s.hidden, device=DEV), torch.zeros(40, s.hidden, device=DEV)
        ctx = B.MoeContext(s, max_tokens=40)
        for path, T in cases:
            ctx.set_path(path)
            with pytest.raises(B.BreadError):
                ctx.forward(t.desc(), x, h, T)
            assert B.lib.bread_last_error().decode().startswith("bread_moe_forward:")
            with pytest.raises(B.BreadError):
                ctx.forward_by_rule(t.desc(), B.RouteRule(), x, h, T)
            assert B.lib.bread_last_error().decode().startswith("bread_moe_forward_by_rule:")
        torch.cuda.synchronize()
        assert torch.all(h == 0)
