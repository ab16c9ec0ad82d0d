"""Tensors that the operators' Python calls refuse, on the CPU."""
import ctypes

import pytest
import torch

import breadv2_amd as B
from breadv2_amd import _lib, api


@pytest.mark.parametrize("qtype,cols,size", [(12, 256, 144), (14, 256, 210), (8, 256, 272), (1, 256, 512)])
def test_matmul_takes_dense_weights_only(qtype, cols, size):
    x = torch.zeros(2, cols, dtype=torch.float16)
    y = torch.zeros(2, 16, dtype=torch.float16)
    wide = torch.zeros(16, size + 16, dtype=torch.uint8)
    for w in (wide[:, :size], torch.zeros(2 * 16 * size, dtype=torch.uint8)[::2], torch.zeros(size, 16, dtype=torch.uint8).t(),
              torch.zeros(1, dtype=torch.uint8).expand(16 * size)):
        with pytest.raises(ValueError, match="dense"):
            B.bread_matmul(w, x, y, 16, cols, qtype)


def test_block_by_rule_takes_whole_dense_rows():
    """x and hidden with fewer rows than n_tokens, of another type or strided: nothing would be there to read."""
    ctx = B.MoeContext.__new__(B.MoeContext)  # (its library context needs a GPU; the tensors are looked at first)
    ctx.shape, ctx.max_tokens, ctx._h = api.shape(256, 256, 256, 8, 2), 8, ctypes.c_void_p()
    layer, rule, good = _lib.MoeLayer(), B.RouteRule(), torch.zeros(4, 256)
    for bad in (good[:3], good.half(), good.double(), torch.zeros(4, 512)[:, :256], torch.zeros(256, 4).t(),
                torch.zeros(4, 255)):
        with pytest.raises(ValueError, match="x must be dense float32"):
            ctx.route_by_rule(layer, rule, bad, 4)
        with pytest.raises(ValueError, match="x must be dense float32"):
            ctx.forward_by_rule(layer, rule, bad, good, 4)
        with pytest.raises(ValueError, match="hidden must be dense float32"):
            ctx.forward_by_rule(layer, rule, good, bad, 4)
