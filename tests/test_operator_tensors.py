"""Tensors that the operators' Python calls refuse, on the CPU."""
import pytest
import torch

import breadv2_amd as B


@pytest.mark.parametrize("qtype,cols,size", [(12, 256, 144), (14, 256, 210), (8, 256, 272), (1, 256, 512)])
def test_matmul_takes_dense_weights_only(qtype, cols, size):
    x = torch.zeros(2, cols, dtype=torch.float16)
    y = torch.zeros(2, 16, dtype=torch.float16)
    wide = torch.zeros(16, size + 16, dtype=torch.uint8)
    for w in (wide[:, :size], torch.zeros(2 * 16 * size, dtype=torch.uint8)[::2], torch.zeros(size, 16, dtype=torch.uint8).t(),
              torch.zeros(1, dtype=torch.uint8).expand(16 * size)):
        with pytest.raises(ValueError, match="dense"):
            B.bread_matmul(w, x, y, 16, cols, qtype)
