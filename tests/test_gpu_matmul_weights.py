"""bread_matmul: Q6_K weights keep every bit, through each kernel that the sizes choose.

A weight's integer is scale times code, up to 4096, and fp16 holds 11 bits.  Half of the columns carry the code 31
against x = a, the others the code 30 against x = -a, with odd scales sc near 127: a row's sum is
a (cols / 2) sc d, and integers rounded to 11 bits would be off by 1 / sc of that (31 sc is odd and above 2048).
The fp32 sums' bound is 61 sc / 2 times (270 + 2 cols / 256) 2^-23 of it, a quarter; an fp16 result adds half a step.
"""
import numpy as np
import pytest
import torch

import breadv2_amd as B

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
Q6 = 14


def q6_bytes(codes, scales, d):
    """Q6_K superblocks from codes 0 to 63 [n][256], int8 scales [n][16] and fp16 d [n]."""
    n = len(codes)
    b = np.zeros((n, 210), np.uint8)
    for e in range(256):
        h, j = divmod(e, 128)
        quarter, at = divmod(j, 32)
        b[:, 64 * h + at + 32 * (quarter % 2)] |= ((codes[:, e] & 15) << (0 if quarter < 2 else 4)).astype(np.uint8)
        b[:, 128 + 32 * h + at] |= ((codes[:, e] >> 4) << (2 * quarter)).astype(np.uint8)
    b[:, 192:208] = scales.astype(np.int8).view(np.uint8)
    b[:, 208:210] = d.astype(np.float16).reshape(-1, 1).view(np.uint8)
    return b.reshape(-1)


def tiles(T, rows, m, n):
    return -(-T // m) * -(-rows // n)


# by rows (activations held, two sets, two chunks, not held), 32 x 64, 32 x 32, 64 x 64, 128 x 128, 128 x 256
SIZES = [(1, 50, 256), (9, 50, 2048), (20, 50, 512), (9, 16403, 2304), (17, 50, 2560), (40, 96, 512), (40, 96, 1280),
         (300, 2700, 512), (1537, 2100, 512), (2049, 3300, 256)]


@pytest.mark.parametrize("half", [True, False], ids=["y16", "y32"])
@pytest.mark.parametrize("T,rows,cols", SIZES)
def test_six_bit_weights_keep_every_bit(T, rows, cols, half):
    if T == 300:
        assert tiles(T, rows, 64, 64) >= 200 > tiles(T, rows, 128, 128)
    if T == 1537:
        assert tiles(T, rows, 128, 128) >= 200 > tiles(T, rows, 128, 256)
    if T == 2049:
        assert tiles(T, rows, 128, 256) >= 200
    plus = np.random.default_rng(rows).permutation(cols) % 2 == 0
    codes = np.broadcast_to(np.where(plus, 63, 62), (rows, cols)).reshape(-1, 256)
    sc = (127 - 2 * (np.arange(rows) % 9)) * np.where(np.arange(rows) % 4 < 2, 1, -1)
    scales = np.repeat(np.repeat(sc, cols // 256)[:, None], 16, 1)
    d = np.full(len(codes), 2.0 ** -10)
    a = (1.0 + np.arange(T) % 3) / 8
    x = np.where(plus, 1.0, -1.0) * a[:, None]
    y = torch.empty(T, rows, dtype=torch.float16 if half else torch.float32, device=DEV)
    w = torch.from_numpy(q6_bytes(codes, scales, d)).to(DEV)
    B.bread_matmul(w, torch.from_numpy(x.astype(np.float16)).to(DEV), y, rows, cols, Q6)
    want = a[:, None] * (cols // 2 * 2.0 ** -10) * sc
    tol = (270 + 2 * cols / 256) * 2.0 ** -23 * 61 / 2 * cols * 2.0 ** -10 * np.abs(a[:, None] * sc)
    assert np.all(2.5 * tol < np.abs(want) / 97)
    if half:
        tol = tol + 2.0 ** -11 * (np.abs(want) + tol)
    assert np.all(np.abs(y.cpu().numpy().astype(np.float64) - want) <= tol)
