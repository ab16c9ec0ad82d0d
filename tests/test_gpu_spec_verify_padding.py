"""bread_spec_verify in buffers of a fixed size: rows before the first request and behind the last are no request's,
whatever they hold, and their log-probabilities stay as they were."""
import ctypes

import numpy as np
import pytest
import torch

import breadv2_amd as B
from breadv2_amd import _lib

from test_gpu_spec_verify import DEV, dev, plain, round_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("probs", [True, False], ids=["model", "lookup"])
@pytest.mark.parametrize("before,behind", [(0, 3), (2, 0), (5, 40)])
def test_rows_of_no_request(before, behind, probs):
    counts, V = [3, 0, 5], 5000
    z, tokens, off, u, q = round_of(counts, V, 9, True, probs)
    rows = before + len(tokens) + behind
    rng = np.random.default_rng(1)

    def pad(a, n, fill):
        out = np.resize(np.asarray(fill, a.dtype), (n,) + a.shape[1:]).copy()
        out[before:before + len(a)] = a
        return dev(out)

    temp = np.array([0.7, 0.0, 1.3], np.float32)
    junk = np.where(rng.random(V) < 0.5, np.nan, np.inf)
    d = dict(z=pad(z, rows, junk), tokens=pad(tokens.astype(np.int32), rows, [-7, 2 ** 30]),
             off=dev((off + before).astype(np.int32)), u=pad(u, rows, [np.nan, 7.0]), temp=dev(temp))
    if probs:
        d["q"] = pad(q, rows - len(counts), [np.nan])
    acc, nxt = (torch.empty(3, dtype=torch.int32, device=DEV) for _ in range(2))
    lp = torch.full((rows,), 5.0, device=DEV)
    ctx = B.MoeContext(B.shape(), max_tokens=64)
    p = {k: v.data_ptr() for k, v in d.items()}
    a = _lib.VerifyArgs(p["z"], V, _lib.QTYPE_F16, V, rows, 3, p["tokens"], p["off"], p["u"], p.get("q"), V, p["temp"],
                        -1, acc.data_ptr(), nxt.data_ptr(), lp.data_ptr())
    assert B.lib.bread_spec_verify(ctx.handle, ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert ctx.check_device() == 0
    ra, rn, rl = plain(z, tokens, off, u, q, temp)
    assert np.array_equal(acc.cpu().numpy(), ra) and np.array_equal(nxt.cpu().numpy(), rn)
    got = lp.cpu().numpy()
    assert np.all(np.abs(got[before:before + len(tokens)] - rl) <= 2.0 ** -24 * np.abs(rl) + 1e-12)
    assert np.all(got[:before] == 5.0) and np.all(got[before + len(tokens):] == 5.0)
