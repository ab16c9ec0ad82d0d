"""bread_rmsnorm_fp8 with hidden in place of x or of the residual, of the same stride and of another."""
import ctypes

import pytest
import torch

import breadv2_amd as B
from breadv2_amd import _lib
from test_fp8_args import P, norm

F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("kw", [dict(hidden=P, hidden_stride=512), dict(hidden=P, x_stride=272),
                                dict(hidden=2 * P, residual=2 * P, residual_stride=512),
                                dict(hidden=2 * P, residual=2 * P, hidden_stride=260, x_stride=260)])
def test_another_stride_is_refused(kw):
    assert norm(**kw) == _lib.ERR_ARG
    assert "bread_rmsnorm_fp8" in _lib.lib.bread_last_error().decode()


@pytest.mark.gpu
def test_in_place():
    def call(x, residual, hidden):
        T, n = x.shape
        codes, scales = torch.empty(T, n, dtype=F8, device="cuda"), torch.empty(T, n // 128, device="cuda")
        B.bread_rmsnorm_fp8(x, None, codes, scales, 1e-6, residual=residual, hidden=hidden)
        return codes.view(torch.uint8), scales

    g = torch.Generator().manual_seed(1)
    buf, r = torch.randn(4, 512, generator=g).cuda(), torch.randn(4, 256, generator=g).cuda()
    x = buf[:, :256]
    want = x + r
    apart = call(x.clone(), r, None)
    with pytest.raises(B.BreadError) as e:  # hidden's rows would lie where x's are
        call(x, r, buf.view(-1)[:1024].view(4, 256))
    assert e.value.status == _lib.ERR_ARG
    for a, b in zip(apart, call(x, r, x)):
        assert torch.equal(a, b)
    assert torch.equal(buf[:, :256], want)
    # one row has no stride
    one = torch.randn(1, 256, generator=g).cuda()
    codes, scales = torch.empty(1, 256, dtype=F8, device="cuda"), torch.empty(1, 2, device="cuda")
    a = _lib.RmsnormFp8Args()
    a.x = a.hidden = one.data_ptr()
    a.x_type, a.n, a.n_tokens, a.eps, a.hidden_stride = 0, 256, 1, 1e-6, 512
    a.codes, a.scales = codes.data_ptr(), scales.data_ptr()
    st = torch.cuda.current_stream().cuda_stream
    assert _lib.lib.bread_rmsnorm_fp8(ctypes.byref(a), st) == _lib.OK
    torch.cuda.synchronize()
