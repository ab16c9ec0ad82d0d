"""What the 8-bit floating point entry points refuse, on the CPU: before any HIP call."""
import ctypes

import pytest
import torch

import breadv2_amd as B
from breadv2_amd import _lib, api

lib = _lib.lib
P = 0x1000  # an aligned address that is never read
F8 = torch.float8_e4m3fn


def fill(cls, base, kw):
    a = cls()
    for k, v in {**base, **kw}.items():
        assert any(k == f[0] for f in cls._fields_), k
        setattr(a, k, v)
    return a


def norm(**kw):
    base = dict(x=P, x_type=0, eps=1e-6, n=256, n_tokens=2, codes=P, scales=P)
    return lib.bread_rmsnorm_fp8(ctypes.byref(fill(_lib.RmsnormFp8Args, base, kw)), None)


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), _lib.ERR_ARG), (dict(codes=None), _lib.ERR_ARG), (dict(scales=None), _lib.ERR_ARG),
    (dict(n=0), _lib.ERR_ARG), (dict(n=-16), _lib.ERR_ARG), (dict(n_tokens=-1), _lib.ERR_ARG),
    (dict(x_type=8), _lib.ERR_QTYPE), (dict(x_type=0x1000), _lib.ERR_QTYPE), (dict(normed=P, normed_type=12), _lib.ERR_QTYPE),
    (dict(n=250), _lib.ERR_SHAPE), (dict(n=32784), _lib.ERR_SHAPE), (dict(n_tokens=(1 << 22) + 1), _lib.ERR_SHAPE),
    (dict(x_stride=255), _lib.ERR_SHAPE), (dict(residual_stride=255), _lib.ERR_SHAPE),
    (dict(hidden_stride=-256), _lib.ERR_SHAPE), (dict(codes_stride=240), _lib.ERR_SHAPE),
    (dict(scales_stride=1), _lib.ERR_SHAPE), (dict(normed_stride=1), _lib.ERR_SHAPE),
    (dict(codes=P + 8), _lib.ERR_ALIGN), (dict(codes_stride=264), _lib.ERR_ALIGN), (dict(x=P + 2), _lib.ERR_ALIGN),
    (dict(x=P + 1, x_type=1), _lib.ERR_ALIGN), (dict(residual=P + 2), _lib.ERR_ALIGN), (dict(hidden=P + 1), _lib.ERR_ALIGN),
    (dict(weight=P + 2), _lib.ERR_ALIGN), (dict(scales=P + 2), _lib.ERR_ALIGN),
    (dict(normed=P + 1, normed_type=30), _lib.ERR_ALIGN)])
def test_norm_refuses(kw, want):
    assert norm(**kw) == want
    assert "bread_rmsnorm_fp8" in lib.bread_last_error().decode()


def test_norm_refuses_more_rows_than_a_launch_holds():
    """2^22 rows of 1024 threads each are 2^32 threads, one more than a launch counts."""
    assert norm(n=32768, n_tokens=1 << 22) == _lib.ERR_SHAPE


def matmul(groups=None, **kw):
    base = dict(w=P, w_scale=P, x=P, x_scale=P, y=P, y_type=0, rows=64, cols=256, n_tokens=2)
    a = fill(_lib.MatmulFp8Args, base, kw)
    if groups is None:
        return lib.bread_matmul_fp8(ctypes.byref(a), None)
    g = fill(_lib.Fp8Groups, dict(n_groups=4, offsets=P), groups)
    return lib.bread_matmul_fp8_grouped(ctypes.byref(a), ctypes.byref(g), None)


BAD = [
    (dict(w=None), _lib.ERR_ARG), (dict(w_scale=None), _lib.ERR_ARG), (dict(x=None), _lib.ERR_ARG),
    (dict(x_scale=None), _lib.ERR_ARG), (dict(y=None), _lib.ERR_ARG), (dict(up=P), _lib.ERR_ARG),
    (dict(y_type=0x1000), _lib.ERR_ARG), (dict(rows=-1), _lib.ERR_ARG), (dict(cols=0), _lib.ERR_ARG),
    (dict(n_tokens=-1), _lib.ERR_ARG), (dict(act=5), _lib.ERR_ARG), (dict(act=-1), _lib.ERR_ARG),
    (dict(y_type=8), _lib.ERR_QTYPE), (dict(y_type=12), _lib.ERR_QTYPE), (dict(cols=264), _lib.ERR_SHAPE),
    (dict(cols=(1 << 20) + 16), _lib.ERR_SHAPE), (dict(rows=(1 << 24) + 1), _lib.ERR_SHAPE),
    (dict(n_tokens=(1 << 24) + 1), _lib.ERR_SHAPE), (dict(rows=1 << 20, n_tokens=(1 << 13) + 1), _lib.ERR_SHAPE),
    (dict(rows=(1 << 20) + 1, cols=1 << 20), _lib.ERR_SHAPE), (dict(x_stride=(1 << 22) + 16), _lib.ERR_SHAPE),
    (dict(x_scale_stride=(1 << 20) + 1), _lib.ERR_SHAPE), (dict(x_stride=240), _lib.ERR_SHAPE),
    (dict(x_scale_stride=1), _lib.ERR_SHAPE), (dict(y_stride=63), _lib.ERR_SHAPE),
    (dict(y_type=0x1000, y_scale=P, rows=65), _lib.ERR_SHAPE), (dict(y_type=0x1000, y_scale=P, rows=256, y_scale_stride=1), _lib.ERR_SHAPE),
    (dict(y_type=0x1000, y_scale=P, residual=P), _lib.ERR_ARG), (dict(up=P, up_scale=P, bias=P), _lib.ERR_ARG),
    (dict(w=P + 8), _lib.ERR_ALIGN), (dict(up=P + 8, up_scale=P), _lib.ERR_ALIGN), (dict(x=P + 8), _lib.ERR_ALIGN),
    (dict(x_stride=264), _lib.ERR_ALIGN), (dict(y=P + 2), _lib.ERR_ALIGN), (dict(y=P + 1, y_type=1), _lib.ERR_ALIGN),
    (dict(y=P + 8, y_type=0x1000, y_scale=P), _lib.ERR_ALIGN), (dict(y_stride=72, y_type=0x1000, y_scale=P), _lib.ERR_ALIGN),
    (dict(residual=P + 2), _lib.ERR_ALIGN), (dict(bias=P + 2), _lib.ERR_ALIGN), (dict(w_scale=P + 2), _lib.ERR_ALIGN),
    (dict(x_scale=P + 1), _lib.ERR_ALIGN)]


@pytest.mark.parametrize("kw,want", BAD)
def test_matmul_refuses(kw, want):
    assert matmul(**kw) == want
    assert "bread_matmul_fp8:" in lib.bread_last_error().decode()
    if "bias" not in kw and "residual" not in kw:
        assert matmul(groups={}, **kw) == want
        assert "bread_matmul_fp8_grouped" in lib.bread_last_error().decode()


@pytest.mark.parametrize("groups,kw,want", [
    (dict(n_groups=-1), {}, _lib.ERR_ARG), (dict(n_groups=1025), {}, _lib.ERR_SHAPE), (dict(offsets=None), {}, _lib.ERR_ARG),
    (dict(x_rows=P, n_x=(1 << 23) + 1), {}, _lib.ERR_SHAPE), (dict(x_rows=P, n_x=1 << 23), dict(x_scale_stride=65), _lib.ERR_SHAPE),
    (dict(n_groups=1024), dict(rows=(1 << 18) + 1), _lib.ERR_SHAPE), (dict(offsets=P + 2), {}, _lib.ERR_ALIGN), (dict(x_rows=P + 2, n_x=2), {}, _lib.ERR_ALIGN),
    (dict(y_rows=P + 1, n_y=2), {}, _lib.ERR_ALIGN), (dict(x_rows=P, n_x=-1), {}, _lib.ERR_ARG),
    (dict(y_rows=P, n_y=-1), {}, _lib.ERR_ARG), ({}, dict(bias=P), _lib.ERR_ARG), ({}, dict(residual=P), _lib.ERR_ARG)])
def test_groups_refuse(groups, kw, want):
    assert matmul(groups=groups, **kw) == want


def test_of_nothing():
    assert norm(n_tokens=0, x=None, codes=None, scales=None) == _lib.OK
    assert matmul(rows=0, w=None, x=None, y=None) == _lib.OK and matmul(n_tokens=0, y=None) == _lib.OK
    assert matmul(groups={}, n_tokens=0) == _lib.OK and matmul(groups=dict(n_groups=0, offsets=None), w=None) == _lib.OK
    for call in (lambda: lib.bread_rmsnorm_fp8(None, None), lambda: lib.bread_matmul_fp8(None, None),
                 lambda: lib.bread_matmul_fp8_grouped(None, None, None),
                 lambda: lib.bread_moe_expert_block_fp8(None, None, P, P, P, P, 0, 1, P, P, None)):
        assert call() == _lib.ERR_ARG


def f8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(F8)


def test_python_norm_refuses():
    x, codes, scales = torch.zeros(2, 256), f8(2, 256), torch.zeros(2, 2)
    good = dict(x=x, w=None, codes=codes, scales=scales, eps=1e-6)
    for kw in (dict(x=x.double()), dict(x=x[0]), dict(x=torch.zeros(2, 512)[:, ::2]), dict(codes=f8(3, 256)), dict(codes=f8(2, 255)),
               dict(codes=torch.zeros(2, 256, dtype=torch.uint8)), dict(scales=torch.zeros(2, 3)), dict(scales=torch.zeros(1, 2)),
               dict(scales=scales.half()), dict(w=torch.zeros(255)), dict(w=torch.zeros(256).half()), dict(residual=x.half()),
               dict(residual=x[:1]), dict(hidden=x.half()), dict(hidden=torch.zeros(2, 255)), dict(normed=x.double()),
               dict(normed=x[:1]), dict(x=x[:1].expand(2, 256))):
        with pytest.raises(ValueError):
            B.bread_rmsnorm_fp8(**{**good, **kw})


def test_python_matmul_refuses():
    w, ws, x, xs, y = f8(64, 256), torch.zeros(1, 2), f8(3, 256), torch.zeros(3, 2), torch.zeros(3, 64)
    good = dict(w=w, w_scale=ws, x=x, x_scale=xs, y=y)
    for kw in (dict(act="swish"), dict(w=w.view(torch.uint8)), dict(w=f8(64, 512)[:, :256]), dict(w=f8(256, 64).t()), dict(w=w[0]),
               dict(w_scale=torch.zeros(2, 1)), dict(w_scale=ws.half()), dict(w_scale=None), dict(x=x.view(torch.uint8)), dict(x=f8(3, 272)),
               dict(x=f8(3, 512)[:, ::2]), dict(x_scale=xs[:2]), dict(x_scale=torch.zeros(3, 3)), dict(x_scale=xs.half()),
               dict(y=y.double()), dict(y=y[:2]), dict(y=torch.zeros(3, 65)), dict(y=torch.zeros(64, 3).t()), dict(y=f8(3, 64)),
               dict(y=f8(3, 64), y_scale=torch.zeros(3, 2)), dict(y_scale=torch.zeros(3, 1)), dict(up=w),
               dict(up=f8(32, 256), up_scale=ws), dict(up=w, up_scale=torch.zeros(2, 2)), dict(bias=torch.zeros(63)),
               dict(bias=torch.zeros(64).half()), dict(residual=y.half()), dict(residual=y[:2]),
               dict(residual=torch.zeros(3, 65)[:, :64]), dict(x=x[:1].expand(3, 256))):
        with pytest.raises(ValueError):
            B.bread_matmul_fp8(**{**good, **kw})


def test_python_groups_refuse():
    w, ws, x, xs, y = f8(4, 64, 256), torch.zeros(4, 1, 2), f8(3, 256), torch.zeros(3, 2), torch.zeros(3, 64)
    off = torch.zeros(5, dtype=torch.int32)
    good = dict(w=w, w_scale=ws, x=x, x_scale=xs, offsets=off, y=y)
    rows = torch.zeros(3, dtype=torch.int32)
    for kw in (dict(w=w[0]), dict(w_scale=ws[:3]), dict(offsets=off[:4]), dict(offsets=off.long()), dict(offsets=torch.zeros(10, dtype=torch.int32)[::2]),
               dict(x_rows=rows.long()), dict(x_rows=rows[None]), dict(x_rows=torch.zeros(4, dtype=torch.int32)), dict(y_rows=rows[:2]),
               dict(y_rows=rows.float()), dict(y=y[:2]), dict(x_scale=xs[:2])):
        with pytest.raises(ValueError):
            B.bread_matmul_fp8_grouped(**{**good, **kw})


def test_python_block_refuses():
    E, I, H, K = 4, 256, 512, 2
    gate, gs, down, ds = f8(E, I, H), torch.zeros(E, 2, 4), f8(E, H, I), torch.zeros(E, 4, 2)
    for t in ((gate[0], gs, gate, gs, down, ds), (gate, gs[:3], gate, gs, down, ds), (gate, gs, f8(E, I, 256), gs, down, ds),
              (gate, gs, gate, gs, gate, gs), (gate, gs, gate, gs, down, gs), (gate.view(torch.uint8), gs, gate, gs, down, ds)):
        with pytest.raises(ValueError):
            B.Fp8Experts(*t)
    ctx = B.MoeContext.__new__(B.MoeContext)  # (its library context needs a GPU; the tensors are looked at first)
    ctx.shape, ctx.max_tokens, ctx._h = api.shape(H, I, I, E, K), 8, ctypes.c_void_p()
    ex = B.Fp8Experts(gate, gs, gate, gs, down, ds)
    good = dict(experts=ex, x=f8(3, H), x_scale=torch.zeros(3, 4), hidden=torch.zeros(3, H), idx=torch.zeros(3, K, dtype=torch.int32),
                w=torch.zeros(3, K))
    for kw in (dict(x=f8(3, 256)), dict(x=torch.zeros(3, H)), dict(x=f8(3, 2 * H)[:, :H]), dict(x_scale=torch.zeros(3, 3)), dict(x_scale=torch.zeros(2, 4)),
               dict(hidden=torch.zeros(3, H).double()), dict(hidden=torch.zeros(2, H)), dict(residual=torch.zeros(3, H).half()),
               dict(residual=torch.zeros(2, H)), dict(idx=torch.zeros(3, K)), dict(idx=torch.zeros(3, 3, dtype=torch.int32)),
               dict(w=torch.zeros(3, K).half()), dict(w=torch.zeros(2, 3).t()), dict(experts=B.Fp8Experts(gate[:2], gs[:2], gate[:2], gs[:2], down[:2], ds[:2]))):
        with pytest.raises(ValueError):
            ctx.expert_block_fp8(**{**good, **kw})


def test_packed_arguments_are_the_structures():
    """The bytes that the Python calls pass lie as the C structures of the header do."""
    for packed, cls in ((api._NORM_ARGS, _lib.RmsnormFp8Args), (api._MATMUL_ARGS, _lib.MatmulFp8Args),
                        (api._GROUP_ARGS, _lib.Fp8Groups)):
        values = [i + 1 for i in range(len(cls._fields_))]
        s = cls.from_buffer_copy(packed.pack(*values).ljust(ctypes.sizeof(cls), b"\0"))
        assert packed.size <= ctypes.sizeof(cls) and packed.size > getattr(cls, cls._fields_[-1][0]).offset
        assert [getattr(s, name) for name, _ in cls._fields_] == values
