"""Argument checks of bread_matmul, bread_route_select, the rule entry points
and bread_spec_verify, on the CPU: they refuse before any HIP call."""
import ctypes

import pytest
import torch

import breadv2_amd as B
from breadv2_amd import _lib

lib = _lib.lib
P = 0x1000  # an aligned address that is never read


def matmul(w=P, x=P, y=P, rows=16, cols=256, qtype=12, T=2, **opts):
    o = _lib.MatmulOpts(opts.get("bias"), opts.get("residual"), opts.get("act", 0), opts.get("y_type", 1),
                        opts.get("xs", 0), opts.get("ys", 0))
    return lib.bread_matmul(w, x, y, rows, cols, qtype, T, ctypes.byref(o), None)


@pytest.mark.parametrize("kw,want", [
    (dict(w=None), _lib.ERR_ARG), (dict(x=None), _lib.ERR_ARG), (dict(y=None), _lib.ERR_ARG),
    (dict(rows=-1), _lib.ERR_ARG), (dict(cols=0), _lib.ERR_ARG), (dict(T=-1), _lib.ERR_ARG),
    (dict(qtype=2), _lib.ERR_QTYPE), (dict(qtype=0), _lib.ERR_QTYPE), (dict(y_type=8), _lib.ERR_QTYPE),
    (dict(act=5), _lib.ERR_ARG), (dict(act=-1), _lib.ERR_ARG),
    (dict(cols=255), _lib.ERR_SHAPE), (dict(cols=40, qtype=8), _lib.ERR_SHAPE), (dict(cols=12, qtype=1), _lib.ERR_SHAPE),
    (dict(xs=248), _lib.ERR_SHAPE), (dict(ys=15), _lib.ERR_SHAPE), (dict(xs=-256), _lib.ERR_SHAPE),
    (dict(xs=260), _lib.ERR_ALIGN), (dict(x=P + 8), _lib.ERR_ALIGN), (dict(w=P + 8), _lib.ERR_ALIGN),
    (dict(w=P + 2, qtype=14), _lib.ERR_ALIGN), (dict(w=P + 2, qtype=8), _lib.ERR_ALIGN),
    (dict(w=P + 8, qtype=1), _lib.ERR_ALIGN), (dict(y=P + 1), _lib.ERR_ALIGN),
    (dict(y=P + 2, y_type=0), _lib.ERR_ALIGN), (dict(residual=P + 1), _lib.ERR_ALIGN),
    (dict(bias=P + 2), _lib.ERR_ALIGN)])
def test_matmul_refuses(kw, want):
    assert matmul(**kw) == want
    assert "bread_matmul" in lib.bread_last_error().decode()


@pytest.mark.parametrize("kw", [dict(rows=(1 << 30) + 1), dict(cols=(1 << 30) + 256), dict(T=(1 << 28) + 1),
                                dict(rows=1 << 30, cols=32, qtype=8, T=1 << 20)])
def test_matmul_refuses_sizes_that_no_launch_has(kw):
    assert matmul(**kw) == _lib.ERR_SHAPE
    assert select(T=(1 << 26) + 1) == _lib.ERR_SHAPE


def test_matmul_of_nothing():
    assert matmul(rows=0) == _lib.OK and matmul(T=0) == _lib.OK
    assert matmul(rows=0, w=None, x=None, y=None) == _lib.OK


def select(E=64, K=8, T=3, stride=0, logits=P, idx=P, w=P, **rule):
    r = _lib.RouteRuleDesc(rule.get("bias"), rule.get("score", 0), rule.get("n_groups", 1), rule.get("top_groups", 1),
                           rule.get("group_top", 1), 1, 1.0)
    return lib.bread_route_select(ctypes.byref(r), logits, stride, E, K, T, idx, w, None)


@pytest.mark.parametrize("kw,want", [
    (dict(logits=None), _lib.ERR_ARG), (dict(idx=None), _lib.ERR_ARG), (dict(w=None), _lib.ERR_ARG),
    (dict(T=-1), _lib.ERR_ARG), (dict(E=0), _lib.ERR_SHAPE), (dict(E=1025), _lib.ERR_SHAPE), (dict(K=0), _lib.ERR_SHAPE),
    (dict(K=33), _lib.ERR_SHAPE), (dict(E=4, K=5), _lib.ERR_SHAPE), (dict(stride=63), _lib.ERR_SHAPE),
    (dict(score=2), _lib.ERR_ARG), (dict(n_groups=0), _lib.ERR_SHAPE), (dict(n_groups=7), _lib.ERR_SHAPE),
    (dict(n_groups=8, top_groups=0), _lib.ERR_ARG), (dict(n_groups=8, top_groups=9), _lib.ERR_ARG),
    (dict(n_groups=16, top_groups=1), _lib.ERR_SHAPE), (dict(group_top=0), _lib.ERR_ARG),
    (dict(group_top=3), _lib.ERR_ARG), (dict(bias=P + 2), _lib.ERR_ALIGN), (dict(logits=P + 2), _lib.ERR_ALIGN)])
def test_route_select_refuses(kw, want):
    assert select(**kw) == want


def test_route_select_of_nothing():
    assert select(T=0, logits=None, idx=None, w=None) == _lib.OK
    assert lib.bread_route_select(None, P, 0, 64, 8, 1, P, P, None) == _lib.ERR_ARG


def test_null_contexts():
    rule = _lib.RouteRuleDesc(None, 0, 1, 1, 1, 1, 1.0)
    layer = _lib.MoeLayer()
    assert lib.bread_route_by_rule(None, ctypes.byref(layer), ctypes.byref(rule), P, 1, P, P, P, None) == _lib.ERR_ARG
    assert lib.bread_moe_forward_by_rule(None, ctypes.byref(layer), ctypes.byref(rule), P, P, 1, None, None, None,
                                         None) == _lib.ERR_ARG
    assert lib.bread_spec_verify(None, ctypes.byref(_lib.VerifyArgs()), None) == _lib.ERR_ARG


def test_python_layer_refuses():
    w = torch.zeros(16 * 144, dtype=torch.uint8)
    x = torch.zeros(2, 256, dtype=torch.float16)
    y = torch.zeros(2, 16, dtype=torch.float16)
    for kw in (dict(act="swish"), dict(bias=torch.zeros(15)), dict(bias=torch.zeros(16, dtype=torch.float16)),
               dict(residual=torch.zeros(2, 16)), dict(residual=torch.zeros(2, 17, dtype=torch.float16)[:, :16])):
        with pytest.raises(ValueError):
            B.bread_matmul(w, x, y, 16, 256, 12, **kw)
    for a, b, c, rows, cols in ((w, x.float(), y, 16, 256), (w, x, y.double(), 16, 256), (w, x, y[:1], 16, 256),
                                (w, x[:, ::2], y, 16, 128), (w, x, y, 17, 256), (w[:-1], x, y, 16, 256),
                                (w, x[:1].expand(2, 256), y, 16, 256), (w, x, y[:1].expand(2, 16), 16, 256)):
        with pytest.raises(ValueError):
            B.bread_matmul(a, b, c, rows, cols, 12)
    with pytest.raises(ValueError):
        B.RouteRule(score="tanh")
    with pytest.raises(ValueError):
        B.RouteRule(bias=torch.zeros(4, dtype=torch.float64))
    with pytest.raises(ValueError):
        B.route_select(torch.zeros(2, 8, dtype=torch.float16), 2, B.RouteRule())
    with pytest.raises(ValueError):
        B.route_select(torch.zeros(2, 8), 2, B.RouteRule(bias=torch.zeros(9)))
