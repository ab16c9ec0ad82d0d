"""Python host layer over the C ABI: device memory and streams come from
PyTorch (plumbing); every computation is a call into libbread_moe.so.

Names mirror the reference's interface for this path (kernels.cu:289
bread_matvec, one_layer.cu:937 route_layer, the MoE block of
one_layer_forward one_layer.cu:1800-1986), with the reference's exit(1)
replaced by a raised BreadError carrying the status code.

A call goes to torch's current stream, or to `stream`.  Tensors that it
returns are of that stream's memory, as if it had been the current one:
another stream that uses them waits for it and records itself on them
(Tensor.record_stream).
"""
from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import BreadError, MoeLayer, MoeShape, check, lib

QTYPE_Q8_0 = _lib.QTYPE_Q8_0
QTYPE_Q4_K = _lib.QTYPE_Q4_K
QTYPE_Q6_K = _lib.QTYPE_Q6_K
PATH_AUTO = _lib.PATH_AUTO
PATH_DECODE = _lib.PATH_DECODE
PATH_GROUPED = _lib.PATH_GROUPED
PATH_PER_TOKEN = _lib.PATH_PER_TOKEN
PATH_SMALL = _lib.PATH_SMALL
QTYPE_F16 = _lib.QTYPE_F16
QTYPE_BF16 = _lib.QTYPE_BF16
QTYPE_E4M3 = _lib.QTYPE_E4M3


def _p(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _s(stream) -> ctypes.c_void_p:
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def _need(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def _on(stream, tensors) -> int:
    """The raw stream a call on these tensors (or None) goes to (default: torch's
    current one).  A launch goes to the current device, so they have to be there."""
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"a tensor is on {t.device}, the current device is cuda:{dev}")
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(dev)
    if stream.device_index != dev:
        raise ValueError(f"the stream is on cuda:{stream.device_index}, the current device is cuda:{dev}")
    return stream.cuda_stream


def _empty(stream):
    """torch.empty for the outputs of a call on `stream`, from that stream's memory:
    a block of the current stream's may still be waiting for work queued there
    before it was freed, and would be handed on there before the call is done
    with it."""
    if stream is None:
        return torch.empty

    def empty(*size, dtype, device):
        with torch.cuda.stream(stream):
            return torch.empty(*size, dtype=dtype, device=device)

    return empty


_HIP = None


def device_copy(dst: int, src: int, nbytes: int) -> None:
    """Synchronous device-to-device copy between raw device pointers (HIP
    runtime of the process, which torch has loaded)."""
    global _HIP
    if _HIP is None:
        _HIP = ctypes.CDLL("libamdhip64.so")
        _HIP.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
        _HIP.hipMemcpy.restype = ctypes.c_int
    torch.cuda.synchronize()
    rc = _HIP.hipMemcpy(dst, src, nbytes, 3)  # hipMemcpyDeviceToDevice
    if rc != 0:
        raise RuntimeError(f"hipMemcpy failed: {rc}")


def row_bytes(qtype: int, cols: int) -> int:
    if qtype == QTYPE_Q4_K:
        return cols // 256 * 144
    if qtype == QTYPE_Q6_K:
        return cols // 256 * 210
    if qtype == QTYPE_Q8_0:
        return cols // 32 * 34
    raise ValueError(f"qtype {qtype}")


# ---------------------------------------------------------------- matvec


def bread_matvec(w, x, y, rows: int, cols: int, qtype: int, stream=None) -> None:
    """fp16 in / fp16 out (kernels.cu:289). x, y: torch.float16 device tensors."""
    check(lib.bread_matvec(_p(w), _p(x), _p(y), rows, cols, qtype, _s(stream)), "bread_matvec")


def bread_matvec_f32(w, x, y, rows: int, cols: int, qtype: int, stream=None) -> None:
    check(lib.bread_matvec_f32(_p(w), _p(x), _p(y), rows, cols, qtype, _s(stream)), "bread_matvec_f32")


ACTS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU,
        "gelu_tanh": _lib.ACT_GELU_TANH, "relu": _lib.ACT_RELU}
_Y_TYPES = {torch.float16: _lib.QTYPE_F16, torch.float32: _lib.QTYPE_F32}


def _rows_of(t: torch.Tensor, name: str, cols: int) -> int:
    """Elements from one row of a 2-d tensor to the next (rows themselves dense)."""
    if t.dim() != 2 or t.shape[1] != cols:
        raise ValueError(f"{name} must be 2-d with {cols} columns, is {tuple(t.shape)}")
    step, one = t.stride()
    if one != 1 and cols > 1:
        raise ValueError(f"{name}'s rows must be dense")
    if t.shape[0] <= 1:
        return cols
    if step < cols:
        raise ValueError(f"{name}'s rows overlap")
    return step


def bread_matmul(w, x, y, rows: int, cols: int, qtype: int, bias=None, act=None, residual=None, stream=None) -> None:
    """y[t] = act(W x[t] + bias) + residual[t] for the rows t of x: torch.float16
    [n_tokens][cols], y (and residual, which may be y) float16 or float32
    [n_tokens][rows], bias float32 [rows]; rows of x and y may be strided.
    act: None, "silu", "gelu", "gelu_tanh" or "relu"."""
    a = ACTS.get(act)
    if a is None:
        raise ValueError(f"unknown activation {act!r}")
    if x.dtype != torch.float16:
        raise ValueError("x must be float16")
    kind = y.dtype
    y_type = _Y_TYPES.get(kind)
    if y_type is None:
        raise ValueError("y must be float16 or float32")
    xs, ys = _rows_of(x, "x", cols), _rows_of(y, "y", rows)
    T = x.shape[0]
    if y.shape[0] != T:
        raise ValueError("x and y must have a row a token")
    block = _WEIGHT_BLOCKS.get(qtype)
    if block and rows > 0 and cols > 0 and w.numel() * w.element_size() < rows * -(-cols // block[0]) * block[1]:
        raise ValueError("w holds fewer than rows x cols weights")
    if not w.is_contiguous():
        raise ValueError("w must be dense")
    bp = rp = None
    if bias is not None:
        if bias.dtype != torch.float32 or not bias.is_contiguous() or bias.numel() != rows:
            raise ValueError("bias must be float32 [rows]")
        bp = bias.data_ptr()
    if residual is not None:
        if residual.dtype != kind or residual.shape[0] != T or _rows_of(residual, "residual", rows) != ys:
            raise ValueError("residual must have y's type, shape and stride")
        rp = residual.data_ptr()
    st = _on(stream, (w, x, y, bias, residual))
    rc = lib.bread_matmul(w.data_ptr(), x.data_ptr(), y.data_ptr(), rows, cols, qtype, T,
                          ctypes.byref(_lib.MatmulOpts(bp, rp, a, y_type, xs, ys)), st)
    if rc:
        check(rc, "bread_matmul")


def bread_dequant_rows(w, qtype: int, rows: int, cols: int, out=None, stream=None) -> torch.Tensor:
    if out is None:
        empty = _empty(stream)
        out = empty(rows * cols, dtype=torch.float32, device=w.device)
    check(lib.bread_dequant_rows(_p(w), qtype, rows, cols, _p(out), _s(stream)), "bread_dequant_rows")
    return out


def bread_rmsnorm_f32(x, w, out, n: int, n_tokens: int, eps: float, stream=None) -> None:
    check(lib.bread_rmsnorm_f32(_p(x), _p(w), _p(out), n, n_tokens, eps, _s(stream)), "bread_rmsnorm_f32")


# ---------------------------------------------------------------- 8-bit floating point

_F8 = torch.float8_e4m3fn
_WIDE_TYPES = {torch.float16: _lib.QTYPE_F16, torch.bfloat16: _lib.QTYPE_BF16, torch.float32: _lib.QTYPE_F32}
# The argument structs as bytes, field by field (a ctypes structure takes longer to make than a small call runs)
_NORM_ARGS = struct.Struct("@PPPiqqqPfiiPqPqPiq")
_MATMUL_ARGS = struct.Struct("@PPPPPPqqPPqqiPPiiii")
_GROUP_ARGS = struct.Struct("@iPPiPi")


def _step(t: torch.Tensor, name: str, kind, n: int, cols: int) -> int:
    """Elements from one row of an [n][cols] tensor of a type to the next (rows themselves dense)."""
    if t.dtype != kind or t.shape != (n, cols):
        raise ValueError(f"{name} must be {kind} [{n}][{cols}], is {t.dtype} {list(t.shape)}")
    return cols if t.is_contiguous() else _rows_of(t, name, cols)


def _weights_of(w, scale, name: str, shape, scale_shape) -> None:
    """Dense codes and scales of matrices."""
    if w.dtype != _F8 or w.shape != shape or not w.is_contiguous():
        raise ValueError(f"{name} must be dense float8_e4m3fn {list(shape)}")
    if scale is None or scale.dtype != torch.float32 or scale.shape != scale_shape or not scale.is_contiguous():
        raise ValueError(f"{name}'s scales must be dense float32 {list(scale_shape)}")


def bread_rmsnorm_fp8(x, w, codes, scales, eps: float, residual=None, hidden=None, normed=None, stream=None) -> None:
    """bread_rmsnorm_fp8: h = x + residual and v = h / sqrt(mean(h^2) + eps) * w for the
    rows of x (float16, bfloat16 or float32 [n_tokens][n], n a multiple of 16);
    codes float8_e4m3fn [n_tokens][n] and scales float32 [n_tokens][ceil(n / 128)]
    receive v quantised, hidden (x's type; may be x or residual) h, normed
    (float16, bfloat16 or float32) v.  w: float32 [n] or None.  Rows may be strided."""
    kind = x.dtype
    x_type = _WIDE_TYPES.get(kind)
    if x_type is None or x.dim() != 2:
        raise ValueError("x must be float16, bfloat16 or float32 [n_tokens][n]")
    T, n = x.shape
    xs = n if x.is_contiguous() else _rows_of(x, "x", n)
    cs, ss = _step(codes, "codes", _F8, T, n), _step(scales, "scales", torch.float32, T, (n + 127) // 128)
    wp = rp = hp = op = rs = hs = os = out_type = 0
    if w is not None:
        if w.dtype != torch.float32 or w.shape != (n,) or not w.is_contiguous():
            raise ValueError("w must be float32 [n]")
        wp = w.data_ptr()
    if residual is not None:
        rs, rp = _step(residual, "residual", kind, T, n), residual.data_ptr()
    if hidden is not None:
        hs, hp = _step(hidden, "hidden", kind, T, n), hidden.data_ptr()
    if normed is not None:
        out_type = _WIDE_TYPES.get(normed.dtype)
        if out_type is None:
            raise ValueError("normed must be float16, bfloat16 or float32")
        os, op = _step(normed, "normed", normed.dtype, T, n), normed.data_ptr()
    st = _on(stream, (x, w, codes, scales, residual, hidden, normed))
    rc = lib.bread_rmsnorm_fp8(_NORM_ARGS.pack(x.data_ptr(), rp, hp, x_type, xs, rs, hs, wp, eps, n, T,
                                               codes.data_ptr(), cs, scales.data_ptr(), ss, op, out_type, os), st)
    if rc:
        check(rc, "bread_rmsnorm_fp8")


def _matmul_fp8_args(w, w_scale, x, x_scale, y, y_scale, up, up_scale, act, shape, n_x, n_y, T, bp, rp):
    """bread_matmul_fp8_t of checked tensors; shape: the weights'."""
    rows, cols = shape[-2:]
    nb, nr = (cols + 127) // 128, (rows + 127) // 128
    a = ACTS.get(act)
    if a is None:
        raise ValueError(f"unknown activation {act!r}")
    scale_shape = (*shape[:-2], nr, nb)
    _weights_of(w, w_scale, "w", shape, scale_shape)
    upp = usp = ysp = yss = 0
    if up is not None:
        _weights_of(up, up_scale, "up", shape, scale_shape)
        upp, usp = up.data_ptr(), up_scale.data_ptr()
    xs, ss = _step(x, "x", _F8, n_x, cols), _step(x_scale, "x_scale", torch.float32, n_x, nb)
    kind = y.dtype
    if kind == _F8:
        y_type = _lib.QTYPE_E4M3
        if y_scale is None:
            raise ValueError("quantised results need y_scale")
        yss, ysp = _step(y_scale, "y_scale", torch.float32, n_y, nr), y_scale.data_ptr()
    else:
        y_type = _WIDE_TYPES.get(kind)
        if y_type is None:
            raise ValueError("y must be float16, bfloat16, float32 or float8_e4m3fn")
        if y_scale is not None:
            raise ValueError("y_scale is for quantised results")
    ys = _step(y, "y", kind, n_y, rows)
    return _MATMUL_ARGS.pack(w.data_ptr(), w_scale.data_ptr(), upp, usp, x.data_ptr(), x_scale.data_ptr(), xs, ss,
                             y.data_ptr(), ysp, ys, yss, y_type, bp, rp, a, rows, cols, T)


def bread_matmul_fp8(w, w_scale, x, x_scale, y, y_scale=None, up=None, up_scale=None, bias=None, act=None,
                     residual=None, stream=None) -> None:
    """bread_matmul_fp8: y[t] = act(W x[t] + bias) + residual[t], or act(W x[t]) *
    (Up x[t]) + residual[t], for codes w, up float8_e4m3fn [rows][cols] with scales
    float32 [ceil(rows / 128)][ceil(cols / 128)] and x float8_e4m3fn
    [n_tokens][cols] with x_scale float32 [n_tokens][ceil(cols / 128)].  y
    [n_tokens][rows]: float16, bfloat16, float32, or float8_e4m3fn with y_scale
    float32 [n_tokens][ceil(rows / 128)].  residual (may be y) has y's type, bias
    is float32 [rows]; rows of x, y and the scales of tokens may be strided."""
    shape = w.shape
    if len(shape) != 2 or x.dim() != 2:
        raise ValueError("w and x must be 2-d")
    T = x.shape[0]
    bp = rp = 0
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != shape[:1] or not bias.is_contiguous():
            raise ValueError("bias must be float32 [rows]")
        bp = bias.data_ptr()
    if residual is not None:
        if (residual.dtype != y.dtype or residual.shape != y.shape
                or (residual.stride() != y.stride() if T > 1 else not residual.is_contiguous())):
            raise ValueError("residual must have y's type, shape and stride")
        rp = residual.data_ptr()
    a = _matmul_fp8_args(w, w_scale, x, x_scale, y, y_scale, up, up_scale, act, shape, T, T, T, bp, rp)
    rc = lib.bread_matmul_fp8(a, _on(stream, (w, w_scale, x, x_scale, y, y_scale, up, up_scale, bias, residual)))
    if rc:
        check(rc, "bread_matmul_fp8")


def _rows_index(t, name: str) -> int:
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be dense int32")
    return t.shape[0]


def bread_matmul_fp8_grouped(w, w_scale, x, x_scale, offsets, y, y_scale=None, up=None, up_scale=None, act=None,
                             x_rows=None, y_rows=None, stream=None) -> None:
    """bread_matmul_fp8_grouped: row i of offsets[g] <= i < offsets[g + 1] (int32
    [n_groups + 1]) is row x_rows[i] of x through matrix g of w [n_groups][rows][cols],
    written to row y_rows[i] of y (int32, None: i itself); scales and results as
    bread_matmul_fp8.  There are as many rows i as x_rows, y_rows or else x has."""
    shape = w.shape
    if len(shape) != 3 or x.dim() != 2 or y.dim() != 2:
        raise ValueError("w must be 3-d, x and y 2-d")
    G = shape[0]
    if _rows_index(offsets, "offsets") != G + 1:
        raise ValueError("offsets must hold n_groups + 1 values")
    T = n_x = x.shape[0]
    xrp = yrp = 0
    if x_rows is not None:
        T, xrp = _rows_index(x_rows, "x_rows"), x_rows.data_ptr()
    n_y = T
    if y_rows is not None:
        if _rows_index(y_rows, "y_rows") != T:
            raise ValueError("y_rows must name a row of y for every row")
        n_y, yrp = y.shape[0], y_rows.data_ptr()
    a = _matmul_fp8_args(w, w_scale, x, x_scale, y, y_scale, up, up_scale, act, shape, n_x, n_y, T, 0, 0)
    rc = lib.bread_matmul_fp8_grouped(
        a, _GROUP_ARGS.pack(G, offsets.data_ptr(), xrp, n_x, yrp, n_y),
        _on(stream, (w, w_scale, x, x_scale, offsets, y, y_scale, up, up_scale, x_rows, y_rows)))
    if rc:
        check(rc, "bread_matmul_fp8_grouped")


class Fp8Experts:
    """bread_fp8_experts_t: a layer's routed experts as float8_e4m3fn codes, gate and
    up [n_experts][inter][hidden], down [n_experts][hidden][inter], each with float32
    scales [n_experts][ceil(rows / 128)][ceil(cols / 128)].  Holds the tensors."""

    def __init__(self, gate, gate_scale, up, up_scale, down, down_scale):
        if gate.dim() != 3:
            raise ValueError("gate must be 3-d")
        E, I, H = gate.shape
        i, h = -(-I // 128), -(-H // 128)
        _weights_of(gate, gate_scale, "gate", (E, I, H), (E, i, h))
        _weights_of(up, up_scale, "up", (E, I, H), (E, i, h))
        _weights_of(down, down_scale, "down", (E, H, I), (E, h, i))
        self.shape = (E, I, H)
        self.tensors = (gate, up, down, gate_scale, up_scale, down_scale)
        self.desc = _lib.Fp8ExpertsDesc(*(t.data_ptr() for t in self.tensors))
        self.ref = ctypes.byref(self.desc)


# ---------------------------------------------------------------- synth


def synth_q4k(dst, n_blocks: int, seed: int, stream=None) -> None:
    check(lib.bread_synth_q4k(_p(dst), n_blocks, seed, _s(stream)), "bread_synth_q4k")


def synth_q6k(dst, n_blocks: int, seed: int, stream=None) -> None:
    check(lib.bread_synth_q6k(_p(dst), n_blocks, seed, _s(stream)), "bread_synth_q6k")


def synth_normal_f32(dst, n: int, seed: int, mean: float, std: float, stream=None) -> None:
    check(lib.bread_synth_normal_f32(_p(dst), n, seed, mean, std, _s(stream)), "bread_synth_normal_f32")


def synth_normal_f16(dst, n: int, seed: int, mean: float, std: float, stream=None) -> None:
    check(lib.bread_synth_normal_f16(_p(dst), n, seed, mean, std, _s(stream)), "bread_synth_normal_f16")


# ---------------------------------------------------------------- shape / layers


def shape(hidden=2048, expert_inter=512, shared_inter=512, n_experts=256, top_k=8, rms_eps=1e-6) -> MoeShape:
    return MoeShape(hidden, expert_inter, shared_inter, n_experts, top_k, rms_eps)


# Expert tensor types of a layer: gate, up, down, gate_shexp, up_shexp,
# down_shexp.  STANDARD_TYPES is the mix the reference GPU path hardcodes and
# the specialised kernels take; each entry may be Q4_K or Q6_K.
STANDARD_TYPES = (QTYPE_Q4_K, QTYPE_Q4_K, QTYPE_Q6_K, QTYPE_Q4_K, QTYPE_Q4_K, QTYPE_Q6_K)
BLOCK_BYTES = {QTYPE_Q4_K: 144, QTYPE_Q6_K: 210}
_WEIGHT_BLOCKS = {QTYPE_Q4_K: (256, 144), QTYPE_Q6_K: (256, 210), QTYPE_Q8_0: (32, 34), QTYPE_F16: (1, 2)}


def row_bytes(qtype: int, cols: int) -> int:
    """Bytes of one Q4_K or Q6_K row of cols columns."""
    return (cols // 256) * BLOCK_BYTES[qtype]


def layer_types(d: MoeLayer) -> tuple:
    return (d.gate_type, d.up_type, d.down_type, d.gate_shexp_type, d.up_shexp_type, d.down_shexp_type)


def shape_bytes(s: MoeShape, types=STANDARD_TYPES) -> dict:
    """Byte sizes of one layer's tensors (native GGUF layout)."""
    H, I, Ish, E = s.hidden, s.expert_inter, s.shared_inter, s.n_experts
    g, u, d, gs, us, ds = types
    return {
        "gate_expert": I * row_bytes(g, H),
        "up_expert": I * row_bytes(u, H),
        "down_expert": H * row_bytes(d, I),
        "gate_sh": Ish * row_bytes(gs, H),
        "up_sh": Ish * row_bytes(us, H),
        "down_sh": H * row_bytes(ds, Ish),
        "router": E * H * 4,
        "shgate": H * 2,
    }


def synth_quant(dst, qtype: int, nbytes: int, seed: int, stream=None) -> None:
    """Fill nbytes of Q4_K or Q6_K superblocks with the device generator."""
    fn = synth_q4k if qtype == QTYPE_Q4_K else synth_q6k
    fn(dst, nbytes // BLOCK_BYTES[qtype], seed, stream)


def route_noalloc(s: MoeShape, layer: MoeLayer, x: torch.Tensor, n_tokens: int, stream=None):
    """bread_route_noalloc: routing without a context (the library's static
    device workspace holds the logits; n_tokens * n_experts <= 1048576)."""
    K = s.top_k
    empty = _empty(stream)
    idx = empty((n_tokens, K), dtype=torch.int32, device=x.device)
    w = empty((n_tokens, K), dtype=torch.float32, device=x.device)
    gsh = empty((n_tokens,), dtype=torch.float32, device=x.device)
    check(lib.bread_route_noalloc(ctypes.byref(s), ctypes.byref(layer), _p(x), n_tokens, _p(idx), _p(w), _p(gsh),
                                  _s(stream)), "bread_route_noalloc")
    return idx, w, gsh


class RouteRule:
    """bread_route_rule_t: how experts are chosen from router logits (scores by
    "softmax" or "sigmoid", a bias float32 [n_experts] that only steers the
    choice, top_groups of n_groups groups by their group_top largest choices,
    weights renormalised and scaled).  Holds the bias tensor."""

    def __init__(self, score: str = "softmax", bias: torch.Tensor | None = None, n_groups: int = 1,
                 top_groups: int = 1, group_top: int = 1, renorm: bool = True, scale: float = 1.0):
        _need(score in ("softmax", "sigmoid"), f"unknown score {score!r}")
        _need(bias is None or (bias.dtype == torch.float32 and bias.dim() == 1 and bias.is_contiguous()),
              "bias must be float32 [n_experts]")
        self.bias = bias
        self.desc = _lib.RouteRuleDesc(
            None if bias is None else bias.data_ptr(),
            _lib.SCORE_SIGMOID if score == "sigmoid" else _lib.SCORE_SOFTMAX, n_groups, top_groups, group_top,
            int(renorm), scale)
        self.ref = ctypes.byref(self.desc)

    def check(self, n_experts: int) -> None:
        if self.bias is not None and self.bias.shape[0] != n_experts:
            raise ValueError("the rule's bias must have n_experts values")


def route_select(logits: torch.Tensor, top_k: int, rule: RouteRule, stream=None):
    """bread_route_select over the rows of a 2-d float32 device tensor (rows
    may be strided): (indices int32, weights float32), each [n_tokens][top_k]."""
    if logits.dtype != torch.float32 or logits.dim() != 2:
        raise ValueError("logits must be float32 [n_tokens][n_experts]")
    T, E = logits.shape
    rule.check(E)
    ls = _rows_of(logits, "logits", E)
    st = _on(stream, (logits, rule.bias))
    dev = logits.device
    empty = _empty(stream)
    idx = empty(T, top_k, dtype=torch.int32, device=dev)
    w = empty(T, top_k, dtype=torch.float32, device=dev)
    rc = lib.bread_route_select(rule.ref, logits.data_ptr(), ls, E, top_k, T, idx.data_ptr(), w.data_ptr(), st)
    if rc:
        check(rc, "bread_route_select")
    return idx, w


@dataclass
class LayerTensors:
    """One layer's weights as device tensors (keeps them alive)."""

    shape: MoeShape
    gate_exps: torch.Tensor
    up_exps: torch.Tensor
    down_exps: torch.Tensor
    gate_sh: torch.Tensor
    up_sh: torch.Tensor
    down_sh: torch.Tensor
    router: torch.Tensor
    shgate: torch.Tensor | None
    types: tuple = STANDARD_TYPES

    def desc(self) -> MoeLayer:
        b = shape_bytes(self.shape, self.types)
        g, u, d, gs, us, ds = self.types
        return MoeLayer(
            self.gate_exps.data_ptr(), self.up_exps.data_ptr(), self.down_exps.data_ptr(),
            b["gate_expert"], b["up_expert"], b["down_expert"],
            g, u, d,
            self.gate_sh.data_ptr(), self.up_sh.data_ptr(), self.down_sh.data_ptr(),
            gs, us, ds,
            self.router.data_ptr(),
            self.shgate.data_ptr() if self.shgate is not None else None,
            None,
        )


def layer_seeds(seed: int, layer: int) -> dict:
    base = (seed * 1_000_003 + layer * 101) & ((1 << 63) - 1)
    names = ["gate_exps", "up_exps", "down_exps", "gate_sh", "up_sh", "down_sh", "router", "shgate"]
    return {n: base + i for i, n in enumerate(names)}


def synth_layer_tensors(s: MoeShape, seed: int, layer: int = 0, router_std: float = 0.02,
                        shgate_std: float = 0.02, device="cuda", stream=None, types=STANDARD_TYPES) -> LayerTensors:
    """Allocate one layer with torch and fill it with the device generator
    (types: the six expert tensor types, each Q4_K or Q6_K)."""
    types = tuple(types)
    b = shape_bytes(s, types)
    E = s.n_experts
    sd = layer_seeds(seed, layer)
    u8 = dict(dtype=torch.uint8, device=device)
    t = LayerTensors(
        s,
        torch.empty(E * b["gate_expert"], **u8),
        torch.empty(E * b["up_expert"], **u8),
        torch.empty(E * b["down_expert"], **u8),
        torch.empty(b["gate_sh"], **u8),
        torch.empty(b["up_sh"], **u8),
        torch.empty(b["down_sh"], **u8),
        torch.empty(E * s.hidden, dtype=torch.float32, device=device),
        torch.empty(s.hidden, dtype=torch.float16, device=device),
        types,
    )
    g, u, d, gs, us, ds = types
    synth_quant(t.gate_exps, g, E * b["gate_expert"], sd["gate_exps"], stream)
    synth_quant(t.up_exps, u, E * b["up_expert"], sd["up_exps"], stream)
    synth_quant(t.down_exps, d, E * b["down_expert"], sd["down_exps"], stream)
    synth_quant(t.gate_sh, gs, b["gate_sh"], sd["gate_sh"], stream)
    synth_quant(t.up_sh, us, b["up_sh"], sd["up_sh"], stream)
    synth_quant(t.down_sh, ds, b["down_sh"], sd["down_sh"], stream)
    synth_normal_f32(t.router, E * s.hidden, sd["router"], 0.0, router_std, stream)
    synth_normal_f16(t.shgate, s.hidden, sd["shgate"], 0.0, shgate_std, stream)
    return t


def argmax_f16(logits: torch.Tensor, stream=None) -> torch.Tensor:
    """bread_argmax_f16 over the rows of a 2-d fp16 device tensor."""
    assert logits.dtype == torch.float16 and logits.dim() == 2 and logits.is_contiguous()
    empty = _empty(stream)
    out = empty((logits.shape[0],), dtype=torch.int32, device=logits.device)
    check(lib.bread_argmax_f16(_p(logits), logits.shape[1], logits.shape[0], _p(out), _s(stream)),
          "bread_argmax_f16")
    return out


def spec_accept(pred, draft, eos: int, max_accept: int):
    """bread_spec_accept on host lists: (n_accept, next token)."""
    pred = list(pred)
    draft = list(draft)
    assert len(pred) == len(draft) + 1
    pa = (ctypes.c_int32 * len(pred))(*pred)
    da = (ctypes.c_int32 * max(1, len(draft)))(*draft)
    na, nx = ctypes.c_int(), ctypes.c_int32()
    check(lib.bread_spec_accept(pa, da, len(draft), eos, max_accept, ctypes.byref(na), ctypes.byref(nx)),
          "bread_spec_accept")
    return na.value, nx.value


class Gguf:
    """A parsed GGUF v2/v3 file (bread_gguf_*): metadata and tensor index over
    a read-only mapping; weights are read when loaded into an Arena."""

    def __init__(self, path: str):
        self._h = ctypes.c_void_p()
        check(lib.bread_gguf_open(path.encode(), ctypes.byref(self._h)), "bread_gguf_open")

    def info(self) -> dict:
        v, a = ctypes.c_uint32(), ctypes.c_uint32()
        nt, nk, off = ctypes.c_uint64(), ctypes.c_uint64(), ctypes.c_uint64()
        check(lib.bread_gguf_info(self._h, ctypes.byref(v), ctypes.byref(nt), ctypes.byref(nk), ctypes.byref(off),
                                  ctypes.byref(a)), "bread_gguf_info")
        return {"version": v.value, "n_tensors": nt.value, "n_kv": nk.value, "data_offset": off.value,
                "alignment": a.value}

    @staticmethod
    def _t(t: _lib.GgufTensor) -> dict:
        return {"name": t.name.decode(), "type": t.type, "dims": list(t.dims[: t.n_dims]), "offset": t.offset,
                "size": t.size, "n_elems": t.n_elems, "data": t.data}

    def tensor(self, i: int) -> dict:
        t = _lib.GgufTensor()
        check(lib.bread_gguf_tensor(self._h, i, ctypes.byref(t)), "bread_gguf_tensor")
        return self._t(t)

    def tensors(self) -> list:
        return [self.tensor(i) for i in range(self.info()["n_tensors"])]

    def find(self, name: str):
        t = _lib.GgufTensor()
        return self._t(t) if lib.bread_gguf_find(self._h, name.encode(), ctypes.byref(t)) == 0 else None

    def kv_int(self, key: str):
        v = ctypes.c_int64()
        return v.value if lib.bread_gguf_kv_int(self._h, key.encode(), ctypes.byref(v)) == 0 else None

    def kv_float(self, key: str):
        v = ctypes.c_double()
        return v.value if lib.bread_gguf_kv_float(self._h, key.encode(), ctypes.byref(v)) == 0 else None

    def kv_str(self, key: str):
        b = ctypes.create_string_buffer(4096)
        return b.value.decode() if lib.bread_gguf_kv_str(self._h, key.encode(), b, 4096) == 0 else None

    def moe_shape(self, layer: int) -> MoeShape:
        sh = MoeShape()
        check(lib.bread_gguf_moe_shape(self._h, layer, ctypes.byref(sh)), "bread_gguf_moe_shape")
        return sh

    def close(self) -> None:
        if self._h:
            lib.bread_gguf_close(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Arena:
    """All experts of n_layers layers resident in HBM (bread_arena_*)."""

    def __init__(self, s: MoeShape, n_layers: int):
        self.shape = s
        self.n_layers = n_layers
        self._h = ctypes.c_void_p()
        check(lib.bread_arena_create(ctypes.byref(s), n_layers, ctypes.byref(self._h)), "bread_arena_create")

    @property
    def layer_bytes(self) -> int:
        return int(lib.bread_arena_layer_bytes(self._h))

    def layer(self, l: int) -> MoeLayer:
        d = MoeLayer()
        check(lib.bread_arena_layer(self._h, l, ctypes.byref(d)), "bread_arena_layer")
        return d

    def set_layer_types(self, l: int, types) -> None:
        """bread_arena_set_layer_types: the six expert tensor types of layer l
        (gate, up, down, gate_shexp, up_shexp, down_shexp; Q4_K or Q6_K)."""
        check(lib.bread_arena_set_layer_types(self._h, l, *[int(t) for t in types]), "bread_arena_set_layer_types")

    def synth_layer(self, l: int, seed: int, router_std=0.02, shgate_std=0.02, stream=None) -> None:
        d = self.layer(l)
        s = self.shape
        types = layer_types(d)
        b = shape_bytes(s, types)
        E = s.n_experts
        sd = layer_seeds(seed, l)
        st = _s(stream)

        def q(qtype, ptr, nbytes, sv):
            fn = lib.bread_synth_q4k if qtype == QTYPE_Q4_K else lib.bread_synth_q6k
            check(fn(ctypes.c_void_p(ptr), nbytes // BLOCK_BYTES[qtype], sv, st), fn.__name__)

        g, u, dn, gs, us, ds = types
        q(g, d.gate_exps, E * b["gate_expert"], sd["gate_exps"])
        q(u, d.up_exps, E * b["up_expert"], sd["up_exps"])
        q(dn, d.down_exps, E * b["down_expert"], sd["down_exps"])
        q(gs, d.gate_shexp, b["gate_sh"], sd["gate_sh"])
        q(us, d.up_shexp, b["up_sh"], sd["up_sh"])
        q(ds, d.down_shexp, b["down_sh"], sd["down_sh"])
        check(lib.bread_synth_normal_f32(ctypes.c_void_p(d.router), E * s.hidden, sd["router"], 0.0, router_std, st),
              "bread_synth_normal_f32")
        if d.shexp_gate:
            check(lib.bread_synth_normal_f16(ctypes.c_void_p(d.shexp_gate), s.hidden, sd["shgate"], 0.0, shgate_std,
                                             st), "bread_synth_normal_f16")

    def load_gguf(self, l: int, g: "Gguf", gguf_layer: int) -> None:
        """bread_arena_load_gguf: block gguf_layer's MoE tensors into layer l."""
        check(lib.bread_arena_load_gguf(self._h, l, g._h, gguf_layer), "bread_arena_load_gguf")

    def set_router_column(self, l: int, col: int, values) -> None:
        """Overwrite column col of layer l's fp32 router [E][H] with values[E]
        (e.g. a routing bias carried by a constant activation feature)."""
        d = self.layer(l)
        E, H = self.shape.n_experts, self.shape.hidden
        r = torch.empty(E * H, dtype=torch.float32, device=torch.device("cuda", torch.cuda.current_device()))
        device_copy(r.data_ptr(), d.router, E * H * 4)
        r.view(E, H)[:, col] = torch.as_tensor(values, dtype=torch.float32).to(r.device)
        device_copy(d.router, r.data_ptr(), E * H * 4)

    def close(self) -> None:
        if self._h:
            lib.bread_arena_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class MoeContext:
    """bread_moe_ctx_t: scratch for MoE calls on one stream."""

    def __init__(self, s: MoeShape, max_tokens: int = 1):
        self.shape = s
        self.max_tokens = max_tokens
        self._h = ctypes.c_void_p()
        check(lib.bread_moe_ctx_create(ctypes.byref(s), max_tokens, ctypes.byref(self._h)), "bread_moe_ctx_create")

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def set_path(self, path: int) -> None:
        """bread_moe_ctx_set_path: PATH_AUTO, PATH_DECODE, PATH_GROUPED, PATH_PER_TOKEN or PATH_SMALL."""
        check(lib.bread_moe_ctx_set_path(self._h, path), "bread_moe_ctx_set_path")

    def set_spin_limit(self, n_sleeps: int) -> None:
        """bread_moe_ctx_set_spin_limit: bound every wait of the decode and
        small-batch kernels at n_sleeps sleeps after the first look (< 0: the
        kernels' defaults).  A small bound forces the time-out error paths."""
        check(lib.bread_moe_ctx_set_spin_limit(self._h, n_sleeps), "bread_moe_ctx_set_spin_limit")

    def route(self, layer: MoeLayer, x: torch.Tensor, n_tokens: int, stream=None):
        K = self.shape.top_k
        empty = _empty(stream)
        idx = empty((n_tokens, K), dtype=torch.int32, device=x.device)
        w = empty((n_tokens, K), dtype=torch.float32, device=x.device)
        gsh = empty((n_tokens,), dtype=torch.float32, device=x.device)
        check(lib.bread_route(self._h, ctypes.byref(layer), _p(x), n_tokens, _p(idx), _p(w), _p(gsh), _s(stream)),
              "bread_route")
        return idx, w, gsh

    def route_layer(self, layer: MoeLayer, x: torch.Tensor, stream=None):
        """route_layer shim (one_layer.cu:937): host lists and the raw gate logit."""
        K = self.shape.top_k
        idx = (ctypes.c_int32 * K)()
        w = (ctypes.c_float * K)()
        g = ctypes.c_float()
        check(lib.bread_route_layer(self._h, ctypes.byref(layer), _p(x), idx, w, ctypes.byref(g), _s(stream)),
              "bread_route_layer")
        return list(idx), list(w), g.value

    def route_layer_f16(self, layer: MoeLayer, normed16: torch.Tensor, stream=None):
        """route_layer on the reference's own input (one_layer.cu:937-939):
        fp16 d_normed2 [H], widened on the device; host lists and the raw
        shared-gate logit."""
        assert normed16.dtype == torch.float16 and normed16.is_contiguous()
        K = self.shape.top_k
        idx = (ctypes.c_int32 * K)()
        w = (ctypes.c_float * K)()
        g = ctypes.c_float()
        check(lib.bread_route_layer_f16(self._h, ctypes.byref(layer), _p(normed16), idx, w, ctypes.byref(g),
                                        _s(stream)), "bread_route_layer_f16")
        return list(idx), list(w), g.value

    def forward(self, layer: MoeLayer, x: torch.Tensor, hidden: torch.Tensor, n_tokens: int,
                want_routing: bool = False, stream=None):
        K = self.shape.top_k
        idx = w = gsh = None
        if want_routing:
            empty = _empty(stream)
            idx = empty((n_tokens, K), dtype=torch.int32, device=x.device)
            w = empty((n_tokens, K), dtype=torch.float32, device=x.device)
            gsh = empty((n_tokens,), dtype=torch.float32, device=x.device)
        check(lib.bread_moe_forward(self._h, ctypes.byref(layer), _p(x), _p(hidden), n_tokens, _p(idx), _p(w),
                                    _p(gsh), _s(stream)), "bread_moe_forward")
        return idx, w, gsh

    def _check_rows(self, name: str, t: torch.Tensor, n_tokens: int) -> None:
        if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < n_tokens * self.shape.hidden:
            raise ValueError(f"{name} must be dense float32 with n_tokens rows of the context's hidden size")

    def route_by_rule(self, layer: MoeLayer, rule: RouteRule, x: torch.Tensor, n_tokens: int, stream=None):
        """bread_route_by_rule: route() with the experts and weights of a rule."""
        K = self.shape.top_k
        rule.check(self.shape.n_experts)
        self._check_rows("x", x, n_tokens)
        st = _on(stream, (x, rule.bias))
        empty = _empty(stream)
        idx = empty((n_tokens, K), dtype=torch.int32, device=x.device)
        w = empty((n_tokens, K), dtype=torch.float32, device=x.device)
        gsh = empty((n_tokens,), dtype=torch.float32, device=x.device)
        check(lib.bread_route_by_rule(self._h, ctypes.byref(layer), rule.ref, _p(x), n_tokens, _p(idx),
                                      _p(w), _p(gsh), st), "bread_route_by_rule")
        return idx, w, gsh

    def forward_by_rule(self, layer: MoeLayer, rule: RouteRule, x: torch.Tensor, hidden: torch.Tensor, n_tokens: int,
                        want_routing: bool = False, stream=None):
        """bread_moe_forward_by_rule: forward() with the experts and weights of a rule."""
        K = self.shape.top_k
        rule.check(self.shape.n_experts)
        self._check_rows("x", x, n_tokens)
        self._check_rows("hidden", hidden, n_tokens)
        st = _on(stream, (x, hidden, rule.bias))
        idx = w = gsh = None
        if want_routing:
            empty = _empty(stream)
            idx = empty((n_tokens, K), dtype=torch.int32, device=x.device)
            w = empty((n_tokens, K), dtype=torch.float32, device=x.device)
            gsh = empty((n_tokens,), dtype=torch.float32, device=x.device)
        check(lib.bread_moe_forward_by_rule(self._h, ctypes.byref(layer), rule.ref, _p(x), _p(hidden),
                                            n_tokens, _p(idx), _p(w), _p(gsh), st), "bread_moe_forward_by_rule")
        return idx, w, gsh

    def spec_verify(self, logits: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor, u: torch.Tensor,
                    draft_probs: torch.Tensor | None = None, temperature: torch.Tensor | None = None, eos: int = -1,
                    want_logprob: bool = True, stream=None):
        """bread_spec_verify: (accepted drafts int32 [n_requests], next tokens int32
        [n_requests], log-probabilities float32 [n_rows] or None).  logits
        [n_rows][vocab] float16 or float32, tokens int32 and u float32 [n_rows],
        offsets int32 [n_requests + 1], draft_probs float32
        [n_rows - n_requests][vocab] or None, temperature float32 [n_requests]."""
        z_type = _Y_TYPES.get(logits.dtype)
        if z_type is None or logits.dim() != 2:
            raise ValueError("logits must be float16 or float32 [n_rows][vocab]")
        R, V = logits.shape
        B = offsets.shape[0] - 1
        for t, name, kind, n in ((tokens, "tokens", torch.int32, R), (offsets, "offsets", torch.int32, B + 1),
                                 (u, "u", torch.float32, R)):
            if t.dtype != kind or t.shape != (n,) or n > 1 and t.stride(0) != 1:
                raise ValueError(f"{name} must be dense {kind} [{n}]")
        if B < 0:
            raise ValueError("offsets must hold n_requests + 1 values")
        qp = tp = lp = None
        qs = 0
        if draft_probs is not None and R > B:
            if draft_probs.dtype != torch.float32 or draft_probs.shape != (R - B, V):
                raise ValueError("draft_probs must be float32 [n_rows - n_requests][vocab]")
            qp, qs = draft_probs.data_ptr(), _rows_of(draft_probs, "draft_probs", V)
        if temperature is not None:
            if temperature.dtype != torch.float32 or temperature.shape != (B,) or B > 1 and temperature.stride(0) != 1:
                raise ValueError("temperature must be dense float32 [n_requests]")
            tp = temperature.data_ptr()
        st = _on(stream, (logits, tokens, offsets, u, draft_probs, temperature))
        empty = _empty(stream)
        accepted = empty((B,), dtype=torch.int32, device=logits.device)
        following = empty((B,), dtype=torch.int32, device=logits.device)
        logp = None
        if want_logprob:
            logp = empty((R,), dtype=torch.float32, device=logits.device)
            lp = logp.data_ptr()
        a = _lib.VerifyArgs(logits.data_ptr(), _rows_of(logits, "logits", V), z_type, V, R, B, tokens.data_ptr(),
                            offsets.data_ptr(), u.data_ptr(), qp, qs, tp, eos, accepted.data_ptr(),
                            following.data_ptr(), lp)
        rc = lib.bread_spec_verify(self._h, ctypes.byref(a), st)
        if rc:
            check(rc, "bread_spec_verify")
        return accepted, following, logp

    def expert_block(self, layer: MoeLayer, x: torch.Tensor, hidden: torch.Tensor, n_tokens: int,
                     idx: torch.Tensor, w: torch.Tensor, stream=None) -> None:
        """bread_moe_expert_block: hidden += sum_k w[t][k] * expert_{idx[t][k]}(x_t),
        routed experts only, with the caller's routing (device int32 / fp32 [n_tokens][K])."""
        assert idx.dtype == torch.int32 and w.dtype == torch.float32
        check(lib.bread_moe_expert_block(self._h, ctypes.byref(layer), _p(x), _p(hidden), n_tokens, _p(idx),
                                         _p(w), _s(stream)), "bread_moe_expert_block")

    def expert_block_fp8(self, experts: Fp8Experts, x: torch.Tensor, x_scale: torch.Tensor, hidden: torch.Tensor,
                         idx: torch.Tensor, w: torch.Tensor, residual: torch.Tensor | None = None,
                         stream=None) -> None:
        """bread_moe_expert_block_fp8: hidden = residual + sum_k w[t][k] * expert_{idx[t][k]}(x_t)
        with 8-bit experts and the caller's routing (residual None: hidden itself, which the sum
        is added to).  x float8_e4m3fn [n_tokens][H], x_scale float32 [n_tokens][H / 128], hidden and
        residual float16, bfloat16 or float32 [n_tokens][H], idx int32 and w float32
        [n_tokens][K], all dense."""
        s = self.shape
        if experts.shape != (s.n_experts, s.expert_inter, s.hidden):
            raise ValueError("the experts are of another shape than the context")
        T, H, K = x.shape[0], s.hidden, s.top_k
        h_type = _WIDE_TYPES.get(hidden.dtype)
        if h_type is None:
            raise ValueError("hidden must be float16, bfloat16 or float32")
        if residual is None:
            residual = hidden
        for t, name, kind, cols in ((x, "x", _F8, H), (x_scale, "x_scale", torch.float32, -(-H // 128)),
                                    (hidden, "hidden", hidden.dtype, H), (residual, "residual", hidden.dtype, H),
                                    (idx, "idx", torch.int32, K), (w, "w", torch.float32, K)):
            if t.dtype != kind or t.shape != (T, cols) or not t.is_contiguous():
                raise ValueError(f"{name} must be dense {kind} [{T}][{cols}]")
        st = _on(stream, (x, x_scale, hidden, residual, idx, w, *experts.tensors))
        rc = lib.bread_moe_expert_block_fp8(self._h, experts.ref, x.data_ptr(), x_scale.data_ptr(),
                                            residual.data_ptr(), hidden.data_ptr(), h_type, T, idx.data_ptr(),
                                            w.data_ptr(), st)
        if rc:
            check(rc, "bread_moe_expert_block_fp8")

    def forward_f16(self, layer: MoeLayer, hidden: torch.Tensor, normed: torch.Tensor, n_tokens: int,
                    norm_w=None, want_routing: bool = False, stream=None):
        """bread_moe_forward_f16: the MoE block on fp16 hidden / normed
        [n_tokens][H] (one_layer.cu:1800-1986).  norm_w: a float32 device
        tensor or raw device pointer (e.g. layer.post_norm_w); None takes
        `normed` as the input instead of computing it."""
        assert hidden.dtype == torch.float16 and normed.dtype == torch.float16
        K = self.shape.top_k
        idx = w = gsh = None
        if want_routing:
            empty = _empty(stream)
            idx = empty((n_tokens, K), dtype=torch.int32, device=hidden.device)
            w = empty((n_tokens, K), dtype=torch.float32, device=hidden.device)
            gsh = empty((n_tokens,), dtype=torch.float32, device=hidden.device)
        nw = norm_w if isinstance(norm_w, int) or norm_w is None else norm_w.data_ptr()
        check(lib.bread_moe_forward_f16(self._h, ctypes.byref(layer), nw, _p(hidden), _p(normed), n_tokens, _p(idx),
                                        _p(w), _p(gsh), _s(stream)), "bread_moe_forward_f16")
        return idx, w, gsh

    def decode_layers(self, layers, hidden: torch.Tensor, want_routing: bool = False, stream=None):
        """bread_moe_decode_layers: one token through len(layers) layers,
        h <- h + MoE_l(RMSNorm(h) * w_l), in one launch."""
        n = len(layers)
        arr = (MoeLayer * n)(*layers)
        K = self.shape.top_k
        idx = w = gsh = None
        if want_routing:
            empty = _empty(stream)
            idx = empty((n, K), dtype=torch.int32, device=hidden.device)
            w = empty((n, K), dtype=torch.float32, device=hidden.device)
            gsh = empty((n,), dtype=torch.float32, device=hidden.device)
        check(lib.bread_moe_decode_layers(self._h, arr, n, _p(hidden), _p(idx), _p(w), _p(gsh), _s(stream)),
              "bread_moe_decode_layers")
        return idx, w, gsh

    def decode_launcher(self, layers, hidden: torch.Tensor, stream=None):
        """A callable f(i) that runs bread_moe_decode_layers on the single
        layer layers[i % len(layers)] with every ctypes argument built once:
        a launch costs one foreign call (for loops that time the kernel)."""
        arrs = [(MoeLayer * 1)(l) for l in layers]
        n = len(arrs)
        fn = lib.bread_moe_decode_layers
        h, hp, sp = self._h, _p(hidden), _s(stream)

        def launch(i: int) -> None:
            rc = fn(h, arrs[i % n], 1, hp, None, None, None, sp)
            if rc:
                check(rc, "bread_moe_decode_layers")

        return launch

    def stack_forward(self, layers, hidden: torch.Tensor, n_tokens: int, want_routing: bool = False, stream=None):
        """bread_moe_stack_forward: n_tokens tokens through len(layers) MoE
        layers, h <- h + MoE_l(RMSNorm(h) * w_l): one batched call per layer,
        or one decode-stack launch per token for up to
        bread_stack_loop_tokens() tokens (automatic choice)."""
        n = len(layers)
        arr = (MoeLayer * n)(*layers)
        K = self.shape.top_k
        idx = w = gsh = None
        if want_routing:
            empty = _empty(stream)
            idx = empty((n, n_tokens, K), dtype=torch.int32, device=hidden.device)
            w = empty((n, n_tokens, K), dtype=torch.float32, device=hidden.device)
            gsh = empty((n, n_tokens), dtype=torch.float32, device=hidden.device)
        check(lib.bread_moe_stack_forward(self._h, arr, n, _p(hidden), n_tokens, _p(idx), _p(w), _p(gsh),
                                          _s(stream)), "bread_moe_stack_forward")
        return idx, w, gsh

    def greedy_head(self, hidden: torch.Tensor, norm_w: torch.Tensor | None, w_out: torch.Tensor, qtype: int,
                    vocab: int, n_tokens: int, stream=None):
        """bread_moe_greedy_head: (tokens int32 [n_tokens], fp16 logits
        [n_tokens][vocab]) of the output norm + lm_head + greedy argmax."""
        empty = _empty(stream)
        logits = empty((n_tokens, vocab), dtype=torch.float16, device=hidden.device)
        tokens = empty((n_tokens,), dtype=torch.int32, device=hidden.device)
        check(lib.bread_moe_greedy_head(self._h, _p(hidden), _p(norm_w), _p(w_out), qtype, vocab, n_tokens,
                                        _p(logits), _p(tokens), _s(stream)), "bread_moe_greedy_head")
        return tokens, logits

    def set_trace(self, buf: torch.Tensor | None) -> int:
        """Record the decode kernel's timeline into buf (int64 device tensor)."""
        g = ctypes.c_int(0)
        n = 0 if buf is None else buf.numel()
        check(lib.bread_moe_ctx_set_trace(self._h, _p(buf), n, ctypes.byref(g)), "bread_moe_ctx_set_trace")
        self._trace = buf
        return g.value

    ROUTE_STAT_NAMES = ("decode_radius", "decode_per_expert", "decode_pair", "decode_exact",
                        "multi_certified", "multi_candidates", "multi_exact")

    def route_stats(self, reset: bool = False) -> dict:
        """bread_moe_ctx_route_stats: how often exact routing took each path
        (decode layers by certificate outcome, multi-token tokens certified
        or recomputed), since creation or the last reset."""
        n = len(self.ROUTE_STAT_NAMES)
        out = (ctypes.c_uint64 * n)()
        check(lib.bread_moe_ctx_route_stats(self._h, out, n, 1 if reset else 0), "bread_moe_ctx_route_stats")
        return dict(zip(self.ROUTE_STAT_NAMES, (int(v) for v in out)))

    def check_device(self) -> int:
        """bread_moe_ctx_check: 0, or BreadError carrying the kernels' error
        word in .device_error (the call clears it and resets the context)."""
        e = ctypes.c_int(0)
        rc = lib.bread_moe_ctx_check(self._h, ctypes.byref(e))
        if rc != _lib.OK:
            raise BreadError(int(rc), "bread_moe_ctx_check", e.value)
        return e.value

    def close(self) -> None:
        if self._h:
            lib.bread_moe_ctx_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
