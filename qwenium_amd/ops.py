"""The 8-bit float feed-forward's operators over libqmoe's C ABI (include/qmoe.h).

For expert weights that come as e4m3 (torch.float8_e4m3fn) with one f32 scale per
block of 128 x 128; the layers of moe.py take GGUF Q4_0/Q8_0.  One block is

    n = residual_norm(x, y, w, eps, quantize=True)          # x', its norm, the norm in e4m3
    idx, weights = ...                                       # the router on n.h
    o = sort_tokens(idx, n_experts)
    gu = fp8_matmul(n.q, n.q_scale, w_gate_up, s_gate_up, offsets=o.offsets, rows=o.tokens)
    h, hs = fp8_quantize(gu, act="swiglu")
    ys = fp8_matmul(h, hs, w_down, s_down, offsets=o.offsets)
    y = combine_tokens(ys, o, weights)                       # the next block's y

Rows are torch.float32 or torch.bfloat16.  As with moe.py, work goes to the given
stream or the current stream of the operands' device, outputs are allocated on it,
strided rows are copied first, and wrong arguments raise ValueError, or QmoeError where
the C ABI refuses them (sizes, overlapping buffers), before a launch.
The calls stand outside autograd: none records a gradient (gather_tokens_backward and
combine_tokens_backward are called by the training program), and an operand that requires
grad is refused unless gradients are off (torch.no_grad()).
"""
from __future__ import annotations

import contextlib
import ctypes
import dataclasses
from typing import Optional, Union

import torch

from ._lib import TYPE_BF16, TYPE_F32, QmoeNormArgs, check, lib
from .moe import _describe

FP8 = torch.float8_e4m3fn
BLOCK = 128  # columns of one scale
_TYPES = {torch.float32: TYPE_F32, torch.bfloat16: TYPE_BF16}
_ACTS = {None: 0, "swiglu": 1, "geglu": 2}
_GATES = {None: 0, "sigmoid": 1, "silu": 2}


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _want(name: str, what: str, got) -> ValueError:
    return ValueError(f"{name} expected {what}, got {_describe(got)}")


def _no_grad(name: str) -> None:
    if torch.is_grad_enabled():
        raise ValueError(f"{name} expected a tensor outside autograd (detach() it, or call within torch.no_grad()), "
                         "got one that requires grad")


def _rows(name: str, t, device=None, shape=None, dtype=None) -> torch.Tensor:
    """A read-only cuda [R, C] operand, made contiguous."""
    if getattr(t, "requires_grad", False):
        _no_grad(name)
    if (not isinstance(t, torch.Tensor) or t.dim() != 2 or not t.is_cuda
            or (t.dtype not in _TYPES if dtype is None else t.dtype != dtype)
            or (device is not None and t.device != device) or (shape is not None and t.shape != shape)):
        kind = "float32 or bfloat16" if dtype is None else str(dtype).replace("torch.", "")
        size = "[rows, columns]" if shape is None else list(shape)
        raise _want(name, f"a cuda {kind} {size} tensor" + (f" on {device}" if device is not None else ""), t)
    return t if t.is_contiguous() else t.contiguous()


def _kept(name: str, t, device, shape, dtype) -> torch.Tensor:
    """An operand or output that is used in place: contiguous as it is."""
    if getattr(t, "requires_grad", False):
        _no_grad(name)
    if (not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape or t.device != device
            or not t.is_contiguous()):
        raise _want(name, f"a contiguous {str(dtype).replace('torch.', '')} {list(shape)} tensor on {device}", t)
    return t


def _out(name: str, t, device, shape, dtype) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=device) if t is None else _kept(name, t, device, shape, dtype)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# torch.cuda.current_stream(i).cuda_stream without the Stream object around it (1.9 us of a 5 us call), and the
# current device, by torch's own bindings where they are
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device

_NO_STREAM = contextlib.nullcontext()


def _on(stream):
    return _NO_STREAM if stream is None else torch.cuda.stream(stream)


def _launch(fn, device, stream, *args) -> None:
    """Calls fn(*args, stream) with the operands' device current."""
    index = device.index
    if stream is None:
        handle = _raw_stream(index)
    elif stream.device != device:
        raise ValueError(f"stream expected one of {device}, got one of {stream.device}")
    else:
        handle = stream.cuda_stream
    if index == _current_device():
        rc = fn(*args, handle)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, handle)
    if rc:
        check(rc)


def fp8_quantize(x: torch.Tensor, act: Optional[str] = None, *, q: Optional[torch.Tensor] = None,
                 scale: Optional[torch.Tensor] = None, stream=None):
    """(q, scale): the rows of x [R, C] in e4m3, with one f32 scale per block of 128
    columns (scale = max|v| / 448; q * scale stands for v).  act "swiglu" or "geglu":
    of the activation of x [R, 2C]'s halves (gate columns first) instead.
    q [R, C] and scale [R, ceil(C/128)] may be given."""
    with _on(stream):
        if act not in _ACTS:
            raise ValueError(f"act expected None, \"swiglu\" or \"geglu\", got {act!r}")
        x = _rows("x", x)
        R, C = x.shape
        if act is not None:
            if C % 2:
                raise _want("x", "an even number of columns (gate and up halves)", x)
            C //= 2
        if C < 1:
            raise _want("x", "at least one column", x)
        q = _out("q", q, x.device, (R, C), FP8)
        scale = _out("scale", scale, x.device, (R, _blocks(C)), torch.float32)
        _launch(lib().qmoe_fp8_quantize, x.device, stream, x.data_ptr(), _TYPES[x.dtype], R, C, _ACTS[act],
                q.data_ptr(), scale.data_ptr())
    return q, scale


def fp8_matmul(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, *,
               offsets: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32, stream=None) -> torch.Tensor:
    """y = (a * a_scale) @ (w * w_scale)^T with e4m3 operands and f32 sums, k a multiple of 16.

    a [A, k], a_scale [A, ceil(k/128)] (fp8_quantize's); w [n, k], w_scale
    [ceil(n/128), ceil(k/128)].  Grouped: w [E, n, k], w_scale [E, ...] and offsets
    (int32 [E+1], a TokenOrder's): row r is multiplied by expert e's matrix for
    offsets[e] <= r < offsets[e+1]; rows of no expert are left as they were (in a new
    result: uninitialised).
    rows (int32 [R], a TokenOrder's tokens): row r is a[rows[r]]; an index outside a
    gives zeros.  out [R, n] may be given, float32 or bfloat16; else out_dtype is its type."""
    with _on(stream):
        a = _rows("a", a, dtype=FP8)
        dev = a.device
        A, k = a.shape
        if k % 16 or k < 16:
            raise _want("a", "a multiple of 16 columns", a)
        kb = _blocks(k)
        a_scale = _rows("a_scale", a_scale, dev, (A, kb), torch.float32)
        grouped = offsets is not None
        if not isinstance(w, torch.Tensor) or w.dim() != (3 if grouped else 2) or w.shape[-1] != k:
            raise _want("w", f"[experts, n, {k}] with offsets" if grouped else f"[n, {k}] without offsets", w)
        E, n = (w.shape[0] if grouped else 1), w.shape[-2]
        lead = (E,) if grouped else ()
        _kept("w", w, dev, lead + (n, k), FP8)
        _kept("w_scale", w_scale, dev, lead + (_blocks(n), kb), torch.float32)
        if grouped:
            _kept("offsets", offsets, dev, (E + 1,), torch.int32)
        R = A
        if rows is not None:
            if not isinstance(rows, torch.Tensor) or rows.dim() != 1:
                raise _want("rows", "an int32 [R] tensor", rows)
            R = rows.shape[0]
            _kept("rows", rows, dev, (R,), torch.int32)
        if out is not None:
            out_dtype = out.dtype
        if out_dtype not in _TYPES:
            raise ValueError(f"out_dtype expected torch.float32 or torch.bfloat16, got {out_dtype}")
        out = _out("out", out, dev, (R, n), out_dtype)
        _launch(lib().qmoe_fp8_matmul, dev, stream, a.data_ptr(), a_scale.data_ptr(), A, w.data_ptr(),
                w_scale.data_ptr(), E, n, k, _ptr(offsets), _ptr(rows), R, out.data_ptr(), _TYPES[out_dtype])
    return out


class TokenOrder:
    """The lists of a routing topk_idx [T, k] (assignment a = t * k + j), int32:
    offsets [E+1] each expert's first row and the number of rows; rows [T*k] the
    assignments grouped by expert, ascending within one; tokens [T*k] their tokens;
    place [T, k] each assignment's index in rows.  Dropped assignments (ids outside
    [0, E)) have place -1; rows and tokens are -1 from offsets[E] on.  Read-only:
    the tensors are checked once, here."""
    __slots__ = ("_offsets", "_rows", "_tokens", "_place", "_dims")

    def __init__(self, offsets: torch.Tensor, rows: torch.Tensor, tokens: torch.Tensor, place: torch.Tensor):
        if not isinstance(place, torch.Tensor) or place.dim() != 2:
            raise _want("place", "an int32 [T, k] tensor", place)
        if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 2:
            raise _want("offsets", "an int32 [n_experts + 1] tensor", offsets)
        T, k = place.shape
        _kept("place", place, place.device, (T, k), torch.int32)
        _kept("offsets", offsets, place.device, tuple(offsets.shape), torch.int32)
        _kept("rows", rows, place.device, (T * k,), torch.int32)
        _kept("tokens", tokens, place.device, (T * k,), torch.int32)
        self._set(offsets, rows, tokens, place)

    def _set(self, offsets, rows, tokens, place):
        self._offsets, self._rows, self._tokens, self._place = offsets, rows, tokens, place
        self._dims = (*place.shape, offsets.shape[0] - 1)
        return self

    offsets = property(lambda self: self._offsets)
    rows = property(lambda self: self._rows)
    tokens = property(lambda self: self._tokens)
    place = property(lambda self: self._place)
    n_experts = property(lambda self: self._dims[2])


def sort_tokens(topk_idx: torch.Tensor, n_experts: int, *, stream=None) -> TokenOrder:
    """The experts' lists of topk_idx (int32 [T, k]); ids outside [0, n_experts) are dropped."""
    with _on(stream):
        idx = _rows("topk_idx", topk_idx, dtype=torch.int32)
        T, k = idx.shape
        n_experts = int(n_experts)
        if n_experts < 1:
            raise ValueError(f"n_experts expected at least 1, got {n_experts}")
        A = T * k
        place, rows, tokens, offsets = torch.empty(3 * A + n_experts + 1, dtype=torch.int32, device=idx.device).split(
            (A, A, A, n_experts + 1))  # one allocation
        place = place.view(T, k)
        _launch(lib().qmoe_sort_tokens, idx.device, stream, idx.data_ptr(), T, k, n_experts, offsets.data_ptr(),
                rows.data_ptr(), tokens.data_ptr(), place.data_ptr())
    return object.__new__(TokenOrder)._set(offsets, rows, tokens, place)


def _order(order: TokenOrder, device) -> tuple:
    """(T, k, E) of an order on `device`."""
    if not isinstance(order, TokenOrder) or order._place.device != device:
        raise _want("order", f"a TokenOrder on {device}", order._place if isinstance(order, TokenOrder) else order)
    return order._dims


def gather_tokens(x: torch.Tensor, order: TokenOrder, *, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """The rows of x [T, C] in the experts' order, [T*k, C]; rows from offsets[E] on are
    zeros.  x may also be e4m3 rows or their scales."""
    with _on(stream):
        x = _rows("x", x, dtype=x.dtype if isinstance(x, torch.Tensor) and x.dtype == FP8 else None)
        T, k, E = _order(order, x.device)
        if x.shape[0] != T:
            raise _want("x", f"[{T}, columns]", x)
        C = x.shape[1]
        out = _out("out", out, x.device, (T * k, C), x.dtype)
        _launch(lib().qmoe_gather_tokens, x.device, stream, x.data_ptr(), x.element_size(), T, C, k, E,
                order.offsets.data_ptr(), order.place.data_ptr(), out.data_ptr())
    return out


def _combine(ys, order, weights, residual, out, stream) -> torch.Tensor:
    with _on(stream):
        ys = _rows("ys", ys)
        T, k, _ = _order(order, ys.device)
        if ys.shape[0] != T * k:
            raise _want("ys", f"[{T * k}, columns]", ys)
        C = ys.shape[1]
        if weights is not None:
            weights = _rows("weights", weights, ys.device, (T, k), torch.float32)
        if residual is not None:
            residual = _rows("residual", residual, ys.device, (T, C), ys.dtype)
        out = _out("out", out, ys.device, (T, C), ys.dtype)
        _launch(lib().qmoe_combine_tokens, ys.device, stream, ys.data_ptr(), _TYPES[ys.dtype], T, C, k,
                order.place.data_ptr(), _ptr(weights), _ptr(residual), out.data_ptr())
    return out


def combine_tokens(ys: torch.Tensor, order: TokenOrder, weights: torch.Tensor, *, residual: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """y[t] = residual[t] + sum_j weights[t, j] ys[place[t, j]]: the experts' rows
    ys [T*k, C] back to tokens [T, C], j in order in f32, rounded once.  weights
    float32 [T, k]; dropped assignments add nothing; out may be residual."""
    if weights is None:
        raise ValueError("weights expected a float32 [T, k] tensor, got None")
    return _combine(ys, order, weights, residual, out, stream)


def gather_tokens_backward(dxs: torch.Tensor, order: TokenOrder, *, out: Optional[torch.Tensor] = None,
                           stream=None) -> torch.Tensor:
    """gather_tokens' gradient: dx[t] = sum_j dxs[place[t, j]]."""
    return _combine(dxs, order, None, None, out, stream)


def combine_tokens_backward(dy: torch.Tensor, ys: torch.Tensor, order: TokenOrder, weights: torch.Tensor, *,
                            stream=None):
    """combine_tokens' gradients (dys [T*k, C], dweights float32 [T, k]); the residual's
    is dy.  dys[place[t, j]] = weights[t, j] dy[t], dweights[t, j] = <dy[t], ys[place[t, j]]>;
    a dropped assignment's dweight is 0, dys rows from offsets[E] on are zeros."""
    with _on(stream):
        ys = _rows("ys", ys)
        T, k, E = _order(order, ys.device)
        C = ys.shape[1]
        if ys.shape[0] != T * k:
            raise _want("ys", f"[{T * k}, columns]", ys)
        dy = _rows("dy", dy, ys.device, (T, C), ys.dtype)
        weights = _rows("weights", weights, ys.device, (T, k), torch.float32)
        dys = torch.empty((T * k, C), dtype=ys.dtype, device=ys.device)
        dw = torch.empty((T, k), dtype=torch.float32, device=ys.device)
        _launch(lib().qmoe_combine_tokens_backward, ys.device, stream, dy.data_ptr(), ys.data_ptr(), _TYPES[ys.dtype],
                T, C, k, E, order.offsets.data_ptr(), order.place.data_ptr(), weights.data_ptr(), dys.data_ptr(),
                dw.data_ptr())
    return dys, dw


@dataclasses.dataclass
class NormOut:
    """residual_norm's rows: x (the residual rows), h (their norm), and with quantize
    q (h in e4m3) and q_scale."""
    x: torch.Tensor
    h: torch.Tensor
    q: Optional[torch.Tensor] = None
    q_scale: Optional[torch.Tensor] = None


def residual_norm(x: torch.Tensor, y: Optional[torch.Tensor], w: Optional[torch.Tensor], eps: float, *,
                  post_w: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  gate_act: Optional[str] = None, scale: Union[float, torch.Tensor] = 1.0, quantize: bool = False,
                  out: Optional[torch.Tensor] = None, stream=None) -> NormOut:
    """The norms between two blocks in one pass over [T, H] rows (H <= 16384):

        u  = y / sqrt(mean(y^2) + eps) * post_w     (post_w: the norm after the block)
        u  = u * sigmoid(gate) or u * silu(gate)    (gate [T, H], gate_act)
        x' = x + scale * u                          (scale: a number or float32 [H])
        h  = x' / sqrt(mean(x'^2) + eps) * w        (w None: not scaled)

    and with quantize fp8_quantize of h.  y None: x' = x.  h is made of the f32 x'
    before its rounding to x's type.  out receives x' and may be x or y."""
    with _on(stream):
        x = _rows("x", x)
        T, H = x.shape
        dev, dt = x.device, x.dtype
        if not 1 <= H <= 16384:
            raise _want("x", "1 to 16384 columns", x)
        if gate_act not in _GATES or (gate is None) != (gate_act is None):
            raise ValueError(f"gate_act expected \"sigmoid\" or \"silu\" with a gate and None without, got {gate_act!r}")
        vector = isinstance(scale, torch.Tensor)
        if y is None and (post_w is not None or gate is not None or vector or scale != 1.0 or out is not None):
            raise ValueError("y expected the block's output with post_w, gate, scale or out, got None")
        if y is not None:
            y = _rows("y", y, dev, x.shape, dt)
        if gate is not None:
            gate = _rows("gate", gate, dev, x.shape, dt)
        for name, v in (("w", w), ("post_w", post_w), ("scale", scale if vector else None)):
            if v is not None:
                _kept(name, v, dev, (H,), torch.float32)
        x_out = x if y is None else torch.empty_like(x) if out is None else _kept("out", out, dev, (T, H), dt)
        h = torch.empty_like(x)
        q = q_scale = None
        if quantize:
            q = torch.empty((T, H), dtype=FP8, device=dev)
            q_scale = torch.empty((T, _blocks(H)), dtype=torch.float32, device=dev)
        args = QmoeNormArgs(x.data_ptr(), _ptr(y), _ptr(gate), _ptr(post_w), scale.data_ptr() if vector else None,
                            _ptr(w), None if y is None else x_out.data_ptr(), h.data_ptr(), _ptr(q), _ptr(q_scale),
                            1.0 if vector else float(scale), float(eps), _TYPES[dt], _GATES[gate_act])
        _launch(lib().qmoe_residual_norm, dev, stream, ctypes.byref(args), T, H)
    return NormOut(x_out, h, q, q_scale)
