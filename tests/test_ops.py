"""The 8-bit float feed-forward's operators (qwenium_amd/ops.py): against plain forms in
64 bits on the CPU, their refusals, and a block of them together.

Tolerances count roundings: u(t) is half a step of type t relative to the value (f32
2^-24, bf16 2^-8; e4m3 2^-4, and 2^-10 below its smallest normal number)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import qwenium_amd as qa
from qwenium_amd import _lib
from qwenium_amd._lib import QMOE_ERR_NULL, QMOE_ERR_TYPE, QMOE_ERR_VALUE, QMOE_OK, TYPE_BF16, TYPE_F32, TYPE_Q8_0
from qwenium_amd.ops import NormOut, TokenOrder

FAKE = 0x10000000
FP8 = torch.float8_e4m3fn
U32 = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
MIB = 1 << 20


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g)


def blocks(n):
    return -(-n // 128)


# ---- plain forms -----------------------------------------------------------------------------------

def plain_quantize(v):
    """The definition on the CPU: the scale one f32 quotient, the value v * 448 / m in 64 bits (off by 2^-51
    of it: f32 values lie no nearer to a border unless on it) rounded to e4m3's steps, ties to even."""
    R, C = v.shape
    b = blocks(C)
    p = torch.zeros(R, b * 128, dtype=torch.float32)
    p[:, :C] = v.float()
    p = p.view(R, b, 128)
    m = p.abs().amax(2).clamp_min(1e-30)  # (amax and clamp_min keep a NaN)
    z = p.double() * 448 / m.double()[:, :, None]
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.where(torch.isnan(z), z, torch.round(z / step) * step).to(FP8)
    return q.view(R, b * 128)[:, :C].contiguous(), m / 448


def fp8_rows(g, R, C):
    return plain_quantize(randn(g, R, C) * (1 + 10 * (torch.rand(C, generator=g) < 0.02)))


def fp8_weights(g, *shape):
    w = (100 * randn(g, *shape)).clamp(-448, 448).to(FP8)
    s = 2e-4 * (0.5 + torch.rand(*shape[:-2], blocks(shape[-2]), blocks(shape[-1]), generator=g))
    return w, s


def whole(q, s, line=1):
    n, k = q.shape[-2:]
    s = s.double().repeat_interleave(128, -1)[..., :k]
    if line > 1:
        s = s.repeat_interleave(line, -2)[..., :n, :]
    return q.double() * s


def plain_order(idx, E):
    """offsets, rows, tokens, place with numpy, dropped ids last."""
    idx = idx.numpy().astype(np.int64)
    T, k = idx.shape
    flat = idx.reshape(-1)
    valid = (flat >= 0) & (flat < E)
    order = np.argsort(np.where(valid, flat, E), kind="stable")[:valid.sum()]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[valid], minlength=E)[:E])])
    rows = np.full(T * k, -1)
    rows[:len(order)] = order
    tokens = np.where(rows >= 0, rows // k, -1)
    place = np.full(T * k, -1)
    place[order] = np.arange(len(order))
    return offsets, rows, tokens, place.reshape(T, k)


def routing(g, T, E, k, kind="even"):
    if kind == "one":  # every token to the same experts
        return torch.arange(k, dtype=torch.int32).repeat(T, 1)
    logits = randn(g, T, E)
    if kind == "skew":
        logits -= 2 * torch.log(torch.arange(1, E + 1).float())
    idx = torch.topk(logits, k, dim=1).indices.to(torch.int32)
    if kind == "drop":  # ids that no expert has
        bad = torch.tensor([-1, E, 2 ** 31 - 1, -2 ** 31], dtype=torch.int64)
        at = torch.rand(T, k, generator=g) < 0.3
        idx = torch.where(at, bad[torch.randint(0, 4, (T, k), generator=g)], idx.long()).to(torch.int32)
    return idx


def near(got, want, tol, what=""):
    """Every value within its own tolerance; NaN and infinities where they belong."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} != {tuple(want.shape)}"
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {off.max().item():.3e} over its tolerance"


# ---- refusals (no GPU) ------------------------------------------------------------------------------

def rc_quantize(x=FAKE, t=TYPE_F32, R=4, C=256, act=0, q=FAKE + MIB, s=FAKE + 2 * MIB):
    return _lib.lib().qmoe_fp8_quantize(x, t, R, C, act, q, s, None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(t=TYPE_Q8_0), QMOE_ERR_TYPE, "x_type"), (dict(R=-1), QMOE_ERR_VALUE, "n_rows"),
    (dict(C=0), QMOE_ERR_VALUE, "n_cols"), (dict(act=3), QMOE_ERR_VALUE, "act"), (dict(act=-1), QMOE_ERR_VALUE, "act"),
    (dict(x=None), QMOE_ERR_NULL, "x"), (dict(q=None), QMOE_ERR_NULL, "q"), (dict(s=None), QMOE_ERR_NULL, "scale"),
    (dict(x=FAKE + 2), QMOE_ERR_VALUE, "aligned"), (dict(q=FAKE), QMOE_ERR_VALUE, "distinct"),
    (dict(q=FAKE + 4095), QMOE_ERR_VALUE, "q expected a buffer distinct from x"), (dict(s=FAKE - 28), QMOE_ERR_VALUE, "distinct"),
    (dict(s=FAKE + MIB + 1020), QMOE_ERR_VALUE, "scale expected a buffer distinct from q"),
    (dict(R=2 ** 31 - 1, C=2 ** 28), QMOE_ERR_VALUE, "ceil(n_cols/128)"), (dict(R=2 ** 28, C=1), QMOE_ERR_VALUE, "ceil(n_cols/128)"),
])
def test_quantize_refusals(kw, code, needle):
    assert rc_quantize(**kw) == code
    assert needle in _lib.last_error() and "expected" in _lib.last_error()


def test_quantize_blocks_of_one_launch():
    """16 threads a block in whole workgroups of 16 blocks, below 2^32 threads: up to 2^28 - 16 blocks."""
    for R, C in ((2 ** 28 - 15, 1), (2 ** 28 - 1, 128), (2 ** 27 - 7, 129)):
        assert rc_quantize(R=R, C=C, x=None) == QMOE_ERR_VALUE
        assert f"ceil(n_cols/128) expected 0..{2 ** 28 - 16}" in _lib.last_error()
    for R, C in ((2 ** 28 - 16, 1), (2 ** 27 - 8, 129)):  # (the next check's answer)
        assert rc_quantize(R=R, C=C, x=None) == QMOE_ERR_NULL


def test_no_rows_is_a_no_op_without_gpu():
    L = _lib.lib()
    assert rc_quantize(R=0, x=None, q=None, s=None) == QMOE_OK
    assert rc_matmul(R=0, A=0, a=None, y=None) == QMOE_OK
    assert L.qmoe_gather_tokens(None, 4, 0, 8, 2, 4, None, None, None, None) == QMOE_OK
    assert L.qmoe_combine_tokens(None, TYPE_F32, 0, 8, 2, None, None, None, None, None) == QMOE_OK
    assert L.qmoe_combine_tokens_backward(None, None, TYPE_F32, 0, 8, 2, 4, None, None, None, None, None, None) == QMOE_OK
    assert L.qmoe_residual_norm(ctypes.byref(norm_args()), 0, 64, None) == QMOE_OK


def rc_matmul(a=FAKE, sa=FAKE + 0x100, A=4, w=FAKE + MIB, sw=FAKE + 2 * MIB, E=1, n=64, k=128, offsets=None, rows=None,
              R=4, y=FAKE + 3 * MIB, t=TYPE_F32):
    return _lib.lib().qmoe_fp8_matmul(a, sa, A, w, sw, E, n, k, offsets, rows, R, y, t, None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(t=TYPE_Q8_0), QMOE_ERR_TYPE, "y_type"), (dict(R=-1), QMOE_ERR_VALUE, "n_rows"),
    (dict(n=0), QMOE_ERR_VALUE, "n expected"), (dict(k=0), QMOE_ERR_VALUE, "k expected"),
    (dict(k=120), QMOE_ERR_VALUE, "multiple of 16"), (dict(E=2), QMOE_ERR_VALUE, "n_experts"),
    (dict(E=0, offsets=FAKE), QMOE_ERR_VALUE, "n_experts"), (dict(E=1025, offsets=FAKE), QMOE_ERR_VALUE, "n_experts"),
    (dict(A=3), QMOE_ERR_VALUE, "a_rows"), (dict(A=0, rows=FAKE), QMOE_ERR_VALUE, "a_rows"),
    (dict(a=None), QMOE_ERR_NULL, "a expected"), (dict(sa=None), QMOE_ERR_NULL, "a_scale"),
    (dict(w=None), QMOE_ERR_NULL, "w expected"), (dict(sw=None), QMOE_ERR_NULL, "w_scale"),
    (dict(y=None), QMOE_ERR_NULL, "y expected"), (dict(a=FAKE + 8), QMOE_ERR_VALUE, "16-byte"),
    (dict(w=FAKE + MIB + 4), QMOE_ERR_VALUE, "16-byte"), (dict(y=FAKE + MIB), QMOE_ERR_VALUE, "distinct"),
    (dict(y=FAKE + MIB + 2), QMOE_ERR_VALUE, "aligned"), (dict(y=FAKE + 508), QMOE_ERR_VALUE, "distinct from a"),
    (dict(y=FAKE + MIB - 1020), QMOE_ERR_VALUE, "distinct from w"), (dict(R=2 ** 30 + 1, A=2 ** 30 + 1), QMOE_ERR_VALUE, "n_rows"),
    (dict(offsets=FAKE + 3 * MIB + 1020), QMOE_ERR_VALUE, "distinct from offsets"),
])
def test_matmul_refusals(kw, code, needle):
    assert rc_matmul(**kw) == code
    assert needle in _lib.last_error()


def test_matmul_larger_than_a_launch():
    """1024 experts with a row each and 2^23 columns are 2^26 workgroups or more: refused by name, before the launch."""
    a, b, c, d, e, f = (FAKE + (i << 40) for i in range(6))
    assert rc_matmul(a=a, sa=b, A=1024, w=c, sw=d, E=1024, n=2 ** 23, k=16, offsets=e, R=1024, y=f) == QMOE_ERR_VALUE
    assert "n_rows x n expected fewer than 2^32 threads" in _lib.last_error() and "1024 x 8388608" in _lib.last_error()


def test_token_refusals():
    L = _lib.lib()
    a, b, c, d, e = (FAKE + i * MIB for i in range(5))
    assert L.qmoe_sort_tokens(a, -1, 2, 4, b, c, d, e, None) == QMOE_ERR_VALUE
    assert L.qmoe_sort_tokens(a, 4, 0, 4, b, c, d, e, None) == QMOE_ERR_VALUE and "top_k" in _lib.last_error()
    assert L.qmoe_sort_tokens(a, 4, 65, 4, b, c, d, e, None) == QMOE_ERR_VALUE
    assert L.qmoe_sort_tokens(a, 4, 2, 1025, b, c, d, e, None) == QMOE_ERR_VALUE and "n_experts" in _lib.last_error()
    assert L.qmoe_sort_tokens(a, 2 ** 30, 2, 4, b, c, d, e, None) == QMOE_ERR_VALUE and "n_tokens * top_k" in _lib.last_error()
    assert L.qmoe_sort_tokens(a, 4, 2, 4, None, c, d, e, None) == QMOE_ERR_NULL and "offsets" in _lib.last_error()
    assert L.qmoe_sort_tokens(a, 4, 2, 4, b, c, d, a, None) == QMOE_ERR_VALUE and "distinct" in _lib.last_error()
    assert L.qmoe_gather_tokens(a, 3, 4, 8, 2, 4, b, c, d, None) == QMOE_ERR_VALUE and "elem_bytes" in _lib.last_error()
    assert L.qmoe_gather_tokens(a, 4, 4, 0, 2, 4, b, c, d, None) == QMOE_ERR_VALUE and "n_cols" in _lib.last_error()
    assert L.qmoe_gather_tokens(a, 4, 4, 8, 2, 4, b, None, d, None) == QMOE_ERR_NULL and "place" in _lib.last_error()
    assert L.qmoe_gather_tokens(a, 4, 4, 8, 2, 4, b, c, a, None) == QMOE_ERR_VALUE
    assert L.qmoe_gather_tokens(a + 2, 4, 4, 8, 2, 4, b, c, d, None) == QMOE_ERR_VALUE and "aligned" in _lib.last_error()
    assert L.qmoe_combine_tokens(a, TYPE_Q8_0, 4, 8, 2, b, c, d, e, None) == QMOE_ERR_TYPE
    assert L.qmoe_combine_tokens(a, TYPE_F32, 4, 8, 2, b, c, d, a, None) == QMOE_ERR_VALUE
    assert L.qmoe_combine_tokens(None, TYPE_F32, 4, 8, 2, b, c, d, e, None) == QMOE_ERR_NULL
    assert L.qmoe_combine_tokens_backward(a, b, TYPE_F32, 4, 8, 2, 4, c, d, e, a, a + 64, None) == QMOE_ERR_VALUE
    assert L.qmoe_combine_tokens_backward(a, b, TYPE_F32, 4, 8, 2, 4, c, d, None, e, a + 64, None) == QMOE_ERR_NULL


def test_rows_of_one_launch():
    """A launch holds below 2^32 threads: more rows are refused."""
    L, T = _lib.lib(), 1 << 22
    a, b, c, d, e, f, g = (FAKE + (i << 40) for i in range(7))
    assert L.qmoe_gather_tokens(a, 4, T, 8, 1, 4, b, c, d, None) == QMOE_ERR_VALUE and "n_tokens" in _lib.last_error()
    assert L.qmoe_combine_tokens(a, TYPE_F32, T, 8, 1, b, c, d, e, None) == QMOE_ERR_VALUE and "n_tokens" in _lib.last_error()
    assert L.qmoe_combine_tokens_backward(a, b, TYPE_F32, T, 8, 1, 4, c, d, e, f, g, None) == QMOE_ERR_VALUE
    assert "n_tokens" in _lib.last_error()
    norm = norm_args(x=a, y=b, x_out=c, h=d)
    assert L.qmoe_residual_norm(ctypes.byref(norm), T, 8, None) == QMOE_ERR_VALUE and "n_tokens" in _lib.last_error()


def norm_args(**kw):
    d = dict(x=FAKE, y=FAKE + MIB, gate=None, post_w=None, scale_v=None, w=None, x_out=FAKE + 2 * MIB, h=FAKE + 3 * MIB,
             q=None, q_scale=None, scale=1.0, eps=1e-6, x_type=TYPE_F32, gate_act=0)
    return _lib.QmoeNormArgs(**{**d, **kw})


@pytest.mark.parametrize("kw,code,needle", [
    (dict(x_type=TYPE_Q8_0), QMOE_ERR_TYPE, "x_type"), (dict(x=None), QMOE_ERR_NULL, "x expected"),
    (dict(h=None), QMOE_ERR_NULL, "h expected"), (dict(x_out=None), QMOE_ERR_NULL, "x_out"),
    (dict(gate=FAKE + 4 * MIB), QMOE_ERR_VALUE, "gate_act"), (dict(gate_act=1), QMOE_ERR_VALUE, "gate_act"),
    (dict(gate_act=3), QMOE_ERR_VALUE, "gate_act"), (dict(y=None, post_w=FAKE), QMOE_ERR_VALUE, "y expected"),
    (dict(q=FAKE + 5 * MIB), QMOE_ERR_NULL, "q_scale"), (dict(eps=-1.0), QMOE_ERR_VALUE, "eps"),
    (dict(eps=float("nan")), QMOE_ERR_VALUE, "eps"), (dict(h=FAKE), QMOE_ERR_VALUE, "distinct"),
    (dict(x_out=FAKE + 3 * MIB), QMOE_ERR_VALUE, "distinct"), (dict(x_out=FAKE + 1020), QMOE_ERR_VALUE, "distinct from x"),
    (dict(w=FAKE + 3 * MIB + 1020), QMOE_ERR_VALUE, "distinct from w"), (dict(h=FAKE + 2), QMOE_ERR_VALUE, "aligned"),
])
def test_norm_refusals(kw, code, needle):
    assert _lib.lib().qmoe_residual_norm(ctypes.byref(norm_args(**kw)), 4, 64, None) == code
    assert needle in _lib.last_error()


def test_norm_width_refusals():
    L = _lib.lib()
    assert L.qmoe_residual_norm(None, 4, 64, None) == QMOE_ERR_NULL
    for H in (0, 16385):
        assert L.qmoe_residual_norm(ctypes.byref(norm_args()), 4, H, None) == QMOE_ERR_VALUE
        assert "n_embd" in _lib.last_error()
    assert L.qmoe_residual_norm(ctypes.byref(norm_args()), -1, 64, None) == QMOE_ERR_VALUE


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 128)
    order = TokenOrder(*(torch.zeros(n, dtype=torch.int32) for n in (5, 8, 8)), torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="place expected"):
        TokenOrder(order.offsets, order.rows, order.tokens, order.rows)
    with pytest.raises(ValueError, match="x expected a cuda"):
        qa.fp8_quantize(x)
    with pytest.raises(ValueError, match="act expected"):
        qa.fp8_quantize(x, act="relu")
    with pytest.raises(ValueError, match="a expected a cuda"):
        qa.fp8_matmul(x, x, x, x)
    with pytest.raises(ValueError, match="topk_idx expected a cuda"):
        qa.sort_tokens(torch.zeros(4, 2, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="x expected a cuda"):
        qa.gather_tokens(x, order)
    with pytest.raises(ValueError, match="ys expected a cuda"):
        qa.combine_tokens(x, order, x)
    with pytest.raises(ValueError, match="weights expected"):
        qa.combine_tokens(x, order, None)
    with pytest.raises(ValueError, match="ys expected a cuda"):
        qa.combine_tokens_backward(x, x, order, x)
    with pytest.raises(ValueError, match="x expected a cuda"):
        qa.residual_norm(x, x, None, 1e-6)


GRAD_CALLS = {
    "fp8_quantize": lambda x, y, w: qa.fp8_quantize(x),
    "gather_tokens": lambda x, y, w: qa.gather_tokens(x, None),
    "combine_tokens": lambda x, y, w: qa.combine_tokens(x, None, w),
    "gather_tokens_backward": lambda x, y, w: qa.gather_tokens_backward(x, None),
    "combine_tokens_backward": lambda x, y, w: qa.combine_tokens_backward(y, x, None, w),
    "residual_norm": lambda x, y, w: qa.residual_norm(x, y, w, 1e-6),
}  # (fp8_matmul's first operand is e4m3: on the device, below)


@pytest.mark.parametrize("name", GRAD_CALLS)
def test_operands_that_require_grad_are_refused(name):
    """No call records a gradient: an operand that asks for one is refused rather than its gradient lost."""
    x, y, w = torch.zeros(4, 128, requires_grad=True), torch.zeros(4, 128), torch.zeros(128)
    with pytest.raises(ValueError, match="(x|ys) expected a tensor outside autograd .* requires grad"):
        GRAD_CALLS[name](x, y, w)
    with torch.no_grad(), pytest.raises(ValueError, match="expected a cuda"):
        GRAD_CALLS[name](x, y, w)


@pytest.mark.gpu
def test_operands_that_require_grad_on_device(gpu):
    """Every operand that a gradient could be asked of; within no_grad the calls run and give what they gave."""
    g = gen(8)
    T, k, E, H = 6, 2, 4, 128
    x, ys, w = randn(g, T, H).to(gpu), randn(g, T * k, H).to(gpu), torch.rand(T, k, generator=g).to(gpu)
    o = device_order(gpu, routing(g, T, E, k), E)
    q, s = qa.fp8_quantize(x)
    m, sm = (t.to(gpu) for t in fp8_weights(g, 64, H))
    vec = torch.rand(H, generator=g).to(gpu)
    for call, args in ((lambda a: qa.gather_tokens(a, o), (x,)), (lambda a, b: qa.combine_tokens(a, o, b), (ys, w)),
                       (lambda a, b, c: qa.combine_tokens(a, o, b, residual=c), (ys, w, x)),
                       (lambda a: qa.gather_tokens_backward(a, o), (ys,)),
                       (lambda a, b, c: qa.combine_tokens_backward(a, b, o, c)[0], (x, ys, w)),
                       (lambda a: qa.fp8_quantize(a)[1], (x,)), (lambda a, b: qa.fp8_matmul(q, a, m, b), (s, sm)),
                       (lambda a, b, c: qa.residual_norm(a, b, c, 1e-6).h, (x, x.clone(), vec)),
                       (lambda a, b, c: qa.residual_norm(x, x.clone(), None, 1e-6, post_w=a, scale=b, gate=c, gate_act="silu").h,
                        (vec, vec.clone(), x.clone()))):
        want = call(*args)
        assert not want.requires_grad
        for i in range(len(args)):
            asks = [a.detach().clone().requires_grad_(j == i) for j, a in enumerate(args)]
            with pytest.raises(ValueError, match="outside autograd"):
                call(*asks)
            with torch.no_grad():
                assert torch.equal(call(*asks), want)
            with torch.inference_mode():
                assert torch.equal(call(*asks), want)


@pytest.mark.gpu
def test_python_refusals_on_device(gpu):
    x = torch.zeros(4, 128, device=gpu)
    q, s = qa.fp8_quantize(x)
    w, sw = torch.zeros(64, 128, device=gpu).to(FP8), torch.zeros(1, 1, device=gpu)
    for bad in (dict(a=q[:, :120]), dict(a_scale=s[:2]), dict(a_scale=s.double()), dict(w=w[:, :64]), dict(w=w[None]),
                dict(w=w.t().contiguous().t()), dict(w_scale=sw.repeat(2, 1)), dict(out_dtype=torch.float16),
                dict(offsets=torch.zeros(2, dtype=torch.int32, device=gpu)), dict(rows=torch.zeros(4, device=gpu)),
                dict(out=torch.zeros(4, 63, device=gpu)), dict(out=torch.zeros(4, 64)),
                dict(w=w[None], w_scale=sw[None], offsets=torch.zeros(3, dtype=torch.int32, device=gpu))):
        kw = dict(a=q, a_scale=s, w=w, w_scale=sw)
        kw.update(bad)
        with pytest.raises(ValueError, match="expected"):
            qa.fp8_matmul(kw.pop("a"), kw.pop("a_scale"), kw.pop("w"), kw.pop("w_scale"), **kw)
    o = qa.sort_tokens(torch.zeros(4, 2, dtype=torch.int32, device=gpu), 3)
    for call in (lambda: qa.sort_tokens(torch.zeros(4, 2, dtype=torch.int64, device=gpu), 3),
                 lambda: qa.sort_tokens(torch.zeros(4, 2, dtype=torch.int32, device=gpu), 0),
                 lambda: qa.gather_tokens(x[:3], o), lambda: qa.combine_tokens(x, o, torch.ones(4, 2, device=gpu)),
                 lambda: qa.combine_tokens(x.repeat(2, 1), o, torch.ones(4, 3, device=gpu)),
                 lambda: qa.combine_tokens(x.repeat(2, 1), o, torch.ones(4, 2, device=gpu), residual=x.bfloat16()),
                 lambda: qa.combine_tokens_backward(x[:3], x.repeat(2, 1), o, torch.ones(4, 2, device=gpu)),
                 lambda: qa.fp8_quantize(x.half()), lambda: qa.fp8_quantize(x[:, :5], act="swiglu"),
                 lambda: qa.fp8_quantize(x, scale=s.t()), lambda: qa.residual_norm(x, x[:3], None, 1e-6),
                 lambda: qa.residual_norm(x, None, None, 1e-6, scale=0.5),
                 lambda: qa.residual_norm(x, x, x[0].bfloat16(), 1e-6), lambda: qa.residual_norm(x, x, None, 1e-6, gate=x),
                 lambda: qa.residual_norm(x, x, None, 1e-6, gate_act="silu")):
        with pytest.raises(ValueError, match="expected"):
            call()
    with pytest.raises(qa.QmoeError, match="n_experts"):
        qa.sort_tokens(torch.zeros(4, 2, dtype=torch.int32, device=gpu), 2000)


# ---- quantization -----------------------------------------------------------------------------------

def check_fp8(q, s, v, err=0.0, what=""):
    """q and s stand for v (64 bits, itself known to err): the scale to err and two roundings, each
    value to half an e4m3 step."""
    R, C = v.shape
    b = blocks(C)
    pad = torch.zeros(R, b * 128, dtype=torch.float64)
    pad[:, :C] = v.abs()
    m = pad.view(R, b, 128).amax(2)
    near(s, (m / 448).clamp_min(1e-30 / 448), (2 * U32 + err) * m / 448 + 1e-38, what + " scale")
    ss = s.cpu().double().repeat_interleave(128, 1)[:, :C]
    near(q.cpu().double() * ss, v, (2.0 ** -4 * (1 + 2.0 ** -10) + 2 * err) * v.abs() + 2.0 ** -10 * (1 + 2.0 ** -10) * ss, what)


SIZES = [(1, 1), (1, 128), (3, 127), (5, 129), (2, 2048), (33, 704), (17, 8), (130, 100), (7, 1000), (64, 512), (1, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,C", SIZES)
def test_quantize_bits(gpu, R, C, dtype):
    """The definition's bits: values over many magnitudes, a block of zeros, the ends of f32."""
    g = gen(R * 31 + C)
    x = randn(g, R, C) * torch.exp(4 * randn(g, R, 1))
    x[0, :min(C, 128)] = 0
    if R > 2:
        x[1] *= 1e30
        x[2] *= 1e-36
    x = x.to(dtype)
    q, s = qa.fp8_quantize(x.to(gpu))
    want_q, want_s = plain_quantize(x)
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().view(torch.uint8), want_q.view(torch.uint8))


@pytest.mark.gpu
def test_quantize_non_finite(gpu):
    x = torch.ones(4, 384)
    x[0, 5], x[1, 130], x[2, 383], x[3, 0] = math.nan, math.inf, -math.inf, math.nan
    x[3, 1] = math.inf
    q, s = (t.cpu() for t in qa.fp8_quantize(x.to(gpu)))
    v = q.float() * s.repeat_interleave(128, 1)
    assert torch.isnan(v[0, :128]).all() and torch.isnan(v[3, :128]).all()
    assert torch.isinf(s[1, 1]) and torch.isnan(v[1, 128:256]).all() and torch.isinf(s[2, 2])
    near(v[:3, 128:256][[0, 2]], torch.ones(2, 128, dtype=torch.float64), 2.0 ** -4)
    assert torch.isfinite(v[1, :128]).all() and torch.isfinite(v[1, 256:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["swiglu", "geglu"])
@pytest.mark.parametrize("R,C", SIZES)
def test_quantize_activation(gpu, R, C, act, dtype):
    g = gen(R + C)
    x = (3 * randn(g, R, 2 * C)).to(dtype)
    x[0, 0] = -80.0
    gate, up = x.double()[:, :C], x.double()[:, C:]
    z = gate if act == "swiglu" else 2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
    v = gate * torch.sigmoid(z) * up
    # exp(-z): |z| <= 88 where it is finite, and z itself carries 5 roundings: 88 * 5 u, then a
    # handful more; where exp overflows both are 0 to f32's smallest numbers
    q, s = qa.fp8_quantize(x.to(gpu), act=act)
    check_fp8(q, s, v, 460 * U32, act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["swiglu", "geglu"])
@pytest.mark.parametrize("R,C", [(600, 1024), (700, 333), (3, 70001)])
def test_quantize_activation_rounds_once(gpu, R, C, act, dtype):
    """q is the 64-bit formula's nearest e4m3, unless its quotient is the middle of two to within 64 bits' own error
    (some 20 roundings of 2^-53, and those that gelu's z multiplies by |z| <= 60: 1e-13)."""
    x = (2 * randn(gen(R * C), R, 2 * C)).to(dtype)
    q, _ = qa.fp8_quantize(x.to(gpu), act=act)
    g, u = x.double()[:, :C], x.double()[:, C:]
    z = g if act == "swiglu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    v = torch.nn.functional.pad(u * g * torch.sigmoid(z), (0, -C % 128)).view(R, -1, 128)
    p = (v / (v.abs().amax(2, keepdim=True).clamp_min(1e-30) / 448)).view(R, -1)[:, :C]
    step = torch.exp2(torch.floor(torch.log2(p.abs().clamp_min(2.0 ** -6))) - 3)
    want, got = torch.round(p / step) * step, q.cpu().double()
    off = (got - want).abs()
    middle = (p - (got + want) / 2).abs() <= 1e-13 * p.abs()
    assert ((off == 0) | ((off <= step) & middle)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["swiglu", "geglu"])
@pytest.mark.parametrize("low,high", [(-9, -7), (-9, -5), (-14, -9), (-30, 4), (-1, 12)])
def test_quantize_activation_rounds_once_far_gates(gpu, low, high, act, dtype):
    """As above for blocks whose gates all lie between low and high: far below zero z's own roundings count |z| times in
    the value and in the block's maximum.  (64 bits: where |v| counts beside 1e-30 / 448, z > -81, and up to
    20 roundings of 2^-53 of it are 2e-13.)"""
    R, C = 3001, 4096
    g = torch.Generator(device=gpu).manual_seed(1000 - 31 * low + high)
    x = torch.empty(R, 2 * C, device=gpu)
    x[:, :C] = low + (high - low) * torch.rand(R, C, generator=g, device=gpu)
    x[:, C:] = 2 * torch.randn(R, C, generator=g, device=gpu)
    x = x.to(dtype)
    q, s = qa.fp8_quantize(x, act=act)
    gate, up = x.double()[:, :C], x.double()[:, C:]
    z = gate if act == "swiglu" else 2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
    v = (up * gate * torch.sigmoid(z)).view(R, -1, 128)
    m = v.abs().amax(2, keepdim=True).clamp_min(1e-30)
    p = (v * 448 / m).view(R, C)
    step = torch.exp2(torch.floor(torch.log2(p.abs().clamp_min(2.0 ** -6))) - 3)
    want, got = torch.round(p / step) * step, q.double()
    off = (got - want).abs()
    middle = (p - (got + want) / 2).abs() <= 4e-13 * p.abs()
    assert ((off == 0) | ((off <= step) & middle)).all(), f"{int(((off > 0) & ~middle).sum())} of {R * C} values"
    # the scale: z's 6 roundings counted |z| times, 8 others, 2 of its own
    far = 0.0 if act == "swiglu" else float(6 * z.abs().max())
    assert ((s.double() - m[:, :, 0] / 448).abs() <= (10 + far) * U32 * m[:, :, 0] / 448).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["swiglu", "geglu"])
def test_quantize_activation_non_finite(gpu, act):
    """An infinite product gives its block an infinite scale, NaN a NaN one; a far negative gate gives zeros."""
    x = torch.ones(6, 2, 256)
    x[0, 0, 3], x[1, 1, 130], x[2, 0, 200], x[3, 1, 7] = math.inf, -math.inf, -1000.0, math.nan
    x[4, 0, :128] = -1000.0
    x[5, 0, 1], x[5, 1, 1] = 3e38, 3e38
    _, s = (t.cpu() for t in qa.fp8_quantize(x.view(6, 512).to(gpu), act=act))
    one = s[2, 0]
    assert torch.isfinite(one) and one > 0
    assert math.isinf(s[0, 0]) and math.isinf(s[1, 1]) and math.isnan(s[3, 0]) and math.isinf(s[5, 0])
    assert s[4, 0] == torch.tensor(1e-30) / 448
    for r, b in ((0, 1), (1, 0), (2, 1), (3, 1), (4, 1), (5, 1)):
        assert s[r, b] == one


# ---- products --------------------------------------------------------------------------------------

def check_product(y, a, s, w, sw, dtype, what=""):
    """Against 64 bits: each block's 128 products are exact and summed in f32 (a truncating step
    loses two half steps), then scaled (2 roundings) and summed over the blocks and the waves.
    bf16 results may come from the e4m3 MFMA, which aligns the products of a group of 8 to the
    largest, P, and drops what is below 2^-13 P of each of the 7 others: 7 2^-13 P a group, P at most
    the group's part of sum |a w|."""
    A, W = whole(a, s), whole(w, sw, 128)
    want = A @ W.T
    size = A.abs() @ W.abs().T
    tol = (2 * 128 + blocks(a.shape[1]) + 8) * U32 + (7 * 2.0 ** -13 if dtype == torch.bfloat16 else 0)
    near(y, want, tol * size * (1 + 2.0 ** -8) + U[dtype] * want.abs(), what)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 2048, 2048), (2, 33, 144), (15, 127, 128), (16, 128, 256), (17, 129, 240),
                                   (33, 200, 1040), (64, 64, 704), (65, 130, 512), (127, 96, 2064), (128, 256, 1024),
                                   (130, 257, 384), (200, 384, 640), (257, 500, 272), (300, 1024, 128), (1000, 272, 400),
                                   (520, 640, 2048)])
def test_matmul_dense(gpu, M, N, K, dtype):
    g = gen(M + N + K)
    a, s = fp8_rows(g, M, K)
    w, sw = fp8_weights(g, N, K)
    y = qa.fp8_matmul(a.to(gpu), s.to(gpu), w.to(gpu), sw.to(gpu), out_dtype=dtype)
    check_product(y, a, s, w, sw, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("T,E,k,N,K,kind", [
    (1, 8, 2, 64, 128, "even"), (10, 64, 8, 100, 256, "even"), (3, 300, 8, 48, 144, "even"), (40, 16, 4, 128, 704, "even"),
    (64, 4, 2, 130, 272, "one"), (100, 8, 3, 200, 384, "skew"), (257, 5, 1, 257, 512, "even"), (50, 8, 4, 64, 256, "drop"),
    (700, 12, 4, 256, 640, "skew"), (90, 700, 2, 32, 128, "drop"), (600, 3, 2, 384, 1040, "drop"), (300, 2, 2, 96, 16, "even")])
def test_matmul_experts(gpu, T, E, k, N, K, kind, gather, dtype):
    g = gen(T + E + N)
    idx = routing(g, T, E, k, kind)
    offsets, rows, tokens, _ = plain_order(idx, E)
    R, live = T * k, int(offsets[-1])
    a, s = fp8_rows(g, T if gather else R, K)
    w, sw = fp8_weights(g, E, N, K)
    off = torch.tensor(offsets, dtype=torch.int32)
    tok = torch.tensor(tokens, dtype=torch.int32)
    y = torch.full((R, N), 7.0, dtype=dtype, device=gpu)
    got = qa.fp8_matmul(a.to(gpu), s.to(gpu), w.to(gpu), sw.to(gpu), offsets=off.to(gpu), rows=tok.to(gpu) if gather else None,
                        out=y)
    assert got is y
    y = y.cpu()
    for e in range(E):
        i, j = int(offsets[e]), int(offsets[e + 1])
        if j > i:
            at = tok[i:j].long() if gather else slice(i, j)
            check_product(y[i:j], a[at], s[at], w[e], sw[e], dtype, f"expert {e}")
    assert (y[live:] == 7).all(), "rows of no expert were written"


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 40, 300])
def test_matmul_index_values(gpu, M):
    """Indices outside a give zeros, repeated ones the same row; offsets outside the rows count as their ends."""
    g = gen(M)
    K, N = 272, 160
    a, s = fp8_rows(g, M, K)
    w, sw = fp8_weights(g, 2, N, K)
    rows = torch.randint(0, M, (M,), generator=g).to(torch.int32)
    rows[0], rows[M // 2], rows[M - 1] = -1, M, 2 ** 31 - 1
    bad = (rows < 0) | (rows >= M)
    d = [t.to(gpu) for t in (a, s, w, sw)]
    y = qa.fp8_matmul(d[0], d[1], d[2][0].contiguous(), d[3][0].contiguous(), rows=rows.to(gpu)).cpu()
    assert (y[bad] == 0).all()
    at = rows[~bad].long()
    check_product(y[~bad], a[at], s[at], w[0], sw[0], torch.float32)
    half = M // 2
    for off in ([-5, half, 2 ** 31 - 1], [-2 ** 31, half, M + 1]):
        y = qa.fp8_matmul(*d, offsets=torch.tensor(off, dtype=torch.int32, device=gpu)).cpu()
        check_product(y[:half], a[:half], s[:half], w[0], sw[0], torch.float32)
        check_product(y[half:], a[half:], s[half:], w[1], sw[1], torch.float32)
    keep = torch.full((M, N), 3.0, device=gpu)
    for off in ([M, 0, M // 3], [M // 3, M // 3, M // 3], [2 ** 31 - 1, -1, -1]):  # falling and empty: within bounds
        qa.fp8_matmul(*d, offsets=torch.tensor(off, dtype=torch.int32, device=gpu), out=keep)
    assert torch.isfinite(keep).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [3, 150, 1500])
def test_matmul_nan_stays_in_its_row(gpu, M, dtype):
    g = gen(7)
    a, s = fp8_rows(g, M, 144)
    w, sw = fp8_weights(g, 72, 144)
    a.view(torch.uint8)[1, 143] = 0x7F  # a NaN in the last, short block
    s2 = s.clone()
    s2[2, 0] = math.inf
    y = qa.fp8_matmul(a.to(gpu), s2.to(gpu), w.to(gpu), sw.to(gpu), out_dtype=dtype).cpu()
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    keep = [i for i in range(M) if i not in (1, 2)]
    check_product(y[keep], a[keep], s[keep], w, sw, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,R,N,K", [(0, 4100, 4104, 144), (0, 2050, 4100, 272), (0, 600, 2100, 528), (0, 300, 520, 144),
                                     (8, 1500, 5128, 144), (8, 2000, 1704, 272), (16, 1280, 2696, 144), (24, 700, 2000, 656),
                                     (8, 900, 1000, 1040), (40, 600, 1000, 1040), (40, 700, 900, 400), (60, 700, 900, 656), (2, 4500, 3000, 128), (300, 2400, 260, 256), (70, 20000, 256, 528)])
def test_matmul_tile_sizes(gpu, E, R, N, K, dtype):
    """Every tile, at its edges: sizes that fill the device, odd rows, columns and blocks; against 64 bits on
    the device, the whole result."""
    g = gen(R + N)
    a, s = (t.to(gpu) for t in fp8_rows(g, R, K))
    w, sw = (t.to(gpu) for t in fp8_weights(g, max(E, 1), N, K))
    order = torch.randperm(R, generator=g).to(torch.int32)
    order[R // 3] = -1
    bounds = [0, R]
    kw = {}
    if E:
        cut = torch.sort(torch.randint(0, R - 5, (E - 1,), generator=g)).values.tolist()
        bounds = [3] + [max(3, c) for c in cut] + [R - 2]
        kw["offsets"] = torch.tensor(bounds, dtype=torch.int32, device=gpu)
    else:
        w, sw = w[0], sw[0]
    y = torch.full((R, N), 7.0, dtype=dtype, device=gpu)
    qa.fp8_matmul(a, s, w, sw, rows=order.to(gpu), out=y, **kw)
    assert (y[:bounds[0]] == 7).all() and (y[bounds[-1]:] == 7).all()
    y = y.double()
    at = order.long().to(gpu)
    A = whole(a.float(), s)[at.clamp_min(0)] * (at >= 0)[:, None]
    loss = (2 * 128 + blocks(K) + 8) * U32 + (7 * 2.0 ** -13 if dtype == torch.bfloat16 else 0)  # as check_product
    for e in range(max(E, 1)):
        i, j = bounds[e], bounds[e + 1]
        if j > i:
            W = whole((w[e] if E else w).float(), sw[e] if E else sw, 128)
            want = A[i:j] @ W.T
            size = A[i:j].abs() @ W.abs().T
            off = (y[i:j] - want).abs() - loss * size * (1 + 2.0 ** -8) - U[dtype] * want.abs()
            assert off.max() <= 0, f"expert {e}: {off.max().item():.3e} over its tolerance"


# experts (0: dense), rows, n, k: the kernel of few rows, then every tile
SUMS = [(0, 3, 200, 144), (0, 40, 520, 1040), (0, 300, 520, 1024), (0, 600, 2100, 528), (0, 2050, 4100, 400), (0, 4100, 4104, 400),
        (3, 9, 64, 272), (8, 1500, 5128, 272), (8, 2000, 1704, 272), (16, 1280, 2696, 400), (8, 900, 1000, 1040), (40, 700, 900, 656),
        (300, 2400, 260, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,R,N,K", SUMS)
def test_matmul_large_products_that_cancel(gpu, E, R, N, K, dtype):
    """Of every 8 columns two hold 448 x 448 and 448 x -448, the others whole numbers up to 3.  All products are whole
    and those of a block of 128 add up to less than 32 x 448^2 + 96 x 9 < 2^23, so sums of 24 bits are exact in any
    order, whatever the number of rows: y is the small numbers' sum, rounded to its type once."""
    g = gen(R + N + K)

    def small(*shape):
        return torch.randint(-3, 4, shape, generator=g).float()

    a, w = small(R, K), small(max(E, 1), N, K)
    pair = torch.argsort(torch.rand(K // 8, 8, generator=g), 1)[:, :2] + 8 * torch.arange(K // 8)[:, None]
    a[:, pair] = 0
    w[:, :, pair] = 0
    bounds = torch.linspace(0, R, max(E, 1) + 1).int()
    want = torch.cat([a[bounds[e]:bounds[e + 1]].to(gpu) @ w[e].to(gpu).T for e in range(max(E, 1))]).to(dtype)
    a[:, pair] = 448.0
    w[:, :, pair[:, 0]], w[:, :, pair[:, 1]] = 448.0, -448.0
    s, sw = torch.ones(R, blocks(K), device=gpu), torch.ones(max(E, 1), blocks(N), blocks(K), device=gpu)
    a, w = a.to(gpu).to(FP8), w.to(gpu).to(FP8)
    if E:
        y = qa.fp8_matmul(a, s, w, sw, offsets=bounds.to(gpu), out_dtype=dtype)
    else:
        y = qa.fp8_matmul(a, s, w[0], sw[0], out_dtype=dtype)
    assert torch.equal(y, want)


# tile, experts (0: dense), rows, n, k, rows an expert: many steps of 128 columns through each tile's buffers, their number
# a multiple of 4 (row scales in 16 bytes) and not, k whole blocks (weights of one row tile past the caches) and not
STEADY = [("256x256", 0, 4100, 4104, 1040, ""), ("256x256", 0, 4100, 4104, 1024, ""), ("256x256", 0, 4096, 4096, 2048, ""),
          ("128x256", 0, 2050, 4100, 1040, ""), ("128x256", 0, 2050, 4100, 1024, ""), ("64x128", 0, 1000, 2600, 1040, ""),
          ("64x128", 0, 1000, 2600, 1536, ""), ("32x128", 0, 600, 2100, 1040, ""), ("32x128", 0, 600, 2100, 2048, ""),
          ("256x256", 8, 10000, 2100, 1040, "any"), ("256x256", 8, 10000, 2100, 1536, "any"), ("256x256", 16, 3600, 5000, 1024, "any"),
          ("256x256", 16, 3600, 5000, 1152, "even"), ("160x128", 40, 5200, 1000, 1024, "even"), ("160x128", 40, 5200, 1000, 1040, "any"),
          ("160x128", 40, 5200, 1000, 1152, "any"), ("128x128", 20, 1600, 2000, 1024, "even"), ("128x128", 20, 1600, 2000, 1040, "any"),
          ("64x128", 40, 1400, 1000, 1024, "even"), ("64x128", 40, 1400, 1000, 1040, "any"), ("64x128, two buffers", 40, 1400, 1000, 512, "any"),
          ("32x64, four buffers", 300, 2400, 260, 1024, "any"), ("32x64, four buffers", 300, 2400, 260, 2064, "any"),
          ("32x64, three buffers", 40, 500, 1000, 896, "any")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tile,E,R,N,K,cuts", STEADY, ids=["-".join(map(str, c)) for c in STEADY])
def test_matmul_tiles_over_many_steps(gpu, tile, E, R, N, K, cuts, dtype):
    """Against 64 bits on the device, the whole result, with f32 sums for either type (check_product's roundings without
    its allowance for the e4m3 instruction).  Uneven experts hold few rows, none, and more than a tile's, so that waves
    of a workgroup make different numbers of subtiles."""
    g = gen(R + N + K)
    a, s = (t.to(gpu) for t in fp8_rows(g, R, K))
    w, sw = (t.to(gpu) for t in fp8_weights(g, max(E, 1), N, K))
    rows = torch.randperm(R, generator=g).to(torch.int32)
    rows[R // 2] = R
    bounds, kw = [0, R], {}
    if E:
        cut = torch.linspace(0, R, E + 1).int()[1:-1] if cuts == "even" else \
            torch.sort(torch.randint(0, R, (E - 1,), generator=g)).values.int()
        bounds = [0] + cut.tolist() + [R]
        kw["offsets"] = torch.tensor(bounds, dtype=torch.int32, device=gpu)
    else:
        w, sw = w[0], sw[0]
    y = qa.fp8_matmul(a, s, w, sw, rows=rows.to(gpu), out_dtype=dtype, **kw)
    assert torch.equal(y, qa.fp8_matmul(a, s, w, sw, rows=rows.to(gpu), out_dtype=dtype, **kw))
    y = y.double()
    at = rows.long().to(gpu)
    A = whole(a.float(), s)[at % R] * (at < R)[:, None]
    loss = (2 * 128 + blocks(K) + 8) * U32
    for e in range(max(E, 1)):
        i, j = bounds[e], bounds[e + 1]
        if j > i:
            W = whole((w[e] if E else w).float(), sw[e] if E else sw, 128)
            want = A[i:j] @ W.T
            off = (y[i:j] - want).abs() - loss * (A[i:j].abs() @ W.abs().T) * (1 + 2.0 ** -8) - U[dtype] * want.abs()
            assert off.max() <= 0, f"{tile}, expert {e}: {off.max().item():.3e} over its tolerance"


@pytest.mark.gpu
def test_matmul_beyond_32_bit_offsets(gpu):
    """Rows, experts and outputs whose byte offsets pass 2^32."""
    K, N = 1024, 32
    A = (1 << 22) + 5
    a = torch.zeros((A, K), dtype=torch.uint8, device=gpu).view(FP8)
    s = torch.ones((A, K // 128), device=gpu)
    g = gen(3)
    few, fs = fp8_rows(g, 3, K)
    w, sw = fp8_weights(g, N, K)
    at = torch.tensor([A - 1, 0, 1 << 22], dtype=torch.int32)
    a.view(torch.uint8)[at.long().to(gpu)] = few.view(torch.uint8).to(gpu)
    s[at.long().to(gpu)] = fs.to(gpu)
    y = qa.fp8_matmul(a, s, w.to(gpu), sw.to(gpu), rows=at.to(gpu))
    check_product(y, few, fs, w, sw, torch.float32, "far rows")
    wide = (1 << 20) // 32 + 40  # 128 x n x 1024 bytes pass 2^32
    big = torch.zeros((128, wide, K), dtype=torch.uint8, device=gpu).view(FP8)
    big.view(torch.uint8)[127, wide - N:] = w.view(torch.uint8).to(gpu)
    bs = torch.ones((128, blocks(wide), K // 128), device=gpu)
    off = torch.zeros(129, dtype=torch.int32)
    off[128] = 3
    y = qa.fp8_matmul(few.to(gpu), fs.to(gpu), big, bs, offsets=off.to(gpu))
    want = whole(few, fs) @ w.double().T
    near(y[:, wide - N:], want, 300 * U32 * (whole(few, fs).abs() @ w.double().abs().T), "far expert")
    assert (y[:, :wide - N] == 0).all()
    del big
    y = qa.fp8_matmul(a, s, w.to(gpu), sw.to(gpu), out_dtype=torch.float32)
    y = torch.cat([y[A - 1:], y[:1], y[1 << 22:(1 << 22) + 1]])
    check_product(y, few, fs, w, sw, torch.float32, "many rows")


# ---- tokens ---------------------------------------------------------------------------------------

ORDERS = [(1, 1, 1, "even"), (1, 8, 8, "even"), (10, 256, 8, "even"), (3, 1024, 2, "even"), (64, 4, 2, "one"), (65, 7, 3, "skew"),
          (500, 64, 6, "skew"), (1000, 33, 10, "even"), (40, 16, 4, "drop"), (1021, 500, 5, "drop"), (17, 64, 64, "even"),
          (4099, 256, 8, "skew")]


def device_order(gpu, idx, E):
    return qa.sort_tokens(idx.to(gpu), E)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,kind", ORDERS + [(20000, 256, 8, "even"), (70001, 3, 2, "drop"), (30000, 1024, 4, "skew"),
                                               (2000, 1024, 3, "drop"), (66000, 256, 8, "even"), (341, 64, 3, "drop"),
                                               (342, 64, 3, "even")])
def test_sort_tokens(gpu, T, E, k, kind):
    idx = routing(gen(T), T, E, k, kind)
    o = device_order(gpu, idx, E)
    for got, want, name in zip((o.offsets, o.rows, o.tokens, o.place), plain_order(idx, E), ("offsets", "rows", "tokens", "place")):
        assert np.array_equal(got.cpu().numpy(), want), name
    assert o.n_experts == E


@pytest.mark.gpu
def test_sort_tokens_many(gpu):
    """33 million assignments, a chunk of many rounds a workgroup; checked on the device."""
    T, k, E = (1 << 23) + 5, 4, 200
    g = torch.Generator(device=gpu).manual_seed(3)
    idx = torch.randint(-1, E + 1, (T, k), generator=g, device=gpu, dtype=torch.int32)
    o = qa.sort_tokens(idx, E)
    flat = idx.view(-1)
    valid = (flat >= 0) & (flat < E)
    counts = torch.bincount(flat[valid].long(), minlength=E)
    assert torch.equal(o.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))
    live = int(o.offsets[E])
    rows = o.rows[:live].long()
    key = flat[rows].long() * (T * k) + rows
    assert (key[1:] > key[:-1]).all() and valid[rows].all()  # by expert, ascending within one: each assignment once
    assert (o.rows[live:] == -1).all() and (o.tokens[live:] == -1).all() and torch.equal(o.tokens[:live].long(), rows // k)
    place = o.place.view(-1)
    assert torch.equal(place[rows], torch.arange(live, device=gpu, dtype=torch.int32)) and (place[~valid] == -1).all()


@pytest.mark.gpu
def test_sort_tokens_ends(gpu):
    """No tokens: the offsets are still written.  All dropped.  A token with one expert twice."""
    o = qa.sort_tokens(torch.zeros((0, 4), dtype=torch.int32, device=gpu), 9)
    assert o.offsets.tolist() == [0] * 10 and o.rows.numel() == 0
    assert qa.gather_tokens(torch.zeros((0, 16), device=gpu), o).shape == (0, 16)
    o = device_order(gpu, torch.full((5, 3), -1, dtype=torch.int32), 4)
    assert o.offsets.tolist() == [0] * 5 and (o.rows == -1).all() and (o.place == -1).all()
    x = torch.ones(5, 6, device=gpu)
    assert (qa.gather_tokens(x, o) == 0).all()
    assert torch.equal(qa.combine_tokens(torch.full((15, 6), math.nan, device=gpu), o, torch.ones(5, 3, device=gpu), residual=x), x)
    dys, dw = qa.combine_tokens_backward(x, torch.full((15, 6), math.nan, device=gpu), o, torch.ones(5, 3, device=gpu))
    assert (dys == 0).all() and (dw == 0).all()
    o = device_order(gpu, torch.tensor([[1, 1], [0, 1]], dtype=torch.int32), 2)
    assert o.rows.tolist() == [2, 0, 1, 3] and o.place.tolist() == [[1, 2], [0, 3]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [1, 33, 128, 2048, 4100])
@pytest.mark.parametrize("T,E,k,kind", ORDERS[:-1])
def test_tokens_there_and_back(gpu, T, E, k, kind, H, dtype):
    g = gen(T + H)
    idx = routing(g, T, E, k, kind)
    offsets, _, tokens, place = plain_order(idx, E)
    o = device_order(gpu, idx, E)
    R, live = T * k, int(offsets[-1])
    x, ys, dxs = (randn(g, n, H).to(dtype) for n in (T, R, R))
    res, dy = randn(g, T, H).to(dtype), randn(g, T, H).to(dtype)
    w = torch.rand(T, k, generator=g)
    xs = qa.gather_tokens(x.to(gpu), o).cpu()
    assert torch.equal(xs[:live], x[torch.tensor(tokens[:live])]) and (xs[live:] == 0).all()
    pl = torch.tensor(place)
    has = (pl >= 0)[:, :, None]
    at = pl.clamp_min(0)
    picked = torch.where(has, ys.double()[at], 0.0)
    terms = w.double()[:, :, None] * picked
    for r in (None, res):
        base = 0.0 if r is None else r.double()
        want = base + terms.sum(1)
        y = qa.combine_tokens(ys.to(gpu), o, w.to(gpu), residual=None if r is None else r.to(gpu))
        size = terms.abs().sum(1) + (0.0 if r is None else r.double().abs())
        near(y, want, (k + 2) * U32 * size + U[dtype] * want.abs(), "combine")
    back = torch.where(has, dxs.double()[at], 0.0)
    near(qa.gather_tokens_backward(dxs.to(gpu), o), back.sum(1), (k + 1) * U32 * back.abs().sum(1) + U[dtype] * back.sum(1).abs(), "dx")
    dys, dw = qa.combine_tokens_backward(dy.to(gpu), ys.to(gpu), o, w.to(gpu))
    want = torch.zeros(R, H, dtype=torch.float64)
    want[pl[has[:, :, 0]]] = (w.double()[:, :, None] * dy.double()[:, None, :])[has[:, :, 0]]
    near(dys, want, (U[dtype] + (U32 if dtype != torch.float32 else 0)) * want.abs(), "dys")
    each = picked * dy.double()[:, None, :]
    near(dw, each.sum(2), (H + 8) * U32 * each.abs().sum(2), "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [1, 3, 5, 9, 131, 1027, 2047])
def test_combine_into_its_residual(gpu, H, dtype):
    """Rows that end inside a 16-byte piece, the output in the residual's place: the same bits as apart."""
    T, k, E = 37, 9, 7
    g = gen(H)
    o = qa.sort_tokens(torch.randint(0, E + 1, (T, k), generator=g, dtype=torch.int32).to(gpu), E)
    ys, r = randn(g, T * k, H).to(dtype).to(gpu), randn(g, T, H).to(dtype).to(gpu)
    w = torch.rand(T, k, generator=g).to(gpu)
    want = qa.combine_tokens(ys, o, w, residual=r)
    for _ in range(3):
        y = r.clone()
        assert qa.combine_tokens(ys, o, w, residual=y, out=y) is y
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_token_gradients_against_differences(gpu):
    """L = <dy, combine(ys, w)> and L = <dxs, gather(x)> are linear in each operand, so a difference over
    any step is its derivative: (L(p + d) - L(p - d)) / 2 = <grad, d>, to the roundings of the two L."""
    g = gen(11)
    T, E, k, H = 37, 9, 3, 130
    o = device_order(gpu, routing(g, T, E, k, "drop"), E)
    x, dx_ = randn(g, T, H).to(gpu), randn(g, T, H).to(gpu)
    ys, dys_, dxs = (randn(g, T * k, H).to(gpu) for _ in range(3))
    w, dw_ = torch.rand(T, k, generator=g).to(gpu), randn(g, T, k).to(gpu)
    dy = randn(g, T, H).to(gpu)

    def loss(m, n):
        return (m.double() * n.double()).sum().item()

    def size(m, n):
        return (m.double().abs() * n.double().abs()).sum().item()

    gys, gw = qa.combine_tokens_backward(dy, ys, o, w)
    gx = qa.gather_tokens_backward(dxs, o)
    for f, p, d, grad, up in ((lambda v: qa.combine_tokens(v, o, w), ys, dys_, gys, dy),
                              (lambda v: qa.combine_tokens(ys, o, v), w, dw_, gw, dy),
                              (lambda v: qa.gather_tokens(v, o), x, dx_, gx, dxs)):
        hi, lo = p + d, p - d
        slope = (loss(up, f(hi)) - loss(up, f(lo))) / 2
        # p + d and p - d round once each, the sums of a forward k + 2 times, those of a gradient H + 8 times
        tol = (H + 2 * k + 16) * U32 * (size(up, f(hi)) + size(up, f(lo)) + size(grad, d) + size(grad, p)) * 4
        assert abs(slope - loss(grad, d)) <= tol


@pytest.mark.gpu
def test_token_outputs_given(gpu):
    """Outputs in the caller's buffers, the sum into its residual; orders made by hand are checked."""
    g = gen(6)
    o = device_order(gpu, routing(g, 30, 8, 2), 8)
    x, ys, w = randn(g, 30, 72).to(gpu), randn(g, 60, 72).to(gpu), torch.rand(30, 2, generator=g).to(gpu)
    buf = torch.empty(60, 72, device=gpu)
    assert qa.gather_tokens(x, o, out=buf) is buf and torch.equal(buf, qa.gather_tokens(x, o))
    want = qa.combine_tokens(ys, o, w, residual=x)
    res = x.clone()
    assert qa.combine_tokens(ys, o, w, residual=res, out=res) is res and torch.equal(res, want)
    back = torch.empty(30, 72, device=gpu)
    assert qa.gather_tokens_backward(ys, o, out=back) is back
    assert torch.equal(back, qa.combine_tokens(ys, o, torch.ones(30, 2, device=gpu)))
    again = TokenOrder(o.offsets, o.rows, o.tokens, o.place)
    assert torch.equal(qa.gather_tokens(x, again), buf) and again.n_experts == 8
    for bad in ((o.offsets.long(), o.rows, o.tokens, o.place), (o.offsets[:1], o.rows, o.tokens, o.place),
                (o.offsets, o.rows[:-1], o.tokens, o.place), (o.offsets, o.rows, o.tokens.cpu(), o.place),
                (o.offsets, o.rows, o.tokens, o.place.t()), (o.offsets, o.rows, o.tokens, o.place.view(-1))):
        with pytest.raises(ValueError, match="expected"):
            TokenOrder(*bad)
    with pytest.raises(ValueError, match="order expected"):
        qa.gather_tokens(x, (o.offsets, o.place))
    for out in (ys[:30], ys[7:37], ys[30:]):
        with pytest.raises(qa.QmoeError, match="y expected a buffer distinct from ys, got an overlapping one"):
            qa.combine_tokens(ys, o, w, out=out)
    both = torch.zeros(40, 72, device=gpu)
    with pytest.raises(qa.QmoeError, match="distinct from residual"):
        qa.combine_tokens(ys, o, w, residual=both[:30], out=both[10:])
    with pytest.raises(qa.QmoeError, match="distinct from x"):
        qa.residual_norm(both[:30], both[10:], None, 1e-6, out=both[5:35])


@pytest.mark.gpu
def test_gather_fp8_rows_and_scales(gpu):
    g = gen(5)
    idx = routing(g, 50, 8, 3, "drop")
    o = device_order(gpu, idx, 8)
    for C in (64, 100, 7):
        q, s = fp8_rows(g, 50, C)
        live = int(o.offsets[-1])
        at = o.tokens[:live].long().cpu()
        got = qa.gather_tokens(q.to(gpu), o).cpu().view(torch.uint8)
        assert torch.equal(got[:live], q.view(torch.uint8)[at]) and (got[live:] == 0).all()
        assert torch.equal(qa.gather_tokens(s.to(gpu), o).cpu()[:live], s[at])


@pytest.mark.gpu
def test_token_index_values(gpu):
    """Places outside the rows are skipped, never followed."""
    place = torch.tensor([[0, -7], [2 ** 31 - 1, 3], [-2 ** 31, 6]], dtype=torch.int32, device=gpu)
    rows = torch.zeros(6, dtype=torch.int32, device=gpu)
    o = TokenOrder(torch.tensor([0, 6], dtype=torch.int32, device=gpu), rows, rows, place)
    ys = torch.arange(6, device=gpu).float()[:, None].repeat(1, 8) + 1
    y = qa.combine_tokens(ys, o, torch.ones(3, 2, device=gpu))
    assert y[:, 0].tolist() == [1.0, 4.0, 0.0]
    xs = torch.full((6, 8), 9.0, device=gpu)
    qa.gather_tokens(torch.tensor([[1.0], [2.0], [3.0]], device=gpu).repeat(1, 8), o, out=xs)
    assert xs[:, 0].tolist() == [1.0, 9.0, 9.0, 2.0, 9.0, 9.0]
    dys, dw = qa.combine_tokens_backward(torch.ones(3, 8, device=gpu), ys, o, torch.ones(3, 2, device=gpu))
    assert dw.tolist() == [[8.0, 0.0], [0.0, 32.0], [0.0, 0.0]]


@pytest.mark.gpu
def test_tokens_beyond_32_bit_offsets(gpu):
    T, H, k = (1 << 20) + 3, 1024, 2  # 2 T rows of 2048 bytes pass 2^32
    idx = torch.stack([torch.arange(T) % 3, torch.arange(T) % 3], 1).to(torch.int32)
    o = device_order(gpu, idx, 3)
    x = (torch.arange(T, device=gpu) % 251).to(torch.bfloat16)[:, None].repeat(1, H)
    xs = qa.gather_tokens(x, o)
    assert torch.equal(xs[:, 5], x[o.tokens.long(), 5]) and torch.equal(xs[:, H - 1], x[o.tokens.long(), 5])
    y = qa.combine_tokens(xs, o, torch.full((T, k), 0.5, device=gpu))
    assert torch.equal(y, x)
    dys, dw = qa.combine_tokens_backward(torch.ones_like(x), xs, o, torch.full((T, k), 0.5, device=gpu))
    assert (dys == 0.5).all() and torch.equal(dw[:, 1], x[:, 0].float() * H)


# ---- norms ---------------------------------------------------------------------------------------

def plain_norm(x, y, w, eps, post_w=None, gate=None, gate_act=None, scale=1.0):
    """(x', h, error of x', error of h) in 64 bits; the errors bound the f32 roundings behind them."""
    x = x.double()
    ex = torch.zeros_like(x)
    if y is not None:
        u, n = y.double(), 1
        if post_w is not None:
            u = u / torch.sqrt((u * u).mean(1, keepdim=True) + eps) * post_w.double()
            n += 7  # the mean, the sum with eps, the root, the quotient, two products; squares half as much
        if gate is not None:
            gd = gate.double()
            u = u * torch.sigmoid(gd) * (gd if gate_act == "silu" else 1.0)
            n = n + 8 + gd.abs()  # exp(-g) carries |g| roundings of its argument
        u = u * (scale.double() if isinstance(scale, torch.Tensor) else scale)
        x = x + u
        ex = (n + 2) * U32 * u.abs() + U32 * x.abs()
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    wd = 1.0 if w is None else w.double()
    h = x * r * wd
    # the root mean square is off by at most x's own relative error in the 2-norm, and its roundings
    off = ex.norm(dim=1, keepdim=True) / x.norm(dim=1, keepdim=True).clamp_min(1e-300)
    eh = (ex * r + (x * r).abs() * (off + 8 * U32)) * (wd if isinstance(wd, float) else wd.abs())
    return x, h, ex, eh


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("post,gate,vector,quantize", [(False, None, False, False), (True, None, True, True),
                                                       (False, "sigmoid", False, True), (True, "silu", True, False),
                                                       (True, "sigmoid", True, True)])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 2048), (3, 127), (5, 129), (10, 2816), (4, 4096), (7, 8191), (2, 16384),
                                 (65, 64), (300, 1000), (2, 5120)])
def test_residual_norm(gpu, T, H, post, gate, vector, quantize, dtype):
    g = gen(T * 7 + H)
    x, y, gt = (randn(g, T, H).to(dtype) for _ in range(3))
    w, pw = 1 + 0.2 * randn(g, H), 1 + 0.2 * randn(g, H)
    scale = 0.5 + 0.2 * randn(g, H) if vector else 0.7
    kw = dict(post_w=pw if post else None, gate=gt if gate else None, gate_act=gate, scale=scale)
    # f32 of 0.7 is what the call takes
    want_x, want_h, ex, eh = plain_norm(x, y, w, 1e-6, **{**kw, "scale": scale if vector else float(np.float32(0.7))})
    n = qa.residual_norm(x.to(gpu), y.to(gpu), w.to(gpu), 1e-6, quantize=quantize,
                         **{a: v.to(gpu) if isinstance(v, torch.Tensor) else v for a, v in kw.items()})
    assert isinstance(n, NormOut) and (n.q is not None) == quantize
    u = 0.0 if dtype == torch.float32 else U[dtype]
    near(n.x, want_x, ex + u * want_x.abs() * (1 + 2.0 ** -8), "x")
    near(n.h, want_h, eh + U32 * want_h.abs() + u * want_h.abs() * (1 + 2.0 ** -8), "h")
    if quantize:
        err = float(((eh + U32 * want_h.abs()) / want_h.abs().clamp_min(1e-3)).max())
        ss = n.q_scale.cpu().double().repeat_interleave(128, 1)[:, :H]
        near(n.q.cpu().double() * ss, want_h, 2.0 ** -4 * (1 + 2.0 ** -9) * want_h.abs() + 2.0 ** -10 * (1 + 2.0 ** -9) * ss + 2 * eh, "q")
        b = blocks(H)
        pad = torch.zeros(T, b * 128, dtype=torch.float64)
        pad[:, :H] = want_h.abs()
        m = pad.view(T, b, 128).amax(2)
        near(n.q_scale, m / 448, (err + 3 * U32) * m / 448 + 1e-38, "q_scale")
        if dtype == torch.float32:  # the bits of the operator by itself
            q, s = qa.fp8_quantize(n.h)
            assert torch.equal(q.view(torch.uint8), n.q.view(torch.uint8)) and torch.equal(s, n.q_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mag,eps", [(1e25, 1e-6), (3e38, 1e-6), (2e19, 0.0), (1e-25, 0.0), (2e-38, 0.0), (1e-17, 1e-38),
                                     (1e-25, 1e-6), (1e-20, 1e-38), (1.0, 3e38)])
@pytest.mark.parametrize("T,H", [(3, 1), (5, 200), (4, 2816), (2, 16384)])
def test_residual_norm_magnitudes(gpu, T, H, mag, eps, dtype):
    """Rows whose squares leave f32's range, in the residual rows and before the norm after the block; a row of each beside
    ordinary ones, which keep their bits."""
    g = gen(T + H)
    big = ((2 * torch.rand(T, H, generator=g) - 1) * mag).to(dtype)
    big[:, 0] = mag
    one, w = randn(g, T, H).to(dtype), 1 + 0.2 * randn(g, H)
    eps = float(np.float32(eps))  # what the call takes
    u = 0.0 if dtype == torch.float32 else U[dtype]
    rows = one.clone()
    rows[::2] = big[::2]
    n = qa.residual_norm(rows.to(gpu), None, w.to(gpu), eps, quantize=True)
    _, want, _, eh = plain_norm(rows, None, w, eps)
    tiny = 2.0 ** -149  # (f32's and bf16's smallest steps: 2^-149, 2^-133)
    near(n.h, want, eh + (U32 + u * (1 + 2.0 ** -8)) * want.abs() + (tiny if dtype == torch.float32 else 2.0 ** -133), "h")
    assert torch.equal(n.h[1::2].cpu(), qa.residual_norm(one.to(gpu), None, w.to(gpu), eps).h[1::2].cpu())
    y = one.clone()
    y[::2] = big[::2]
    n = qa.residual_norm(one.to(gpu), y.to(gpu), w.to(gpu), eps, post_w=w.to(gpu), scale=0.5)
    yd = y.double()
    v = 0.5 * yd / torch.sqrt((yd * yd).mean(1, keepdim=True) + eps) * w.double()
    want = one.double() + v
    near(n.x, want, 12 * U32 * v.abs() + (U32 + u * (1 + 2.0 ** -8)) * want.abs() + tiny, "x")


@pytest.mark.gpu
def test_residual_norm_alone_and_in_place(gpu):
    g = gen(2)
    x, y, w = randn(g, 9, 777), randn(g, 9, 777), randn(g, 777)
    dx, dy = x.to(gpu), y.to(gpu)
    n = qa.residual_norm(dx, None, w.to(gpu), 1e-5, quantize=True)
    _, want, _, eh = plain_norm(x, None, w, 1e-5)
    near(n.h, want, eh + U32 * want.abs(), "h")
    assert n.x.data_ptr() == dx.data_ptr() and torch.equal(dx.cpu(), x)
    first = qa.residual_norm(dx, dy, w.to(gpu), 1e-5, scale=0.25)
    assert torch.equal(qa.residual_norm(dx, None, None, 1e-5).h, qa.rms_norm(dx, None, 1e-5))
    for target in ("x", "y"):
        a, b = dx.clone(), dy.clone()
        m = qa.residual_norm(a, b, w.to(gpu), 1e-5, scale=0.25, out=a if target == "x" else b)
        assert m.x is (a if target == "x" else b) and torch.equal(m.x, first.x) and torch.equal(m.h, first.h)
    z = torch.zeros(3, 130, device=gpu)
    n = qa.residual_norm(z, z.clone(), None, 1e-6, post_w=torch.ones(130, device=gpu), quantize=True)
    assert (n.x == 0).all() and (n.h == 0).all() and (n.q.float() == 0).all()


@pytest.mark.gpu
def test_residual_norm_gate_ends(gpu):
    """Gates at the ends: an infinite or far negative gate closes it, a far positive one opens it; a NaN row stays alone."""
    y = torch.full((4, 256), 2.0)
    x = torch.ones(4, 256)
    gate = torch.zeros(4, 256)
    gate[0], gate[1], gate[2] = -1000.0, 1000.0, -math.inf
    y[3, 9] = math.nan
    for act in ("sigmoid", "silu"):
        n = qa.residual_norm(x.to(gpu), y.to(gpu), None, 1e-6, gate=gate.to(gpu), gate_act=act).x.cpu()
        assert (n[0] == 1).all() and (n[1] == (3 if act == "sigmoid" else 2001)).all()
        assert (n[2] == 1).all() if act == "sigmoid" else True
        assert torch.isnan(n[3, 9]) and torch.isfinite(n[3, :9]).all()
    h = qa.residual_norm(x.to(gpu), y.to(gpu), None, 1e-6).h.cpu()
    assert torch.isnan(h[3]).all() and torch.isfinite(h[:3]).all()


# ---- strides, streams, graphs ----------------------------------------------------------------------

@pytest.mark.gpu
def test_strided_operands_and_other_alignments(gpu):
    g = gen(21)
    big = randn(g, 40, 600).to(gpu)
    for x in (big[:, 3:259], big[::2, :256], big.t()[:256], big[:, 1:130]):
        q, s = qa.fp8_quantize(x)
        q2, s2 = qa.fp8_quantize(x.clone(memory_format=torch.contiguous_format))
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    flat = randn(g, 4 * 256 + 8).to(gpu)
    for off in (0, 1, 2, 3):  # rows that start at 4-byte steps
        x = flat[off:off + 4 * 256].view(4, 256)
        q, s = qa.fp8_quantize(x)
        wq, wsc = plain_quantize(x.cpu())
        assert torch.equal(q.cpu().view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s.cpu(), wsc)
        n = qa.residual_norm(x, x.clone(), None, 1e-6)
        m = qa.residual_norm(x.clone(), x.clone(), None, 1e-6)
        assert torch.equal(n.x, m.x) and torch.equal(n.h, m.h)
        o = qa.sort_tokens(torch.tensor([[0, 1], [1, 0], [0, 1], [1, 0]], dtype=torch.int32, device=gpu), 2)
        assert torch.equal(qa.gather_tokens(x, o), x[o.tokens.long()])
        ys = x.repeat(2, 1)
        assert torch.equal(qa.combine_tokens(ys[:, 1:], o, torch.ones(4, 2, device=gpu)),
                           qa.combine_tokens(ys, o, torch.ones(4, 2, device=gpu))[:, 1:])
    a, sa = fp8_rows(g, 24, 512)
    w, sw = fp8_weights(g, 64, 256)
    a = a.to(gpu)
    y = qa.fp8_matmul(a[::2, 256:], sa.to(gpu)[::2, 2:], w.to(gpu), sw.to(gpu))
    check_product(y, a.cpu()[::2, 256:], sa[::2, 2:], w, sw, torch.float32)
    odd = torch.empty(12 * 64 + 1, device=gpu)[1:].view(12, 64)  # rows that start 4 bytes off
    assert torch.equal(qa.fp8_matmul(a[::2, 256:], sa.to(gpu)[::2, 2:], w.to(gpu), sw.to(gpu), out=odd), y)


def block_inputs(g, T, H, F, E, k, dtype, dev):
    x, y = (randn(g, T, H).to(dtype).to(dev) for _ in range(2))
    wn = (1 + 0.1 * randn(g, H)).to(dev)
    gu, sgu = (t.to(dev) for t in fp8_weights(g, E, 2 * F, H))
    dn, sdn = (t.to(dev) for t in fp8_weights(g, E, H, F))
    idx = routing(g, T, E, k).to(dev)
    w = torch.softmax(randn(g, T, k), 1).to(dev)
    return x, y, wn, gu, sgu, dn, sdn, idx, w


def block(x, y, wn, gu, sgu, dn, sdn, idx, w, stream=None):
    """One feed-forward as a user of the operators runs it: (x', the experts' sum)."""
    n = qa.residual_norm(x, y, wn, 1e-6, quantize=True, stream=stream)
    o = qa.sort_tokens(idx, gu.shape[0], stream=stream)
    h = qa.fp8_matmul(n.q, n.q_scale, gu, sgu, offsets=o.offsets, rows=o.tokens, out_dtype=x.dtype, stream=stream)
    q, s = qa.fp8_quantize(h, act="swiglu", stream=stream)
    ys = qa.fp8_matmul(q, s, dn, sdn, offsets=o.offsets, out_dtype=x.dtype, stream=stream)
    return n.x, qa.combine_tokens(ys, o, w, stream=stream)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,F,E,k", [(1, 256, 128, 8, 2), (13, 512, 96, 16, 4), (150, 384, 256, 4, 2)])
def test_block(gpu, T, H, F, E, k, dtype):
    """The operators together against the same feed-forward in 64 bits.  Both quantizations are off by up
    to half an e4m3 step per value (2^-4 of it), independently over a row's values: of a sum of n terms a
    value's share is 1 / sqrt(n), so the rows are compared in the 2-norm, where the first moves the result
    by at most 2^-4 through the gate and again through the up half, the second by 2^-4: 3 2^-4, and the
    types' own roundings on top."""
    x, y, wn, gu, sgu, dn, sdn, idx, w = (t.cpu() for t in block_inputs(gen(T), T, H, F, E, k, dtype, "cpu"))
    xo, got = block(*(t.to(gpu) for t in (x, y, wn, gu, sgu, dn, sdn, idx, w)))
    wx, h, ex, _ = plain_norm(x, y, wn, 1e-6)
    near(xo, wx, ex + U[dtype] * wx.abs() * (1 + 2.0 ** -8), "x")
    G, D = whole(gu, sgu, 128), whole(dn, sdn, 128)
    want = torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            e = int(idx[t, j])
            z = G[e] @ h[t]
            want[t] += w[t, j].double() * (D[e] @ (z[:F] * torch.sigmoid(z[:F]) * z[F:]))
    off = (got.cpu().double() - want).norm(dim=1) / want.norm(dim=1)
    assert off.max() <= 3 * 2.0 ** -4 + 8 * U[dtype], off.max()


@pytest.mark.gpu
def test_other_stream_and_same_bits(gpu):
    args = block_inputs(gen(4), 40, 256, 128, 8, 2, torch.float32, gpu)
    first = block(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    second = block(*args, stream=side)
    with torch.cuda.stream(side):
        third = block(*args)
    side.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    dy = torch.randn(40, 256, device=gpu)
    ys = torch.randn(80, 256, device=gpu)
    o = qa.sort_tokens(args[7], 8)
    one = qa.combine_tokens_backward(dy, ys, o, args[8])
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(one, qa.combine_tokens_backward(dy, ys, o, args[8])))


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """Blocks on two streams with nothing between them give what they give one after the other."""
    both = [block_inputs(gen(s), 130, 512, 256, 16, 4, dt, gpu) for s, dt in ((14, torch.bfloat16), (15, torch.float32))]
    want = [block(*args) for args in both]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    got = [[block(*args, stream=stream) for args, stream in zip(both, streams)] for _ in range(10)]
    torch.cuda.synchronize()
    for pair in got:
        for a, b in zip(pair, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_streams_and_devices_without_torchs_bindings(gpu, monkeypatch):
    """The stream handle is the current stream's, by either way to it; with another device current the operands' own is
    set for the launch."""
    from qwenium_amd import ops
    x = randn(gen(5), 9, 300).to(gpu)
    want = qa.fp8_quantize(x)[0].view(torch.uint8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            assert ops._raw_stream(0) == stream.cuda_stream and ops._current_device() == 0
    monkeypatch.setattr(ops, "_raw_stream", lambda i: torch.cuda.current_stream(i).cuda_stream)
    monkeypatch.setattr(ops, "_current_device", lambda: 1)
    assert torch.equal(qa.fp8_quantize(x)[0].view(torch.uint8), want)
    with torch.cuda.stream(side):
        got = qa.fp8_quantize(x)[0].view(torch.uint8)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 200])
def test_graph_replays(gpu, T):
    """Two captured blocks, replayed in turn on changed inputs with eager work between: the eager results."""
    def make(seed):
        args = block_inputs(gen(seed), T, 256, 128, 8, 2, torch.bfloat16, gpu)
        warm = torch.cuda.Stream()
        warm.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(warm):
            block(*args)
        torch.cuda.current_stream().wait_stream(warm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(*args)
        return args, graph, out

    both = [make(1), make(2)]
    g = gen(9)
    for step in range(4):
        for args, graph, out in both:
            args[0].copy_(randn(g, T, 256))
            args[7].copy_(routing(g, T, 8, 2, "drop" if step == 2 else "even"))
        for _, graph, _ in both:
            graph.replay()
        torch.cuda.synchronize()
        for args, _, out in both:
            for a, b in zip(out, block(*args)):
                assert torch.equal(a, b)
