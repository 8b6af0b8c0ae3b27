"""The operators around and inside a mixture-of-experts feed-forward whose expert weights are
8-bit floats, as cases that can be timed and checked.

A case's "op":
  product   rows in e4m3 (one f32 scale per row and block of 128 columns) times weights in e4m3 (one f32
            scale per block of 128 x 128): fp8_matmul. experts 0: one weight matrix and `rows` rows (a linear
            projection); otherwise each of `rows` tokens goes to `top_k` of `experts` matrices, the rows
            grouped by expert, read through the token index ("gather": the gate/up projection) or in place (the
            down projection). n, k: the weight's rows and columns; out: the output's type
  quantize  rows to e4m3 with their scales: fp8_quantize. act: nothing, or the SwiGLU / GeGLU of (gate, up) halves
  order     tokens sorted by expert and back: sort_tokens, gather_tokens, combine_tokens; train: also the
            gradients (of the gathered rows, of the experts' outputs and of the weights)
  norm      residual_norm: a block's output normed and gated, the scaled residual add, and the next
            block's normed input, quantize: in e4m3 too

skew: a few experts take most of the tokens.
"""
import math

import torch

own = False

BLOCK = 128
EPS = 1e-6
TOP = 448.0       # the largest e4m3 value
TINY = 1e-30      # the smallest block maximum that sets a scale
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


def _product(name, experts, top_k, rows, n, k, out, gather=False, skew=False):
    return {"name": name, "op": "product", "experts": experts, "top_k": top_k, "rows": rows, "n": n, "k": k,
            "out": out, "gather": gather, "skew": skew}


def listed():
    return [
        # one user's decode step on the 256-expert layer: 8 experts' gate and up matrices
        _product("experts decode 1", 256, 8, 1, 1024, 2048, "f32", gather=True),
        # ten users' decode step: about 70 experts' matrices for 80 rows
        _product("experts decode 10", 256, 8, 10, 1024, 2048, "bf16", gather=True),
        # a short prompt's down projection, 13 rows per expert, 5.5 blocks of 128 columns
        _product("experts down 211", 128, 8, 211, 2816, 704, "f32"),
        # a long prompt's gate/up projection: every expert, 128 rows each
        _product("experts prompt 4096", 256, 8, 4096, 1024, 2048, "bf16", gather=True),
        # a linear projection of a long batch: bound by arithmetic
        _product("linear 8192", 0, 1, 8192, 4096, 4096, "bf16"),
        # the activations of a prompt in the layer's own type
        {"name": "quantize prompt", "op": "quantize", "rows": 4096, "cols": 2048, "in": "f32", "act": "none"},
        # between gate/up and down of a long prompt: 32768 rows
        {"name": "quantize swiglu", "op": "quantize", "rows": 32768, "cols": 512, "in": "bf16", "act": "swiglu"},
        # a decode batch: three launches, latency
        {"name": "order decode 10", "op": "order", "tokens": 10, "top_k": 8, "experts": 256, "hidden": 2048,
         "in": "f32", "train": False, "skew": False},
        # a long prompt
        {"name": "order prompt 4096", "op": "order", "tokens": 4096, "top_k": 8, "experts": 256, "hidden": 2048,
         "in": "bf16", "train": False, "skew": False},
        # a fine-tuning step's tokens with routing as unbalanced as trained models show it
        {"name": "order train 2000", "op": "order", "tokens": 2000, "top_k": 6, "experts": 64, "hidden": 1536,
         "in": "f32", "train": True, "skew": True},
        # a decode batch before its experts, with the e4m3 rows that they read
        {"name": "norm decode 10", "op": "norm", "tokens": 10, "hidden": 2048, "in": "f32", "post": False,
         "gate": "none", "vector": False, "quantize": True},
        # a prompt between two blocks with norms on both sides, a gate and a scale per column
        {"name": "norm prompt 4096", "op": "norm", "tokens": 4096, "hidden": 2816, "in": "bf16", "post": True,
         "gate": "sigmoid", "vector": True, "quantize": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("product", "product", "quantize", "order", "norm"))
    if op == "product":
        k = 16 * _log(rng, 4, 256)
        n = _log(rng, 33, 4096)
        out = rng.choice(("f32", "bf16"))
        if rng.random() < 0.3:
            rows = _log(rng, 1, 8192)
            return {"op": op, "experts": 0, "top_k": 1, "rows": rows, "n": n, "k": k, "out": out, "gather": False,
                    "skew": False}
        experts = _log(rng, 4, 256)
        top_k = rng.randint(1, min(8, experts))
        rows = _log(rng, 1, 4096)
        experts = max(4, min(experts, 256 * 1024 * 2048 // (n * k)))
        top_k = min(top_k, experts)
        rows = max(1, min(rows, 4096 * 8 * 1024 * 2048 // (top_k * n * k)))
        return {"op": op, "experts": experts, "top_k": top_k, "rows": rows, "n": n, "k": k, "out": out,
                "gather": rng.random() < 0.5, "skew": rng.random() < 0.25}
    if op == "quantize":
        cols = _log(rng, 32, 8192)
        rows = min(_log(rng, 1, 32768), 32768 * 512 // cols + 1)
        return {"op": op, "rows": rows, "cols": cols, "in": rng.choice(("f32", "bf16")),
                "act": rng.choice(("none", "swiglu", "geglu"))}
    if op == "order":
        experts = _log(rng, 4, 512)
        top_k = rng.randint(1, min(10, experts))
        hidden = _log(rng, 128, 4096)
        tokens = max(1, min(_log(rng, 1, 8192), 4096 * 8 * 2048 // (top_k * hidden)))
        return {"op": op, "tokens": tokens, "top_k": top_k, "experts": experts, "hidden": hidden,
                "in": rng.choice(("f32", "bf16")), "train": rng.random() < 0.4, "skew": rng.random() < 0.4}
    hidden = _log(rng, 64, 8192)
    tokens = max(1, min(_log(rng, 1, 8192), 4096 * 2816 // hidden))
    return {"op": op, "tokens": tokens, "hidden": hidden, "in": rng.choice(("f32", "bf16")),
            "post": rng.random() < 0.5, "gate": rng.choice(("none", "sigmoid", "silu")),
            "vector": rng.random() < 0.5, "quantize": rng.random() < 0.5}


def _blocks(n):
    return -(-n // BLOCK)


# ---- inputs ----------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _routing(g, tokens, experts, top_k, skew):
    """(ids [T, k] int32 in the order of falling logits, softmax weights [T, k])."""
    logits = _randn(g, tokens, experts)
    if skew:  # half of the tokens' choices on an eighth of the experts
        bias = -0.7 * torch.log(torch.arange(1, experts + 1, device="cuda").float())
        logits = logits + bias[torch.randperm(experts, generator=g, device="cuda")]
    top = torch.topk(logits, top_k, dim=1)
    return top.indices.to(torch.int32), torch.softmax(top.values, dim=1)


def _activations(g, rows, cols):
    """Rows as a model has them: unit columns, a few of them far larger."""
    x = _randn(g, rows, cols)
    return x * (1 + 15 * (torch.rand(cols, generator=g, device="cuda") < 0.01))


def _fp8_rows(g, rows, cols):
    x = _activations(g, rows, cols)
    return _quantize(x)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "product":
        e, n, k = case["experts"], case["n"], case["k"]
        s["a"], s["a_scale"] = _fp8_rows(g, case["rows"] * (1 if case["gather"] else case["top_k"]), k)
        # weights N(0, 0.02): a block's largest value maps to 448, a value's spread to about 100
        w = torch.empty((max(1, e), n, k), dtype=torch.float8_e4m3fn, device="cuda")
        for i in range(max(1, e)):
            w[i] = (100 * _randn(g, n, k)).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
        sw = 2e-4 * (0.8 + 0.4 * torch.rand((max(1, e), _blocks(n), _blocks(k)), generator=g, device="cuda"))
        rows = case["rows"] * case["top_k"]
        s["out"] = torch.empty((rows, n), dtype=DTYPES[case["out"]], device="cuda")
        if not e:
            s["w"], s["w_scale"] = w[0], sw[0]
            return s
        s["w"], s["w_scale"] = w, sw
        ids, _ = _routing(g, case["rows"], e, case["top_k"], case["skew"])
        offsets, order, _ = _sorted(ids, e)
        s["offsets"] = offsets
        s["rows"] = (order // case["top_k"]).to(torch.int32) if case["gather"] else None
        s["most"] = int((offsets[1:] - offsets[:-1]).max())  # the plain form's padded length
    elif case["op"] == "quantize":
        cols = case["cols"] * (1 if case["act"] == "none" else 2)
        s["x"] = _activations(g, case["rows"], cols).to(DTYPES[case["in"]])
        s["q"] = torch.empty((case["rows"], case["cols"]), dtype=torch.float8_e4m3fn, device="cuda")
        s["scale"] = torch.empty((case["rows"], _blocks(case["cols"])), dtype=torch.float32, device="cuda")
    elif case["op"] == "order":
        t, k, h, dt = case["tokens"], case["top_k"], case["hidden"], DTYPES[case["in"]]
        s["ids"], s["weights"] = _routing(g, t, case["experts"], k, case["skew"])
        s["x"] = _randn(g, t, h).to(dt)
        s["ys"] = (0.1 * _randn(g, t * k, h)).to(dt)  # what the experts make of the sorted rows
        s["residual"] = _randn(g, t, h).to(dt)
        if case["train"]:
            s["dy"] = (0.01 * _randn(g, t, h)).to(dt)
            s["dxs"] = (0.01 * _randn(g, t * k, h)).to(dt)
    else:
        t, h, dt = case["tokens"], case["hidden"], DTYPES[case["in"]]
        s["x"] = _activations(g, t, h).to(dt)
        s["y"] = (0.3 * _randn(g, t, h)).to(dt)
        s["w"] = 1 + 0.1 * _randn(g, h)
        s["post_w"] = 1 + 0.1 * _randn(g, h) if case["post"] else None
        s["gate"] = _randn(g, t, h).to(dt) if case["gate"] != "none" else None
        s["scale"] = 0.5 + 0.1 * _randn(g, h) if case["vector"] else 0.75
    return s


# ---- the plain forms: 32 bits, rounded once ------------------------------------------------------------

def _quantize(v):
    """v [R, C] f32 -> (e4m3 [R, C], scales [R, blocks])."""
    rows, cols = v.shape
    b = _blocks(cols)
    v = torch.nn.functional.pad(v, (0, b * BLOCK - cols)).view(rows, b, BLOCK)
    top = v.abs().amax(2).clamp_min(TINY)
    q = (v * (TOP / top)[:, :, None]).to(torch.float8_e4m3fn)
    return q.view(rows, b * BLOCK)[:, :cols].contiguous(), top / TOP


def _activate(x, act):
    x = x.float()
    if act == "none":
        return x
    g, u = x.chunk(2, dim=1)
    if act == "swiglu":
        return g / (1 + torch.exp(-g)) * u
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))) * u


def _whole(q, scale, rows_per_scale):
    """The values that e4m3 numbers and their block scales stand for, in f32."""
    n, k = q.shape[-2:]
    s = scale.repeat_interleave(BLOCK, dim=-1)[..., :k]
    if rows_per_scale > 1:
        s = s.repeat_interleave(rows_per_scale, dim=-2)[..., :n, :]
    return q.float() * s


def _sorted(ids, experts):
    """(offsets [E + 1], assignments in the experts' order, each assignment's place in it), int32."""
    flat = ids.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    bounds = torch.searchsorted(flat[order], torch.arange(experts + 1, device=ids.device))
    return bounds.to(torch.int32), order.to(torch.int32), place.view(ids.shape).to(torch.int32)


def _plain_product(s):
    case = s["case"]
    a = _whole(s["a"], s["a_scale"], 1)
    dt = DTYPES[case["out"]]
    if not case["experts"]:
        return (a @ _whole(s["w"], s["w_scale"], BLOCK).t()).to(dt)
    offsets, rows = s["offsets"].long(), case["rows"] * case["top_k"]
    r = torch.arange(rows, device=a.device)
    e = torch.searchsorted(offsets[1:], r, right=True)
    if rows <= case["experts"]:  # each row's own matrix: no more than all of them
        w = _whole(s["w"].view(torch.uint8)[e].view(torch.float8_e4m3fn), s["w_scale"][e], BLOCK)
        return torch.bmm(w, (a[s["rows"].long()] if case["gather"] else a)[:, :, None])[:, :, 0].to(dt)
    w = _whole(s["w"], s["w_scale"], BLOCK)
    at = (offsets[:-1, None] + torch.arange(s["most"], device=a.device)).clamp_max(rows - 1)
    padded = a[s["rows"].long()[at] if case["gather"] else at]
    y = torch.bmm(padded, w.transpose(1, 2).contiguous())
    return y[e, r - offsets[e]].to(dt)


def _plain_order(s):
    case = s["case"]
    t, k, dt = case["tokens"], case["top_k"], DTYPES[case["in"]]
    offsets, order, place = _sorted(s["ids"], case["experts"])
    tokens = order // k
    xs = s["x"][tokens.long()]
    at = place.long()
    rows = s["ys"][at].float()
    y = (s["residual"].float() + (s["weights"][:, :, None] * rows).sum(1)).to(dt)
    got = {"offsets": offsets, "rows": order, "place": place, "xs": xs, "y": y}
    if case["train"]:
        dy = s["dy"].float()
        got["dx"] = s["dxs"][at].float().sum(1).to(dt)
        dys = (s["weights"][:, :, None] * dy[:, None, :]).to(dt)
        got["dys"] = dys.reshape(t * k, -1)[order.long()]
        got["dw"] = (rows * dy[:, None, :]).sum(2)
    return got


def _rms(v):
    return v / torch.sqrt(v.square().mean(1, keepdim=True) + EPS)


def _plain_norm(s):
    case = s["case"]
    dt = DTYPES[case["in"]]
    y = s["y"].float()
    if case["post"]:
        y = _rms(y) * s["post_w"]
    if case["gate"] != "none":
        g = s["gate"].float()
        y = y / (1 + torch.exp(-g)) * (g if case["gate"] == "silu" else 1.0)
    x = s["x"].float() + s["scale"] * y
    h = _rms(x) * s["w"]
    got = {"x": x.to(dt), "h": h.to(dt)}
    if case["quantize"]:
        got["q"], got["scale"] = _quantize(h)
    return got


# ---- one pass ------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        import qwenium_amd as qa
        if op == "product":
            return qa.fp8_matmul(s["a"], s["a_scale"], s["w"], s["w_scale"], offsets=s.get("offsets"),
                                 rows=s.get("rows"), out=s["out"])
        if op == "quantize":
            q, scale = qa.fp8_quantize(s["x"], act=None if case["act"] == "none" else case["act"], q=s["q"],
                                       scale=s["scale"])
            return {"q": q, "scale": scale}
        if op == "order":
            o = qa.sort_tokens(s["ids"], case["experts"])
            xs = qa.gather_tokens(s["x"], o)
            y = qa.combine_tokens(s["ys"], o, s["weights"], residual=s["residual"])
            got = {"offsets": o.offsets, "rows": o.rows, "place": o.place, "xs": xs, "y": y}
            if case["train"]:
                got["dx"] = qa.gather_tokens_backward(s["dxs"], o)
                got["dys"], got["dw"] = qa.combine_tokens_backward(s["dy"], s["ys"], o, s["weights"])
            return got
        n = qa.residual_norm(s["x"], s["y"], s["w"], EPS, post_w=s["post_w"], gate=s["gate"],
                             gate_act=case["gate"] if case["gate"] != "none" else None, scale=s["scale"],
                             quantize=case["quantize"])
        got = {"x": n.x, "h": n.h}
        if case["quantize"]:
            got["q"], got["scale"] = n.q, n.q_scale
        return got
    if op == "product":
        return _plain_product(s)
    if op == "quantize":
        q, scale = _quantize(_activate(s["x"], case["act"]))
        return {"q": q, "scale": scale}
    return _plain_order(s) if op == "order" else _plain_norm(s)


# ---- bytes and operations ------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "product":
        r, n, k, e = case["rows"] * case["top_k"], case["n"], case["k"], case["experts"]
        # the experts that at least one token takes, were they taken evenly
        used = e * (1 - (1 - case["top_k"] / e) ** case["rows"]) if e else 1
        a = case["rows"] if case["gather"] else r
        b = a * (k + 4 * _blocks(k)) + used * (n * k + 4 * _blocks(n) * _blocks(k)) + r * n * SIZE[case["out"]]
        b += (4 * (e + 1) if e else 0) + (4 * r if case["gather"] else 0)
        return {"bytes": b, "flops": 2 * r * n * k}
    if op == "quantize":
        v = case["rows"] * case["cols"]
        b = v * (SIZE[case["in"]] * (1 if case["act"] == "none" else 2) + 1) + 4 * case["rows"] * _blocks(case["cols"])
        return {"bytes": b, "flops": v * (4 if case["act"] == "none" else 10)}
    if op == "order":
        t, k, h, z = case["tokens"], case["top_k"], case["hidden"], SIZE[case["in"]]
        r = t * k
        b = 4 * (3 * r + case["experts"] + 1) + 4 * r + z * h * (t + r + r + 2 * t)
        f = 2 * r * h
        if case["train"]:
            b += z * h * (r + t + r + r + t) + 8 * r  # dx; then dys and dw
            f += r * h + 3 * r * h
        return {"bytes": b, "flops": f}
    t, h, z = case["tokens"], case["hidden"], SIZE[case["in"]]
    b = t * h * z * (4 + (case["gate"] != "none")) + 4 * h * (1 + case["post"] + case["vector"])
    if case["quantize"]:
        b += t * (h + 4 * _blocks(h))
    return {"bytes": b, "flops": t * h * 12}


# ---- the definitions in 64 bits ------------------------------------------------------------------------

def _exact_quantize(v):
    rows, cols = v.shape
    b = _blocks(cols)
    wide = torch.zeros((rows, b * BLOCK), dtype=torch.float64, device=v.device)
    wide[:, :cols] = v
    wide = wide.view(rows, b, BLOCK)
    scale = torch.maximum(wide.abs().amax(2), torch.tensor(TINY, dtype=torch.float64, device=v.device)) / TOP
    z = wide / scale[:, :, None]
    # the e4m3 grid: steps of 2^(e-3) from 2^-6 up, of 2^-9 below
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
    q = (torch.round(z / step) * step).clamp(-TOP, TOP)
    return q.reshape(rows, b * BLOCK)[:, :cols].contiguous(), scale


def _exact_product(s):
    case = s["case"]
    n, k = case["n"], case["k"]
    col = torch.arange(k, device="cuda") // BLOCK
    line = torch.arange(n, device="cuda") // BLOCK
    a = s["a"].double() * s["a_scale"].double()[:, col]
    if not case["experts"]:
        return a @ (s["w"].double() * s["w_scale"].double()[line][:, col]).t()
    bounds = s["offsets"].tolist()
    got = torch.zeros((case["rows"] * case["top_k"], n), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        i, j = bounds[e], bounds[e + 1]
        if j > i:
            w = s["w"][e].double() * s["w_scale"][e].double()[line][:, col]
            rows = a[s["rows"][i:j].long()] if case["gather"] else a[i:j]
            got[i:j] = rows @ w.t()
    return got


def _exact_order(s):
    case = s["case"]
    t, k, e = case["tokens"], case["top_k"], case["experts"]
    # each assignment's place: those of lower experts, and those of its own before it
    key = s["ids"].reshape(-1).long() * (t * k) + torch.arange(t * k, device="cuda")
    order = torch.sort(key).values % (t * k)
    place = torch.argsort(order).view(t, k)
    counts = torch.bincount(s["ids"].reshape(-1).long(), minlength=e)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(counts, 0)])
    xs = s["x"].double()[order // k]
    y = s["residual"].double()
    w = s["weights"].double()
    for j in range(k):
        y = y + w[:, j:j + 1] * s["ys"].double()[place[:, j]]
    got = {"offsets": offsets.to(torch.int32), "rows": order.to(torch.int32), "place": place.to(torch.int32),
           "xs": xs, "y": y}
    if case["train"]:
        dy = s["dy"].double()
        got["dx"] = torch.zeros_like(dy).index_add_(0, order // k, s["dxs"].double())
        got["dys"] = w.reshape(-1)[order][:, None] * dy[order // k]
        dw = torch.empty(t * k, dtype=torch.float64, device="cuda")
        dw[order] = (s["ys"].double() * dy[order // k]).sum(1)
        got["dw"] = dw.view(t, k)
    return got


def _exact_norm(s):
    case = s["case"]
    x, y = s["x"].double(), s["y"].double()
    h = x.shape[1]
    if case["post"]:
        y = y * torch.rsqrt((y * y).sum(1) / h + EPS)[:, None] * s["post_w"].double()
    if case["gate"] == "sigmoid":
        y = y * torch.sigmoid(s["gate"].double())
    elif case["gate"] == "silu":
        y = y * s["gate"].double() * torch.sigmoid(s["gate"].double())
    x = x + y * (s["scale"].double() if case["vector"] else s["scale"])
    n = x * torch.rsqrt((x * x).sum(1) / h + EPS)[:, None] * s["w"].double()
    got = {"x": x, "h": n}
    if case["quantize"]:
        got["q"], got["scale"] = _exact_quantize(n)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "product":
        return _exact_product(s)
    if op == "quantize":
        v = s["x"].double()
        if case["act"] != "none":
            g, u = v[:, :case["cols"]], v[:, case["cols"]:]
            if case["act"] == "swiglu":
                v = u * g * torch.sigmoid(g)
            else:
                v = u * g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        q, scale = _exact_quantize(v)
        return {"q": q, "scale": scale}
    return _exact_order(s) if op == "order" else _exact_norm(s)
