"""Operators of a decoder's training step, as a list of timed cases.

Four operators that stand next to the optimizers and the fused model operations of this package:

``clip``        the norm over every gradient of a model, and the gradients scaled in place to stay below a bound
``embed``       token embedding with a scale, and the dense gradient of its table
``norm``        residual addition + RMSNorm, with its gradients; or with an 8-bit result and a scale per 128 values
``linear``      a linear layer whose products take 8-bit operands with a scale per block of 128, with both gradients; or
                on a weight that is kept in 8 bits

``run`` makes one call; with ``own`` false it computes the same from elementary torch operations in 32 bits.

The 8-bit format is e4m3 with a 32-bit scale per group: for the largest magnitude ``a`` of a group (at least 1e-30), the scale
is ``a / 448`` and a value x is held as ``e4m3(x * (448 / a))``, every step of that rounded to 32 bits.  Groups are runs of 128
along the dimension that a product sums over (the last run may be shorter), and squares of 128 x 128 for weights.
"""

import math
import random

import torch

own = False  # set from outside: true runs the package's operators, false the plain forms

_E4M3 = 448.0
_SMALLEST = 1e-30
_TIGHTEN = 0.9999  # the bound of a gradient norm from one pass to the next


def _layers(d, ffn, count):
    """Parameters of ``count`` SwiGLU decoder layers: four attention matrices, three feed-forward ones, two norms."""
    return [(d, d)] * (4 * count) + [(ffn, d)] * (2 * count) + [(d, ffn)] * count + [(d,)] * (2 * count)


def _spell(shapes):
    return ";".join("x".join(str(n) for n in s) for s in shapes)


def _shapes(text):
    return [tuple(int(n) for n in s.split("x")) for s in text.split(";")]


def listed():
    return [
        # Latency: the gradients of the 784-512-10 perceptron.
        dict(name="clip_perceptron", kind="clip", weights=_spell([(512, 784), (512,), (10, 512), (10,)]), dtype="float32"),
        # Odd sizes packed without padding (most tensors start off any vector boundary), bf16.
        dict(name="clip_ragged", kind="clip", weights=_spell([(1000, 1337), (333, 1000), (77, 333), (1337,), (333,)] * 6), dtype="bfloat16"),
        # Four decoder layers of the 1B configuration with its head: 334M gradients.
        dict(name="clip_decoder", kind="clip", weights=_spell(_layers(2048, 8192, 4) + [(32000, 2048)]), dtype="float32"),
        # The table of the 124M decoder, sixteen sequences of 1024 tokens.
        dict(name="embed_gpt2", kind="embed", tokens=16384, vocab=50257, width=768, dtype="float32", out="float32", scale=1.0, pad=0.0),
        # The table of the 1B decoder in bf16, eight sequences of 2048 tokens, scaled by the square root of the width.
        dict(name="embed_llama", kind="embed", tokens=16384, vocab=32000, width=2048, dtype="bfloat16", out="bfloat16", scale=45.25, pad=0.0),
        # A padded batch: three tokens in five are the same one; odd width, small table, fp32 table with bf16 rows.
        dict(name="embed_padded", kind="embed", tokens=4001, vocab=1000, width=333, dtype="float32", out="bfloat16", scale=18.25, pad=0.6),
        # Training, 1B decoder: bf16 branch added to an fp32 residual stream.
        dict(name="norm_train", kind="norm", rows=16384, width=2048, x="bfloat16", residual="float32", fp8=False),
        # Training, odd width, few rows, everything bf16.
        dict(name="norm_ragged", kind="norm", rows=333, width=1337, x="bfloat16", residual="bfloat16", fp8=False),
        # Evaluation of one token: the 8-bit operand of the next product.
        dict(name="norm_token", kind="norm", rows=1, width=2048, x="bfloat16", residual="float32", fp8=True),
        # Training, feed-forward input product of the 1B decoder: 16384 tokens, fp32 weight.
        dict(name="linear_train", kind="linear", rows=16384, inner=2048, outer=8192, x="bfloat16", weight="float32"),
        # Training, odd sizes in every dimension.
        dict(name="linear_ragged", kind="linear", rows=1001, inner=1337, outer=333, x="bfloat16", weight="float32"),
        # Evaluation of four tokens on a weight kept in 8 bits: feed-forward output product of the 1B decoder.
        dict(name="linear_tokens", kind="linear", rows=4, inner=8192, outer=2048, x="bfloat16", weight="e4m3"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng, lo, hi):
    """A width: a multiple of 128, or of 8, or any number."""
    n = _log_int(rng, lo, hi)
    step = rng.choice([128, 128, 8, 1])
    return max(lo, n // step * step) if n >= step else n


def draw(rng: random.Random):
    kind = rng.choice(["clip", "embed", "norm", "norm", "linear", "linear"])
    while True:
        if kind == "clip":
            shapes = []
            for _ in range(_log_int(rng, 1, 120)):
                shapes.append((_dim(rng, 1, 4096), _dim(rng, 1, 4096)) if rng.random() < 0.6 else (_dim(rng, 1, 8192),))
            case = dict(kind="clip", weights=_spell(shapes), dtype=rng.choice(["float32", "float32", "bfloat16"]))
        elif kind == "embed":
            dtype = rng.choice(["float32", "float32", "bfloat16"])
            case = dict(
                kind="embed", tokens=_log_int(rng, 1, 32768), vocab=_log_int(rng, 64, 65536), width=_dim(rng, 16, 4096), dtype=dtype,
                out=dtype if dtype == "bfloat16" else rng.choice(["float32", "bfloat16"]), scale=rng.choice([1.0, 1.0, 27.75]),
                pad=rng.choice([0.0, 0.0, 0.3, 0.9]),
            )
        elif kind == "norm":
            x, residual = rng.choice([("bfloat16", "float32"), ("bfloat16", "bfloat16"), ("float32", "float32")])
            case = dict(kind="norm", rows=_log_int(rng, 1, 16384), width=_dim(rng, 16, 8192), x=x, residual=residual, fp8=rng.random() < 0.4)
        elif rng.random() < 0.6:
            case = dict(kind="linear", rows=_log_int(rng, 1, 16384), inner=_dim(rng, 16, 8192), outer=_dim(rng, 16, 8192),
                        x="bfloat16", weight=rng.choice(["float32", "float32", "bfloat16"]))
        else:
            case = dict(kind="linear", rows=_log_int(rng, 1, 2048), inner=_dim(rng, 16, 8192), outer=_dim(rng, 16, 8192),
                        x="bfloat16", weight="e4m3")
        need = work(case)
        # No larger than the largest listed case.
        if need["bytes"] <= 2.6e9 and need["flops"] <= 1.6e12:
            return case


# ----------------------------------------------------------------------------------------------
# What a program holds before the call
# ----------------------------------------------------------------------------------------------
def _dtype(name):
    return getattr(torch, name)


def _activations(gen, rows, width, spread=0.5):
    """Rows and columns of different scale: a few channels are much larger than the others, as in trained decoders."""
    x = torch.randn(rows, width, device="cuda", generator=gen)
    x *= torch.exp(spread * torch.randn(rows, 1, device="cuda", generator=gen))
    return x.mul_(torch.exp(spread * torch.randn(1, width, device="cuda", generator=gen)))


def _tokens(gen, count, vocab, pad):
    """Token numbers whose frequency falls as one over their rank; a share ``pad`` of them is the padding token."""
    u = torch.rand(count, device="cuda", generator=gen, dtype=torch.float64)
    ids = (torch.pow(float(vocab), u).long() - 1).clamp_(0, vocab - 1)
    return torch.where(torch.rand(count, device="cuda", generator=gen) < pad, vocab - 1, ids)


def _pitched(rows, cols, dtype=torch.float8_e4m3fn):
    """[rows, cols] whose rows start 16 bytes apart or a multiple of that, as the products' operands do."""
    return torch.zeros(rows, (cols + 15) // 16 * 16, device="cuda", dtype=torch.uint8).view(dtype)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "clip":
        shapes = _shapes(case["weights"])
        sizes = [math.prod(s) for s in shapes]
        flat = torch.randn(sum(sizes), device="cuda", generator=gen)
        scales = torch.exp(torch.randn(len(sizes), device="cuda", generator=gen)).tolist()
        for part, s in zip(flat.split(sizes), scales):
            part.mul_(1e-3 * s)
        bound = 0.4 * float(flat.norm())
        flat = flat.to(_dtype(case["dtype"]))
        params = []
        for part, s in zip(flat.split(sizes), shapes):
            params.append(torch.nn.Parameter(torch.empty(s, device="cuda", dtype=flat.dtype)))
            params[-1].grad = part.view(s)
        return dict(case=case, flat=flat, params=params, bound=bound)
    if kind == "embed":
        n, v, c = case["tokens"], case["vocab"], case["width"]
        table = (torch.randn(v, c, device="cuda", generator=gen) * 0.02).to(_dtype(case["dtype"])).requires_grad_()
        ids = _tokens(gen, n, v, case["pad"])
        dy = (_activations(gen, n, c) * 1e-3).to(_dtype(case["out"]))
        return dict(case=case, table=table, ids=ids, dy=dy)
    if kind == "norm":
        r, c = case["rows"], case["width"]
        x = (0.3 * _activations(gen, r, c)).to(_dtype(case["x"]))
        residual = _activations(gen, r, c).to(_dtype(case["residual"]))
        weight = 1 + 0.2 * torch.randn(c, device="cuda", generator=gen)
        if case["fp8"]:
            return dict(case=case, x=x, residual=residual, weight=weight)
        dy = (1e-3 * _activations(gen, r, c)).to(x.dtype)
        dh = (1e-3 * _activations(gen, r, c)).to(residual.dtype)
        return dict(case=case, x=x.requires_grad_(), residual=residual.requires_grad_(), weight=weight.requires_grad_(), dy=dy, dh=dh)
    t, k, n = case["rows"], case["inner"], case["outer"]
    x = _activations(gen, t, k).to(_dtype(case["x"]))
    weight = 0.02 * torch.randn(n, k, device="cuda", generator=gen)
    if case["weight"] == "e4m3":
        data = _pitched(n, k)
        q, scale = _squares(weight)
        data.view(torch.uint8).copy_(q.view(torch.uint8))
        return dict(case=case, x=x, data=data, scale=scale)
    dy = (1e-3 * _activations(gen, t, n)).to(x.dtype)
    return dict(case=case, x=x.requires_grad_(), weight=weight.to(_dtype(case["weight"])).requires_grad_(), dy=dy)


# ----------------------------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------------------------
def _padded(x, rows, cols):
    return torch.nn.functional.pad(x.float(), (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))


def _grouped(x, rows, cols):
    """e4m3 values and scales of ``x`` in groups of rows x cols; scales [groups down, groups across]."""
    p = _padded(x, rows, cols)
    blocks = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    top = blocks.abs().amax((1, 3)).clamp_min(_SMALLEST)
    most = torch.full_like(top, _E4M3)  # a number in its place would be divided by as a product with a reciprocal
    q = (blocks * (most / top)[:, None, :, None]).view_as(p).to(torch.float8_e4m3fn)
    return q[: x.shape[0], : x.shape[1]], top / most


def _runs(x):
    return _grouped(x, 1, 128)


def _squares(x):
    return _grouped(x, 128, 128)


def _values(q, scale):
    """The numbers that e4m3 values with scales stand for."""
    rows, cols = q.shape
    down, across = (1, 128) if scale.shape[0] == rows else (128, 128)
    return q.float() * scale.repeat_interleave(down, 0)[:rows].repeat_interleave(across, 1)[:, :cols]


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "clip":
        flat = s["flat"]
        norm = flat.float().square().sum().sqrt()
        factor = (s["bound"] / (norm + 1e-6)).clamp(max=1.0)
        flat.copy_(flat.float() * factor)
        s["bound"] *= _TIGHTEN
        return norm, flat
    if kind == "embed":
        table, ids, dy = s["table"].detach(), s["ids"], s["dy"]
        y = (table[ids].float() * case["scale"]).to(dy.dtype)
        grad = torch.zeros(table.shape, device="cuda").index_add_(0, ids, dy.float()) * case["scale"]
        return y, grad.to(table.dtype)
    if kind == "norm":
        x, residual, w = (s[n].detach() for n in ("x", "residual", "weight"))
        h = (x.float() + residual.float()).to(residual.dtype)
        hf = h.float()
        rstd = torch.rsqrt(hf.square().mean(1, keepdim=True) + 1e-5)
        z = hf * rstd
        if case["fp8"]:
            return (*_runs(z * w), h)
        g, dh = s["dy"].float(), s["dh"].float()
        gw = g * w
        dh = dh + rstd * (gw - z * (gw * z).mean(1, keepdim=True))
        return (z * w).to(x.dtype), h, dh.to(x.dtype), dh.to(residual.dtype), (g * z).sum(0)
    x = s["x"].detach()
    if case["weight"] == "e4m3":
        return (_values(*_runs(x)) @ _values(s["data"], s["scale"]).t()).to(x.dtype)
    w, dy = _values(*_squares(s["weight"].detach())), s["dy"]
    y = (_values(*_runs(x)) @ w.t()).to(x.dtype)
    dx = (_values(*_runs(dy)) @ w).to(x.dtype)
    dw = _values(*_runs(dy.t())) @ _values(*_runs(x.t())).t()
    return y, dx, dw.to(s["weight"].dtype)


def run(s):
    if not own:
        return _plain(s)
    from optimizers_b200 import clip_grad_norm_
    from optimizers_b200.models import fp8, fused_ops

    case, kind = s["case"], s["case"]["kind"]
    if kind == "clip":
        norm = clip_grad_norm_(s["params"], s["bound"])
        s["bound"] *= _TIGHTEN  # the buffers stay, so that a pass finds what the last one left: it has to clip again
        return norm, s["flat"]
    if kind == "embed":
        y = fused_ops.embedding(s["ids"], s["table"], scale=case["scale"], out_dtype=s["dy"].dtype)
        return (y.detach(), *torch.autograd.grad(y, s["table"], s["dy"]))
    if kind == "norm":
        if case["fp8"]:
            rows, h = fp8.add_rms_norm(s["x"], s["residual"], s["weight"], eps=1e-5)
            return rows.data, rows.scale, h
        leaves = (s["x"], s["residual"], s["weight"])
        y, h = fused_ops.add_rms_norm(*leaves, eps=1e-5)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (s["dy"], s["dh"])))
    if case["weight"] == "e4m3":
        return fp8.linear(s["x"], fp8.Weight(s["data"], s["scale"]))
    y = fp8.linear(s["x"], s["weight"])
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"]))


# ----------------------------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------------------------
def work(case):
    size = dict(float32=4, bfloat16=2, e4m3=1)
    kind = case["kind"]
    if kind == "clip":
        n = sum(math.prod(s) for s in _shapes(case["weights"]))
        return {"bytes": 2 * n * size[case["dtype"]], "flops": 3 * n}
    if kind == "embed":
        n, v, c = case["tokens"], case["vocab"], case["width"]
        return {"bytes": 8 * n + (min(n, v) + v) * c * size[case["dtype"]] + 2 * n * c * size[case["out"]], "flops": 3 * n * c}
    if kind == "norm":
        n, c, bx, br = case["rows"] * case["width"], case["width"], size[case["x"]], size[case["residual"]]
        if case["fp8"]:
            return {"bytes": n * (bx + 2 * br + 1) + 4 * case["rows"] * -(-c // 128) + 4 * c, "flops": 8 * n}
        return {"bytes": n * (4 * bx + 4 * br) + 8 * c, "flops": 16 * n}
    t, k, n = case["rows"], case["inner"], case["outer"]
    bx, bw = size[case["x"]], size[case["weight"]]
    if case["weight"] == "e4m3":
        return {"bytes": bx * t * (k + n) + n * k + 4 * -(-n // 128) * -(-k // 128), "flops": 2 * t * n * k}
    return {"bytes": 2 * bx * t * (k + n) + 2 * bw * n * k, "flops": 6 * t * n * k}


# ----------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ----------------------------------------------------------------------------------------------
def _to_e4m3(v):
    """The nearest e4m3 value (ties to even): three binary digits after the leading one, exponents from -6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    return torch.round(v / step) * step


def _held(x, rows, cols):
    """What ``x`` is after a trip through the 8-bit format, in 64 bits (the factor, the scaled value and the scale are 32-bit numbers)."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for j in range(0, x.shape[1], cols):  # one column of groups at a time
        part = x[:, j : j + cols].double()
        top = part.abs().amax(1)
        if rows > 1:
            top = torch.cat([t.amax().expand(len(t)) for t in top.split(rows)])
        top = top.clamp_min(float(torch.tensor(_SMALLEST))).unsqueeze(1)
        factor, scale = (_E4M3 / top).float().double(), (top / _E4M3).float().double()
        out[:, j : j + cols] = _to_e4m3((part * factor).float().double()) * scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "clip":
        g = s["flat"].double()
        norm = torch.linalg.vector_norm(g)
        return norm, g * min(1.0, s["bound"] / (float(norm) + 1e-6))
    if kind == "embed":
        table, dy = s["table"].detach().double(), s["dy"].double()
        order = torch.argsort(s["ids"], stable=True)
        sums = torch.zeros(case["vocab"] + 1, case["width"], dtype=torch.float64, device="cuda")
        ends = torch.bincount(s["ids"], minlength=case["vocab"]).cumsum(0)
        running = torch.cat([torch.zeros_like(dy[:1]), dy[order].cumsum(0)])
        sums[1:] = running[ends]
        return table.index_select(0, s["ids"]) * case["scale"], (sums[1:] - sums[:-1]) * case["scale"]
    if kind == "norm":
        x, r, w = (s[n].detach().double() for n in ("x", "residual", "weight"))
        h = x + r
        held = h.to(s["residual"].dtype).double()  # the normalisation reads the stream as it is handed on
        length = torch.sqrt(torch.linalg.vector_norm(held, dim=1, keepdim=True) ** 2 / case["width"] + 1e-5)
        y = held / length * w
        if case["fp8"]:
            groups = torch.nn.functional.pad(y, (0, -y.shape[1] % 128)).unflatten(1, (-1, 128))
            return None, groups.abs().amax(2).clamp_min(_SMALLEST) / _E4M3, h  # an 8-bit value next to a border has no single answer
        dy, dh = s["dy"].double(), s["dh"].double()
        along = (dy * y).sum(1, keepdim=True) / case["width"]
        dh = dh + (dy * w - held / length * along) / length
        return y, h, dh, dh, (dy * held / length).sum(0)
    x = s["x"].detach()
    if case["weight"] == "e4m3":
        scale = s["scale"].double()
        w = s["data"].to(torch.float64)
        at = [torch.arange(n, device="cuda") // 128 for n in w.shape]
        return _held(x, 1, 128) @ (w * scale[at[0]][:, at[1]]).T
    w = _held(s["weight"].detach(), 128, 128)
    dw = _held(s["dy"].T, 1, 128) @ _held(x.T, 1, 128).T
    return _held(x, 1, 128) @ w.T, _held(s["dy"], 1, 128) @ w, dw
