"""The quantised-serving operators, as cases that can be timed and compared.

Three operators: the root-mean-square norm with the residual's addition (output in the input's type, or in 8 bits with
a scale for each row), the linear layer on 8-bit operands, and the linear layer with 4-bit weights in groups.

A case is a dict of plain values; prepare(case, seed) makes what a program has in hand before the call, run(state) is
one pass, either in plain torch operations (own = False) or through rokoko_b200.linear (own = True).
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
Q8_MAX = 448.0      # largest finite value of the 8-bit type (4 exponent bits, 3 mantissa bits)
AMAX_FLOOR = 1e-30  # rows below it keep this scale: no division by zero


def listed():
    return [
        # the phonemizer's norm before its projections, one word of 11 characters: a launch, nothing else
        dict(name="norm_word_f32", op="norm", rows=11, cols=256, type="f32", residual=True, q8=False),
        # one token of a wide model, in 8 bits for the projection that follows
        dict(name="norm_q8_token_bf16", op="norm", rows=1, cols=8192, type="bf16", residual=True, q8=True),
        # the phonemizer over 256 sentences in one call
        dict(name="norm_q8_sentences_f32", op="norm", rows=31000, cols=256, type="f32", residual=True, q8=True),
        # a long prompt of a wide model: bound by memory
        dict(name="norm_q8_long_bf16", op="norm", rows=16384, cols=8192, type="bf16", residual=True, q8=True),
        # one token through a square projection: the weights' bytes are the cost
        dict(name="q8_token_bf16", op="q8", rows=1, n=8192, k=8192, type="bf16", bias=False, residual=False),
        # the phonemizer's gate and up projections over 256 sentences: a short reduction, a large output
        dict(name="q8_sentences_f32", op="q8", rows=31000, n=2048, k=256, type="f32", bias=True, residual=False),
        # nothing divides anything
        dict(name="q8_ragged_f16", op="q8", rows=1531, n=4099, k=2037, type="f16", bias=True, residual=True),
        # a long prompt: bound by the matrix instructions
        dict(name="q8_long_bf16", op="q8", rows=8192, n=8192, k=8192, type="bf16", bias=False, residual=False),
        # the phonemizer's gate and up projections, one word
        dict(name="q4_word_f32", op="q4", rows=11, n=2048, k=256, type="f32", scale="f32", group=64, zeros=False,
             bias=True, residual=False),
        # one token through a square projection
        dict(name="q4_token_bf16", op="q4", rows=1, n=8192, k=8192, type="bf16", scale="bf16", group=128, zeros=False,
             bias=False, residual=True),
        # four tokens through a wide one, with zero points: 128 MiB of weights
        dict(name="q4_wide_f16", op="q4", rows=4, n=16384, k=16384, type="f16", scale="f16", group=128, zeros=True,
             bias=False, residual=False),
        # a small batch, small groups, odd sizes, 32-bit activations
        dict(name="q4_batch_f32", op="q4", rows=24, n=5003, k=4001, type="f32", scale="f16", group=32, zeros=True,
             bias=True, residual=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; a quarter of them multiples of 64."""
    v = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
    return max(lo, min(hi, v // 64 * 64)) if v > 128 and rng.random() < 0.25 else max(lo, min(hi, v))


def draw(rng):
    op, t = rng.choice(("norm", "q8", "q4")), rng.choice(("f32", "f16", "bf16"))
    if op == "norm":
        cols = _log(rng, 64, 16384)
        return dict(op=op, rows=_log(rng, 1, max(1, min(32768, (1 << 26) // cols))), cols=cols, type=t,
                    residual=rng.random() < 0.7, q8=rng.random() < 0.6)
    if op == "q8":
        n, k = _log(rng, 64, 12288), _log(rng, 64, 12288)
        return dict(op=op, rows=_log(rng, 1, max(1, min(32768, (1 << 37) // (n * k)))), n=n, k=k, type=t,
                    bias=rng.random() < 0.5, residual=rng.random() < 0.4)
    n = _log(rng, 64, 16384)
    return dict(op=op, rows=_log(rng, 1, 32), n=n, k=_log(rng, 64, max(64, min(16384, (1 << 27) // n))), type=t,
                scale=rng.choice(("f32", t)), group=rng.choice((32, 64, 128, 256)), zeros=rng.random() < 0.5,
                bias=rng.random() < 0.4, residual=rng.random() < 0.4)


# ------------------------------------------------------------------ inputs

def _to_q8(x):
    """Rows in 8 bits with a scale each (32-bit x): codes [rows, cols] in rows of a multiple of 16 bytes, scales [rows]."""
    scale = x.abs().amax(1).clamp_min(AMAX_FLOOR) / Q8_MAX
    rows, cols = x.shape
    q = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.float8_e4m3fn, device=x.device)[:, :cols]
    q.copy_((x / scale[:, None]).clamp(-Q8_MAX, Q8_MAX).to(torch.float8_e4m3fn))
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    t = TYPES[case["type"]]
    s = {"op": case["op"], "type": t, "residual": None, "bias": None}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        spread = torch.exp(0.7 * normal(cols))  # channels differ in size, as those of a residual stream do
        s["x"] = normal(rows, cols).mul_(spread).to(t)
        s["weight"] = (1 + 0.2 * normal(cols)).to(t)
        s["q8"] = case["q8"]
        if case["residual"]:
            s["residual"] = normal(rows, cols).mul_(spread).mul_(0.5).to(t)
        return s
    rows, n, k = case["rows"], case["n"], case["k"]
    if case["op"] == "q8":
        s["x"], s["x_scale"] = _to_q8(normal(rows, k))
        s["w"], s["w_scale"] = _to_q8(normal(n, k).mul_(k ** -0.5))
    else:
        groups = -(-k // case["group"])
        s["x"] = normal(rows, k).to(t)
        s["group"] = case["group"]
        # two weights a byte, the even column in the low half; rows of a multiple of 16 bytes
        s["w"] = torch.randint(0, 256, (n, (k + 31) // 32 * 16), generator=g, device=DEVICE, dtype=torch.uint8)
        s["w_scale"] = ((0.5 + torch.rand(n, groups, generator=g, device=DEVICE)) * (0.2 * k ** -0.5)).to(
            TYPES[case["scale"]])
        s["zeros"] = None
        if case["zeros"]:
            s["zeros"] = torch.randint(4, 12, (n, groups), generator=g, device=DEVICE, dtype=torch.uint8)
    if case["bias"]:
        s["bias"] = normal(n)
    if case["residual"]:
        s["residual"] = normal(rows, n).to(t)
    return s


# ------------------------------------------------------------------ one pass

def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
    out = [h.to(s["type"])] if s["residual"] is not None else []
    if not s["q8"]:
        return [y.to(s["type"])] + out
    scale = y.abs().amax(1).clamp_min(AMAX_FLOOR) / Q8_MAX
    return [(y / scale[:, None]).clamp(-Q8_MAX, Q8_MAX).to(torch.float8_e4m3fn), scale] + out


def _plain_finish(s, y):
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return [y.to(s["type"])]


def _plain_q8(s):
    x = s["x"].float() * s["x_scale"][:, None]
    w = s["w"].float() * s["w_scale"][:, None]
    return _plain_finish(s, x @ w.t())


def _plain_q4(s):
    k = s["x"].shape[1]
    q = torch.stack((s["w"] & 15, s["w"] >> 4), 2).flatten(1)[:, :k].float()
    at = torch.arange(k, device=q.device) // s["group"]
    zero = s["zeros"].float()[:, at] if s["zeros"] is not None else 8.0
    return _plain_finish(s, s["x"].float() @ ((q - zero) * s["w_scale"].float()[:, at]).t())


def run(state):
    s = state
    if not own:
        return {"norm": _plain_norm, "q8": _plain_q8, "q4": _plain_q4}[s["op"]](s)
    from rokoko_b200 import linear
    if s["op"] == "norm":
        f = linear.rms_norm_q8 if s["q8"] else linear.rms_norm
        out = f(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return list(out) if isinstance(out, tuple) else [out]
    if s["op"] == "q8":
        return [linear.linear_q8(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"], residual=s["residual"],
                                 dtype=s["type"])]
    return [linear.linear_q4(s["x"], s["w"], s["w_scale"], s["group"], zeros=s["zeros"], bias=s["bias"],
                             residual=s["residual"])]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e = SIZE[case["type"]]
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        n = rows * cols
        moved = n * e * (3 if case["residual"] else 1) + cols * e + (n + 4 * rows if case["q8"] else n * e)
        return {"bytes": moved, "flops": (8 if case["q8"] else 5) * n}
    rows, n, k = case["rows"], case["n"], case["k"]
    moved = rows * n * e * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0)
    if case["op"] == "q8":
        return {"bytes": moved + (rows + n) * (k + 4), "flops": 2 * rows * n * k}
    groups = -(-k // case["group"])
    weights = n * ((k + 1) // 2) + n * groups * (SIZE[case["scale"]] + (1 if case["zeros"] else 0))
    return {"bytes": moved + rows * k * e + weights, "flops": 2 * rows * n * k}


# ------------------------------------------------------------------ the definition in 64 bits

def _nearest_q8(v):
    """The nearest value of the 8-bit type, halves to the even one: steps of 2^(e-3) within [2^e, 2^(e+1)), e >= -6."""
    _, e = torch.frexp(v)  # v = m 2^e with m in [0.5, 1)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return ((v / step).round() * step).clamp(-Q8_MAX, Q8_MAX)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h += s["residual"].double()
        y = h / ((h * h).sum(1) / h.shape[1] + EPS).sqrt()[:, None]
        y *= s["weight"].double()
        out = [h] if s["residual"] is not None else []
        if not case["q8"]:
            return [y] + out
        top = torch.maximum(y.amax(1), -y.amin(1)).clamp_min(AMAX_FLOOR)
        return [_nearest_q8(y * (Q8_MAX / top)[:, None]), top / Q8_MAX] + out
    if case["op"] == "q8":  # the scales leave the sum
        y = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
        y *= s["x_scale"].double()[:, None]
        y *= s["w_scale"].double()
    else:  # group by group, the zero point by the group's sum of x: scale (sum q x - zero sum x)
        x, low, high = s["x"].double(), (s["w"] % 16).double(), (s["w"] // 16).double()
        y, k, half = 0, case["k"], case["group"] // 2
        for i in range(s["w_scale"].shape[1]):
            a, b = i * case["group"], min(k, (i + 1) * case["group"])
            even, odd = x[:, a:b:2], x[:, a + 1:b:2]
            part = even @ low[:, i * half:i * half + even.shape[1]].t()
            part += odd @ high[:, i * half:i * half + odd.shape[1]].t()
            zero = s["zeros"][:, i].double() if s["zeros"] is not None else 8
            y = y + (part - x[:, a:b].sum(1)[:, None] * zero) * s["w_scale"][:, i].double()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return [y]
