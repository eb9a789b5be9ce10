"""What is measured of the 4-bit and the distillation operators.

``own = False``: ``run`` computes them in elementary torch operations, in 32 bits, rounded once at the end.
``own = True``:  ``run`` makes the calls a program makes of ``lira_amd``.

Kinds of case:

* ``store``    rows packed to microscaled 4-bit floats and read back (what a 4-bit index does on ``add`` and
               ``reconstruct``); the packed values are returned as the numbers they stand for
* ``linear``   act(alpha * Q(x) W^T + bias) with W packed beforehand and x packed on the way
* ``distill``  loss from a teacher's top logits, and the gradient of the student's logits: ``autograd`` through
               the loss function, or ``fused`` in one call

Packed layout (both sides take it): rows padded with zeros to P planes of 128 elements, codes (P, n, 64) uint8 with
element 2i in the low half of byte i, one e8m0 scale per 32 elements, (P, n, 4) uint8.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _lira():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "lira-ann-search_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import lira_amd
    return lira_amd


def listed():
    return [
        # one query packed on its own: the latency of a call
        {"name": "store-one-query", "kind": "store", "n": 1, "k": 128, "dtype": "fp32"},
        # rows whose length fills neither a block nor a plane, in the type that models hold
        {"name": "store-odd-bf16", "kind": "store", "n": 4099, "k": 1000, "dtype": "bf16"},
        # a whole base set of the SIFT1M shape
        {"name": "store-sift1m", "kind": "store", "n": 1000000, "k": 128, "dtype": "fp32"},
        # a wide layer for a single row: a stream over the weights
        {"name": "linear-1row-8192", "kind": "linear", "m": 1, "n": 8192, "k": 8192, "dtype": "bf16",
         "bias": False, "act": "", "alpha": 1.0},
        # one query scored against the SIFT1M base set, squared norms as the bias
        {"name": "scores-1q-sift1m", "kind": "linear", "m": 1, "n": 1000000, "k": 128, "dtype": "fp32",
         "bias": True, "act": "", "alpha": -1.0},
        # a small batch through a wide layer with odd sizes everywhere
        {"name": "linear-ragged-37row", "kind": "linear", "m": 37, "n": 11111, "k": 5000, "dtype": "fp16",
         "bias": True, "act": "relu", "alpha": 1.0},
        # the probing model's last layer: 10 k queries, 128 hidden units, 1024 partitions
        {"name": "linear-probe-head", "kind": "linear", "m": 10000, "n": 1024, "k": 128, "dtype": "fp32",
         "bias": True, "act": "sigmoid", "alpha": 1.0},
        # a wide layer for a long batch: bound by the matrix cores
        {"name": "linear-8192", "kind": "linear", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16",
         "bias": False, "act": "", "alpha": 1.0},
        # a few rows of an odd number of partitions: the latency of a step
        {"name": "distill-few-odd", "kind": "distill", "rows": 64, "vocab": 257, "top": 8, "dtype": "fp32",
         "ids": "int32", "t": 1.0, "masked": False, "mode": "fused"},
        # a training batch of the probing model at BIGANN-100M's 1024 partitions, taught by the 32 nearest
        {"name": "distill-probe", "kind": "distill", "rows": 4096, "vocab": 1024, "top": 32, "dtype": "fp32",
         "ids": "int32", "t": 1.0, "masked": False, "mode": "autograd"},
        # a wide output layer in training, with masked entries and rows without a teacher
        {"name": "distill-wide-autograd", "kind": "distill", "rows": 4096, "vocab": 32768, "top": 64, "dtype": "bf16",
         "ids": "int64", "t": 2.0, "masked": True, "mode": "autograd"},
        # the widest: an odd number of outputs, loss and gradient in one call
        {"name": "distill-widest-fused", "kind": "distill", "rows": 2048, "vocab": 131071, "top": 64, "dtype": "bf16",
         "ids": "int64", "t": 2.0, "masked": True, "mode": "fused"},
    ]


def _size(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "linear", "linear", "distill"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "store":
        k = _size(rng, 16, 1024)
        return {"kind": kind, "n": _size(rng, 1, min(1000000, 128000000 // k)), "k": k, "dtype": dtype}
    if kind == "linear":
        k = _size(rng, 32, 8192)
        n = _size(rng, 32, 16384)
        m = _size(rng, 1, min(8192, 8192 ** 3 // (n * k), 2 ** 26 // n))
        return {"kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5,
                "act": rng.choice(["", "relu", "sigmoid"]), "alpha": rng.choice([1.0, -1.0, 0.125])}
    vocab = _size(rng, 17, 131072)
    most = 2048 * 131071 if dtype != "fp32" else 1024 * 131071
    return {"kind": kind, "rows": _size(rng, 1, min(8192, most // vocab)), "vocab": vocab,
            "top": _size(rng, 1, min(64, vocab // 2)), "dtype": dtype, "ids": rng.choice(["int32", "int64"]),
            "t": rng.choice([1.0, 2.0, 4.0]), "masked": rng.random() < 0.5, "mode": rng.choice(["autograd", "fused"])}


def _planes(k):
    return (k + 127) // 128


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["kind"] == "store":
        x = normal(case["n"], case["k"])
        # rows of different lengths, as vectors of one set have
        x *= torch.exp(0.5 * normal(case["n"], 1))
        return {"case": case, "x": x.to(dt)}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = normal(m, k).to(dt)
        codes, scales = _pack(*_quantize(normal(n, k) * k ** -0.5))
        bias = normal(n) if case["bias"] else None
        return {"case": case, "x": x, "codes": codes, "scales": scales, "bias": bias}
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    z = (2.0 * normal(rows, vocab)).to(dt)
    tv, ti = torch.topk(z.float() + 1.5 * normal(rows, vocab), top, dim=1)
    if case["masked"]:
        # a share of the outputs is unavailable to the student, and short teacher lists end in -1;
        # every 16th row has no teacher at all
        hide = torch.rand((rows, vocab), generator=g, device="cuda") < 0.125
        hide.scatter_(1, ti, False)
        z.masked_fill_(hide, float("-inf"))
        length = torch.randint(1, top + 1, (rows, 1), generator=g, device="cuda")
        length[15::16] = 0
        ti.masked_fill_(torch.arange(top, device="cuda") >= length, -1)
    ti = ti.to(torch.int32 if case["ids"] == "int32" else torch.int64)
    weight = torch.rand(rows, generator=g, device="cuda") / rows
    z.requires_grad_(case["mode"] == "autograd")
    return {"case": case, "z": z, "ti": ti, "tv": tv, "weight": weight}


# ------------------------------------------------------------- plain forms
def _quantize(x):
    """Elements' magnitudes and signs on the 4-bit grid, (n, 4P, 32), and the blocks' exponents (n, 4P)."""
    n, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, _planes(k) * 128 - k)).view(n, -1, 32)
    top = x.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127, dtype=torch.int32))
    e = e.clamp_(min=-127)
    half = e.div(2, rounding_mode="floor")  # (two steps: 2^127 times 2^3 would not fit 32 bits)
    y = torch.ldexp(torch.ldexp(x, -half[..., None]), (half - e)[..., None])
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    v = (torch.round(a / step) * step).clamp_(max=6.0)
    return torch.copysign(v, y), e


def _pack(v, e):
    n, b, _ = v.shape
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code + 8 * torch.signbit(v).to(torch.uint8)).view(n, b // 4, 64, 2)
    codes = (code[..., 0] + 16 * code[..., 1]).transpose(0, 1).contiguous()
    return codes, (e + 127).to(torch.uint8).view(n, b // 4, 4).transpose(0, 1).contiguous()


def _values(codes, scales, dtype):
    p, n, _ = codes.shape
    c = torch.stack((codes & 15, codes >> 4), dim=-1).view(p, n, 4, 32).int()
    a = (c & 7).to(dtype)
    a = torch.where(a < 4, a / 2, torch.where(a < 6, a - 2, 2 * a - 8)) * (1 - 2 * (c >> 3)).to(dtype)
    a = torch.ldexp(a, scales[..., None].int() - 127)
    return a.transpose(0, 1).reshape(n, p * 128)


def _plain_store(x):
    v, e = _quantize(x)
    return torch.ldexp(v, e[..., None]).view(x.shape[0], -1)[:, :x.shape[1]].to(x.dtype)


def _plain_linear(s):
    case = s["case"]
    v, e = _quantize(s["x"])
    x = torch.ldexp(v, e[..., None]).view(case["m"], -1)
    y = case["alpha"] * (x @ _values(s["codes"], s["scales"], torch.float32).t())
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["act"] == "relu":
        y = y.clamp(min=0)
    elif case["act"] == "sigmoid":
        y = 1 / (1 + torch.exp(-y))
    return y.to(s["x"].dtype)


def _plain_distill(s):
    case, t = s["case"], s["case"]["t"]
    z, ti = s["z"].detach().float() / t, s["ti"].long()
    used = ti >= 0
    at = ti.clamp(min=0)
    lse = torch.log(torch.exp(z - z.amax(1, keepdim=True)).sum(1, keepdim=True)) + z.amax(1, keepdim=True)
    tv = (s["tv"] / t).masked_fill(~used, float("-inf"))
    most = tv.amax(1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(tv - most)
    total = p.sum(1, keepdim=True)
    some = total > 0
    logp = (tv - most) - torch.log(torch.where(some, total, 1.0))
    p = p / torch.where(some, total, 1.0)
    loss = t * t * torch.where(p > 0, p * (logp - (z.gather(1, at) - lse)), 0.0).sum(1)
    grad = torch.exp(z - lse) * some
    grad = t * grad.scatter_add_(1, at, -p) * s["weight"][:, None]
    return loss, grad.to(s["z"].dtype)


def run(state):
    case = state["case"]
    if own:
        lira = _lira()
        if case["kind"] == "store":
            return lira.mx4_quantize(state["x"]).dequantize(state["x"].dtype)
        if case["kind"] == "linear":
            w = lira.MX4Tensor(state["codes"], state["scales"], case["k"])
            return lira.mx4_linear(state["x"], w, state["bias"], activation=case["act"] or None, alpha=case["alpha"])
        if case["mode"] == "fused":
            return lira.distill_topk_loss_and_grad(state["z"], state["ti"], state["tv"], temperature=case["t"],
                                                   row_weight=state["weight"])
        loss = lira.distill_topk_loss(state["z"], state["ti"], state["tv"], temperature=case["t"], reduction="none")
        (grad,) = torch.autograd.grad(loss, state["z"], state["weight"])
        return loss.detach(), grad
    if case["kind"] == "store":
        return _plain_store(state["x"])
    if case["kind"] == "linear":
        return _plain_linear(state)
    return _plain_distill(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "store":
        # rows in, packed rows out, rows out
        return {"bytes": case["n"] * (2 * case["k"] * size + 68 * _planes(case["k"])), "flops": 0}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m * k + m * n) * size + n * (68 * _planes(k) + 4 * case["bias"]), "flops": 2 * m * n * k}
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    ids = 4 if case["ids"] == "int32" else 8
    return {"bytes": rows * (2 * vocab * size + top * (4 + ids) + 8), "flops": 6 * rows * vocab}


# ------------------------------------------------------------ 64-bit values
def _round64(x):
    """Rows on the 4-bit grid by comparison with the midpoints between neighbours, in 64 bits."""
    n, k = x.shape
    x = torch.nn.functional.pad(x.double(), (0, _planes(k) * 128 - k)).view(n, -1, 32)
    top = x.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -125))) - 2)
    # (a logarithm next to a whole number may round to it)
    unit = torch.where(top >= 8 * unit, 2 * unit, torch.where(top < 4 * unit, unit / 2, unit)).clamp(min=2.0 ** -127)
    a = x.abs() / unit
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    place = (a > mid[0]).long()  # a tie goes to the neighbour of even place
    for i in range(1, 7):
        place += (a > mid[i]) if i % 2 == 0 else (a >= mid[i])
    return (torch.sign(x) * grid[place] * unit).view(n, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return _round64(s["x"])
    if case["kind"] == "linear":
        w = _values(s["codes"], s["scales"], torch.float64)[:, :case["k"]]
        y = case["alpha"] * torch.matmul(_round64(s["x"]), w.t().contiguous())
        if s["bias"] is not None:
            y += s["bias"].double()
        return y.relu() if case["act"] == "relu" else torch.sigmoid(y) if case["act"] == "sigmoid" else y
    t, ti = case["t"], s["ti"].long()
    logq = torch.log_softmax(s["z"].detach().double() / t, dim=1)
    used = ti >= 0
    some = used.any(1, keepdim=True)
    tv = (s["tv"].double() / t).masked_fill(~used, float("-inf")).masked_fill(~some, 0.0)
    logp = torch.log_softmax(tv, dim=1).masked_fill(~some, float("-inf"))
    p = logp.exp()
    at = ti.clamp(min=0)
    loss = t * t * torch.where(p > 0, p * (logp - logq.gather(1, at)), 0.0).sum(1)
    grad = logq.exp_().mul_(some).scatter_add_(1, at, -p)
    return loss, grad.mul_(t * s["weight"].double()[:, None])
