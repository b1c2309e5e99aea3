"""The measured operators of a block that is kept in 8 bits, served and trained
through: its products, the norm of the residual stream in front of them, and the
clipping of the gradients that the weight updates take.

Kinds of case (``kind``):

* ``product`` -- ``y = x w^T`` of 8-bit operands with a scale for each block of
                 128 (``fp8.product``), and the gradient of ``x`` from that of
                 ``y`` (``fp8.product_grad``);
* ``norm``    -- the residual's addition and the RMS norm of the sum, written in
                 16 or 32 bits or in 8 with scales (``norm.add_rms_norm``), and
                 its gradients (``norm.add_rms_norm_grad``);
* ``block``   -- the two together (``norm.normed_product``) and their gradients;
* ``clip``    -- the norm of all gradients of a step, and their clipping
                 (``clip.clip_grads``).

Blocks: 128 values along a row (the last one of a row may be short) share a scale
``2^e``, ``e`` the least integer with ``max |x| <= 448 * 2^e`` (0 for a block of
zeros), and are rounded to e4m3 after the division by it; a weight has one scale
for each 128 x 128 values.  Sizes are those of the PLE block (``n_embd`` 2560, four
streams, packed sequences of 2,047 positions) or odd ones.
"""
from __future__ import annotations

import math

import torch

own = False  # False: the plain form of every operator; True: the framework's kernels

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK, LARGEST = 128, 448.0
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # one decoded token through the key projection
        dict(name="product_one_token", kind="product", m=1, k=2560, n=10_240, dtype="bf16", train=False),
        # a few sequences decoded together, fp32 activations
        dict(name="product_few_rows_f32", kind="product", m=24, k=2560, n=10_240, dtype="f32", train=False),
        # one packed sequence
        dict(name="product_packed", kind="product", m=2047, k=2560, n=10_240, dtype="bf16", train=False),
        # eight packed sequences of a prompt batch
        dict(name="product_prompts_f16", kind="product", m=16_376, k=2560, n=10_240, dtype="f16", train=False),
        # a small projection of odd sizes: rows end inside a block, tiles past the last row and column
        dict(name="product_odd_f32", kind="product", m=777, k=1000, n=1111, dtype="f32", train=True),
        # a step of the rows' training through the frozen projection: the product and the gradient of its input
        dict(name="product_train", kind="product", m=2047, k=2560, n=10_240, dtype="bf16", train=True),
        # the four streams of one decoded token
        dict(name="norm_one_token", kind="norm", rows=4, d=2560, dtype="bf16", out="fp8", train=False),
        # the four streams of a packed sequence, in 8 bits for the products behind
        dict(name="norm_packed_fp8", kind="norm", rows=8188, d=2560, dtype="bf16", out="fp8", train=False),
        # the same in fp32 in training, all gradients
        dict(name="norm_train_f32", kind="norm", rows=8188, d=2560, dtype="f32", out="f32", train=True),
        # residual, norm and projection of a packed sequence with all gradients
        dict(name="block_train", kind="block", m=2047, k=2560, n=10_240, dtype="bf16", train=True),
        # the gradients of the block's norm and convolution weights
        dict(name="clip_norm_weights", kind="clip", sizes="10240 10240 10240 40960", dtype="f32"),
        # the gradients of the whole block
        dict(name="clip_block", kind="clip", sizes="26214400 6553600 10240 10240 10240 40960",
             dtype="f32"),
    ]


def draw(rng) -> dict:
    def span(lo: int, hi: int) -> int:  # log-uniform, odd sizes among them
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["product", "product", "norm", "block", "clip"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "clip":
        # a few large gradients that share most values, and smaller ones
        left, sizes = span(200, 32_000_000), []
        for i in range(span(1, 60) - 1):
            sizes.append(max(1, int(left * (0.6 if i % 3 == 0 else rng.uniform(0.0, 0.05)))))
            left = max(1, left - sizes[-1])
        return dict(kind=kind, sizes=" ".join(str(x) for x in sizes + [left]), dtype=dtype)
    if kind == "norm":
        d = rng.choice([2560, span(16, 16_384)])
        return dict(kind=kind, rows=min(span(1, 16_376), 40_000_000 // d), d=d, dtype=dtype,
                    out=rng.choice(["fp8", dtype]), train=rng.choice([False, True]))
    k, n = rng.choice([2560, span(32, 10_240)]), rng.choice([2560, span(32, 10_240)])
    m = min(span(1, 16_376), 16_376 * 2560 * 10_240 // (2 * k * n))
    if kind == "block":
        return dict(kind=kind, m=m, k=k, n=n, dtype=rng.choice(["bf16", "f16"]), train=rng.choice([False, True]))
    return dict(kind=kind, m=m, k=k, n=n, dtype=dtype, train=rng.choice([False, True]))


# ---- inputs -----------------------------------------------------------------------------------

def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEV)


def _activations(g, rows: int, cols: int) -> torch.Tensor:
    """Rows about N(0, 1), a few columns much larger than the others, as a residual stream has them."""
    x = _randn(g, rows, cols)
    x *= torch.exp(0.5 * _randn(g, cols))
    x[:, torch.rand(cols, generator=g, device=DEV) < 0.005] *= 20.0
    return x


def _sizes(case: dict) -> list[int]:
    return [int(x) for x in case["sizes"].split()]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed((seed * 1_000_003 + 77) % (1 << 62))
    s = dict(case=case)
    t = TYPES[case["dtype"]]
    if case["kind"] == "clip":
        # gradients of a step, some much larger than others, together above the bound or below it (fp16 ones are scaled,
        # as they are trained with)
        scale = 10.0 ** (_randn(g, len(_sizes(case))).clamp(-2.0, 1.5) - 3.0) * (4096.0 if case["dtype"] == "f16" else 1.0)
        s["grads"] = [(_randn(g, size) * c).to(t) for size, c in zip(_sizes(case), scale)]
        s["out"] = [torch.empty_like(x) for x in s["grads"]]
        total = torch.stack([x.double().square().sum() for x in s["grads"]]).sum().sqrt()
        s["max_norm"] = float(total) * (0.01 + 1.2 * float(torch.rand((), generator=g, device=DEV)))
        return s
    if case["kind"] != "product":
        rows, d = (case["rows"], case["d"]) if case["kind"] == "norm" else (case["m"], case["k"])
        s["x"] = (_activations(g, rows, d) * 0.3).to(t)
        s["residual"] = _activations(g, rows, d).to(t)
        s["norm_weight"] = 1.0 + 0.2 * _randn(g, d)
        if case["train"]:
            width = d if case["kind"] == "norm" else case["n"]
            s["d_y"] = (_randn(g, rows, width) * 1e-2).to(t)
            s["d_h"] = (_randn(g, rows, d) * 1e-2).to(t)
    else:
        s["x"] = _activations(g, case["m"], case["k"]).to(t)
        if case["train"]:
            s["d_y"] = (_randn(g, case["m"], case["n"]) * 1e-2).to(t)
    if case["kind"] != "norm":
        # the projection as a program keeps it: e4m3 values, their scales, and both of the transpose
        w = _randn(g, case["n"], case["k"]) * (0.02 * torch.exp(0.3 * _randn(g, case["n"], 1)))
        s["q"], s["scales"] = _weight_blocks(w)
        if case["train"]:
            bytes_, e = s["q"].view(torch.uint8), s["scales"].view(torch.uint8)
            s["q_t"], s["scales_t"] = _padded(bytes_[:, :case["k"]].T, e[:, :-(-case["k"] // BLOCK)].T)
    return s


def _padded(q, e):
    """Rows of whole blocks (zeros behind the last value), and scales to a multiple of four a row (1 behind the last)."""
    whole = torch.zeros((q.shape[0], -(-q.shape[1] // BLOCK) * BLOCK), dtype=torch.uint8, device=DEV)
    whole[:, :q.shape[1]] = q
    scales = torch.full((e.shape[0], -(-e.shape[1] // 4) * 4), 127, dtype=torch.uint8, device=DEV)
    scales[:, :e.shape[1]] = e
    return whole.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def _exponents(top: torch.Tensor) -> torch.Tensor:
    """The least e with top <= 448 * 2^e, from top = m * 2^x with m in [1/2, 1) and 448 = 7/8 * 2^9."""
    m, x = torch.frexp(top)
    return torch.where(top > 0, x - 9 + (m > 0.875).to(x.dtype), 0)


def _weight_blocks(w: torch.Tensor):
    n, k = w.shape
    full = torch.zeros((-(-n // BLOCK) * BLOCK, -(-k // BLOCK) * BLOCK), device=DEV)
    full[:n, :k] = w
    tiles = full.reshape(-1, BLOCK, full.shape[1] // BLOCK, BLOCK)
    e = _exponents(tiles.abs().amax((1, 3)))
    q = torch.ldexp(tiles, -e[:, None, :, None]).reshape(full.shape)[:n, :k].to(torch.float8_e4m3fn)
    return _padded(q.view(torch.uint8), (e + 127).to(torch.uint8))


# ---- one pass ---------------------------------------------------------------------------------

def run(s: dict):
    if own:
        import __graft_entry__

        __graft_entry__.load_package()
        return _run_own(s, s["case"])
    return {"product": _plain_product, "norm": _plain_norm, "block": _plain_block, "clip": _plain_clip}[s["case"]["kind"]](s, s["case"])


def _weight(s, case):
    """The handle that a program keeps of its projection."""
    if "weight" not in s:
        from engraft_ngram_amd import fp8

        s["weight"] = fp8.Fp8Weight(s["q"], s["scales"], case["k"], s.get("q_t"), s.get("scales_t"))
    return s["weight"]


def _run_own(s, case):
    kind, t = case["kind"], TYPES[case["dtype"]]
    if kind == "clip":
        from engraft_ngram_amd import clip

        return dict(norm=clip.clip_grads(s["grads"], s["max_norm"], out=s["out"]), grads=s["out"])
    if kind == "product":
        from engraft_ngram_amd import fp8

        w = _weight(s, case)
        y = fp8.product(s["x"], w)
        return dict(y=y, d_x=fp8.product_grad(s["d_y"], w)) if case["train"] else y
    from engraft_ngram_amd import norm

    if kind == "norm":
        y, h, rstd = norm.add_rms_norm_stats(s["x"], s["residual"], s["norm_weight"], eps=EPS,
                                             out_dtype="fp8" if case["out"] == "fp8" else t)
        r = dict(y=y.dequantize() if case["out"] == "fp8" else y, h=h)
        if case["train"]:
            r["d_h"], r["d_weight"] = norm.add_rms_norm_grad(s["d_y"], h, rstd, s["norm_weight"], d_residual=s["d_h"])
        return r
    w = _weight(s, case)
    if not case["train"]:
        y, h = norm.normed_product(s["x"], s["residual"], s["norm_weight"], w, eps=EPS)
        return dict(y=y, h=h)
    x, nw = s["x"].detach().requires_grad_(), s["norm_weight"].detach().requires_grad_()
    y, h = norm.normed_product(x, s["residual"], nw, w, eps=EPS)
    d_h, d_weight = torch.autograd.grad((y, h), (x, nw), (s["d_y"], s["d_h"]))
    return dict(y=y.detach(), h=h.detach(), d_h=d_h, d_weight=d_weight)


def _rounded(x: torch.Tensor) -> torch.Tensor:
    """The values that the blocks of fp32 rows stand for."""
    rows, cols = x.shape
    full = torch.zeros((rows, -(-cols // BLOCK) * BLOCK), device=DEV)
    full[:, :cols] = x
    parts = full.reshape(rows, -1, BLOCK)
    e = _exponents(parts.abs().amax(2, keepdim=True))
    q = torch.ldexp(parts, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).reshape(rows, -1)[:, :cols]


def _weight_values(s, case) -> torch.Tensor:
    k, n = case["k"], case["n"]
    scale = s["scales"].float().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return s["q"][:, :k].float() * scale


def _plain_product(s, case):
    w, t = _weight_values(s, case), TYPES[case["dtype"]]
    y = (_rounded(s["x"].float()) @ w.T).to(t)
    return dict(y=y, d_x=(_rounded(s["d_y"].float()) @ w).to(t)) if case["train"] else y


def _sum_and_norm(s):
    """h as it is kept, its values in fp32, 1 / rms and the normed rows in fp32."""
    h = (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
    v = h.float()
    rstd = (v.square().mean(1, keepdim=True) + EPS).rsqrt()
    return h, v, rstd, v * rstd * s["norm_weight"]


def _norm_grads(s, v, rstd, d_y):
    """The gradients of h and of the norm's weight from fp32 d_y."""
    u = v * rstd
    p = d_y * s["norm_weight"]
    d_h = s["d_h"].float() + rstd * (p - u * (p * u).mean(1, keepdim=True))
    return d_h.to(s["residual"].dtype), (d_y * u).sum(0)


def _plain_norm(s, case):
    h, v, rstd, y = _sum_and_norm(s)
    r = dict(y=_rounded(y).to(torch.bfloat16) if case["out"] == "fp8" else y.to(TYPES[case["out"]]), h=h)
    if case["train"]:
        r["d_h"], r["d_weight"] = _norm_grads(s, v, rstd, s["d_y"].float())
    return r


def _plain_block(s, case):
    w, t = _weight_values(s, case), TYPES[case["dtype"]]
    h, v, rstd, y = _sum_and_norm(s)
    r = dict(y=(_rounded(y) @ w.T).to(t), h=h)
    if case["train"]:
        r["d_h"], r["d_weight"] = _norm_grads(s, v, rstd, _rounded(s["d_y"].float()) @ w)
    return r


def _plain_clip(s, case):
    total = torch.stack([x.double().square().sum() for x in s["grads"]]).sum().sqrt()
    factor = torch.where(total > s["max_norm"], s["max_norm"] / total, 1.0).float()
    for to, x in zip(s["out"], s["grads"]):
        to.copy_(x.float() * factor)
    return dict(norm=total.float(), grads=s["out"])


# ---- bytes and operations ---------------------------------------------------------------------

def work(case: dict) -> dict:
    size = TYPES[case["dtype"]].itemsize
    if case["kind"] == "clip":
        return {"bytes": 2 * sum(_sizes(case)) * size, "flops": 3 * sum(_sizes(case))}
    if case["kind"] == "norm":
        values = case["rows"] * case["d"]
        kept = 2 * size + size + (1 if case["out"] == "fp8" else size)  # x and residual in, h and y out
        more = 3 * size if case["train"] else 0  # d_y and d_h in, d_h out
        return {"bytes": values * (kept + more), "flops": values * (18 if case["train"] else 8)}
    m, k, n = case["m"], case["k"], case["n"]
    twice = 2 if case["train"] else 1
    values = m * k + m * n
    bytes_ = twice * values * size + n * k
    if case["kind"] == "block":
        bytes_ += twice * 2 * m * k * size  # the residual beside x and h beside y; d_h of both
    return {"bytes": bytes_, "flops": twice * 2 * m * k * n}


# ---- the definition in 64 bits ----------------------------------------------------------------

def _e4m3(v: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value, ties to even: steps of 2^-3 of the binade, 2^-9 at the least."""
    a = v.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(v) * torch.round(a / step) * step


def _exact_rounded(x: torch.Tensor) -> torch.Tensor:
    parts = []
    for p in x.split(BLOCK, 1):
        top = p.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, LARGEST) / LARGEST)))
        parts.append(_e4m3(p / scale) * scale)
    return torch.cat(parts, 1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "clip":
        flat = torch.cat([x.double() for x in s["grads"]])
        total = torch.linalg.vector_norm(flat)
        factor = min(1.0, s["max_norm"] / float(total))
        return dict(norm=total, grads=[x.double() * factor for x in s["grads"]])
    w = None
    if case["kind"] != "norm":
        w = s["q"][:, :case["k"]].double()
        e = s["scales"].double()
        for i in range(0, case["n"], BLOCK):
            for j in range(0, case["k"], BLOCK):
                w[i:i + BLOCK, j:j + BLOCK] *= e[i // BLOCK, j // BLOCK]
    if case["kind"] == "product":
        y = _exact_rounded(s["x"].double()) @ w.T
        return dict(y=y, d_x=_exact_rounded(s["d_y"].double()) @ w) if case["train"] else y
    # the sum is kept in the residual's type, and everything behind it is taken from what is kept
    h = (s["x"].double() + s["residual"].double()).to(s["residual"].dtype).double()
    weight = s["norm_weight"].double()
    rms = torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS)
    y = h / rms * weight
    if case["kind"] == "norm":
        r = dict(y=_exact_rounded(y) if case["out"] == "fp8" else y, h=h)
        d_y = s["d_y"].double() if case["train"] else None
    else:
        r = dict(y=_exact_rounded(y) @ w.T, h=h)
        d_y = _exact_rounded(s["d_y"].double()) @ w if case["train"] else None
    if case["train"]:
        g = d_y * weight
        inner = (g * h).sum(1, keepdim=True)
        r["d_h"] = s["d_h"].double() + g / rms - h * inner / (rms ** 3 * h.shape[1])
        r["d_weight"] = (d_y * h / rms).sum(0)
    return r
