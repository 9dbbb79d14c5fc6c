"""The operators of a DiT fine-tuning step that are timed against their plain forms.

Three operators that one step of a block uses together: the rotation of queries and keys by
their positions, the frozen linear with 8-bit floating-point blocks (activations quantised per
row and 128 columns with powers of two, weights held per 128 x 128 with float32 scales), and the
orthogonalised update of trained matrices. ``run`` computes them in plain float32 torch where ``own`` is false and calls the package's
entry points where it is true.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NORM_EPS = 1e-7


# ------------------------------------------------------------------------------------ cases
def _rotary(name, batch, tokens, q_heads, k_heads, head_dim, rotary_dim, interleaved, dtype, direction, indexed):
    return {"name": name, "op": "rotary", "batch": batch, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads,
            "head_dim": head_dim, "rotary_dim": rotary_dim, "interleaved": interleaved, "dtype": dtype,
            "direction": direction, "indexed": indexed}


def _fp8(name, rows, in_features, out_features, bias, dtype, direction):
    return {"name": name, "op": "fp8", "rows": rows, "in_features": in_features, "out_features": out_features,
            "bias": bias, "dtype": dtype, "direction": direction}


def _orthogonalize(name, count, rows, cols, dtype):
    return {"name": name, "op": "orthogonalize", "count": count, "rows": rows, "cols": cols, "dtype": dtype}


def listed():
    return [
        # one new token of four sequences against a position table: latency of the call
        _rotary("rotary token", 4, 1, 24, 24, 128, 128, False, "bf16", "forward", True),
        # the 24 x 128 heads of one block over two samples of 4096 image and 512 text tokens
        _rotary("rotary block", 2, 4608, 24, 24, 128, 128, True, "bf16", "forward", False),
        # the same heads in training, a packed stream of odd length, half of each head rotated
        _rotary("rotary train", 1, 12287, 24, 8, 128, 64, False, "f16", "train", True),
        # a long stream in training, both gradients
        _rotary("rotary long train", 1, 32768, 24, 24, 128, 128, True, "bf16", "train", False),
        # the adaLN modulation linear: one row for each sample
        _fp8("fp8 adaln", 2, 3072, 18432, True, "bf16", "forward"),
        # the 512 text tokens of one sample through a projection, and a ragged caption batch
        _fp8("fp8 text", 512, 3072, 3072, False, "bf16", "forward"),
        _fp8("fp8 ragged train", 1003, 1090, 2050, True, "f16", "train"),
        # the MLP of one block over 9216 tokens: forward, and the gradient of its second half
        _fp8("fp8 mlp", 9216, 3072, 12288, True, "bf16", "forward"),
        _fp8("fp8 mlp grad", 9216, 12288, 3072, False, "bf16", "grad"),
        # the rank-32 adapter factors of q, k, v and o in 36 blocks
        _orthogonalize("muon adapters", 144, 32, 3072, "f32"),
        # a tall odd projection on its own
        _orthogonalize("muon odd", 1, 1000, 521, "bf16"),
        # q, k, v and o of a block trained in full
        _orthogonalize("muon qkvo", 4, 3072, 3072, "bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rotary", "fp8", "orthogonalize"))
    if op == "rotary":
        head_dim = rng.choice((64, 80, 96, 128, 256))
        rotary_dim = rng.choice((head_dim, head_dim, head_dim // 2, head_dim - 16))
        k_heads = rng.choice((1, 2, 4, 8, 24))
        q_heads = k_heads * rng.choice((1, 1, 2, 3, 5))
        direction = rng.choice(("forward", "train"))
        most = min(32768, (100 << 20) // ((q_heads + k_heads) * head_dim))
        tokens = _spread(rng, 1, most)
        batch = rng.randint(1, max(1, min(8, most // tokens)))
        return {"op": "rotary", "batch": batch, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads,
                "head_dim": head_dim, "rotary_dim": rotary_dim, "interleaved": rng.random() < 0.5,
                "dtype": rng.choice(("bf16", "f16", "f32")), "direction": direction, "indexed": rng.random() < 0.5}
    if op == "fp8":
        direction = rng.choice(("forward", "grad", "train"))
        rows, k, n = _spread(rng, 1, 16384), _spread(rng, 64, 12288), _spread(rng, 64, 18432)
        if rng.random() < 0.6:  # widths that models have; the others stay as odd as they fell
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        most = 9216 * 3072 * 12288 // (2 if direction == "train" else 1)
        rows = max(1, min(rows, most // (k * n)))
        return {"op": "fp8", "rows": rows, "in_features": k, "out_features": n, "bias": rng.random() < 0.5,
                "dtype": rng.choice(("bf16", "f16")), "direction": direction}
    short = _spread(rng, 4, 3072)
    long = _spread(rng, short, 12288)
    cost = short * short * (3 * long + short)
    most = 4 * 4 * 3072 ** 3
    if cost > most:
        long = short
    count = max(1, min(_spread(rng, 1, 256), most // (short * short * (3 * long + short)), (64 << 20) // (short * long)))
    rows, cols = (short, long) if rng.random() < 0.5 else (long, short)
    return {"op": "orthogonalize", "count": count, "rows": rows, "cols": cols, "dtype": rng.choice(("bf16", "f16", "f32"))}


# ----------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _prepare_rotary(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    b, s, d = case["batch"], case["tokens"], case["head_dim"]
    hq, hk = case["q_heads"], case["k_heads"]
    # queries and keys are views of one fused projection, as a block has them
    fused = _randn(gen, b, s, (hq + hk) * d).to(dtype)
    q = fused[..., : hq * d].unflatten(-1, (hq, d))
    k = fused[..., hq * d :].unflatten(-1, (hk, d))
    half = case["rotary_dim"] // 2
    rows = 4 * s + 64 if case["indexed"] else s
    frequencies = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angles = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * frequencies[None]
    state = {"case": case, "q": q, "k": k, "cos": angles.cos().float(), "sin": angles.sin().float(), "positions": None}
    if case["indexed"]:  # every sequence starts somewhere of its own in the table
        start = torch.randint(0, rows - s + 1, (b, 1), generator=gen, device="cuda")
        state["positions"] = start + torch.arange(s, device="cuda")[None]
    if case["direction"] == "train":
        state["grads"] = (_randn(gen, b, s, hq, d).to(dtype), _randn(gen, b, s, hk, d).to(dtype))
    return state


def _weight_codes(weight):
    """Codes [out, in] (rows 16 bytes apart or a multiple of it) and one scale for each 128 x 128 block."""
    n, k = weight.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    padded = torch.zeros(nb * BLOCK, kb * BLOCK, device=weight.device)
    padded[:n, :k] = weight
    blocks = padded.view(nb, BLOCK, kb, BLOCK)
    scale = blocks.abs().amax(dim=(1, 3)).clamp_min(AMAX_FLOOR) / E4M3_MAX
    codes = (blocks / scale[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:n, :k].to(torch.float8_e4m3fn)
    held = torch.zeros(n, -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device=weight.device)
    held.view(torch.uint8)[:, :k] = codes.view(torch.uint8)
    return held[:, :k], scale


def _prepare_fp8(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    m, k, n = case["rows"], case["in_features"], case["out_features"]
    weight, scale = _weight_codes(0.02 * _randn(gen, n, k) * torch.exp(0.3 * _randn(gen, n, 1)))
    state = {"case": case, "weight": weight, "scale": scale, "bias": None}
    # activations after a modulated norm: some channels are larger than others
    if case["direction"] != "grad":
        state["x"] = (_randn(gen, m, k) * torch.exp(0.5 * _randn(gen, 1, k))).to(dtype)
    if case["direction"] != "forward":  # gradients are small, and differ from token to token
        state["grad"] = (1e-3 * _randn(gen, m, n) * torch.exp(0.5 * _randn(gen, m, 1))).to(dtype)
    if case["bias"]:
        state["bias"] = (0.1 * _randn(gen, n)).to(dtype)
    return state


def _prepare_orthogonalize(case, seed):
    gen = _generator(seed)
    b, m, n = case["count"], case["rows"], case["cols"]
    # momentum of a weight's gradient: rows and columns of different size over a few strong directions
    update = _randn(gen, b, m, n) * torch.exp(0.5 * _randn(gen, b, m, 1)) * torch.exp(0.5 * _randn(gen, b, 1, n))
    strong = min(4, m, n)
    update += 2.0 * _randn(gen, b, m, strong) @ _randn(gen, b, strong, n)
    return {"case": case, "update": (1e-3 * update).to(DTYPES[case["dtype"]])}


def prepare(case, seed):
    return {"rotary": _prepare_rotary, "fp8": _prepare_fp8, "orthogonalize": _prepare_orthogonalize}[case["op"]](case, seed)


# ------------------------------------------------------------------------------ plain forms
def _plain_rotate(x, cos, sin, interleaved, inverse):
    half = cos.shape[-1]
    v = x.float()
    if interleaved:
        a, b = v[..., 0 : 2 * half : 2], v[..., 1 : 2 * half : 2]
    else:
        a, b = v[..., :half], v[..., half : 2 * half]
    if inverse:
        sin = -sin
    first, second = a * cos - b * sin, a * sin + b * cos
    if interleaved:
        rotated = torch.stack((first, second), -1).flatten(-2)
    else:
        rotated = torch.cat((first, second), -1)
    return torch.cat((rotated, v[..., 2 * half :]), -1).to(x.dtype)


def _plain_rotary(s):
    cos, sin = s["cos"], s["sin"]
    if s["positions"] is not None:
        cos, sin = cos[s["positions"]], sin[s["positions"]]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    interleaved = s["case"]["interleaved"]
    out = [_plain_rotate(x, cos, sin, interleaved, False) for x in (s["q"], s["k"])]
    if s["case"]["direction"] == "train":
        out += [_plain_rotate(g, cos, sin, interleaved, True) for g in s["grads"]]
    return out


def _plain_rows(x):
    """What the rows of x are after the trip through their 8-bit codes: one scale for each 128 columns,
    the least power of two that brings them within the format's range (dividing by it is exact)."""
    m, k = x.shape
    padded = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).view(m, -1, BLOCK)
    fraction, exponent = torch.frexp(padded.abs().amax(-1, keepdim=True).clamp_min(AMAX_FLOOR))
    scale = torch.ldexp(torch.ones_like(fraction), exponent - 9 + (fraction > E4M3_MAX / 512).int())
    return ((padded / scale).to(torch.float8_e4m3fn).float() * scale).view(m, -1)[:, :k]


def _plain_weight(weight, scale):
    n, k = weight.shape
    spread = scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return weight.float() * spread


def _plain_fp8(s):
    weight = _plain_weight(s["weight"], s["scale"])
    out = []
    if "x" in s:
        y = _plain_rows(s["x"]) @ weight.t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        out.append(y.to(s["x"].dtype))
    if "grad" in s:
        out.append((_plain_rows(s["grad"]) @ weight).to(s["grad"].dtype))
    return out


def _plain_orthogonalize(s):
    x = s["update"].float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    x = x / x.square().sum(dim=(-2, -1), keepdim=True).sqrt().clamp_min(NORM_EPS)
    a, b, c = COEFFICIENTS
    for _ in range(5):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    if tall:
        x = x.transpose(-2, -1)
    return [x.to(torch.bfloat16)]


# ------------------------------------------------------------------------------- the package
def _own_rotary(s):
    from moss_image_b200.rotary import apply_rotary

    interleaved = s["case"]["interleaved"]
    if s["case"]["direction"] == "forward":
        return apply_rotary(s["q"], s["k"], s["cos"], s["sin"], interleaved=interleaved, positions=s["positions"])
    q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
    out = apply_rotary(q, k, s["cos"], s["sin"], interleaved=interleaved, positions=s["positions"])
    return [*(y.detach() for y in out), *torch.autograd.grad(out, (q, k), s["grads"])]


def _own_fp8(s):
    from moss_image_b200 import fp8

    direction = s["case"]["direction"]
    if direction == "forward":
        return [fp8.fp8_linear_forward(s["x"], s["weight"], s["scale"], s["bias"])]
    if direction == "grad":
        return [fp8.fp8_linear_backward(s["grad"], s["weight"], s["scale"])]
    x = s["x"].detach().requires_grad_()
    y = fp8.fp8_linear(x, s["weight"], s["scale"], s["bias"])
    return [y.detach(), *torch.autograd.grad(y, x, s["grad"])]


def _own_orthogonalize(s):
    from moss_image_b200.muon import orthogonalize

    return [orthogonalize(s["update"], steps=5, coefficients=COEFFICIENTS, eps=NORM_EPS)]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "fp8": _own_fp8, "orthogonalize": _own_orthogonalize}[op](state)
    return {"rotary": _plain_rotary, "fp8": _plain_fp8, "orthogonalize": _plain_orthogonalize}[op](state)


# --------------------------------------------------------------------------- exact, and work
def _exact_rotate(x, cos, sin, interleaved, sign):
    """Each pair as a complex number, times cos + i sin (or its conjugate)."""
    half = cos.shape[-1]
    v = x.double()
    order = torch.arange(2 * half, device=x.device)
    order = order.view(half, 2) if interleaved else order.view(2, half).t()
    pairs = torch.complex(v[..., order[:, 0]], v[..., order[:, 1]])
    turned = pairs * torch.complex(cos, sign * sin)
    out = v.clone()
    out[..., order[:, 0]], out[..., order[:, 1]] = turned.real, turned.imag
    return out


def _exact_rotary(s):
    cos, sin = s["cos"].double(), s["sin"].double()
    if s["positions"] is not None:
        cos, sin = cos.index_select(0, s["positions"].flatten()), sin.index_select(0, s["positions"].flatten())
        cos, sin = (t.view(*s["positions"].shape, -1) for t in (cos, sin))
    cos, sin = cos[..., None, :], sin[..., None, :]
    interleaved = s["case"]["interleaved"]
    out = [_exact_rotate(s[key], cos, sin, interleaved, 1.0) for key in ("q", "k")]
    if s["case"]["direction"] == "train":
        out += [_exact_rotate(g, cos, sin, interleaved, -1.0) for g in s["grads"]]
    return out


def _exact_rows(x):
    """The quantised rows from the number format itself: 3 fraction bits, exponents from -6, ties to even."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[1], BLOCK):
        v = x[:, at : at + BLOCK].double()
        scale = torch.exp2(torch.log2(v.abs().amax(1, keepdim=True).clamp_min(AMAX_FLOOR) / E4M3_MAX).ceil())
        v = v / scale
        exponent = torch.frexp(v.abs())[1].sub(1).clamp_min(-6)
        step = torch.exp2(exponent.double() - 3)
        out[:, at : at + BLOCK] = (v / step).round() * step * scale
    return out


def _exact_weight(weight, scale):
    out = weight.to(torch.float32).double()
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            out[i * BLOCK : (i + 1) * BLOCK, j * BLOCK : (j + 1) * BLOCK] *= scale[i, j].double()
    return out


def _exact_fp8(s):
    weight = _exact_weight(s["weight"], s["scale"])
    out = []
    if "x" in s:
        y = torch.einsum("mk,nk->mn", _exact_rows(s["x"]), weight)
        out.append(y if s["bias"] is None else y + s["bias"].double())
    if "grad" in s:
        out.append(torch.einsum("mn,nk->mk", _exact_rows(s["grad"]), weight))
    return out


def _exact_orthogonalize(s):
    a, b, c = COEFFICIENTS
    x = s["update"].double()
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp_min(NORM_EPS)
    tall = x.shape[-2] > x.shape[-1]
    for _ in range(5):
        if tall:
            gram = x.mT @ x
            x = x @ torch.diag_embed(torch.full_like(x[..., 0, :], a)) + b * (x @ gram) + c * ((x @ gram) @ gram)
        else:
            gram = x @ x.mT
            x = a * x + b * (gram @ x) + c * (gram @ (gram @ x))
    return [x]


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "fp8": _exact_fp8, "orthogonalize": _exact_orthogonalize}[case["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        rows = case["batch"] * case["tokens"]
        values = rows * (case["q_heads"] + case["k_heads"])
        passes = 2 if case["direction"] == "train" else 1
        table = (rows if case["indexed"] else case["tokens"]) * case["rotary_dim"] * 4 + (8 * rows if case["indexed"] else 0)
        return {"bytes": passes * (2 * values * case["head_dim"] * size + table), "flops": passes * 3 * values * case["rotary_dim"]}
    if case["op"] == "fp8":
        m, k, n = case["rows"], case["in_features"], case["out_features"]
        passes = 2 if case["direction"] == "train" else 1
        weight = n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK)
        extra = size * n if case["bias"] and case["direction"] != "grad" else 0
        return {"bytes": passes * (size * m * (k + n) + weight) + extra, "flops": passes * 2 * m * k * n}
    b, short, long = case["count"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # the Gram matrix and its square are symmetric: half of their products; with a long side of many times
    # the short one, the iteration can stay in the short side's square
    each = 5 * short * short * (3 * long + short)
    gram = 3 * short * short * long + 5 * 4 * short ** 3
    return {"bytes": b * short * long * (size + 2), "flops": b * min(each, gram)}
