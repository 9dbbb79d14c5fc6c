"""More operators of a DiT fine-tuning step that are timed against their plain forms.

Three that a block with a text branch uses together: layer norm with the gradients of its gain and
offset, attention of image tokens to a text encoder's states (another length, masked or packed), and
activations kept as 8-bit codes between the forward and the backward pass, with the weight gradients
that read them. ``run`` computes them in plain float32 torch where ``own`` is false and calls the
package's entry points where it is true.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
CODE_BLOCK = 32  # values that share a power of two
CODE_MAX = 127
LEAST_POWER = -126
MOST_POWER = {"bf16": 121, "f16": 9, "f32": 121}


# ------------------------------------------------------------------------------------ cases
def _norm(name, rows, dim, dtype, gain, direction):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "gain": gain, "direction": direction}


def _codes(name, rows, dim, out_features, dtype, direction):
    return {"name": name, "op": "codes", "rows": rows, "dim": dim, "out_features": out_features, "dtype": dtype,
            "direction": direction}


def _cross(name, batch, q_tokens, k_tokens, q_heads, k_heads, head_dim, dtype, layout, direction):
    return {"name": name, "op": "cross", "batch": batch, "q_tokens": q_tokens, "k_tokens": k_tokens, "q_heads": q_heads,
            "k_heads": k_heads, "head_dim": head_dim, "dtype": dtype, "layout": layout, "direction": direction}


def listed():
    return [
        # the timestep conditions of a small batch: latency of the call
        _norm("norm condition", 4, 3072, "bf16", "same", "forward"),
        # both samples of a block (4096 image and 512 text tokens each), all three gradients
        _norm("norm block train", 9216, 3072, "bf16", "same", "train"),
        # a packed stream of odd length and width under float32 gains
        _norm("norm odd train", 12287, 1090, "f16", "f32", "train"),
        # a long stream in float32 without gain and offset, as before a modulation
        _norm("norm long plain", 32768, 3072, "f32", "none", "forward"),
        # a block's input kept between forward and backward: coded, and decoded again
        _codes("codes block", 9216, 3072, 0, "bf16", "keep"),
        # a ragged caption batch
        _codes("codes odd", 1003, 1090, 0, "f16", "keep"),
        # the weight gradient of a projection trained in full, and of an adapter's first factor (rank 32)
        _codes("codes projection", 9216, 3072, 3072, "bf16", "grad"),
        _codes("codes adapter", 9216, 3072, 32, "bf16", "grad"),
        # one query token of each of four captions: latency
        _cross("cross token", 4, 1, 512, 24, 24, 128, "bf16", "lengths", "forward"),
        # the image tokens of two samples against their 512 text tokens
        _cross("cross text", 2, 4096, 512, 24, 24, 128, "bf16", "dense", "forward"),
        # the same in training, captions of different lengths
        _cross("cross text train", 2, 4096, 512, 24, 24, 128, "bf16", "lengths", "train"),
        # a packed stream of five samples, one without a caption, shared key heads
        _cross("cross packed train", 5, 4099, 777, 24, 8, 64, "f16", "packed", "train"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "codes", "cross", "cross"))
    if op == "norm":
        dim = _spread(rng, 8, 12288)
        if rng.random() < 0.6:  # widths that models have; the others stay as odd as they fell
            dim = -(-dim // 64) * 64
        rows = min(_spread(rng, 1, 65536), 32768 * 3072 // dim)
        return {"op": "norm", "rows": rows, "dim": dim, "dtype": rng.choice(("bf16", "f16", "f32")),
                "gain": rng.choice(("none", "same", "f32")), "direction": rng.choice(("forward", "train"))}
    if op == "codes":
        dim = _spread(rng, 16, 12288)
        if rng.random() < 0.6:
            dim = -(-dim // 64) * 64
        rows = min(_spread(rng, 1, 65536), 32768 * 3072 // (2 * dim))
        if rng.random() < 0.5:
            return {"op": "codes", "rows": rows, "dim": dim, "out_features": 0,
                    "dtype": rng.choice(("bf16", "f16", "f32")), "direction": "keep"}
        out_features = _spread(rng, 4, 12288)
        if rng.random() < 0.6:
            out_features = -(-out_features // 16) * 16
        rows = max(1, min(rows, 9216 * 3072 * 3072 // (dim * out_features), 32768 * 3072 // out_features))
        return {"op": "codes", "rows": rows, "dim": dim, "out_features": out_features,
                "dtype": rng.choice(("bf16", "f16")), "direction": "grad"}
    k_heads = rng.choice((1, 2, 4, 8, 16, 24))
    q_heads = k_heads * rng.choice((1, 1, 1, 2, 3, 4))
    head_dim = rng.choice((64, 72, 80, 96, 128, 128))
    layout = rng.choice(("dense", "lengths", "holes", "packed"))
    batch = rng.randint(1, 8)
    q_tokens, k_tokens = _spread(rng, 1, 8192), _spread(rng, 1, 4096)
    if layout == "packed":  # the whole streams' lengths
        q_tokens, k_tokens = max(q_tokens, batch), max(k_tokens, batch)
    copies = 1 if layout == "packed" else batch
    most = 2 * 24 * 4096 * 400
    q_tokens = max(batch if layout == "packed" else 1, min(q_tokens, most // (copies * q_heads * k_tokens)))
    return {"op": "cross", "batch": batch, "q_tokens": q_tokens, "k_tokens": k_tokens, "q_heads": q_heads,
            "k_heads": k_heads, "head_dim": head_dim, "dtype": rng.choice(("bf16", "f16")), "layout": layout,
            "direction": rng.choice(("forward", "train"))}


# ----------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _activations(gen, rows, dim):
    """A residual stream: channels of different size, some of them away from zero."""
    return _randn(gen, rows, dim) * torch.exp(0.5 * _randn(gen, 1, dim)) + 0.5 * _randn(gen, 1, dim)


def _prepare_norm(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    rows, dim = case["rows"], case["dim"]
    state = {"case": case, "x": _activations(gen, rows, dim).to(dtype), "weight": None, "bias": None}
    gain_dtype = torch.float32 if case["gain"] == "f32" else dtype
    if case["gain"] != "none":
        state["weight"] = (1.0 + 0.2 * _randn(gen, dim)).to(gain_dtype)
        state["bias"] = (0.1 * _randn(gen, dim)).to(gain_dtype)
    if case["direction"] == "train":
        out_dtype = dtype if case["gain"] == "none" else torch.promote_types(dtype, gain_dtype)
        state["grad"] = (1e-2 * _randn(gen, rows, dim)).to(out_dtype)
    return state


def _powers(amax, most):
    """The least power of two with amax <= 127 * 2^p, within the range that codes have."""
    fraction, exponent = torch.frexp(amax)
    power = exponent - 7 + (fraction > CODE_MAX / 128).int()
    return power.clamp(LEAST_POWER, most)


def _plain_code(x, most):
    rows, dim = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -dim % CODE_BLOCK)).view(rows, -1, CODE_BLOCK)
    power = _powers(blocks.abs().amax(-1), most)
    scaled = torch.ldexp(blocks, -power[..., None])
    codes = scaled.round().clamp(-CODE_MAX, CODE_MAX).to(torch.int8).view(rows, -1)[:, :dim]
    return codes, (power + 127).to(torch.uint8)


def _plain_decode(codes, exponents):
    power = (exponents.int() - 127).repeat_interleave(CODE_BLOCK, 1)[:, : codes.shape[1]]
    return torch.ldexp(codes.float(), power)


def _prepare_codes(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    rows, dim, out = case["rows"], case["dim"], case["out_features"]
    x = _activations(gen, rows, dim).to(dtype)
    if case["direction"] == "keep":
        return {"case": case, "x": x}
    # what the forward pass kept: codes whose rows start on 16-byte boundaries, and a byte for each 32 of them
    codes, exponents = _plain_code(x, MOST_POWER[case["dtype"]])
    held = torch.zeros(rows, -(-dim // 16) * 16, dtype=torch.int8, device="cuda")
    held[:, :dim] = codes
    grad = (1e-3 * _randn(gen, rows, out) * torch.exp(0.5 * _randn(gen, rows, 1))).to(dtype)
    return {"case": case, "codes": held[:, :dim], "exponents": exponents, "grad": grad}


def _parts(total, count, salt):
    """`total` tokens in `count` samples of uneven lengths, none empty."""
    rng = random.Random(salt * 1000003 + total * 31 + count)
    cuts = sorted(rng.sample(range(1, total), count - 1)) if count > 1 else []
    return [b - a for a, b in zip([0, *cuts], [*cuts, total])]


def _lengths(case):
    """(query tokens, key tokens) of each sample."""
    batch, q, k = case["batch"], case["q_tokens"], case["k_tokens"]
    if case["layout"] == "packed":
        keys = _parts(k, batch, 2)
        if batch > 2:  # one sample has no caption: its keys go to the next one
            keys[1], keys[2] = 0, keys[1] + keys[2]
        return _parts(q, batch, 1), keys
    if case["layout"] == "lengths":  # captions of several lengths, every fifth one empty
        shares = (0.6, 1.0, 0.25, 0.0, 0.9)
        return [q] * batch, [int(math.ceil(k * shares[i % 5])) for i in range(batch)]
    return [q] * batch, [k] * batch


def _prepare_cross(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    batch, tq, tk, d = case["batch"], case["q_tokens"], case["k_tokens"], case["head_dim"]
    hq, hk = case["q_heads"], case["k_heads"]
    packed = case["layout"] == "packed"
    lead = 1 if packed else batch
    # keys and values are views of one fused projection of the text states
    q = _randn(gen, lead, tq, hq, d).to(dtype)
    fused = _randn(gen, lead, tk, 2, hk, d).to(dtype)
    state = {"case": case, "q": q, "k": fused[:, :, 0], "v": fused[:, :, 1], "mask": None, "scale": d ** -0.5}
    if packed:
        state["q"], state["k"], state["v"] = (t[0] for t in (q, state["k"], state["v"]))
        bounds = [torch.tensor([0, *n], device="cuda").cumsum(0) for n in _lengths(case)]
        state["q_offsets"], state["k_offsets"] = bounds
    elif case["layout"] == "lengths":
        state["mask"] = torch.arange(tk, device="cuda")[None] < torch.tensor(_lengths(case)[1], device="cuda")[:, None]
    elif case["layout"] == "holes":
        state["mask"] = torch.rand(batch, tk, generator=gen, device="cuda") < 0.7
    if case["direction"] == "train":
        state["grad"] = (1e-2 * _randn(gen, lead, tq, hq, d)).to(dtype)
        if packed:
            state["grad"] = state["grad"][0]
    return state


def prepare(case, seed):
    return {"norm": _prepare_norm, "codes": _prepare_codes, "cross": _prepare_cross}[case["op"]](case, seed)


# ------------------------------------------------------------------------------ plain forms
def _plain_norm(s):
    x = s["x"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + EPS)
    normal = centred * rstd
    y, out_dtype = normal, s["x"].dtype
    if s["weight"] is not None:
        y = normal * s["weight"].float() + s["bias"].float()
        out_dtype = torch.promote_types(out_dtype, s["weight"].dtype)
    out = [y.to(out_dtype)]
    if s["case"]["direction"] == "train":
        g = s["grad"].float()
        dn = g if s["weight"] is None else g * s["weight"].float()
        dx = rstd * (dn - dn.mean(-1, keepdim=True) - normal * (dn * normal).mean(-1, keepdim=True))
        out.append(dx.to(s["x"].dtype))
        if s["weight"] is not None:
            out += [(g * normal).sum(0).to(s["weight"].dtype), g.sum(0).to(s["bias"].dtype)]
    return out


def _plain_codes(s):
    if s["case"]["direction"] == "keep":
        codes, exponents = _plain_code(s["x"], MOST_POWER[s["case"]["dtype"]])
        return [_plain_decode(codes, exponents).to(s["x"].dtype)]
    weight_grad = s["grad"].float().t() @ _plain_decode(s["codes"], s["exponents"])
    return [weight_grad.to(s["grad"].dtype)]


def _allowed(s):
    """Which keys a query may look at, broadcast against [batch, heads, queries, keys]; None for all."""
    if s["case"]["layout"] == "packed":
        queries = torch.arange(s["q"].shape[0], device="cuda")
        keys = torch.arange(s["k"].shape[0], device="cuda")
        of_query = torch.searchsorted(s["q_offsets"], queries, right=True)
        of_key = torch.searchsorted(s["k_offsets"], keys, right=True)
        return (of_query[:, None] == of_key[None])[None, None]
    return None if s["mask"] is None else s["mask"][:, None, None]


def _plain_cross(s):
    packed = s["case"]["layout"] == "packed"
    q, k, v = (t[None] if packed else t for t in (s["q"], s["k"], s["v"]))
    batch, tq, hq, d = q.shape
    groups = hq // k.shape[2]
    q, k, v = (t.float().transpose(1, 2) for t in (q, k, v))
    k_all, v_all = k.repeat_interleave(groups, 1), v.repeat_interleave(groups, 1)
    logits = (q @ k_all.transpose(-2, -1)) * s["scale"]
    allowed = _allowed(s)
    if allowed is not None:
        logits = torch.where(allowed, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0.0, 1.0, total)  # a query without keys: zeros
    o = p @ v_all
    out = [o.transpose(1, 2)]
    if s["case"]["direction"] == "train":
        g = (s["grad"][None] if packed else s["grad"]).float().transpose(1, 2)
        dv = p.transpose(-2, -1) @ g
        dp = g @ v_all.transpose(-2, -1)
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * s["scale"]
        dq, dk = ds @ k_all, ds.transpose(-2, -1) @ q
        dk, dv = (t.unflatten(1, (-1, groups)).sum(2) for t in (dk, dv))
        out += [t.transpose(1, 2) for t in (dq, dk, dv)]
    return [(t[0] if packed else t).to(s["q"].dtype).contiguous() for t in out]


# ------------------------------------------------------------------------------- the package
def _own_norm(s):
    from moss_image_b200.norms import layer_norm

    if s["case"]["direction"] == "forward":
        return [layer_norm(s["x"], s["weight"], s["bias"], EPS)]
    leaves = [t.detach().requires_grad_() for t in (s["x"], s["weight"], s["bias"]) if t is not None]
    y = layer_norm(*leaves, eps=EPS)
    return [y.detach(), *torch.autograd.grad(y, leaves, s["grad"])]


def _own_codes(s):
    from moss_image_b200 import activation_codes

    if s["case"]["direction"] == "keep":
        return [activation_codes.decode_activation(activation_codes.encode_activation(s["x"]))]
    return [activation_codes.coded_weight_gradient(s["grad"], s["codes"], s["exponents"])]


def _own_cross(s):
    from moss_image_b200.cross_attention import cross_attention, cross_attention_packed

    train = s["case"]["direction"] == "train"
    q, k, v = (t.detach().requires_grad_(train) for t in (s["q"], s["k"], s["v"]))
    if s["case"]["layout"] == "packed":
        o = cross_attention_packed(q, k, v, s["q_offsets"], s["k_offsets"], scale=s["scale"])
    else:
        o = cross_attention(q, k, v, key_mask=s["mask"], scale=s["scale"])
    if not train:
        return [o]
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), s["grad"])]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "codes": _own_codes, "cross": _own_cross}[op](state)
    return {"norm": _plain_norm, "codes": _plain_codes, "cross": _plain_cross}[op](state)


# --------------------------------------------------------------------------- exact, and work
def _exact_norm(s):
    """The definition, and its derivatives by the chain rule from the normalised values."""
    x = s["x"].double().requires_grad_()
    leaves = [x]
    variance, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(variance + EPS)
    if s["weight"] is not None:
        leaves += [s["weight"].double().requires_grad_(), s["bias"].double().requires_grad_()]
        y = y * leaves[1] + leaves[2]
    if s["case"]["direction"] == "forward":
        return [y.detach()]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["grad"].double())]


def _exact_decode(codes, exponents):
    out = codes.double()
    for at in range(exponents.shape[1]):
        out[:, at * CODE_BLOCK : (at + 1) * CODE_BLOCK] *= torch.exp2(exponents[:, at : at + 1].double() - 127.0)
    return out


def _exact_codes(s):
    if s["case"]["direction"] == "grad":
        return [torch.einsum("mn,mk->nk", s["grad"].double(), _exact_decode(s["codes"], s["exponents"]))]
    most = MOST_POWER[s["case"]["dtype"]]
    out = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
    for at in range(0, s["x"].shape[1], CODE_BLOCK):
        block = s["x"][:, at : at + CODE_BLOCK].double()
        top = block.abs().amax(1, keepdim=True).clamp_min(1e-300)
        power = torch.floor(torch.log2(top)) - 7.0  # a step or two low; raised until the codes fit
        for _ in range(3):
            power = torch.where(top > CODE_MAX * torch.exp2(power), power + 1.0, power)
        step = torch.exp2(power.clamp(LEAST_POWER, most))
        out[:, at : at + CODE_BLOCK] = (block / step).round().clamp(-CODE_MAX, CODE_MAX) * step
    return [out]


def _exact_cross(s):
    """Sample by sample and key head by key head."""
    case = s["case"]
    packed = case["layout"] == "packed"
    names = ("q", "k", "v", "grad") if case["direction"] == "train" else ("q", "k", "v")
    held = {n: s[n].double() for n in names}
    out = [torch.zeros_like(held["q"])] + [torch.zeros_like(held[n]) for n in names[:3] if len(names) == 4]
    groups = case["q_heads"] // case["k_heads"]
    starts = [[sum(n[:i]) for i in range(len(n))] for n in _lengths(case)]
    for b, (nq, nk) in enumerate(zip(*_lengths(case))):
        if packed:
            rows, keys = slice(starts[0][b], starts[0][b] + nq), slice(starts[1][b], starts[1][b] + nk)
        else:
            rows = (b, slice(None))
            keys = (b, torch.arange(case["k_tokens"], device="cuda") if s["mask"] is None else s["mask"][b].nonzero()[:, 0])
        for h in range(case["k_heads"]):
            mine = slice(h * groups, (h + 1) * groups)
            q = held["q"][rows][:, mine].requires_grad_()
            k, v = held["k"][keys][:, h].requires_grad_(), held["v"][keys][:, h].requires_grad_()
            if k.shape[0] == 0:
                continue
            p = torch.softmax(torch.einsum("thd,sd->hts", q, k) * s["scale"], -1)
            o = torch.einsum("hts,sd->thd", p, v)
            out[0][rows][:, mine] = o.detach()
            if len(names) == 4:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), held["grad"][rows][:, mine])
                out[1][rows][:, mine] = dq
                if packed:
                    out[2][keys][:, h], out[3][keys][:, h] = dk, dv
                else:
                    out[2][b][keys[1], h], out[3][b][keys[1], h] = dk, dv
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "codes": _exact_codes, "cross": _exact_cross}[case["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        values = case["rows"] * case["dim"]
        gain = {"none": 0, "same": size, "f32": 4}[case["gain"]]
        y_size = max(size, gain)
        if case["direction"] == "forward":
            return {"bytes": values * (size + y_size) + 2 * gain * case["dim"], "flops": 7 * values}
        return {"bytes": values * (2 * size + 2 * y_size) + 4 * gain * case["dim"], "flops": 18 * values}
    if case["op"] == "codes":
        values = case["rows"] * case["dim"]
        held = values + case["rows"] * -(-case["dim"] // CODE_BLOCK)
        if case["direction"] == "keep":
            return {"bytes": 2 * values * size + 2 * held, "flops": 4 * values}
        out = case["out_features"]
        return {"bytes": held + size * out * (case["rows"] + case["dim"]), "flops": 2 * values * out}
    q_lengths, k_lengths = _lengths(case)
    pairs = sum(a * b for a, b in zip(q_lengths, k_lengths))
    kept = 0.7 if case["layout"] == "holes" else 1.0
    queries = sum(q_lengths) * case["q_heads"] * case["head_dim"]
    keys = sum(k_lengths) * case["k_heads"] * case["head_dim"]
    flops = 4 * kept * pairs * case["q_heads"] * case["head_dim"]
    if case["direction"] == "forward":
        return {"bytes": size * (2 * queries + 2 * keys), "flops": flops}
    written = case["k_tokens"] * (1 if case["layout"] == "packed" else case["batch"]) * case["k_heads"] * case["head_dim"]
    return {"bytes": size * (4 * queries + 2 * keys + 2 * written), "flops": 3.5 * flops}
