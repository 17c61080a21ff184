"""What the block operators of splatx_cuda.network are timed and checked on.

``linear`` (a matrix product with bias, activation and residual in its epilogue, and its gradients)
and ``qk_norm_rotary`` (the norm of queries and keys per head and their rotation by positions with
one or several axes, in one pass, and its gradients) are what a transformer over image patches or
splats needs beside attention, layer norm and AdamW. Each case is one call of one of them: ``run``
makes the call a user makes where ``own`` is true and computes the same thing from elementary torch
operations where it is false, in 32 bits (angles in 64: a far position times a frequency has no
digits left of its turn in 32).
"""
import math

import torch

own = False

DEV = "cuda"
F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
EPS = 1e-6
BASE = 100.0  # image and scene positions: wavelengths from 2 pi to a few hundred
BASE_FAR = 10000.0  # positions in a long sequence


def _linear(name, op, type_, rows, cols_in, cols_out, act, residual, keep=True):
    # keep: the forward is training's and leaves what the activation's gradient needs
    return {"name": name, "op": op, "type": type_, "rows": rows, "in": cols_in, "out": cols_out,
            "act": act, "residual": residual, "keep": keep and act != "none"}


def _rotary(name, op, type_, batch, tokens, heads, kv_heads, dim, axes, pairs, where):
    return {"name": name, "op": op, "type": type_, "batch": batch, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "axes": axes, "pairs": pairs, "where": where}


def listed():
    return [
        # ---- linear, forward
        # one token through the first layer of an MLP: a read-out, a step of generation
        _linear("linear_one_token", "linear_fwd", "bf16", 1, 1024, 4096, "gelu", False, False),
        # a few tokens (one per view) through the second layer, added to the stream
        _linear("linear_few_tokens", "linear_fwd", "f16", 24, 4096, 1024, "none", True),
        # sizes that no tile, no vector and no copy fits
        _linear("linear_odd", "linear_fwd", "bf16", 5001, 333, 777, "silu", True),
        # the colour network's MLP over its splats, in 32 bits
        _linear("linear_f32", "linear_fwd", "f32", 2048, 128, 512, "gelu", False),
        # the tokens of a training step through the first layer of an MLP
        _linear("linear_up", "linear_fwd", "bf16", 32768, 1024, 4096, "gelu", False),
        # ---- linear, backward
        # a short sequence's projection
        _linear("linear_bwd_short", "linear_bwd", "f16", 77, 640, 640, "none", False),
        # an MLP's first layer, ordinary training
        _linear("linear_bwd_up", "linear_bwd", "bf16", 8192, 640, 2560, "gelu", False),
        # an MLP's second layer over many tokens
        _linear("linear_bwd_down", "linear_bwd", "bf16", 32768, 4096, 1024, "none", False),
        # ---- norm and rotation of queries and keys
        # the patches of one small image
        _rotary("rotary_patches", "rotary_fwd", "bf16", 1, 96, 8, 8, 64, "32,32", "axis", "grid"),
        # splats by their place in the scene, shared key-value heads
        _rotary("rotary_splats", "rotary_fwd", "bf16", 4, 8192, 16, 4, 128, "32,48,48", "axis", "scene"),
        # frames of a video, an odd number of tokens, a head size of its own
        _rotary("rotary_bwd_video", "rotary_bwd", "f16", 1, 5001, 12, 4, 80, "16,32,32", "neighbours",
                "grid"),
        # splats, the last values of a head not rotated
        _rotary("rotary_bwd_splats", "rotary_bwd", "bf16", 8, 4096, 16, 16, 64, "16,16,16", "whole",
                "scene"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["linear_fwd", "linear_bwd", "rotary_fwd", "rotary_bwd"])
    if op.startswith("linear"):
        while True:
            sizes = [64, 128, 256, 320, 512, 640, 768, 1024, 1280, 2048, 2560, 4096]
            cols = [rng.choice(sizes) if rng.random() < 0.6 else _log_int(rng, 3, 5000)
                    for _ in range(2)]
            case = {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
                    "rows": _log_int(rng, 1, 32768), "in": cols[0], "out": cols[1],
                    "act": rng.choice(ACTIVATIONS), "residual": op == "linear_fwd" and rng.random() < 0.5}
            case["keep"] = case["act"] != "none" and (op == "linear_bwd" or rng.random() < 0.7)
            # no more than the largest listed case; 32 bits cost many times 16
            most = 32768 * 1024 * 4096 // (16 if case["type"] == "f32" else 1)
            if case["rows"] * cols[0] * cols[1] <= most and case["rows"] * sum(cols) <= 32768 * 5120:
                return case
    while True:
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        n = rng.randint(1, 3)
        if rng.random() < 0.5:  # all of a head, in even shares
            share = dim // n // 2 * 2
            axes = [dim - share * (n - 1)] + [share] * (n - 1)
        else:
            axes = [2 * rng.randint(1, dim // n // 2) for _ in range(n)]
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        case = {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "batch": rng.randint(1, 8),
                "tokens": _log_int(rng, 1, 32768), "heads": kv_heads * rng.choice([1, 1, 2, 4]),
                "kv_heads": kv_heads, "dim": dim, "axes": ",".join(map(str, axes)),
                "pairs": rng.choice(["axis", "whole", "neighbours"]),
                "where": rng.choice(["grid", "scene"] if n > 1 else ["scene", "sequence"])}
        values = case["batch"] * case["tokens"] * (case["heads"] + kv_heads) * dim
        if case["heads"] <= 32 and values * BYTES[case["type"]] <= 4 * 8192 * 20 * 128 * 2:
            return case


# ---------------------------------------------------------------- what a program has in hand

def _axes(case):
    return [int(a) for a in case["axes"].split(",")]


def _base(case):
    return BASE_FAR if case["where"] == "sequence" else BASE


def _rand(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=F32) * std).to(dtype)


def _positions(case, gen):
    """[batch, tokens, axes]: whole numbers of a grid or a sequence, or places in a scene."""
    b, n, axes = case["batch"], case["tokens"], len(_axes(case))
    if case["where"] == "scene":
        return torch.rand((b, n, axes), generator=gen, device=DEV) * 256.0 - 128.0
    i = torch.arange(n, device=DEV)
    if case["where"] == "sequence":  # what is left of a long one: far from zero
        start = torch.randint(0, 1 << 20, (b, 1, 1), generator=gen, device=DEV)
        return start + i[None, :, None]
    side = max(1, math.isqrt(n) if axes == 2 else round(n ** (1 / 3)))
    grid = torch.stack([i // side ** (axes - 1 - a) % (side if a else n + 1) for a in range(axes)], -1)
    return grid[None].expand(b, n, axes).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = TYPES[case["type"]]
    s = {"case": case}
    if case["op"].startswith("linear"):
        m, k, n = case["rows"], case["in"], case["out"]
        s["x"] = _rand(gen, (m, k), dtype)
        s["weight"] = _rand(gen, (n, k), dtype, k ** -0.5)
        s["bias"] = _rand(gen, (n,), F32, 0.2)
        s["residual"] = _rand(gen, (m, n), dtype) if case["residual"] else None
        if case["op"] == "linear_bwd":
            s["v_y"] = _rand(gen, (m, n), dtype, 0.5)
            # what the forward kept of a layer with an activation
            s["pre"] = _rand(gen, (m, n), dtype) if case["keep"] else None
        return s
    b, t, d = case["batch"], case["tokens"], case["dim"]
    # queries and keys as a projection of both and the values leaves them: views of one tensor
    both = case["heads"] + case["kv_heads"]
    qkv = _rand(gen, (b, t, both + case["kv_heads"], d), dtype) * 1.5
    s["q"], s["k"] = qkv[:, :, :case["heads"]], qkv[:, :, case["heads"]:both]
    s["q_weight"], s["k_weight"] = (1.0 + _rand(gen, (d,), F32, 0.1) for _ in range(2))
    s["positions"] = _positions(case, gen)
    if case["op"] == "rotary_bwd":
        s["v_q"], s["v_k"] = (_rand(gen, s[x].shape, dtype) for x in ("q", "k"))
    return s


# ---------------------------------------------------------------- the plain form

def _phi(z):
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _tanh_gate(z):
    """s(2 u) = (1 + tanh u) / 2 of the tanh form of gelu, and the slope of 2 u."""
    c = 2.0 * math.sqrt(2.0 / math.pi)
    return 1.0 / (1.0 + torch.exp(-c * (z + 0.044715 * z * z * z))), c * (1.0 + 3 * 0.044715 * z * z)


def _act_plain(name, z):
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return z * _phi(z)
    if name == "gelu_tanh":
        return z * _tanh_gate(z)[0]
    return z


def _slope_plain(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return g * (1.0 + z * (1.0 - g))
    if name == "gelu":
        return _phi(z) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    g, slope = _tanh_gate(z)
    return g + z * g * (1.0 - g) * slope


def _linear_plain(case, x, weight, bias, residual):
    z = x.float() @ weight.float().T + bias
    y = _act_plain(case["act"], z)
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype), z.to(x.dtype) if case["keep"] else None


def _linear_grad_plain(case, v_y, x, weight, pre):
    g = v_y.float()
    if pre is not None:
        g = g * _slope_plain(case["act"], pre.float())
    return (g @ weight.float()).to(x.dtype), (g.T @ x.float()).to(weight.dtype), g.sum(0)


def _pair_list(case):
    """(first, second, axis, frequency) of the rotated pairs of a head's values."""
    axes, made = _axes(case), []
    rotated, at = sum(axes), 0
    for a, d in enumerate(axes):
        for j in range(d // 2):
            i = at // 2 + j  # the pair's number
            first, second = {"axis": (at + j, at + d // 2 + j), "whole": (i, i + rotated // 2),
                             "neighbours": (2 * i, 2 * i + 1)}[case["pairs"]]
            made.append((first, second, a, _base(case) ** (-2.0 * j / d)))
        at += d
    return made


def _turns(case, positions):
    """Cosines and sines [batch, tokens, 1, pairs], and which values make the pairs."""
    first, second, axis, freq = zip(*_pair_list(case))
    angle = positions.double()[..., list(axis)] * torch.tensor(freq, dtype=F64, device=DEV)
    return torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None], list(first), list(second)


def _rotated(x, turns, back=False):
    c, s, first, second = turns
    s = -s if back else s
    a, b = x[..., first], x[..., second]
    out = x.clone()
    out[..., first] = a * c - b * s
    out[..., second] = a * s + b * c
    return out


def _rotary_plain(x, weight, turns):
    f = x.float()
    rstd = 1.0 / torch.sqrt((f * f).sum(-1, keepdim=True) / f.shape[-1] + EPS)
    return _rotated(f * rstd * weight, turns).to(x.dtype)


def _rotary_grad_plain(g, x, weight, turns):
    f = x.float()
    rstd = 1.0 / torch.sqrt((f * f).sum(-1, keepdim=True) / f.shape[-1] + EPS)
    g = _rotated(g.float(), turns, back=True)
    xhat = f * rstd
    gw = g * weight
    v_x = rstd * (gw - xhat * ((gw * xhat).sum(-1, keepdim=True) / f.shape[-1]))
    return v_x.to(x.dtype), (g * xhat).sum((0, 1, 2))


# ---------------------------------------------------------------- one call

def run(s):
    case, op = s["case"], s["case"]["op"]
    if op == "linear_fwd":
        if own:
            return _network().linear_fwd(s["x"], s["weight"], s["bias"], activation=_name(case),
                                         residual=s["residual"], keep=case["keep"])
        return _linear_plain(case, s["x"], s["weight"], s["bias"], s["residual"])
    if op == "linear_bwd":
        if own:
            return _network().linear_bwd(s["v_y"], s["x"], s["weight"], s["bias"], s["pre"],
                                         activation=_name(case))
        return _linear_grad_plain(case, s["v_y"], s["x"], s["weight"], s["pre"])
    if own:
        how = {"axes": _axes(case), "base": _base(case), "pairs": case["pairs"],
               "q_weight": s["q_weight"], "k_weight": s["k_weight"], "eps": EPS}
        if op == "rotary_fwd":
            return _network().qk_norm_rotary_fwd(s["q"], s["k"], s["positions"], **how)
        return _network().qk_norm_rotary_bwd(s["v_q"], s["v_k"], s["q"], s["k"], s["positions"], **how)
    turns = _turns(case, s["positions"])
    if op == "rotary_fwd":
        return _rotary_plain(s["q"], s["q_weight"], turns), _rotary_plain(s["k"], s["k_weight"], turns)
    v_q, v_qw = _rotary_grad_plain(s["v_q"], s["q"], s["q_weight"], turns)
    v_k, v_kw = _rotary_grad_plain(s["v_k"], s["k"], s["k_weight"], turns)
    return v_q, v_k, v_qw, v_kw


def _name(case):
    return None if case["act"] == "none" else case["act"]


def _network():
    import sys
    if "splatx-metal_b200" not in sys.path:
        sys.path.insert(0, "splatx-metal_b200")
    from splatx_cuda import network
    return network


# ---------------------------------------------------------------- what it cannot do without

def work(case):
    e = BYTES[case["type"]]
    if case["op"].startswith("linear"):
        m, k, n, kept = case["rows"], case["in"], case["out"], case["keep"]
        if case["op"] == "linear_fwd":  # x, weight, bias, residual in; y and what the backward needs out
            mn = m * n * (1 + kept + case["residual"])
            return {"bytes": (m * k + n * k + mn) * e + 4 * n, "flops": 2.0 * m * n * k}
        return {"bytes": (2 * m * k + 2 * n * k + m * n * (1 + kept)) * e + 4 * n, "flops": 4.0 * m * n * k}
    tokens, d = case["batch"] * case["tokens"], case["dim"]
    values = tokens * (case["heads"] + case["kv_heads"]) * d
    size = 4 if case["where"] == "scene" else 8
    where = tokens * len(_axes(case)) * size
    if case["op"] == "rotary_fwd":
        return {"bytes": 2 * values * e + where + 8 * d, "flops": 7.0 * values}
    return {"bytes": 3 * values * e + where + 16 * d, "flops": 14.0 * values}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    """What ``run`` returns, in 64 bits, from the operators' definitions."""
    s = prepare(case, seed)
    if case["op"].startswith("linear"):
        return _exact_linear(case, s)
    weights = [s["q_weight"].double().requires_grad_(), s["k_weight"].double().requires_grad_()]
    xs = [s["q"].double().requires_grad_(), s["k"].double().requires_grad_()]
    outs = [_exact_rotary(case, x, w, s["positions"].double()) for x, w in zip(xs, weights)]
    if case["op"] == "rotary_fwd":
        return tuple(o.detach() for o in outs)
    return torch.autograd.grad(outs, xs + weights, [s["v_q"].double(), s["v_k"].double()])


def _exact_rotary(case, x, weight, positions):
    """Each axis' run of pairs as complex numbers times exp(i angle)."""
    u = x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * weight
    axes, out, at = _axes(case), [None] * x.shape[-1], 0
    rotated = sum(axes)
    for a, d in enumerate(axes):
        ladder = torch.exp(torch.arange(d // 2, device=DEV, dtype=F64) * (-2.0 / d * math.log(_base(case))))
        turn = torch.polar(torch.ones_like(positions[..., :1]), positions[..., a:a + 1] * ladder)[:, :, None]
        if case["pairs"] == "axis":
            one, two = range(at, at + d // 2), range(at + d // 2, at + d)
        elif case["pairs"] == "whole":
            one, two = range(at // 2, (at + d) // 2), range((rotated + at) // 2, (rotated + at + d) // 2)
        else:
            one, two = range(at, at + d, 2), range(at + 1, at + d, 2)
        z = torch.complex(u[..., list(one)], u[..., list(two)]) * turn
        for j, (i, k) in enumerate(zip(one, two)):
            out[i], out[k] = z.real[..., j], z.imag[..., j]
        at += d
    return torch.stack([u[..., i] if o is None else o for i, o in enumerate(out)], -1)


def _exact_linear(case, s):
    x, w, b = (s[k].double() for k in ("x", "weight", "bias"))
    act = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
           "gelu": lambda z: z * torch.special.ndtr(z),
           "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))}[case["act"]]
    if case["op"] == "linear_fwd":
        z = torch.addmm(b, x, w.T)
        y = act(z)
        if s["residual"] is not None:
            y += s["residual"].double()
        return y, z if case["keep"] else None
    g = s["v_y"].double()
    if s["pre"] is not None:
        z = s["pre"].double().requires_grad_()
        if case["act"] == "gelu":  # ndtr' is the normal density
            slope = torch.special.ndtr(z) + z * torch.exp(torch.distributions.Normal(0.0, 1.0).log_prob(z))
            g = g * slope.detach()
        else:
            (g,) = torch.autograd.grad(act(z), z, g)
    return torch.mm(g, w), torch.mm(g.T, x), g.sum(0)
