"""What the network operators of splatx_cuda are timed and checked on.

Attention, layer norm and the multi-tensor AdamW step are what a network that predicts, refines or
conditions splats is trained with beside the rasteriser. Each case below is one call of one of
them: ``run`` makes the call a user makes where ``own`` is true and computes the same thing from
elementary torch operations in 32 bits where it is false.
"""
import math

import torch

own = False

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "f8": 1}
EPS_NORM = 1e-5
ADAM = {"lr": 1e-3, "b1": 0.9, "b2": 0.95, "eps": 1e-8, "weight_decay": 0.1}
ADAM_STEP = 100  # the optimiser is this many steps in: both moments have settled
BLOCK = 256      # values that share one scale of an 8-bit moment
F8_MAX, F8_TINY = 448.0, 2.0 ** -9  # e4m3: the largest value and the smallest above zero
FLUSH = 1e-30    # a block whose largest value is below this is held as zeros

# The optimiser's tensor lists. "splats": the six parameter groups of a Gaussian arena at SH
# degree 3 (means, quaternions, scales, opacities, sh0, shN). "network": the weights of a
# transformer of `layers` blocks of width `width` (norms, attention projections, a 4x MLP).
SPLAT_DIMS = (3, 4, 3, 1, 3, 45)


def tensor_sizes(case):
    if case["tensors"] == "splats":
        return [case["count"] * d for d in SPLAT_DIMS]
    w = case["width"]
    block = [w, w, w * 3 * w, 3 * w, w * w, w, w, w, w * 4 * w, 4 * w, 4 * w * w, w]
    return block * case["layers"] + [w, w, w * 59, 59]


def listed():
    return [
        # ---- attention, forward
        # a handful of tokens per view: the call's own latency
        {"name": "attn_fwd_short", "op": "attention_fwd", "type": "bf16", "batch": 1, "heads": 8,
         "kv_heads": 8, "q_len": 96, "kv_len": 96, "dim": 64, "causal": False, "ragged": False},
        # a padded batch of scenes with different token counts, queries from another view
        {"name": "attn_fwd_ragged", "op": "attention_fwd", "type": "f16", "batch": 6, "heads": 12,
         "kv_heads": 12, "q_len": 1000, "kv_len": 1777, "dim": 64, "causal": False, "ragged": True},
        # one long causal sequence with shared key-value heads
        {"name": "attn_fwd_long", "op": "attention_fwd", "type": "bf16", "batch": 1, "heads": 16,
         "kv_heads": 4, "q_len": 8192, "kv_len": 8192, "dim": 128, "causal": True,
         "ragged": False},
        # one query per scene over a long set of keys: a pooled read-out
        {"name": "attn_fwd_one_query", "op": "attention_fwd", "type": "bf16", "batch": 2,
         "heads": 16, "kv_heads": 8, "q_len": 1, "kv_len": 8000, "dim": 128, "causal": False,
         "ragged": False},
        # ---- attention, backward
        # short sequences of an odd length
        {"name": "attn_bwd_short", "op": "attention_bwd", "type": "f16", "batch": 2, "heads": 6,
         "kv_heads": 6, "q_len": 77, "kv_len": 77, "dim": 64, "causal": True, "ragged": False},
        # ordinary training: image tokens, all of them seen by all
        {"name": "attn_bwd_tokens", "op": "attention_bwd", "type": "bf16", "batch": 8, "heads": 16,
         "kv_heads": 16, "q_len": 1024, "kv_len": 1024, "dim": 64, "causal": False,
         "ragged": False},
        # long causal training with shared key-value heads
        {"name": "attn_bwd_long", "op": "attention_bwd", "type": "bf16", "batch": 2, "heads": 16,
         "kv_heads": 4, "q_len": 4096, "kv_len": 4096, "dim": 128, "causal": True,
         "ragged": False},
        # ---- layer norm
        # the activations of one training step
        {"name": "norm_fwd_tokens", "op": "layer_norm_fwd", "type": "bf16", "rows": 32768,
         "cols": 1024},
        # an odd width in 32 bits
        {"name": "norm_bwd_odd", "op": "layer_norm_bwd", "type": "f32", "rows": 5001, "cols": 777},
        {"name": "norm_bwd_tokens", "op": "layer_norm_bwd", "type": "bf16", "rows": 32768,
         "cols": 1024},
        # ---- AdamW
        # a million Gaussians at SH degree 3, moments in 32 bits
        {"name": "adamw_splats", "op": "adamw", "tensors": "splats", "count": 1_000_000, "width": 0,
         "layers": 0, "type": "f32", "bits": 32},
        # a small network's many tensors, moments in 8 bits
        {"name": "adamw_network8", "op": "adamw", "tensors": "network", "count": 0, "width": 640,
         "layers": 16, "type": "bf16", "bits": 8},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["attention_fwd", "attention_bwd", "layer_norm_fwd", "layer_norm_bwd", "adamw"])
    if op.startswith("attention"):
        # at most the largest listed case's multiplications and key-value bytes
        most = 16 * 8192 * 4096 * 128 if op == "attention_fwd" else 2 * 16 * 4096 * 2048 * 128
        while True:
            kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
            group = rng.choice([1, 1, 2, 4])
            q_len = _log_int(rng, 1, 8192) if op == "attention_fwd" else _log_int(rng, 16, 4096)
            same = rng.random() < 0.6
            kv_len = q_len if same else _log_int(rng, 16, 8192)
            case = {"op": op, "type": rng.choice(["bf16", "bf16", "f16"]),
                    "batch": rng.randint(1, 8), "heads": kv_heads * group, "kv_heads": kv_heads,
                    "q_len": q_len, "kv_len": kv_len, "dim": rng.choice([32, 64, 64, 80, 128, 128]),
                    "causal": kv_len >= q_len and rng.random() < 0.5, "ragged": False}
            case["ragged"] = not case["causal"] and rng.random() < 0.4
            if case["heads"] <= 32 and _pairs(case) * case["heads"] * case["dim"] <= most and \
                    case["batch"] * q_len * case["heads"] <= 262144:
                return case
    if op.startswith("layer_norm"):
        cols = _log_int(rng, 32, 8192)
        if rng.random() < 0.6:
            cols = rng.choice([64, 128, 256, 320, 512, 640, 768, 1024, 1280, 2048, 4096, 8192])
        return {"op": op, "type": rng.choice(["f32", "bf16", "f16"]),
                "rows": _log_int(rng, 1, min(32768, (1 << 25) // cols)), "cols": cols}
    splats = rng.random() < 0.5
    return {"op": op, "tensors": "splats" if splats else "network",
            "count": _log_int(rng, 1000, 1_000_000) if splats else 0,
            "width": 0 if splats else rng.choice([64, 100, 192, 256, 384, 500, 640]),
            "layers": 0 if splats else rng.randint(1, 16),
            "type": rng.choice(["f32", "bf16"]), "bits": rng.choice([8, 32])}


# ---------------------------------------------------------------- what a program has in hand

def _kv_lengths(case):
    """The key counts of a ragged batch: full, and shares of it."""
    shares = (1.0, 0.73, 0.41, 0.9, 0.17, 0.62, 0.35, 0.81)
    if not case["ragged"]:
        return [case["kv_len"]] * case["batch"]
    return [max(1, round(case["kv_len"] * shares[b % 8])) for b in range(case["batch"])]


def _pairs(case):
    """(query, key) pairs of one head that the mask leaves, over the batch."""
    q, k = case["q_len"], case["kv_len"]
    if case["causal"]:
        return case["batch"] * (q * (k - q) + q * (q + 1) // 2)
    return q * sum(_kv_lengths(case))


def _mask(case, kv_lens):
    """True where a key is seen, [batch or 1, 1, q_len or 1, kv_len]; None where all are."""
    j = torch.arange(case["kv_len"], device=DEV)
    if case["causal"]:
        i = torch.arange(case["q_len"], device=DEV)
        return (j[None] <= i[:, None] + (case["kv_len"] - case["q_len"]))[None, None]
    if kv_lens is not None:
        return (j[None] < kv_lens[:, None])[:, None, None]
    return None


def _heads(t, heads):
    """[batch, length, kv_heads, dim] -> [batch, heads, length, dim] in 32 bits."""
    t = t.float().transpose(1, 2)
    return t.repeat_interleave(heads // t.shape[1], dim=1)


def _scores(case, q, k, kv_lens):
    s = _heads(q, case["heads"]) @ _heads(k, case["heads"]).transpose(2, 3)
    s = s * (case["dim"] ** -0.5)
    mask = _mask(case, kv_lens)
    return s if mask is None else s.masked_fill(~mask, -math.inf)


def _attention_plain(case, q, k, v, kv_lens):
    s = _scores(case, q, k, kv_lens)
    top = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(dim=-1, keepdim=True)
    out = (e / total) @ _heads(v, case["heads"])
    lse = (top + torch.log(total)).squeeze(-1)
    return out.transpose(1, 2).contiguous().to(q.dtype), lse


def _shared(g, kv_heads, dtype):
    """Gradients per query head summed over the heads that share a key-value head."""
    b, h, n, d = g.shape
    return g.view(b, kv_heads, h // kv_heads, n, d).sum(2).transpose(1, 2).contiguous().to(dtype)


def _attention_grad_plain(case, q, k, v, out, lse, v_out, kv_lens):
    p = torch.exp(_scores(case, q, k, kv_lens) - lse[..., None])
    g = _heads(v_out, case["heads"])
    delta = (g * _heads(out, case["heads"])).sum(-1, keepdim=True)
    v_v = p.transpose(2, 3) @ g
    ds = p * (g @ _heads(v, case["heads"]).transpose(2, 3) - delta) * (case["dim"] ** -0.5)
    v_q = ds @ _heads(k, case["heads"])
    v_k = ds.transpose(2, 3) @ _heads(q, case["heads"])
    return (v_q.transpose(1, 2).contiguous().to(q.dtype), _shared(v_k, case["kv_heads"], k.dtype),
            _shared(v_v, case["kv_heads"], v.dtype))


def _norm_plain(x, weight, bias):
    x, c = x.float(), x.shape[-1]
    mean = x.sum(-1) / c
    d = x - mean[..., None]
    rstd = 1.0 / torch.sqrt((d * d).sum(-1) / c + EPS_NORM)
    return d * rstd[..., None] * weight.float() + bias.float(), mean, rstd


def _norm_grad_plain(v_y, x, weight, mean, rstd):
    c = x.shape[-1]
    xhat = (x.float() - mean[..., None]) * rstd[..., None]
    g = v_y.float()
    gw = g * weight.float()
    a = gw.sum(-1, keepdim=True) / c
    b = (gw * xhat).sum(-1, keepdim=True) / c
    return ((gw - a - xhat * b) * rstd[..., None]).to(x.dtype), (g * xhat).sum(0), g.sum(0)


def _blocks(t):
    """A flat tensor in rows of BLOCK values, the last one filled up with zeros."""
    n = t.numel()
    return torch.nn.functional.pad(t, (0, -n % BLOCK)).view(-1, BLOCK)


def _pack(t, keep_above_zero):
    """32-bit values -> (e4m3 codes, one scale for every BLOCK of them)."""
    b = _blocks(t)
    top = b.abs().amax(1)
    empty = top < FLUSH
    scale = (top * (1.0 / F8_MAX)).masked_fill(empty, 0.0)
    to = b * (F8_MAX / top).masked_fill(empty, 0.0)[:, None]
    if keep_above_zero:
        to = to.masked_fill((to > 0) & (to < F8_TINY), F8_TINY)
    return to.to(torch.float8_e4m3fn).view(-1)[: t.numel()], scale


def _unpack(codes, scale):
    return (_blocks(codes.float()) * scale[:, None]).view(-1)[: codes.numel()]


def _adamw_moments(g, m, v):
    m = m * ADAM["b1"] + g * (1.0 - ADAM["b1"])
    v = v * ADAM["b2"] + (g * g) * (1.0 - ADAM["b2"])
    return m, v


def _adamw_weights(p, m, v, step):
    c1, c2 = 1.0 - ADAM["b1"] ** step, 1.0 - ADAM["b2"] ** step
    move = m / (torch.sqrt(v) * (1.0 / math.sqrt(c2)) + ADAM["eps"])
    return (p.float() * (1.0 - ADAM["lr"] * ADAM["weight_decay"]) - move * (ADAM["lr"] / c1)).to(p.dtype)


def _adamw32_plain(p, g, m, v, step):
    new_m, new_v = _adamw_moments(g.float(), m, v)
    p.copy_(_adamw_weights(p, new_m, new_v, step))
    m.copy_(new_m)
    v.copy_(new_v)


def _adamw8_plain(p, g, m, v, m_scale, v_scale, step):
    root = _unpack(v, v_scale)  # the second moment is held as its root
    new_m, new_v = _adamw_moments(g.float(), _unpack(m, m_scale), root * root)
    p.copy_(_adamw_weights(p, new_m, new_v, step))
    for to, was in zip((m, m_scale, v, v_scale),
                       (*_pack(new_m, False), *_pack(torch.sqrt(new_v), True))):
        to.copy_(was)


def _rand(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=F32) * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    op, dtype = case["op"], TYPES[case["type"]]
    s = {"case": case}
    if op.startswith("attention"):
        b, d = case["batch"], case["dim"]
        q = _rand(gen, (b, case["q_len"], case["heads"], d), dtype)
        k = _rand(gen, (b, case["kv_len"], case["kv_heads"], d), dtype)
        v = _rand(gen, (b, case["kv_len"], case["kv_heads"], d), dtype)
        lens = None
        if case["ragged"]:
            lens = torch.tensor(_kv_lengths(case), dtype=torch.int32, device=DEV)
        s.update(q=q, k=k, v=v, kv_lens=lens)
        if op == "attention_bwd":
            s["out"], s["lse"] = _attention_plain(case, q, k, v, lens)
            s["v_out"] = _rand(gen, q.shape, dtype)
        return s
    if op.startswith("layer_norm"):
        shape = (case["rows"], case["cols"])
        s["x"] = _rand(gen, shape, dtype) * 1.5 + 0.25
        s["weight"] = 1.0 + _rand(gen, shape[1:], F32, 0.1)
        s["bias"] = _rand(gen, shape[1:], F32, 0.1)
        if op == "layer_norm_bwd":
            _, s["mean"], s["rstd"] = _norm_plain(s["x"], s["weight"], s["bias"])
            s["v_y"] = _rand(gen, shape, dtype)
        return s
    sizes = tensor_sizes(case)
    s["params"] = [_rand(gen, n, dtype, 0.02) for n in sizes]
    # gradients of a training step: each value has a scale of its own, some are zero (a splat that
    # no view saw, a unit that did not fire)
    grads = [_rand(gen, n, F32) * torch.exp(_rand(gen, n, F32, 1.5) - 7.0) for n in sizes]
    grads = [g * (torch.rand(g.shape, generator=gen, device=DEV) < 0.9) for g in grads]
    moments = [_rand(gen, n, F32) * torch.exp(_rand(gen, n, F32, 1.5) - 8.0) for n in sizes]
    squares = [m * m * 4.0 for m in moments]
    s["grads"] = [g.to(dtype) for g in grads]
    s["step"] = ADAM_STEP
    if case["bits"] == 32:
        s["exp_avg"], s["exp_avg_sq"] = moments, squares
    else:
        first = [_pack(m, False) for m in moments]
        second = [_pack(torch.sqrt(v), True) for v in squares]
        s["exp_avg"], s["exp_avg_scale"] = [c for c, _ in first], [x for _, x in first]
        s["exp_avg_sq"], s["exp_avg_sq_scale"] = [c for c, _ in second], [x for _, x in second]
    return s


# ---------------------------------------------------------------- one call

def run(s):
    case, op = s["case"], s["case"]["op"]
    if op == "attention_fwd":
        if own:
            return _network().attention_fwd(s["q"], s["k"], s["v"], causal=case["causal"],
                                            kv_lens=s["kv_lens"])
        return _attention_plain(case, s["q"], s["k"], s["v"], s["kv_lens"])
    if op == "attention_bwd":
        if own:
            return _network().attention_bwd(s["v_out"], s["q"], s["k"], s["v"], s["out"], s["lse"],
                                            causal=case["causal"], kv_lens=s["kv_lens"])
        return _attention_grad_plain(case, s["q"], s["k"], s["v"], s["out"], s["lse"], s["v_out"],
                                     s["kv_lens"])
    if op == "layer_norm_fwd":
        if own:
            return _network().layer_norm_fwd(s["x"], s["weight"], s["bias"], eps=EPS_NORM)
        y, mean, rstd = _norm_plain(s["x"], s["weight"], s["bias"])
        return y.to(s["x"].dtype), mean, rstd
    if op == "layer_norm_bwd":
        if own:
            return _network().layer_norm_bwd(s["v_y"], s["x"], s["weight"], s["mean"], s["rstd"])
        return _norm_grad_plain(s["v_y"], s["x"], s["weight"], s["mean"], s["rstd"])
    if own:
        if "optimizer" not in s:  # a program makes it once and keeps it
            s["optimizer"] = _network().AdamW(
                s["params"], lr=ADAM["lr"], betas=(ADAM["b1"], ADAM["b2"]), eps=ADAM["eps"],
                weight_decay=ADAM["weight_decay"], state_bits=case["bits"],
                state={k: s[k] for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale",
                                         "exp_avg_sq_scale", "step") if k in s})
        s["optimizer"].step(s["grads"])
    else:
        s["step"] += 1
        if case["bits"] == 32:
            [_adamw32_plain(*t, s["step"]) for t in
             zip(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"])]
        else:
            [_adamw8_plain(*t, s["step"]) for t in
             zip(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], s["exp_avg_scale"],
                 s["exp_avg_sq_scale"])]
    return _shown(s)


def _shown(s):
    """The updated tensors; of a network's many, those of its first block and its last layers."""
    keys = ("params", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
    n = len(s["params"])
    at = list(range(n)) if n <= 12 else list(range(8)) + [n - 4, n - 3, n - 2, n - 1]
    return {k: [s[k][i] for i in at] for k in keys if k in s}


def _network():
    import sys
    if "splatx-metal_b200" not in sys.path:
        sys.path.insert(0, "splatx-metal_b200")
    from splatx_cuda import network
    return network


# ---------------------------------------------------------------- what it cannot do without

def work(case):
    op, e = case["op"], BYTES[case["type"]]
    if op.startswith("attention"):
        q = case["batch"] * case["q_len"] * case["heads"]
        kv = sum(_kv_lengths(case)) * case["kv_heads"]
        pairs = _pairs(case) * case["heads"] * case["dim"]
        if op == "attention_fwd":  # two products; q, k, v in, the output and the log-sums out
            return {"bytes": (2 * q + 2 * kv) * case["dim"] * e + 4 * q, "flops": 4.0 * pairs}
        # five products; q, k, v, out, its gradient, log-sums in, three gradients out
        return {"bytes": (4 * q + 4 * kv) * case["dim"] * e + 4 * q, "flops": 10.0 * pairs}
    if op.startswith("layer_norm"):
        n, r, c = case["rows"] * case["cols"], case["rows"], case["cols"]
        if op == "layer_norm_fwd":
            return {"bytes": 2 * n * e + 8 * r + 8 * c, "flops": 8.0 * n}
        return {"bytes": 3 * n * e + 8 * r + 12 * c, "flops": 14.0 * n}
    n = sum(tensor_sizes(case))
    state = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
    return {"bytes": n * (3 * e + state), "flops": 15.0 * n}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    """What ``run`` returns, in 64 bits and head by head, from the operators' definitions."""
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("attention"):
        return _exact_attention(case, s)
    if op == "layer_norm_fwd":
        x, w, b = (s[k].double() for k in ("x", "weight", "bias"))
        mean = x.mean(-1)
        rstd = (x.var(-1, unbiased=False) + EPS_NORM).rsqrt()
        return (x - mean[:, None]) * rstd[:, None] * w + b, mean, rstd
    if op == "layer_norm_bwd":
        x, w, g = (s[k].double() for k in ("x", "weight", "v_y"))
        centred = x - x.mean(-1, keepdim=True)
        inv = (centred.pow(2).mean(-1, keepdim=True) + EPS_NORM).pow(-0.5)
        # y = w c / sqrt(mean(c^2) + eps) + b, by the chain rule through inv and c
        v_c = g * w * inv - centred * inv.pow(3) * (g * w * centred).mean(-1, keepdim=True)
        return v_c - v_c.mean(-1, keepdim=True), (g * centred * inv).sum(0), g.sum(0)
    return _exact_adamw(case, s)


def _exact_attention(case, s):
    group = case["heads"] // case["kv_heads"]
    n, kl = case["q_len"], case["kv_len"]
    seen = torch.ones((n, kl), dtype=torch.bool, device=DEV)
    if case["causal"]:
        seen = torch.tril(seen, diagonal=kl - n)
    lens = _kv_lengths(case)
    shape = (case["batch"], n, case["heads"], case["dim"])
    kv_shape = (case["batch"], kl, case["kv_heads"], case["dim"])
    out = torch.zeros(shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros((case["batch"], case["heads"], n), dtype=torch.float64, device=DEV)
    dk, dv = (torch.zeros(kv_shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for b in range(case["batch"]):
        for h in range(case["heads"]):
            q, k, v = s["q"][b, :, h].double(), s["k"][b, :, h // group].double(), s["v"][b, :, h // group].double()
            logits = torch.einsum("id,jd->ij", q, k) / math.sqrt(case["dim"])
            logits[~(seen & (torch.arange(kl, device=DEV) < lens[b]))] = -math.inf
            weights = torch.softmax(logits, dim=-1)
            if case["op"] == "attention_fwd":
                out[b, :, h] = weights @ v
                lse[b, h] = torch.logsumexp(logits, dim=-1)
                continue
            del logits
            g = s["v_out"][b, :, h].double()
            dv[b, :, h // group] += weights.T @ g
            back = g @ v.T
            back = weights * (back - (weights * back).sum(-1, keepdim=True)) / math.sqrt(case["dim"])
            out[b, :, h] = back @ k
            dk[b, :, h // group] += back.T @ q
    return (out, lse) if case["op"] == "attention_fwd" else (out, dk, dv)


def _exact_adamw(case, s):
    """One step's new weights and moments; an 8-bit moment is what its codes stand for
    (over its scale) before they are rounded."""
    t = s["step"] + 1
    shown = {k: [] for k in ("params", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")}
    eight = case["bits"] == 8

    def real(codes, scale):
        n = codes.numel()
        return codes.double() * scale.double().repeat_interleave(BLOCK)[:n]

    def held(x):
        n = x.numel()
        rows = torch.cat([x, x.new_zeros(-n % BLOCK)]).view(-1, BLOCK)
        top = rows.abs().max(1).values
        ratio = rows / torch.where(top >= FLUSH, top / F8_MAX, math.inf)[:, None]
        return ratio.flatten()[:n], torch.where(top >= FLUSH, top / F8_MAX, 0.0)

    for i in range(len(s["params"])):
        g = s["grads"][i].double()
        m = real(s["exp_avg"][i], s["exp_avg_scale"][i]) if eight else s["exp_avg"][i].double()
        v = real(s["exp_avg_sq"][i], s["exp_avg_sq_scale"][i]) ** 2 if eight else s["exp_avg_sq"][i].double()
        m = ADAM["b1"] * m + (1 - ADAM["b1"]) * g
        v = ADAM["b2"] * v + (1 - ADAM["b2"]) * g ** 2
        mhat, vhat = m / (1 - ADAM["b1"] ** t), v / (1 - ADAM["b2"] ** t)
        p = s["params"][i].double()
        p = p - ADAM["lr"] * (mhat / (vhat ** 0.5 + ADAM["eps"]) + ADAM["weight_decay"] * p)
        shown["params"].append(p)
        (a, sa), (r, sr) = (held(m), held(v ** 0.5)) if eight else ((m, None), (v, None))
        shown["exp_avg"].append(a)
        shown["exp_avg_sq"].append(r)
        if eight:
            shown["exp_avg_scale"].append(sa)
            shown["exp_avg_sq_scale"].append(sr)
    return _shown({k: v for k, v in shown.items() if v})
