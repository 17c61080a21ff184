"""The operators together, as a transformer's block uses them: layer norm, a projection to queries, keys and
values, their norm and rotation, attention, a projection back with the residual, layer norm, an MLP with gelu
and the residual; forward and backward against the same in 64 bits.

Bounds. About twenty operators lie on the way of a gradient, each off by at most 64 2^-24 of its result's size
(float32), or by a rounding of half a step of its type; norms keep sizes. So the whole is off by less than
twenty times that, in the Euclidean norm of each result.
"""
import math
import pathlib
import sys

import pytest

pytestmark = pytest.mark.gpu

BOUND = {"float32": 20 * 64 * 2.0 ** -24, "float16": 20 * 2.0 ** -11, "bfloat16": 20 * 2.0 ** -8}
AXES, BASE = (16, 24, 24), 100.0


def _weights(width, heads, seed=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    w = {"qkv": r(3 * width, width) * width ** -0.5, "proj": r(width, width) * width ** -0.5,
         "up": r(4 * width, width) * width ** -0.5, "down": r(width, 4 * width) * (4 * width) ** -0.5}
    b = {k + "_b": 0.1 * r(v.shape[0]) for k, v in w.items()}
    n = {f"norm{i}_{k}": (1 if k == "w" else 0) + 0.1 * r(width) for i in range(2) for k in "wb"}
    qk = {k: 1 + 0.1 * r(width // heads) for k in ("q_w", "k_w")}
    return w, {**b, **n, **qk}


def _block(x, places, w, p, heads, n_tokens):
    from splatx_cuda import network
    h = network.layer_norm(x, p["norm0_w"], p["norm0_b"])
    qkv = network.linear(h, w["qkv"], p["qkv_b"]).unflatten(-1, (3, heads, -1))
    q, k, v = qkv.unbind(2)
    q, k = network.qk_norm_rotary(q, k, places, axes=AXES, base=BASE, q_weight=p["q_w"], k_weight=p["k_w"])
    o = network.attention(q, k, v, q_lens=n_tokens, kv_lens=n_tokens)
    x = network.linear(o.flatten(2), w["proj"], p["proj_b"], residual=x)
    h = network.layer_norm(x, p["norm1_w"], p["norm1_b"])
    return network.linear(network.linear(h, w["up"], p["up_b"], activation="gelu"), w["down"], p["down_b"], residual=x)


def _norm64(x, w, b, eps=1e-5):
    m = x.mean(-1, keepdim=True)
    return (x - m) * ((x - m).pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w + b


def _turn64(x, w, places):
    import torch
    u = x * (x.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    out, at = u.clone(), 0
    for a, d in enumerate(AXES):
        angle = places[..., a, None].double() * BASE ** (-2.0 / d * torch.arange(d // 2, device=x.device).double())
        c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
        one, two = u[..., at:at + d // 2], u[..., at + d // 2:at + d]
        out[..., at:at + d // 2] = one * c - two * s
        out[..., at + d // 2:at + d] = one * s + two * c
        at += d
    return out


def _block64(x, places, w, p, heads, n_tokens):
    import torch
    h = _norm64(x, p["norm0_w"], p["norm0_b"])
    q, k, v = (h @ w["qkv"].T + p["qkv_b"]).unflatten(-1, (3, heads, -1)).unbind(2)
    q, k = _turn64(q, p["q_w"], places), _turn64(k, p["k_w"], places)
    s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(q.shape[-1])
    j = torch.arange(x.shape[1], device=x.device)
    s = s.masked_fill(~(j < n_tokens[:, None])[:, None, None], -math.inf)
    o = torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v)
    o = o * (j < n_tokens[:, None])[:, :, None, None]  # a query behind the last token sees no key
    x = x + o.flatten(2) @ w["proj"].T + p["proj_b"]
    h = _norm64(x, p["norm1_w"], p["norm1_b"])
    z = h @ w["up"].T + p["up_b"]
    return x + (z * 0.5 * torch.special.erfc(-z / math.sqrt(2))) @ w["down"].T + p["down_b"]


def _case(dtype, tokens, batch=2, width=128, heads=2):
    import torch
    T = getattr(torch, dtype)
    w, p = _weights(width, heads)
    w = {k: v.to(T).cuda() for k, v in w.items()}
    p = {k: v.cuda() for k, v in p.items()}
    g = torch.Generator().manual_seed(tokens)
    x, v_y = (torch.randn(batch, tokens, width, generator=g).to(T).cuda() for _ in range(2))
    places = (torch.rand(batch, tokens, 3, generator=g) * 256 - 128).cuda()
    n = torch.tensor([tokens] + [max(1, tokens - 5)] * (batch - 1), dtype=torch.int32, device="cuda")
    v_y[1:, n[1]:] = 0
    return x, places, w, p, heads, n, v_y


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_block(tokens, dtype):
    import torch
    from splatx_cuda import network
    x, places, w, p, heads, n, v_y = _case(dtype, tokens)
    leaves = [x, *w.values(), *p.values()]
    for t in leaves:
        t.requires_grad_()
    y = _block(x, places, w, p, heads, n)
    grads = torch.autograd.grad(y, leaves, v_y)
    d = [t.detach().double().requires_grad_() for t in leaves]
    want = _block64(d[0], places, dict(zip(w, d[1:5])), dict(zip(p, d[5:])), heads, n)
    want_grads = torch.autograd.grad(want, d, v_y.double())
    live = torch.arange(tokens, device="cuda") < n[:, None]
    for name, a, b in (("y", y * live[..., None], want * live[..., None]), *zip(["x", *w, *p], grads, want_grads)):
        off = float((a.double() - b).norm())
        # a gradient that is nothing but cancellation (of the keys' bias: softmax does not see it) is held to the others' size
        size = max(float(b.norm()), 0.05 * float(v_y.double().norm()))
        assert off <= BOUND[dtype] * size, (name, off / size, BOUND[dtype])
    assert network.attention_status() == 0 and network.linear_status() == 0


def test_block_in_a_graph():
    """Forward and backward captured: every replay gives what the eager call gave, on new values too."""
    import torch
    x, places, w, p, heads, n, v_y = _case("bfloat16", 200)
    leaves = [t.requires_grad_() for t in (x, *w.values(), *p.values())]

    def step():
        y = _block(x, places, w, p, heads, n)
        return (y, *torch.autograd.grad(y, leaves, v_y))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g))
            places.copy_(torch.rand(places.shape, generator=g) * 200)
        graph.replay()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def _example():
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "splatx-metal_b200" / "examples"))
    import color_network
    return color_network


def test_spatial_color_network_gradients():
    """The example's network with places: output and gradients against itself in 64 bits."""
    import torch
    torch.manual_seed(3)
    net = _example().ColorNetwork(11, spatial=True).cuda()
    with torch.no_grad():
        for t in net.qk.values():
            t.add_(0.1 * torch.randn_like(t))
    assert net.axes == (24, 20, 20)
    features, v_y = torch.randn(700, 11, device="cuda"), torch.randn(700, 3, device="cuda").bfloat16().float()
    places = torch.rand(700, 3, device="cuda") * 256 - 128
    out = net(features, places)
    params = dict(net.named_parameters())
    grads = torch.autograd.grad(out, list(params.values()), v_y)
    # weights are rounded to bfloat16 before their products, here as there
    d = {k: (v.detach().bfloat16().double() if k.startswith("w.") else v.detach().double()).requires_grad_() for k, v in params.items()}
    x = features.bfloat16().double()[None] @ d["w.embed"].T
    for i in range(net.layers):
        h = _norm64(x, d[f"scale.attn{i}"], d[f"shift.attn{i}"])
        q, k, v = (h @ d[f"w.qkv{i}"].T).unflatten(-1, (3, net.heads, -1)).unbind(2)
        turned = []
        for t, name in ((q, "q"), (k, "k")):
            u = t * (t.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * d[f"qk.{name}{i}"]
            parts, at = [], 0
            for a, n in enumerate(net.axes):
                angle = places[None, :, a, None].double() * 100.0 ** (-2.0 / n * torch.arange(n // 2, device="cuda").double())
                c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
                one, two = u[..., at:at + n // 2], u[..., at + n // 2:at + n]
                parts += [one * c - two * s, one * s + two * c]
                at += n
            turned.append(torch.cat(parts, -1))
        s = torch.einsum("bihd,bjhd->bhij", *turned) / 8.0
        x = x + torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v).flatten(2) @ d[f"w.proj{i}"].T
        z = _norm64(x, d[f"scale.mlp{i}"], d[f"shift.mlp{i}"]) @ d[f"w.up{i}"].T
        x = x + (z * 0.5 * torch.special.erfc(-z / math.sqrt(2))) @ d[f"w.down{i}"].T
    want = (_norm64(x, d["scale.last"], d["shift.last"]) @ d["w.head"].T)[0]
    want_grads = torch.autograd.grad(want, list(d.values()), v_y.double())
    bound = 2 * BOUND["bfloat16"]  # two blocks
    assert float((out - want).norm()) <= bound * float(want.norm())
    for name, a, b in zip(params, grads, want_grads):
        assert a is not None and bool(torch.isfinite(a).all())
        assert float((a - b).norm()) <= bound * max(float(b.norm()), 0.05 * float(v_y.norm())), name


def test_spatial_color_network_trains():
    import numpy as np
    from splatx_cuda import network
    losses = _example().train(splats=1500, steps=4, state_bits=8, spatial=True)
    assert len(losses) == 4 and np.all(np.isfinite(losses)) and losses[1] != losses[0]
    assert network.attention_status() == 0 and network.linear_status() == 0
