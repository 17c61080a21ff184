"""The norm and rotation of queries and keys, and its gradients, against the definition in 64 bits.

Bounds. A row's sum of squares carries at most 64 roundings a term (16 values a thread, then a tree), its
root and quotient two: rstd is off by E32 / 2 + 2^-23. Products with rstd, weight, cosine and sine and their
sum add one rounding each, and the cosines and sines are off by 2^-22 (2^-25 of the angle, then the library's
function): 2^-21 of |u1| + |u2| in all. Then one rounding to the element type.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}
E32 = 64 * 2.0 ** -24
ANGLE = 2.0 ** -21
name = lambda s: "x".join(map(str, s)) if isinstance(s, (tuple, list)) else str(s)  # noqa: E731


def _pairs(axes, pairs):
    """(first values, second values, axis, pair of the axis)."""
    first, second, axis, order, at, half = [], [], [], [], 0, sum(axes) // 2
    for a, d in enumerate(axes):
        for j in range(d // 2):
            i = len(first)
            one, two = {"axis": (at + j, at + j + d // 2), "whole": (i, i + half), "neighbours": (2 * i, 2 * i + 1)}[pairs]
            first.append(one), second.append(two), axis.append(a), order.append(j)
        at += d
    return first, second, axis, order


def _angles(positions, axes, pairs, base, freqs):
    import torch
    first, second, axis, order = _pairs(axes, pairs)
    f = [base ** (-2.0 * j / axes[a]) for a, j in zip(axis, order)] if freqs is None else list(freqs)
    f = torch.tensor(f, dtype=torch.float64, device=positions.device)
    return positions.double()[..., axis] * f, first, second


def _rotate(x, angles, back=False):
    a, first, second = angles
    a = (-a if back else a)[..., None, :]
    out = x.clone()
    out[..., first] = x[..., first] * torch_cos(a) - x[..., second] * torch_sin(a)
    out[..., second] = x[..., first] * torch_sin(a) + x[..., second] * torch_cos(a)
    return out


def torch_cos(a):
    import torch
    return torch.cos(a)


def torch_sin(a):
    import torch
    return torch.sin(a)


def _both(x, angles):
    """|u1| + |u2| of the pair that each value is in."""
    _, first, second = angles
    x = x.abs()
    out = x.clone()
    out[..., first] = out[..., second] = x[..., first] + x[..., second]
    return out


def _inputs(seed, b, t, h, hk, d, axes, dtype, where="scene", wtype="float32"):
    import torch
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    T = getattr(torch, dtype)
    qkv = (r(b, t, h + 2 * hk, d) * 1.5 + 0.2).to(T).cuda()
    if where == "scene":
        pos = (torch.rand(b, t, axes, generator=g) * 256 - 128).cuda()
    else:
        pos = torch.randint(0, {"grid": 300, "far": 1 << 30}[where], (b, t, axes), generator=g).cuda()
    w = [None, None] if wtype is None else [(1 + 0.2 * r(d)).to(getattr(torch, wtype)).cuda() for _ in range(2)]
    if not hk:
        w[1] = None
    grads = [r(b, t, n, d).to(T).cuda() for n in (h, hk)]
    return qkv[:, :, :h], (qkv[:, :, h:h + hk] if hk else None), pos, w, grads


def _near(label, got, want, bound):
    import torch
    assert got.shape == want.shape, label
    off = (got.double() - want).abs() - bound
    assert off.numel() == 0 or (not torch.isnan(off).any() and float(off.max()) <= 0), (label, float(off.max()))


def _check(q, k, pos, weights, grads, axes, pairs="axis", base=100.0, freqs=None, norm=True, eps=1e-6):
    import torch
    from splatx_cuda import network
    how = {"axes": axes, "pairs": pairs, "base": base, "freqs": freqs, "norm": norm, "q_weight": weights[0],
           "k_weight": weights[1], "eps": eps}
    outs = network.qk_norm_rotary_fwd(q, k, pos, **how)
    back = network.qk_norm_rotary_bwd(grads[0], None if k is None else grads[1], q, k, pos, **how)
    dtype = str(q.dtype).split(".")[1]
    u, tiny = ROUND[dtype], TINY[dtype]
    angles = _angles(pos.expand(q.shape[0], -1, -1) if pos.dim() == 2 else pos, axes, pairs, base, freqs)
    for i, (label, x, w, g) in enumerate((("q", q, weights[0], grads[0]), ("k", k, weights[1], grads[1]))):
        if x is None:
            assert outs[i] is None and back[i] is None and back[2 + i] is None
            continue
        X, G = x.double(), g.double()
        W = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
        r = (X.pow(2).mean(-1, keepdim=True) + eps) ** -0.5 if norm else torch.ones_like(X[..., :1])
        e_r = E32 / 2 + 2.0 ** -23 if norm else 0.0
        U = X * r * W
        want = _rotate(U, angles)
        _near(label, outs[i], want, (e_r + ANGLE) * _both(U, angles) + u * want.abs() + tiny)
        B = _rotate(G, angles, back=True)
        e_b = ANGLE * _both(G, angles)
        if not norm:
            _near("v_" + label, back[i], B, e_b + u * B.abs() + tiny)
            assert back[2 + i] is None
            continue
        H = X * r
        D = B * W
        e_d = e_b * W.abs() + 2.0 ** -24 * D.abs()
        e_h = (e_r + 2.0 ** -24) * H.abs()
        c = (D * H).mean(-1, keepdim=True)
        e_c = (e_d * H.abs() + D.abs() * e_h + E32 * (D * H).abs()).mean(-1, keepdim=True)
        core = D - H * c
        e_core = e_d + e_h * c.abs() + H.abs() * e_c + 2.0 ** -22 * (D.abs() + (H * c).abs())
        VX = core * r
        _near("v_" + label, back[i], VX, (e_core + (e_r + 2.0 ** -24) * core.abs()) * r * (1 + 1e-3) + u * VX.abs() + tiny)
        if w is None:
            assert back[2 + i] is None
            continue
        uw = ROUND[str(w.dtype).split(".")[1]]
        rows = X[..., 0].numel()
        terms = min(rows, rows // 256 + 700) * 2.0 ** -24  # of a thread, of a warp's groups, of CTAs
        VW = (B * H).sum((0, 1, 2))
        bound = (e_b * H.abs() + B.abs() * e_h + terms * (B * H).abs()).sum((0, 1, 2))
        _near(f"v_{label}_weight", back[2 + i], VW, bound + (uw + 2.0 ** -23) * VW.abs())
        assert back[2 + i].dtype == w.dtype
    return outs, back


# head sizes with every number of values a thread takes, odd ones, values that are not rotated
LAYOUTS = [(64, (64,)), (64, (32, 32)), (128, (32, 48, 48)), (80, (16, 32, 32)), (64, (20, 20, 20)), (64, (24, 24, 16)),
           (32, (10, 12, 10)), (96, (32, 32)), (256, (128, 128)), (255, (254,)), (256, (2, 2, 2, 250)), (7, (2, 4)),
           (1, (0,)), (2, (2,)), (48, (0, 16, 0, 16)), (128, (0,)), (72, (72,))]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("pairs", ["axis", "whole", "neighbours"])
@pytest.mark.parametrize("layout", LAYOUTS, ids=name)
def test_layouts(layout, pairs, dtype):
    d, axes = layout
    _check(*_inputs(d, 2, 37, 6, 2, d, len(axes), dtype), axes, pairs)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (1, 1, 32, 8), (3, 1, 5, 0), (1, 2, 1, 7), (2, 96, 8, 8), (1, 5001, 12, 4),
                                  (7, 1000, 16, 16), (1, 20000, 3, 1)], ids=name)
def test_sizes(size, dtype):
    _check(*_inputs(sum(size), *size, 64, 2, dtype, where="grid"), (32, 32))
    _check(*_inputs(sum(size), *size, 128, 3, dtype), (32, 48, 48), pairs="whole")


@pytest.mark.parametrize("wtype", ["float16", "bfloat16", None])
def test_weights(wtype):
    q, k, pos, w, g = _inputs(3, 2, 50, 4, 4, 64, 2, "bfloat16", wtype=wtype)
    _check(q, k, pos, w, g, (32, 32))
    _check(q, k, pos, [w[0], None], g, (32, 32))
    _check(q, k, pos, [None, w[1]], g, (32, 32))


@pytest.mark.parametrize("pairs", ["axis", "whole", "neighbours"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rotation_alone(dtype, pairs):
    q, k, pos, _, g = _inputs(4, 2, 60, 4, 2, 64, 3, dtype)
    _check(q, k, pos, [None, None], g, (16, 24, 24), pairs, norm=False)
    _check(q, k, pos, [None, None], g, (10, 10, 10), pairs, norm=False)


def test_positions():
    """Far whole numbers keep their angle; shared by the batch, strided, of every type."""
    import torch
    from splatx_cuda import network
    q, k, pos, w, g = _inputs(5, 3, 70, 4, 4, 64, 2, "float32", where="far")
    want, _ = _check(q, k, pos, w, g, (32, 32), base=10000.0)
    got, _ = _check(q, k, pos.int(), w, g, (32, 32), base=10000.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    near = (pos % 4096)
    want, _ = _check(q, k, near, w, g, (32, 32), base=10000.0)
    for p in (near.float(), near.transpose(0, 2).contiguous().transpose(0, 2), near.int(),
              torch.stack([near, near], -1)[..., 0]):
        got, _ = _check(q, k, p, w, g, (32, 32), base=10000.0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    shared, _ = _check(q, k, near[0], w, g, (32, 32))
    each, _ = _check(q, k, near[:1].expand(3, -1, -1), w, g, (32, 32))
    assert all(torch.equal(a, b) for a, b in zip(shared, each))
    freqs = torch.rand(32, generator=torch.Generator().manual_seed(1)).tolist()
    _check(q, k, near, w, g, (32, 32), freqs=freqs)
    # zero is no rotation at all
    still = network.qk_norm_rotary_fwd(q, None, torch.zeros_like(pos), axes=(32, 32), norm=False)[0]
    assert torch.equal(still, q.contiguous())


def test_what_is_not_finite():
    """A NaN or infinity stays in its head (a position's in its token's rotated values)."""
    import torch
    from splatx_cuda import network
    q, k, pos, w, g = _inputs(6, 2, 33, 4, 4, 64, 2, "bfloat16")
    how = {"axes": (32, 16), "q_weight": w[0], "k_weight": w[1]}
    want, _ = network.qk_norm_rotary_fwd(q, k, pos, **how)
    q = q.contiguous()
    q[0, 3, 1, 7] = math.nan
    q[1, 5, 2, 60] = math.inf
    got, _ = network.qk_norm_rotary_fwd(q, k, pos, **how)
    rows = torch.ones(2, 33, 4, dtype=torch.bool, device="cuda")
    rows[0, 3, 1] = rows[1, 5, 2] = False
    assert torch.equal(got[rows], want[rows]) and bool(got[0, 3, 1].isnan().all()) and bool(got[1, 5, 2, 60].isnan())
    q = _inputs(6, 2, 33, 4, 4, 64, 2, "bfloat16")[0]
    for value in (math.nan, math.inf):
        p = pos.clone()
        p[1, 4, 1] = value
        got, _ = network.qk_norm_rotary_fwd(q, k, p, **how)
        seen = torch.ones_like(want, dtype=torch.bool)
        seen[1, 4, :, 32:48] = False
        assert torch.equal(got[seen], want[seen]) and bool(got[1, 4, :, 32:48].isnan().all())
    zero = torch.zeros(1, 2, 3, 64, device="cuda")
    out, _ = network.qk_norm_rotary_fwd(zero, None, torch.ones(2, 1, device="cuda"), axes=(64,))
    assert not out.any()


def test_strides():
    import torch
    q, k, pos, w, g = _inputs(7, 2, 40, 4, 4, 64, 2, "bfloat16")
    want = _check(q, k, pos, w, g, (32, 32))

    def same(q, k, g):
        got = _check(q, k, pos, w, g, (32, 32))
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))

    for first, pitch in ((0, 64), (8, 80), (4, 68), (2, 66), (1, 67)):
        wide = torch.full((2, 40, 4, pitch), math.nan, dtype=q.dtype, device="cuda")
        wide[..., first:first + 64] = q
        if pitch % 16 == 0:
            same(wide[..., first:first + 64], k, g)
        else:  # narrower accesses: a row's squares are summed in another order
            _check(wide[..., first:first + 64], k, pos, w, g, (32, 32))
    same(q.transpose(1, 2).contiguous().transpose(1, 2), k, [g[0].transpose(1, 2).contiguous().transpose(1, 2), g[1]])
    same(q.transpose(1, 3).contiguous().transpose(1, 3), k, g)  # copied
    ones = [torch.ones(1, 1, 1, 1, dtype=q.dtype, device="cuda").expand(2, 40, 4, 64) for _ in range(2)]
    _check(q, k, pos, w, ones, (32, 32))


def test_in_place_at_the_c_entry():
    import ctypes as C
    import torch
    from splatx_cuda import _native as n, network
    for dtype, code in (("bfloat16", 2), ("float32", 0)):
        q, k, pos, w, _ = _inputs(8, 2, 300, 8, 2, 64, 2, dtype)
        want = network.qk_norm_rotary_fwd(q, k, pos, axes=(32, 32), q_weight=w[0], k_weight=w[1])
        freqs = (C.c_double * 32)(*[10000.0 ** (-2 * j / 32) for j in range(16)] * 2)
        view = lambda t: n.SxAttentionView(t.data_ptr(), *t.stride()[:3])  # noqa: E731
        ins = n.SxRotaryInputs(view(q), view(k), pos.data_ptr(), *pos.stride(), C.addressof(freqs), w[0].data_ptr(), w[1].data_ptr(),
                               2, 300, 8, 2, 64, 2, (C.c_int32 * 4)(32, 32), 0, code, 0, 0, 1, 1e-6)
        n.check(n.lib().sxcuda_qk_norm_rotary_fwd(C.byref(ins), C.byref(view(q)), C.byref(view(k)), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_no_tokens():
    import torch
    from splatx_cuda import network
    for b, t in ((0, 5), (2, 0)):
        q, k, pos, w, g = _inputs(9, b, t, 4, 4, 64, 2, "bfloat16")
        how = {"axes": (32, 32), "q_weight": w[0], "k_weight": w[1]}
        assert network.qk_norm_rotary_fwd(q, k, pos, **how)[0].shape == (b, t, 4, 64)
        v = network.qk_norm_rotary_bwd(*g, q, k, pos, **how)
        assert v[1].shape == k.shape and not v[2].any() and not v[3].any()


@pytest.mark.parametrize("norm", [True, False])
def test_autograd_and_differences(norm):
    import torch
    from splatx_cuda import network
    q, k, pos, w, g = _inputs(10, 2, 9, 3, 2, 20, 2, "float32")
    ins = [q.contiguous().requires_grad_(), k.contiguous().requires_grad_()]
    ins += [t.requires_grad_() for t in w] if norm else []
    at = lambda t: {"q_weight": t[2], "k_weight": t[3]} if norm else {"norm": False}  # noqa: E731

    def f(*t):
        a, b = network.qk_norm_rotary(t[0], t[1], pos, axes=(8, 12), base=100.0, **at(t))
        return (a.double() * g[0]).sum() + (b.double() * g[1]).sum()

    grads = torch.autograd.grad(f(*ins), ins)
    gen = torch.Generator(device="cuda").manual_seed(2)
    for i, t in enumerate(ins):
        d = torch.randn(t.shape, generator=gen, device="cuda")
        d /= d.norm()
        h = 1e-2
        up, down = ([(u + s * h * d if j == i else u).detach() for j, u in enumerate(ins)] for s in (1, -1))
        slope, want = float(f(*up) - f(*down)) / (2 * h), float((grads[i] * d).sum())
        assert abs(slope - want) <= 2e-3 * float(grads[i].norm()) + 1e-3, (i, slope, want)
    # the rotation keeps lengths: its gradient's gradient is refused, its gradient is the rotation back
    (v,) = torch.autograd.grad(network.qk_norm_rotary(ins[0], None, pos, axes=(8, 12), norm=False)[0].sum(), ins[0], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(v.sum(), ins[0])


def test_streams_graphs_and_repeats():
    import torch
    from splatx_cuda import network
    made = [_inputs(60 + i, 2, 700, 8, 4, 64, 3, "bfloat16") for i in range(2)]

    def both(q, k, pos, w, g):
        how = {"axes": (16, 24, 24), "q_weight": w[0], "k_weight": w[1]}
        return (*network.qk_norm_rotary_fwd(q, k, pos, **how), *network.qk_norm_rotary_bwd(*g, q, k, pos, **how))

    want = [both(*m) for m in made]
    assert all(torch.equal(a, b) for a, b in zip(both(*made[0]), want[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(*made[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs = [], []
    for m in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both(*m))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, v in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, v))


def test_many_batches_of_one_token():
    """More warps than a batch entry has tokens, by far; and a token's many heads cut into units."""
    q, k, pos, w, g = _inputs(12, 9000, 1, 4, 2, 64, 2, "bfloat16")
    _check(q, k, pos, w, g, (32, 32))
    q, k, pos, w, g = _inputs(13, 5000, 2, 1, 1, 16, 1, "float32")
    _check(q, k, pos, w, g, (16,))
    q, k, pos, w, g = _inputs(14, 2, 3000, 70, 50, 32, 2, "bfloat16")
    _check(q, k, pos, w, g, (16, 16))
    q, k, pos, w, g = _inputs(15, 3, 1000, 40, 33, 128, 3, "float32")
    _check(q, k, pos, w, g, (32, 48, 48), pairs="neighbours")


def test_beyond_32_bits():
    """Queries of more than 2^31 values: the last tokens are what they are by themselves."""
    import torch
    from splatx_cuda import network
    n, h, d = 140_001, 128, 128
    q = torch.empty(1, n, h, d, dtype=torch.bfloat16, device="cuda").normal_()
    pos = torch.rand(1, n, 3, device="cuda") * 256
    w = torch.rand(d, device="cuda") + 0.5
    how = {"axes": (32, 48, 48), "q_weight": w}
    out, _ = network.qk_norm_rotary_fwd(q, None, pos, **how)
    for part in (slice(0, 50), slice(n - 50, n)):
        assert torch.equal(out[:, part], network.qk_norm_rotary_fwd(q[:, part], None, pos[:, part], **how)[0])
    v = network.qk_norm_rotary_bwd(out, None, q, None, pos, **how)
    part = slice(n - 50, n)
    assert torch.equal(v[0][:, part], network.qk_norm_rotary_bwd(out[:, part], None, q[:, part], None, pos[:, part], **how)[0])
    assert bool(torch.isfinite(v[2]).all())


def test_refusals():
    import torch
    from splatx_cuda import network
    q, k, pos, w, g = _inputs(11, 2, 8, 4, 2, 64, 2, "bfloat16")
    fwd, bwd = network.qk_norm_rotary_fwd, network.qk_norm_rotary_bwd
    for f in (lambda: fwd(q, k.cpu(), pos, axes=(32, 32)), lambda: fwd(q, k, pos.cpu(), axes=(32, 32)),
              lambda: fwd(q, k, pos, axes=(32, 32), q_weight=w[0].cpu()), lambda: fwd(q.cpu(), k.cpu(), pos.cpu(), axes=(32, 32)),
              lambda: fwd(q, k, pos.requires_grad_(), axes=(32, 32)),
              lambda: bwd(g[0], None, q, k, pos.detach(), axes=(32, 32)), lambda: bwd(*g, q, None, pos.detach(), axes=(32, 32)),
              lambda: bwd(g[1], g[0], q, k, pos.detach(), axes=(32, 32)), lambda: bwd(g[0].float(), g[1], q, k, pos.detach(), axes=(32, 32)),
              lambda: bwd(g[0].cpu(), g[1], q, k, pos.detach(), axes=(32, 32))):
        with pytest.raises(ValueError):
            f()
