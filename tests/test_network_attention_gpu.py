"""Attention forward and backward against the definition in 64 bits, element by element.

Bounds follow from the rounding of each step. With u the unit roundoff of the element type, the
kernels round p and ds to it before the second product (not in float32) and the results once, and
everything else to 32 bits:
  p:    relative error E = u + 2^-20 (exponential) + the error of the score, (dim + 2) 2^-24 scale |q| |k|
  out:  E' sum p|v| + u |out|, where E' holds E twice (the normalising sum has it too)
  v_v:  E sum p|g| + u |v_v|
  ds:   (E + u) |ds| + p (u + 2^-20) |g||out| (out came in rounded) + p (dim 2^-24) |g||v|
  v_q:  scale sum err(ds) |k| + u |v_q|, v_k likewise with |q|.
Sums over n terms in 32 bits add n 2^-24 of the sum of magnitudes.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROUND = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _inputs(seed, b, lq, lk, h, hk, d, dtype, spread=1.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: (torch.randn(*s, generator=g) * spread).to(getattr(torch, dtype)).cuda()  # noqa: E731
    return make(b, lq, h, d), make(b, lk, hk, d), make(b, lk, hk, d), make(b, lq, h, d)


def _seen(b, lq, lk, causal, q_lens, kv_lens):
    import torch
    ql = torch.full((b,), lq) if q_lens is None else q_lens.cpu().long()
    kl = torch.full((b,), lk) if kv_lens is None else kv_lens.cpu().long()
    i, j = torch.arange(lq)[None, :, None], torch.arange(lk)[None, None, :]
    ql, kl = ql[:, None, None], kl[:, None, None]
    seen = (i < ql) & (j < kl)
    return (seen & (j <= i + kl - ql) if causal else seen)[:, None].cuda()


def _definition(q, k, v, g, out, seen, scale, u):
    """Results and error bounds in 64 bits: {name: (value, bound)}."""
    import torch
    group = q.shape[2] // k.shape[2]
    f = lambda t: t.double().transpose(1, 2)  # noqa: E731
    rep = lambda t: f(t).repeat_interleave(group, dim=1)  # noqa: E731
    # rows that no length reaches may hold anything: they are taken as zeros here
    qs, ks = seen.any(3), seen.any(2)
    Q = torch.where(qs[..., None], f(q), 0.0)
    G = torch.where(qs[..., None], f(g), 0.0)
    K, V = (torch.where(ks[..., None], rep(t), 0.0) for t in (k, v))
    b, h, lq, d = Q.shape
    lk = K.shape[2]
    s = (Q @ K.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None]), 0.0)
    A = lambda t: t.abs()  # noqa: E731
    e_s = (d + 2) * 2.0 ** -24 * abs(scale) * (A(Q) @ A(K).transpose(2, 3)) + 2.0 ** -20
    e_p = u + e_s
    n32 = 2.0 ** -24
    res = {}
    o = p @ V
    e_row = (p * e_p).sum(-1, keepdim=True)  # of the normalising sum
    res["out"] = (o, (p * (e_p + e_row + lk * n32)) @ A(V) + (u + 2 * n32) * A(o))
    res["lse"] = (lse, (p * e_s).sum(-1) + 2.0 ** -22 * (1 + A(lse)) + lk * n32)
    # the gradients, whose lse and out are the kernel's own
    e_l = e_row * 0 + ((p * e_s).sum(-1) + 2.0 ** -22 * (1 + A(torch.where(torch.isinf(lse), 0.0, lse))))[..., None]
    e_p = e_p + e_l
    vv = p.transpose(2, 3) @ G
    e_vv = (p * (e_p + lq * n32)).transpose(2, 3) @ A(G) + (u + 2 * n32) * A(vv)
    dp = G @ V.transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_o = res["out"][1]  # what came in as out
    e_delta = (A(G) * e_o).sum(-1, keepdim=True) + (d + 2) * n32 * (A(G) * A(o)).sum(-1, keepdim=True)
    e_ds = (e_p + u) * A(ds) + p * (e_delta + (d + 2) * n32 * (A(G) @ A(V).transpose(2, 3))) * (1 + e_p)
    vq = ds @ K * scale
    e_vq = abs(scale) * ((e_ds + lk * n32 * A(ds)) @ A(K)) + (u + 4 * n32) * A(vq)
    vk = ds.transpose(2, 3) @ Q * scale
    e_vk = abs(scale) * ((e_ds + lq * n32 * A(ds)).transpose(2, 3) @ A(Q)) + (u + 4 * n32) * A(vk)
    shared = lambda t: t.view(b, h // group, group, lk, d).sum(2)  # noqa: E731
    res["v_q"] = (vq, e_vq)
    res["v_k"] = (shared(vk), shared(e_vk) + u * A(shared(vk)))
    res["v_v"] = (shared(vv), shared(e_vv) + u * A(shared(vv)))
    return res


def _check(name, got, want, bound):
    import torch
    got = got.double()
    assert got.shape == want.shape, name
    assert bool((torch.isinf(got) == torch.isinf(want)).all()), name
    fine = torch.isfinite(want)
    assert bool(torch.isfinite(got[fine]).all()), name
    # 2^-24 of magnitude 1: subnormal results of float16
    excess = (got - want).abs()[fine] - bound[fine] - 2.0 ** -24
    assert excess.numel() == 0 or float(excess.max()) <= 0, (name, float(excess.max()))


def _run(q, k, v, g, causal=False, q_lens=None, kv_lens=None, scale=None):
    from splatx_cuda import network
    how = dict(causal=causal, q_lens=q_lens, kv_lens=kv_lens, scale=scale)
    out, lse = network.attention_fwd(q, k, v, **how)
    grads = network.attention_bwd(g, q, k, v, out, lse, **how)
    seen = _seen(q.shape[0], q.shape[1], k.shape[1], causal, q_lens, kv_lens)
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    want = _definition(q, k, v, g, out, seen, scale, ROUND[str(q.dtype).split(".")[1]])
    heads = lambda t: t.transpose(1, 2)  # noqa: E731
    _check("out", heads(out), *want["out"])
    _check("lse", lse, *want["lse"])
    for name, t in zip(("v_q", "v_k", "v_v"), grads):
        _check(name, heads(t), *want[name])
    assert network.attention_status() == 0
    return out, lse, grads


# lengths about the kernels' tiles (64, 128, 256), one token, odd ones; shared heads; dims that fill
# a tile, are padded to it, and (36, 33) cannot be copied in 16-byte pieces
SHAPES = [(1, 1, 1, 1, 1, 64), (2, 1, 300, 4, 2, 128), (1, 127, 129, 2, 2, 64), (2, 128, 128, 2, 1, 128),
          (1, 256, 256, 3, 3, 64), (1, 257, 385, 4, 1, 128), (1, 640, 70, 2, 2, 80), (3, 65, 64, 2, 2, 32),
          (1, 500, 1000, 2, 1, 8), (1, 130, 200, 2, 2, 36), (1, 33, 20, 1, 1, 33), (1, 20, 515, 6, 2, 128),
          (2, 384, 511, 2, 2, 96)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_matches_definition(shape, causal, dtype):
    _run(*_inputs(sum(shape), *shape, dtype), causal=causal)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_padded_batches_ignore_what_lies_beyond_the_lengths(d, causal, dtype):
    """Lengths of zero, one, inside and at tile edges, longer queries than keys (rows that see no
    key); NaN and infinities in every padded row."""
    import torch
    q_lens = torch.tensor([300, 0, 1, 128, 129, 257, 300, 5], dtype=torch.int32, device="cuda")
    kv_lens = torch.tensor([290, 290, 1, 0, 128, 129, 64, 290], dtype=torch.int32, device="cuda")
    q, k, v, g = _inputs(7, 8, 300, 290, 2, 1, d, dtype)
    clean = [t.clone() for t in (q, k, v, g)]
    for b in range(8):
        for t, n in ((q, q_lens[b]), (g, q_lens[b]), (k, kv_lens[b]), (v, kv_lens[b])):
            t[b, int(n):] = math.nan
            t[b, int(n)::3] = math.inf
    _run(*clean, causal=causal, q_lens=q_lens, kv_lens=kv_lens)
    from splatx_cuda import network
    how = dict(causal=causal, q_lens=q_lens, kv_lens=kv_lens)
    a = network.attention_fwd(*clean[:3], **how)
    b = network.attention_fwd(q, k, v, **how)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    ga = network.attention_bwd(clean[3], *clean[:3], *a, **how)
    gb = network.attention_bwd(g, q, k, v, *b, **how)
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))


def test_lengths_outside_the_batch_are_clamped():
    import torch
    from splatx_cuda import network
    q, k, v, _ = _inputs(3, 2, 40, 50, 2, 2, 64, "bfloat16")
    far = torch.tensor([-5, 1 << 30], dtype=torch.int32, device="cuda")
    near = torch.tensor([0, 50], dtype=torch.int32, device="cuda")
    assert torch.equal(network.attention_fwd(q, k, v, kv_lens=far)[0],
                       network.attention_fwd(q, k, v, kv_lens=near)[0])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_scores_of_large_magnitude(dtype):
    """Rows whose maximum grows by far from tile to tile, and one dominated by a single key."""
    import torch
    q, k, v, g = _inputs(11, 1, 200, 700, 2, 2, 64, dtype)
    k *= torch.linspace(0.1, 6.0, 700, device="cuda").to(k.dtype)[None, :, None, None]
    _run(q * 4, k, v, g)
    _run(q * 4, k.flip(1), v, g, causal=True)
    _run(q, k, v, g, scale=-0.3)
    _run(q, k, v, g, scale=0.0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides(dtype):
    """Heads before tokens, a packed qkv projection, an odd offset, a broadcast key-value head, a
    head axis that is not contiguous, a gradient expanded from one row."""
    import torch
    q, k, v, g = _inputs(5, 2, 140, 140, 4, 4, 64, dtype)
    swap = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    _run(swap(q), swap(k), swap(v), swap(g), causal=True)
    qkv = torch.randn(2, 140, 3, 4, 64, device="cuda").to(q.dtype)
    _run(*qkv.unbind(2), g)
    wide = torch.randn(2, 140, 4, 72, device="cuda").to(q.dtype)
    _run(wide[..., 3:67], k, wide[..., 1:65], g)
    _run(q, k[:, :, :1].expand(-1, -1, 4, -1), v[:, :1].expand(-1, 140, -1, -1), g[:1, :1].expand(2, 140, -1, -1))
    _run(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, g.transpose(2, 3).contiguous().transpose(2, 3))


def test_same_result_in_every_call_and_on_another_stream():
    import torch
    from splatx_cuda import network
    q, k, v, g = _inputs(9, 2, 700, 900, 4, 2, 128, "bfloat16")
    out, lse = network.attention_fwd(q, k, v)
    grads = network.attention_bwd(g, q, k, v, out, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [*network.attention_fwd(q, k, v), *network.attention_bwd(g, q, k, v, out, lse)]
    side.synchronize()
    for x, y in zip((out, lse, *grads), again):
        assert torch.equal(x, y)


@pytest.mark.parametrize("lq,lk,h,hk,q_len", [(37, 769, 8, 4, 37), (1, 900, 16, 2, 1), (200, 300, 2, 2, 77), (18, 345, 4, 1, 5)])
def test_rows_of_no_query_change_nothing(lq, lk, h, hk, q_len):
    """The rest of a tile of queries (padding, or what another call left in shared memory where the
    heads of a group share a tile) changes no bit: the same in every call, and with NaN and large
    values behind the length."""
    import torch
    from splatx_cuda import network
    q, k, v, _ = _inputs(lq, 1, lq, lk, h, hk, 128, "bfloat16")
    lens = torch.tensor([q_len], dtype=torch.int32, device="cuda")
    first = network.attention_fwd(q, k, v, q_lens=lens)
    other = [t * 30 for t in _inputs(3, 2, 512, 512, 8, 8, 128, "bfloat16")]
    for fill in (math.nan, 1e4, -1e4):
        network.attention_fwd(*other[:3])
        q[:, q_len:] = fill
        again = network.attention_fwd(q, k, v, q_lens=lens)
        assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_captured_in_a_graph():
    import torch
    from splatx_cuda import network
    q, k, v, g = _inputs(10, 1, 300, 300, 2, 2, 64, "bfloat16")
    want = network.attention_fwd(q, k, v, causal=True)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, lse = network.attention_fwd(q, k, v, causal=True)
        grads = network.attention_bwd(g, q, k, v, out, lse, causal=True)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    direct = network.attention_bwd(g, q, k, v, *want, causal=True)
    assert all(torch.equal(x, y) for x, y in zip(grads, direct))


def test_gradients_against_differences():
    """The directional derivative of sum(out * g) in 64 bits. The central difference's own error is
    h^2 / 6 of the third derivative (h = 1e-4: below 1e-7 of the value here); the kernel's is the
    bounds above summed over the direction."""
    import torch
    from splatx_cuda import network
    q, k, v, g = _inputs(21, 1, 70, 90, 2, 1, 64, "float32")
    out, lse = network.attention_fwd(q, k, v, causal=True)
    grads = network.attention_bwd(g, q, k, v, out, lse, causal=True)
    seen = _seen(1, 70, 90, True, None, None)

    def loss(q, k, v):
        s = q.transpose(1, 2) @ k.transpose(1, 2).repeat_interleave(2, 1).transpose(2, 3) / 8.0
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        return float(((p @ v.transpose(1, 2).repeat_interleave(2, 1)).transpose(1, 2) * g.double()).sum())

    for i in range(3):
        way = torch.randn_like(grads[i]).double()
        plus, minus = ([t.double() + (s * 1e-4 * way if j == i else 0) for j, t in enumerate((q, k, v))]
                       for s in (1, -1))
        diff = (loss(*plus) - loss(*minus)) / 2e-4
        mine = float((grads[i].double() * way).sum())
        size = float((grads[i].double() * way).abs().sum())
        assert abs(diff - mine) <= 1e-5 * size, (i, diff, mine)


def test_autograd():
    import torch
    from splatx_cuda import network
    q, k, v, g = _inputs(22, 2, 50, 60, 4, 2, 64, "bfloat16")
    for t in (q, k, v):
        t.requires_grad_()
    out = network.attention(q, k, v)
    out.backward(g)
    o, lse = network.attention_fwd(q.detach(), k.detach(), v.detach())
    want = network.attention_bwd(g, q.detach(), k.detach(), v.detach(), o, lse)
    assert torch.equal(out, o) and all(torch.equal(t.grad, w) for t, w in zip((q, k, v), want))


@pytest.mark.parametrize("b,lq,lk", [(0, 5, 5), (2, 0, 5), (2, 5, 0)])
def test_empty(b, lq, lk):
    import torch
    q, k, v, g = _inputs(1, b, lq, lk, 2, 2, 64, "bfloat16")
    from splatx_cuda import network
    out, lse = network.attention_fwd(q, k, v)
    assert not out.any() and bool((lse == -math.inf).all())
    for t, like in zip(network.attention_bwd(g, q, k, v, out, lse), (q, k, v)):
        assert t.shape == like.shape and not t.any()
    torch.cuda.synchronize()


def test_offsets_beyond_32_bits():
    """A cache of 2^31 + values: the last head of the last batch entry starts beyond 32-bit offsets."""
    import torch
    from splatx_cuda import network
    b, lk, h, d = 2, 8192, 1040, 128
    k = torch.empty(b, lk, h, d, dtype=torch.bfloat16, device="cuda")
    assert k[1, :, h - 1].data_ptr() - k.data_ptr() > 2 ** 31
    k[:, :, -2:] = torch.randn(b, lk, 2, d, device="cuda").to(k.dtype)
    q = torch.randn(b, 3, 2, d, device="cuda").to(k.dtype)
    view, small = k[:, :, -2:], k[:, :, -2:].contiguous()
    a, c = network.attention_fwd(q, view, view), network.attention_fwd(q, small, small)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    ga = network.attention_bwd(q, q, view, view, *a)
    gc = network.attention_bwd(q, q, small, small, *c)
    assert all(torch.equal(x, y) for x, y in zip(ga, gc))


def test_refusals():
    import torch
    from splatx_cuda import network
    q, k, v, g = _inputs(2, 2, 8, 9, 4, 2, 64, "bfloat16")
    out, lse = network.attention_fwd(q, k, v)
    lens = torch.tensor([8, 8], dtype=torch.int32, device="cuda")
    bad = [
        lambda: network.attention_fwd(q.cpu(), k, v), lambda: network.attention_fwd(q, k.cpu(), v),
        lambda: network.attention_fwd(q.double(), k.double(), v.double()),
        lambda: network.attention_fwd(q, k.float(), v), lambda: network.attention_fwd(q[0], k, v),
        lambda: network.attention_fwd(q[:, :, :3], k, v), lambda: network.attention_fwd(q, k, v[:, :5]),
        lambda: network.attention_fwd(q[:1], k, v), lambda: network.attention_fwd(q, k, v, scale=math.nan),
        lambda: network.attention_fwd(q, k, v, kv_lens=lens.long()),
        lambda: network.attention_fwd(q, k, v, q_lens=lens[:1]),
        lambda: network.attention_fwd(*(torch.cat([t, t, t], -1) for t in (q, k, v))),
        lambda: network.attention_bwd(g, q, k, v, out, lse.double()),
        lambda: network.attention_bwd(g[:, :3], q, k, v, out, lse),
        lambda: network.attention_bwd(g, q, k, v, out[:1], lse),
        lambda: network.attention_bwd(g.float(), q, k, v, out, lse),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_c_entry_refusals():
    """Refusals of the C entry itself; none launches anything."""
    import ctypes as C
    import torch
    from splatx_cuda import _native as n
    L = n.lib()
    t = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    view = n.SxAttentionView(t.data_ptr(), 1024, 64, 64)
    def inputs(**kw):
        d = dict(q=view, k=view, v=view, q_lens=None, kv_lens=None, batch=1, q_len=2, kv_len=2, q_heads=1,
                 kv_heads=1, head_dim=64, dtype=n._SIGNATURES and 2, scale=1.0, causal=0)
        d.update(kw)
        return n.SxAttentionInputs(**d)
    def fwd(ins, out=view, lse=t.data_ptr(), ws=t.data_ptr(), size=1 << 20):
        nb = C.c_size_t(size)
        return L.sxcuda_attention_fwd(C.byref(ins), None if out is None else C.byref(out), lse, ws, C.byref(nb), None)
    null = n.SxAttentionView(None, 0, 0, 0)
    odd = n.SxAttentionView(t.data_ptr() + 1, 1024, 64, 64)
    back = n.SxAttentionView(t.data_ptr(), 1024, -64, 64)
    flat = n.SxAttentionView(t.data_ptr(), 1024, 0, 64)
    cases = [fwd(inputs(head_dim=0)), fwd(inputs(head_dim=129)), fwd(inputs(dtype=7)), fwd(inputs(batch=-1)),
             fwd(inputs(q_heads=3, kv_heads=2)), fwd(inputs(kv_heads=0)), fwd(inputs(q=null)), fwd(inputs(k=odd)),
             fwd(inputs(v=back)), fwd(inputs(), out=None), fwd(inputs(), out=flat), fwd(inputs(), lse=None),
             fwd(inputs(scale=float("inf"))), fwd(inputs(batch=70000)),
             L.sxcuda_attention_fwd(None, C.byref(view), t.data_ptr(), t.data_ptr(), C.byref(C.c_size_t(8)), None),
             L.sxcuda_attention_fwd(C.byref(inputs()), C.byref(view), t.data_ptr(), t.data_ptr(), None, None),
             L.sxcuda_attention_bwd(C.byref(inputs()), None, None, t.data_ptr(), C.byref(C.c_size_t(1 << 20)), None),
             L.sxcuda_attention_bwd(C.byref(inputs()), None, None, t.data_ptr(), C.byref(C.c_size_t(4)), None),
             L.sxcuda_attention_status(None)]
    assert cases == [n.SXCUDA_EINVAL] * len(cases), cases
    assert np.all(t.cpu().float().numpy() == 0)


def _of_two_magnitudes():
    """float16 inputs with key heads that are 2^18 apart in g v."""
    import torch
    q, k, v, g = _inputs(31, 2, 300, 260, 4, 2, 64, "float16")
    g[0, :, :2] *= 2.0 ** 9  # key head 0's two query heads
    v[0, :, 0] *= 2.0 ** 3
    g[0, :, 2:] *= 2.0 ** -6
    return q, k, v, g


@pytest.mark.parametrize("causal", [False, True])
def test_half_gradients_beside_larger_ones(causal):
    _run(*_of_two_magnitudes(), causal=causal)


def test_half_gradients_do_not_depend_on_other_heads_or_entries():
    import torch
    q, k, v, g = _of_two_magnitudes()
    _, _, first = _run(q, k, v, g)
    g[0, :, :2] *= 2.0 ** -12
    v[0, :, 0] = 0
    _, _, again = _run(q, k, v, g)
    for x, y in zip(first, again):
        per = x.shape[2] // 2
        assert torch.equal(x[1], y[1]) and torch.equal(x[0, :, per:], y[0, :, per:])
