"""Linear layers and their gradients against their definition in 64 bits.

Bounds. A sum of K products carries K roundings in 32 bits, each at most 2^-24 of a partial sum, which is
at most S = sum |terms|; taken as independent they stay below 4 sqrt(K) 2^-24 S (6 deviations of K errors
spread evenly over a rounding). Activations have slopes of at most 1.13; their own error is relative to
the value, FAST for 16-bit types (a 16th of half a step of float16) and 2^-21 for float32 (library
functions, some 4 roundings). Slopes are off by SLOPE, absolutely, as they are up to 1.13: a reciprocal and an
exponential of 2^-22 each, and a polynomial's roundings. v_z is rounded to the element type before its products,
but not before the bias' sum.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
FAST = {"float32": 2.0 ** -21, "float16": 2.0 ** -15, "bfloat16": 2.0 ** -15}
SLOPE = 2.0 ** -20
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}  # half a step below the normal numbers
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def _act(name, z):
    import torch
    if name == "relu":
        return torch.relu(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def _slope(name, z):
    import torch
    if name is None:
        return torch.ones_like(z)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    z = z.detach().requires_grad_()
    return torch.autograd.grad(_act(name, z).sum(), z)[0]


def _inputs(seed, rows, k, n, dtype, bias="float32", residual=False):
    import torch
    g = torch.Generator().manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    T = getattr(torch, dtype)
    x, w = t(rows, k).to(T).cuda(), (t(n, k) * k ** -0.5).to(T).cuda()
    b = None if bias is None else (t(n) * 0.3).to(getattr(torch, bias)).cuda()
    return x, w, b, t(rows, n).to(T).cuda() if residual else None, t(rows, n).to(T).cuda()


def _near(name, got, want, bound):
    import torch
    assert got.shape == want.shape, name
    off = (got.double() - want).abs() - bound
    assert off.numel() == 0 or (not torch.isnan(off).any() and float(off.max()) <= 0), (name, float(off.max()))


def _sums(k):
    return (4 * math.sqrt(k) + 4) * 2.0 ** -24


def _check(x, w, b, r, g, act):
    """Forward with everything kept, and backward on what it kept."""
    import torch
    from splatx_cuda import network
    dtype = str(x.dtype).split(".")[1]
    u, fast, tiny = ROUND[dtype], FAST[dtype], TINY[dtype]
    y, pre = network.linear_fwd(x, w, b, activation=act, residual=r, keep=act is not None)
    n, k = w.shape
    X, W, G = x.double().reshape(-1, k), w.double(), g.double().reshape(-1, n)
    B = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
    R = torch.zeros_like(G) if r is None else r.double().reshape(-1, n)
    Z = X @ W.T + B
    e_z = _sums(k) * (X.abs() @ W.abs().T + B.abs())
    A = _act(act, Z)
    Y = A + R
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    _near("y", flat(y), Y, (1.13 * e_z + fast * A.abs() + 2.0 ** -23 * (A.abs() + R.abs())) * (1 + u) + u * Y.abs() + tiny)
    if act is None:
        assert pre is None
        D, e_d = G, torch.zeros_like(G)
        exact = G
    else:
        _near("pre", flat(pre), Z, e_z * (1 + u) + u * Z.abs() + tiny)
        exact = G * _slope(act, flat(pre).double())
        # the sum for the bias takes it before it is rounded
        e_b = SLOPE * G.abs() + 2.0 ** -23 * exact.abs()
        D, e_d = exact, e_b + u * exact.abs() + tiny
    v_x, v_w, v_b = network.linear_bwd(g, x, w, b, pre, activation=act)
    VX, VW, VB = D @ W, D.T @ X, exact.sum(0)
    _near("v_x", flat(v_x), VX, (e_d @ W.abs() + _sums(n) * (D.abs() @ W.abs())) * (1 + u) + u * VX.abs() + tiny)
    m = max(1, X.shape[0])
    _near("v_weight", v_w, VW, (e_d.T @ X.abs() + _sums(m) * (D.abs().T @ X.abs())) * (1 + u) + u * VW.abs() + tiny)
    if b is None:
        assert v_b is None
    else:
        ub = ROUND[str(b.dtype).split(".")[1]]
        e_b = 0.0 if act is None else (SLOPE * G.abs() + 2.0 ** -23 * exact.abs()).sum(0)
        _near("v_bias", v_b, VB, (e_b + _sums(m) * exact.abs().sum(0)) * (1 + ub) + ub * VB.abs() + TINY[str(b.dtype).split(".")[1]])
        assert v_b.dtype == b.dtype
    assert network.linear_status() == 0
    return y, pre, v_x, v_w, v_b


SIZES = [(1, 1, 1), (1, 64, 256), (2, 8, 3), (3, 1000, 17), (7, 4096, 128), (31, 64, 64), (64, 128, 512), (77, 640, 640),
         (127, 63, 129), (128, 64, 128), (129, 65, 257), (256, 256, 256), (257, 72, 264), (300, 333, 777), (1000, 200, 1),
         (1025, 11, 96), (513, 1032, 520), (2048, 128, 512), (4100, 96, 3)]
name = lambda s: "x".join(map(str, s))  # noqa: E731


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("size", SIZES, ids=name)
def test_linear_sizes(size, dtype):
    i = SIZES.index(size)
    act = ACTS[i % 5]
    _check(*_inputs(i, *size, dtype, bias="float32", residual=i % 2 == 0), act)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(act, dtype):
    for residual in (False, True):
        for bias in ("float32", dtype, None):
            _check(*_inputs(5, 200, 136, 328, dtype, bias=bias, residual=residual), act)
            _check(*_inputs(6, 70, 35, 101, dtype, bias=bias, residual=residual), act)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("size", [(5000, 512, 384), (20000, 256, 640), (4096, 1024, 1024), (130, 8192, 96)], ids=name)
def test_linear_larger(size, dtype):
    """More tiles than workers, long sums, tiles that are cut."""
    _check(*_inputs(11, *size, dtype, residual=True), "gelu")
    _check(*_inputs(12, *size, dtype), None)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("act", ACTS[1:])
def test_activation_over_its_range(act, dtype):
    """Weights of one, so that every value of z is met as it is: tails, zeros, the largest."""
    import torch
    from splatx_cuda import network
    T = getattr(torch, dtype)
    z = torch.cat([torch.linspace(-14, 14, 3000, dtype=torch.float64), torch.logspace(-6, 4, 500, dtype=torch.float64),
                   -torch.logspace(-6, 4, 500, dtype=torch.float64), torch.zeros(8, dtype=torch.float64)]).to(T)
    x = torch.zeros(len(z), 8, dtype=T)
    x[:, 0] = z
    w = torch.zeros(16, 8, dtype=T)
    w[:, 0] = 1
    x, w, z = x.cuda(), w.cuda(), z.cuda()
    y, pre = network.linear_fwd(x, w, activation=act, keep=True)
    assert torch.equal(pre, z[:, None].expand(-1, 16))
    u, fast, tiny = ROUND[dtype], FAST[dtype], TINY[dtype]
    A = _act(act, z.double())[:, None].expand(-1, 16)
    if act == "gelu_tanh":  # 1 + tanh of the definition loses the tail that 1 / (1 + exp) keeps
        c = 2 * math.sqrt(2 / math.pi)
        A = (z.double() * torch.sigmoid(c * (z.double() + 0.044715 * z.double() ** 3)))[:, None].expand(-1, 16)
    # an exponential's argument a is rounded: its value is off by 2^-23 |a|, a = z^2 / 2 (twice that for the tanh form)
    a = z.double().abs()[:, None]
    arg = 2.0 ** -23 * {"relu": 0 * a, "silu": a, "gelu": 0.5 * a * a, "gelu_tanh": 1.6 * (a + 0.0448 * a ** 3)}[act].clamp(max=1000)
    # below the least normal number of 32 bits the exponential may end at zero
    _near("y", y, A, (fast + arg) * A.abs() + u * A.abs() + tiny + 2.0 ** -125 * a)
    g = torch.ones(len(z), 16, dtype=T, device="cuda")
    g[:, 1:] = 0
    _, _, v_b = network.linear_bwd(g[:, :16], x, w, torch.zeros(16, device="cuda"), pre, activation=act)
    one = torch.eye(len(z), dtype=T, device="cuda")[:40]
    assert bool(torch.isfinite(v_b).all())
    # one row at a time: its slope is the bias' gradient
    for i in range(0, len(z), 111):
        v = network.linear_bwd(g[i:i + 1], x[i:i + 1], w, torch.zeros(16, device="cuda"), pre[i:i + 1], activation=act)[2]
        want = _slope(act, z[i:i + 1].double())
        assert abs(float(v[0] - want)) <= SLOPE + 2.0 ** -22 * abs(float(want)), (float(z[i]), float(v[0]), float(want))
    assert one.shape[0] == 40


def test_linear_what_is_not_finite():
    """NaN in a row of x stays in that row, an infinite weight's column stays in its column."""
    import torch
    from splatx_cuda import network
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x, w, b, r, g = _inputs(3, 300, 72, 264, str(dtype).split(".")[1], residual=True)
        want, _ = network.linear_fwd(x, w, b, activation="relu", residual=r)
        x[17, 5] = math.nan
        w[100, 3] = math.inf
        y, pre = network.linear_fwd(x, w, b, activation="relu", residual=r, keep=True)
        keep = [i for i in range(300) if i != 17]
        cols = [i for i in range(264) if i != 100]
        assert bool(y[17].isnan().all()) and bool(pre[17].isnan().all())
        assert torch.equal(y[keep][:, cols], want[keep][:, cols])
        assert not bool(torch.isfinite(pre[:, 100]).any())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_linear_strides_and_shapes(dtype):
    import torch
    x, w, b, r, g = _inputs(8, 120, 96, 136, dtype, residual=True)
    want = _check(x, w, b, r, g, "silu")
    wide = torch.full((120, 140), math.nan, dtype=x.dtype, device="cuda")
    for start in (0, 1, 8):
        wide[:, start:start + 96] = x
        got = _check(wide[:, start:start + 96], w, b, r, g, "silu")
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        wide[:] = math.nan
    for pitch, start in ((144, 8), (144, 32), (104, 0)):  # rows that copies reach, between what must not be read
        wide = torch.full((120, pitch), math.nan, dtype=x.dtype, device="cuda")
        wide[:, start:start + 96] = x
        heavy = torch.full((136, pitch), math.nan, dtype=x.dtype, device="cuda")
        heavy[:, start:start + 96] = w
        got = _check(wide[:, start:start + 96], heavy[:, start:start + 96], b, r, g, "silu")
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    got = _check(x.view(2, 5, 12, 96), w, b, r.view(2, 5, 12, 136), g.view(2, 5, 12, 136), "silu")
    assert got[0].shape == (2, 5, 12, 136) and got[2].shape == (2, 5, 12, 96)
    _check(x.t().contiguous().t(), w.t().contiguous().t(), b, r[:1].expand(120, -1), g[:, :1].expand(-1, 136), "silu")
    tall = torch.full((136, 101), math.nan, dtype=x.dtype, device="cuda")
    tall[:, 5:101] = w
    _check(x, tall[:, 5:101], b, r, g, "silu")
    _check(x[0], w, b, r[0], g[0], "gelu")  # one token without a row axis


def test_linear_no_rows():
    import torch
    from splatx_cuda import network
    x, w, b, _, g = _inputs(1, 0, 64, 96, "bfloat16")
    y, pre = network.linear_fwd(x, w, b, activation="gelu", keep=True)
    assert y.shape == pre.shape == (0, 96)
    v_x, v_w, v_b = network.linear_bwd(g, x, w, b, pre, activation="gelu")
    assert v_x.shape == (0, 64) and not v_w.any() and not v_b.any()


def test_linear_only_what_is_needed():
    import torch
    from splatx_cuda import network
    x, w, b, _, g = _inputs(2, 200, 128, 256, "bfloat16")
    every = network.linear_bwd(g, x, w, b)
    assert torch.equal(network.linear_bwd(g, x, w, b, needs_weight=False)[0], every[0])
    some = network.linear_bwd(g, x, w, needs_x=False)
    assert some[0] is None and some[2] is None and torch.equal(some[1], every[1])
    assert network.linear_bwd(g, x, w, needs_x=False, needs_weight=False) == (None, None, None)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_linear_is_the_same_every_time(dtype):
    import torch
    from splatx_cuda import network
    x, w, b, r, g = _inputs(4, 3000, 512, 640, dtype, residual=True)
    runs = []
    for _ in range(3):
        y, pre = network.linear_fwd(x, w, b, activation="gelu", residual=r, keep=True)
        runs.append((y, pre, *network.linear_bwd(g, x, w, b, pre, activation="gelu")))
    assert all(torch.equal(a, c) for run in runs[1:] for a, c in zip(run, runs[0]))


@pytest.mark.parametrize("act", ACTS)
def test_linear_autograd_and_differences(act):
    import torch
    from splatx_cuda import network
    x, w, b, r, g = _inputs(21, 50, 40, 72, "float32", residual=True)
    ins = [t.requires_grad_() for t in (x, w, b, r)]
    y = network.linear(x, w, b, activation=act, residual=r)
    grads = torch.autograd.grad((y * g).sum(), ins)
    D = [t.detach().double().requires_grad_() for t in ins]
    Y = _act(act, D[0] @ D[1].T + D[2]) + D[3]
    for got, want in zip(grads, torch.autograd.grad((Y * g).sum(), D)):
        assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())
    # the forward's own differences along a direction: h^2 of the third derivative, 2^-24 / h of the rounding
    f = lambda *t: (network.linear(t[0], t[1], t[2], activation=act, residual=t[3]).double() * g).sum()  # noqa: E731
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i, t in enumerate(ins):
        d = torch.randn(t.shape, generator=gen, device="cuda")
        d /= d.norm()
        h = 1e-2
        up, down = ([(u + s * h * d if j == i else u).detach() for j, u in enumerate(ins)] for s in (1, -1))
        slope = float(f(*up) - f(*down)) / (2 * h)
        want = float((grads[i] * d).sum())
        scale = float(grads[i].norm())
        if act != "relu":  # a corner has no derivative
            assert abs(slope - want) <= 2e-3 * scale + 1e-3, (i, slope, want)
    y = network.linear(x, w, activation=act)
    (v,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(v.sum(), w)


def test_linear_autograd_of_some_inputs():
    import torch
    from splatx_cuda import network
    x, w, b, r, g = _inputs(22, 64, 64, 64, "bfloat16", residual=True)
    y = network.linear(x, w, b.requires_grad_(), residual=r.requires_grad_(), activation="gelu")
    v_b, v_r = torch.autograd.grad(y, (b, r), g)
    _, pre = network.linear_fwd(x, w, b, activation="gelu", keep=True)
    assert torch.equal(v_b, network.linear_bwd(g, x, w, b, pre, activation="gelu")[2]) and torch.equal(v_r, g)
    with torch.no_grad():
        assert torch.equal(network.linear(x, w, b, residual=r, activation="gelu"), y)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_linear_streams_and_graphs(dtype):
    """On a stream of its own, and captured twice: two graphs that run at the same time."""
    import torch
    from splatx_cuda import network
    made = [_inputs(30 + i, 400, 512, 260, dtype, residual=True) for i in range(2)]

    def both(x, w, b, r, g):
        y, pre = network.linear_fwd(x, w, b, activation="silu", residual=r, keep=True)
        return (y, pre, *network.linear_bwd(g, x, w, b, pre, activation="silu"))

    want = [both(*m) for m in made]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(*made[0])
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want[0]))
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
        for o, w in zip(outs, want):
            assert all(torch.equal(a, c) for a, c in zip(o, w))
            for t in o:
                t.zero_()
    torch.cuda.synchronize()


def test_linear_residual_may_be_the_output():
    """At the C entry y may be written over the residual."""
    import ctypes as C
    import torch
    from splatx_cuda import _native as n, network
    for dtype, size in (("bfloat16", (300, 512, 264)), ("bfloat16", (40, 4096, 101)), ("float32", (300, 512, 264))):
        x, w, b, r, _ = _inputs(40, *size, dtype, residual=True)
        want, _ = network.linear_fwd(x, w, b, activation="gelu", residual=r)
        m, k, o = size
        ins = n.SxLinearInputs(x.data_ptr(), w.data_ptr(), b.data_ptr(), m, k, o, k, k, {"bfloat16": 2, "float32": 0}[dtype], 0, 3)
        outs = n.SxLinearOutputs(r.data_ptr(), o, r.data_ptr(), o, None, 0)
        nbytes = C.c_size_t(0)
        entry, stream = n.lib().sxcuda_linear_fwd, torch.cuda.current_stream().cuda_stream
        n.check(entry(C.byref(ins), C.byref(outs), None, C.byref(nbytes), None))
        ws = torch.empty(max(nbytes.value, 16), dtype=torch.uint8, device="cuda")
        n.check(entry(C.byref(ins), C.byref(outs), ws.data_ptr(), C.byref(nbytes), stream))
        assert torch.equal(r, want)


def test_linear_writes_nothing_else():
    """Guards around outputs of odd sizes, at the C entry with rows further apart than they are long."""
    import ctypes as C
    import torch
    from splatx_cuda import _native as n, network
    for dtype, code, size in ((torch.bfloat16, 2, (131, 72, 101)), (torch.bfloat16, 2, (260, 512, 264)),
                              (torch.float16, 1, (1, 1024, 40)), (torch.float32, 0, (131, 72, 101))):
        m, k, o = size
        x, w, b, _, _ = _inputs(41, *size, str(dtype).split(".")[1])
        want, want_pre = network.linear_fwd(x, w, b, activation="relu", keep=True)
        for pitch, first in ((o + 8, 8), (o + 3, 1)):
            y, pre = (torch.full((m + 2, pitch), 7.0, dtype=dtype, device="cuda") for _ in range(2))
            at = (pitch + first) * y.element_size()
            ins = n.SxLinearInputs(x.data_ptr(), w.data_ptr(), b.data_ptr(), m, k, o, k, k, code, 0, 1)
            outs = n.SxLinearOutputs(None, 0, y.data_ptr() + at, pitch, pre.data_ptr() + at, pitch)
            nbytes = C.c_size_t(0)
            entry, stream = n.lib().sxcuda_linear_fwd, torch.cuda.current_stream().cuda_stream
            n.check(entry(C.byref(ins), C.byref(outs), None, C.byref(nbytes), None))
            ws = torch.empty(max(nbytes.value, 16), dtype=torch.uint8, device="cuda")
            n.check(entry(C.byref(ins), C.byref(outs), ws.data_ptr(), C.byref(nbytes), stream))
            for t, v in ((y, want), (pre, want_pre)):
                rows = torch.as_strided(t, (m, o), (pitch, 1), pitch + first)
                assert torch.equal(rows, v)
                rows.fill_(7.0)
                assert bool((t == 7.0).all())


def test_linear_refusals():
    import torch
    from splatx_cuda import network
    x, w, b, r, g = _inputs(50, 8, 64, 32, "bfloat16", residual=True)
    _, pre = network.linear_fwd(x, w, b, activation="gelu", keep=True)
    for f in (lambda: network.linear_fwd(x, w.cpu()), lambda: network.linear_fwd(x, w, b.cpu()), lambda: network.linear_fwd(x.cpu(), w.cpu()),
              lambda: network.linear_fwd(x, w, residual=r.cpu()), lambda: network.linear_fwd(x, w, residual=r[:4]),
              lambda: network.linear_fwd(x, w, residual=r.float()), lambda: network.linear_fwd(x, w, b.double()),
              lambda: network.linear_bwd(g, x, w, b, pre), lambda: network.linear_bwd(g, x, w, b, activation="gelu"),
              lambda: network.linear_bwd(g[:4], x, w), lambda: network.linear_bwd(g.float(), x, w),
              lambda: network.linear_bwd(g, x, w, b, pre.float(), activation="gelu"),
              lambda: network.linear_bwd(g, x, w, b, pre[:4], activation="gelu"),
              lambda: network.linear_bwd(g.cpu(), x, w)):
        with pytest.raises(ValueError):
            f()


def test_linear_beyond_32_bits():
    """x of more than 2^31 values: its last rows, and all of them in the weight's gradient."""
    import torch
    from splatx_cuda import network
    rows, k, n = 1_100_003, 2048, 24
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    w = (torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5).bfloat16()
    b = torch.randn(n, generator=gen, device="cuda")
    y, _ = network.linear_fwd(x, w, b)
    for part in (slice(0, 300), slice(rows // 2, rows // 2 + 300), slice(rows - 300, rows)):
        X = x[part].double()
        want = X @ w.double().T + b.double()
        bound = _sums(k) * (X.abs() @ w.double().abs().T + b.double().abs()) + ROUND["bfloat16"] * want.abs()
        _near("y", y[part], want, bound * (1 + 2.0 ** -7))
    g = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 5, rows // 2, rows - 2, rows - 1], device="cuda")
    g[at] = torch.randn(5, n, generator=gen, device="cuda").bfloat16()
    v_x, v_w, v_b = network.linear_bwd(g, x, w, b)
    G = g[at].double()
    want = G.T @ x[at].double()
    _near("v_weight", v_w, want, 2.0 ** -21 * (G.abs().T @ x[at].double().abs()) + ROUND["bfloat16"] * want.abs())
    _near("v_bias", v_b, G.sum(0), 2.0 ** -21 * G.abs().sum(0))
    want = G @ w.double()
    _near("v_x", v_x[at], want, _sums(n) * (G.abs() @ w.double().abs()) + ROUND["bfloat16"] * want.abs())
    v_x[at] = 0
    assert not v_x.any()


# float32 in tiles of 128 that are cut along K, forward and in the gradient of x beside one of 64; weight gradients
# of few features and many rows, whose tiles have tens to hundreds of parts.
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("size", [(9700, 700, 1020), (9701, 1019, 701), (30001, 64, 3), (30001, 3, 64), (60000, 48, 64),
                                  (3000, 256, 256), (604, 77, 913)], ids=name)
def test_linear_many_parts(size, dtype):
    x, w, b, r, g = _inputs(31, *size, dtype, residual=True)
    first = _check(x, w, b, r, g, "gelu")
    again = _check(x, w, b, r, g, "gelu")
    for a, c in zip(first, again):
        assert (a == c).all()
    from splatx_cuda import network
    v_x, v_w, v_b = first[2:]
    for needs_x, needs_weight in ((True, False), (False, True)):  # either product without the other
        one = network.linear_bwd(g, x, w, b, first[1], activation="gelu", needs_x=needs_x, needs_weight=needs_weight)
        assert (one[0] is None) != needs_x and (one[1] is None) != needs_weight
        assert (one[2] == v_b).all()
        assert all((a == c).all() for a, c in zip(one[:2], (v_x, v_w)) if a is not None)
