"""Layer norm and the multi-tensor AdamW step against their formulas.

Layer norm's bounds: a row's sums carry at most 64 roundings a term in 32 bits (32 values a thread,
then a tree), so the mean is off by 64 2^-24 mean|x|, and every quantity made from it likewise; the
result is rounded once to the element type. AdamW rounds each operation by itself, so that numpy's
float32 gives every bit of it.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
E32 = 64 * 2.0 ** -24


def _norm_inputs(seed, rows, cols, dtype, wtype, shift=0.5):
    import torch
    g = torch.Generator().manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (t(rows, cols) * 1.5 + shift).to(getattr(torch, dtype)).cuda()
    w, b = ((t(cols) * 0.3 + c).to(getattr(torch, wtype)).cuda() for c in (1.0, 0.0))
    return x, w, b, t(rows, cols).to(x.dtype).cuda()


def _check_norm(x, w, b, g, eps=1e-5):
    import torch
    from splatx_cuda import network
    dtype = str(x.dtype).split(".")[1]
    u, n = ROUND[dtype], x.shape[-1]
    y, mean, rstd = network.layer_norm_fwd(x, w, b, eps=eps)
    v_x, v_w, v_b = network.layer_norm_bwd(g, x, w, mean, rstd)
    X, G = x.double(), g.double()
    W = torch.ones(n, dtype=torch.float64, device="cuda") if w is None else w.double()
    B = torch.zeros_like(W) if b is None else b.double()
    m = X.mean(-1)
    e_m = E32 * X.abs().mean(-1)
    var = X.var(-1, unbiased=False)
    r = (var + eps) ** -0.5
    # a shift of the mean moves the variance by its square and each difference by itself
    e_var = E32 * var + 2 * e_m * (X - m[..., None]).abs().mean(-1) + e_m ** 2
    e_r = r * (0.5 * e_var * r * r + 4 * 2.0 ** -24)
    xhat = (X - m[..., None]) * r[..., None]
    e_x = xhat.abs() * ((e_r / r)[..., None] + 2.0 ** -22) + (e_m * r)[..., None]
    Y = xhat * W + B
    e_y = e_x * W.abs() + (u + 2.0 ** -22) * (Y.abs() + B.abs())

    def near(name, got, want, bound):
        off = ((got.double() - want).abs() - bound - 2.0 ** -25 * (dtype == "float16"))
        assert got.shape == want.shape and (off.numel() == 0 or float(off.max()) <= 0), (name, float(off.max()))

    near("mean", mean, m, e_m + 2.0 ** -24 * m.abs())
    near("rstd", rstd, r, e_r)
    near("y", y, Y, e_y)
    GW = G * W
    a, c = GW.mean(-1, keepdim=True), (GW * xhat).mean(-1, keepdim=True)
    e_a = E32 * GW.abs().mean(-1, keepdim=True)
    e_c = (GW.abs() * (e_x + E32 * xhat.abs())).mean(-1, keepdim=True)
    core = GW - a - xhat * c
    e_core = 2.0 ** -22 * (GW.abs() + a.abs() + (xhat * c).abs()) + e_a + e_x * c.abs() + xhat.abs() * e_c
    VX = core * r[..., None]
    near("v_x", v_x, VX, (e_core + core.abs() * (e_r / r)[..., None]) * r[..., None] * (1 + 1e-3) + (u + 2.0 ** -22) * VX.abs())
    uw = 0.0 if w is None or w.dtype == torch.float32 else ROUND[str(w.dtype).split(".")[1]]
    rows = max(1, X[..., 0].numel())
    flat = lambda t: t.reshape(-1, n).sum(0)  # noqa: E731
    terms = min(rows, rows // 64 + 512) * 2.0 ** -24  # roundings of one column's sum
    VW, VB = flat(G * xhat), flat(G)
    near("v_weight", v_w, VW, flat(G.abs() * (e_x + (terms + 2.0 ** -22) * xhat.abs())) + (uw + 2.0 ** -24) * VW.abs())
    near("v_bias", v_b, VB, flat(G.abs()) * (terms + 2.0 ** -22) + (uw + 2.0 ** -24) * VB.abs())
    return y, v_x, v_w, v_b


# one column, widths about each row group's limit, odd ones, beyond the registers; one row, more
# rows than the grid has groups
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 2), (700, 8), (33, 31), (4000, 64), (3, 257), (1, 1024), (50, 1025),
                                       (6001, 777), (600, 2048), (40, 2049), (301, 4096), (9, 4100), (310, 8192),
                                       (7, 8193), (70, 10001)])
def test_layer_norm(rows, cols, dtype):
    _check_norm(*_norm_inputs(rows + cols, rows, cols, dtype, "float32"))


@pytest.mark.parametrize("wtype", ["float16", "bfloat16", None])
def test_layer_norm_parameter_types(wtype):
    x, w, b, g = _norm_inputs(3, 90, 320, "bfloat16", wtype or "float32")
    if wtype is None:
        w = b = None
    _check_norm(x, w, b, g)


def test_layer_norm_of_a_large_mean_and_of_constant_rows():
    import torch
    x, w, b, g = _norm_inputs(4, 64, 512, "float32", "float32", shift=1000.0)
    _check_norm(x, w, b, g)
    from splatx_cuda import network
    y, mean, rstd = network.layer_norm_fwd(torch.full((3, 512), 0.75, device="cuda"), w, b)
    assert bool((mean == 0.75).all()) and torch.equal(y, b.expand(3, -1))
    assert bool(((rstd - 1e-5 ** -0.5).abs() < 1e-4).all())


def test_layer_norm_strides_and_shapes():
    import torch
    x, w, b, g = _norm_inputs(5, 120, 320, "bfloat16", "float32")
    wide = torch.zeros(120, 330, dtype=x.dtype, device="cuda")
    for start in (0, 3, 8):
        wide[:, start:start + 320] = x
        _check_norm(wide[:, start:start + 320], w, b, g)
    _check_norm(x.view(2, 60, 320).transpose(0, 1), w, b, g.view(60, 2, 320))
    _check_norm(x.t().contiguous().t(), w, b, g[:1].expand(120, -1))


def test_layer_norm_no_rows():
    import torch
    from splatx_cuda import network
    x, w, b, g = _norm_inputs(6, 0, 64, "float32", "float32")
    y, mean, rstd = network.layer_norm_fwd(x, w, b)
    v_x, v_w, v_b = network.layer_norm_bwd(g, x, w, mean, rstd)
    assert y.shape == v_x.shape == (0, 64) and mean.shape == (0,)
    torch.cuda.synchronize()
    assert not v_w.any() and not v_b.any()


def test_layer_norm_same_result_in_every_call_and_autograd():
    import torch
    from splatx_cuda import network
    x, w, b, g = _norm_inputs(7, 5000, 640, "bfloat16", "float32")
    _, mean, rstd = network.layer_norm_fwd(x, w, b)
    one = network.layer_norm_bwd(g, x, w, mean, rstd)
    two = network.layer_norm_bwd(g, x, w, mean, rstd)
    assert all(torch.equal(s, t) for s, t in zip(one, two))
    for t in (x, w, b):
        t.requires_grad_()
    network.layer_norm(x, w, b).backward(g)
    assert torch.equal(x.grad, one[0]) and torch.equal(w.grad, one[1]) and torch.equal(b.grad, one[2])


def test_layer_norm_gradients_against_differences():
    """The directional derivative of sum(y * g) in 64 bits, h = 1e-4."""
    import torch
    from splatx_cuda import network
    x, w, b, g = _norm_inputs(8, 20, 200, "float32", "float32")
    _, mean, rstd = network.layer_norm_fwd(x, w, b)
    grads = network.layer_norm_bwd(g, x, w, mean, rstd)
    def loss(x, w, b):
        d = x - x.mean(-1, keepdim=True)
        return float(((d * (d.pow(2).mean(-1, keepdim=True) + 1e-5) ** -0.5 * w + b) * g.double()).sum())
    for i in range(3):
        way = torch.randn_like(grads[i]).double()
        plus, minus = ([t.double() + (s * 1e-4 * way if j == i else 0) for j, t in enumerate((x, w, b))]
                       for s in (1, -1))
        mine = float((grads[i].double() * way).sum())
        size = float((grads[i].double() * way).abs().sum())
        assert abs((loss(*plus) - loss(*minus)) / 2e-4 - mine) <= 1e-5 * size


def test_layer_norm_refusals():
    import ctypes as C
    import torch
    from splatx_cuda import _native as n, network
    x, w, b, g = _norm_inputs(9, 4, 64, "bfloat16", "float32")
    _, mean, rstd = network.layer_norm_fwd(x, w, b)
    for f in (lambda: network.layer_norm_fwd(x.cpu(), w, b), lambda: network.layer_norm_fwd(x, w[:5], b),
              lambda: network.layer_norm_fwd(x, w, b.half()), lambda: network.layer_norm_fwd(x.double()),
              lambda: network.layer_norm_fwd(x, w, b, eps=-1.0), lambda: network.layer_norm_fwd(x[:, :0]),
              lambda: network.layer_norm_fwd(x, w.cpu(), b), lambda: network.layer_norm_fwd(x.long()),
              lambda: network.layer_norm_bwd(g[:2], x, w, mean, rstd), lambda: network.layer_norm_bwd(g.float(), x, w, mean, rstd),
              lambda: network.layer_norm_bwd(g, x, w, mean.double(), rstd),
              lambda: network.layer_norm_bwd(g, x, w, mean, rstd[:2])):
        with pytest.raises(ValueError):
            f()
    L = n.lib()
    def ins(**kw):
        d = dict(x=x.data_ptr(), weight=None, bias=None, rows=4, cols=64, x_stride=64, dtype=2, param_dtype=0, eps=0.0)
        d.update(kw)
        return n.SxLayerNormInputs(**d)
    y = torch.zeros_like(x)
    fwd = lambda i, y=y.data_ptr(), m=None: L.sxcuda_layer_norm_fwd(C.byref(i), y, 64, m, None, None)  # noqa: E731
    got = [fwd(ins(rows=-1)), fwd(ins(cols=0)), fwd(ins(x_stride=63)), fwd(ins(dtype=9)), fwd(ins(param_dtype=-1)),
           fwd(ins(x=None)), fwd(ins(x=x.data_ptr() + 1)), fwd(ins(eps=math.nan)), fwd(ins(), y=None),
           fwd(ins(), m=mean.data_ptr()),
           L.sxcuda_layer_norm_bwd(C.byref(ins()), None, None, y.data_ptr(), C.byref(C.c_size_t(1)), None),
           L.sxcuda_layer_norm_bwd(C.byref(ins()), None, None, y.data_ptr(), C.byref(C.c_size_t(1 << 30)), None)]
    assert got == [n.SXCUDA_EINVAL] * len(got), got


# ---------------------------------------------------------------- AdamW

F = np.float32
CFG = dict(lr=3e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.05)


def _np(t):
    return t.detach().float().cpu().numpy().ravel()


def _round_to(x, dtype):
    import torch
    return torch.from_numpy(x).to(dtype).float().numpy()


def _pack(x, keep):
    import torch
    n = x.size
    b = np.pad(x, (0, -n % 256)).reshape(-1, 256)
    top = np.abs(b).max(1)
    live = top >= F(1e-30)
    with np.errstate(divide="ignore"):
        to = b * np.where(live, F(1) / top * F(448), F(0))[:, None].astype(F)
    if keep:
        to[(to > 0) & (to < F(2.0 ** -9))] = F(2.0 ** -9)
    codes = torch.from_numpy(to.ravel()[:n].copy()).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, np.where(live, top * F(1.0 / 448.0), F(0)).astype(F)


def _unpack(codes, scale):
    c = codes.float().cpu().numpy().ravel()
    return c * np.repeat(scale, 256)[: c.size]


def _numpy_step(p, g, m, v, step, grad_scale=1.0, lr=None, decay=None):
    b1, b2 = CFG["betas"]
    lr = CFG["lr"] if lr is None else lr
    decay = CFG["weight_decay"] if decay is None else decay
    g = g * F(grad_scale)
    m = m * F(b1) + g * F(1 - b1)
    v = v * F(b2) + (g * g) * F(1 - b2)
    d = np.sqrt(v) * F(1 / math.sqrt(1 - b2 ** step)) + F(CFG["eps"])
    return p * F(1 - lr * decay) - m / d * F(lr / (1 - b1 ** step)), m, v


# no value, one, odd counts, counts about a chunk (4096) and a run (256)
SIZES = [0, 1, 3, 255, 256, 257, 4095, 4096, 4099, 10000, 70001]


def _tensors(seed, ptype, gtype, sizes=SIZES):
    import torch
    g = torch.Generator().manual_seed(seed)
    t = lambda n: torch.randn(n, generator=g)  # noqa: E731
    params = [t(n).to(getattr(torch, ptype)).cuda() for n in sizes]
    grads = [[(t(n) * torch.exp(2 * t(n) - 4) * (t(n) > -1)).to(getattr(torch, gtype)).cuda() for n in sizes] for _ in range(3)]
    return params, grads


@pytest.mark.parametrize("ptype,gtype", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float16"),
                                         ("float32", "bfloat16"), ("bfloat16", "float32"), ("float16", "bfloat16")])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_bit_for_bit(bits, ptype, gtype):
    import torch
    from splatx_cuda.network import AdamW
    params, grads = _tensors(bits, ptype, gtype)
    opt = AdamW(params, state_bits=bits, **CFG)
    P = [_np(p) for p in params]
    M, V = [np.zeros_like(p) for p in P], [np.zeros_like(p) for p in P]
    for t in range(3):
        opt.step(grads[t], grad_scale=0.5)
        st = opt.state()
        assert st["step"] == t + 1
        for i, p in enumerate(params):
            new, m, v = _numpy_step(P[i], _np(grads[t][i]), M[i], V[i], t + 1, 0.5)
            P[i] = _round_to(new, p.dtype)
            assert np.array_equal(_np(p), P[i]), (t, i)
            if bits == 32:
                M[i], V[i] = m, v
                assert np.array_equal(_np(st["exp_avg"][i]), m) and np.array_equal(_np(st["exp_avg_sq"][i]), v)
                continue
            for key, x, keep in (("exp_avg", m, False), ("exp_avg_sq", np.sqrt(v), True)):
                codes, scale = _pack(x, keep)
                assert np.array_equal(_np(st[key][i]), codes.float().numpy()), (key, t, i)
                assert np.array_equal(_np(st[key + "_scale"][i]), scale), (key, t, i)
            M[i] = _unpack(st["exp_avg"][i], _np(st["exp_avg_scale"][i]))
            root = _unpack(st["exp_avg_sq"][i], _np(st["exp_avg_sq_scale"][i]))
            V[i] = root * root
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_bit_for_bit_over_all_magnitudes(bits):
    """Four million gradients from 2^-70 to 2^60, and values beyond both ends of what the kernel's own
    root and quotient are made for: every root and quotient is the rounded one (a quotient may be off
    in its last bit where its residual is below 2^-126: the gradients here keep above that)."""
    import torch
    from splatx_cuda.network import AdamW
    n = 1 << 22
    rng = np.random.default_rng(bits)
    g = (rng.standard_normal(n) * 2.0 ** rng.uniform(-40, 45, n)).astype(F)
    g[: n // 8] = 0
    g[n // 8: n // 4] = (rng.standard_normal(n // 8) * 2.0 ** np.repeat(rng.uniform(-62, 60, n // 8 // 256), 256)).astype(F)
    p = torch.zeros(n, device="cuda")
    opt = AdamW([p], state_bits=bits, **CFG)
    opt.step([torch.from_numpy(g).cuda()])
    new, m, v = _numpy_step(np.zeros(n, F), g, np.zeros(n, F), np.zeros(n, F), 1)
    assert np.array_equal(_np(p), new)
    st = opt.state()
    if bits == 32:
        assert np.array_equal(_np(st["exp_avg"][0]), m) and np.array_equal(_np(st["exp_avg_sq"][0]), v)
    else:
        codes, scale = _pack(np.sqrt(v), True)
        assert np.array_equal(_np(st["exp_avg_sq"][0]), codes.float().numpy())
        assert np.array_equal(_np(st["exp_avg_sq_scale"][0]), scale)


def test_adamw_against_64_bits():
    """Twenty operations of relative error 2^-24 each, against the formula's value and its terms."""
    from splatx_cuda.network import AdamW
    params, grads = _tensors(5, "float32", "float32", [5000])
    opt = AdamW(params, **CFG)
    p, m, v = _np(params[0]).astype(np.float64), 0.0, 0.0
    (b1, b2), lr = CFG["betas"], CFG["lr"]
    for t in range(3):
        opt.step(grads[t])
        g = _np(grads[t][0]).astype(np.float64)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        move = lr * m / (1 - b1 ** (t + 1)) / (np.sqrt(v / (1 - b2 ** (t + 1))) + CFG["eps"])
        p = p * (1 - lr * CFG["weight_decay"]) - move
    # m's terms can cancel: its error is against their size
    assert np.all(np.abs(_np(params[0]) - p) <= 3 * 20 * 2.0 ** -24 * (np.abs(p) + 10 * lr))


def test_adamw_groups_missing_gradients_and_rates():
    import torch
    from splatx_cuda.network import AdamW
    a, b, c = (torch.randn(n, device="cuda", requires_grad=True) for n in (300, 20, 7))
    was = [_np(t) for t in (a, b, c)]
    opt = AdamW([{"params": [a], "lr": 0.1, "weight_decay": 0.0}, {"params": [b, c]}], **CFG)
    a.grad, c.grad = torch.randn_like(a), torch.randn_like(c)
    version = a._version
    opt.step()
    assert a._version >= version and np.array_equal(_np(b), was[1])
    zero = [np.zeros_like(w) for w in was]
    assert np.array_equal(_np(a), _numpy_step(was[0], _np(a.grad), zero[0], zero[0], 1, lr=0.1, decay=0.0)[0])
    assert np.array_equal(_np(c), _numpy_step(was[2], _np(c.grad), zero[2], zero[2], 1)[0])
    opt.set_lr(0.0)
    was = [_np(t) for t in (a, b, c)]
    opt.step()
    assert all(np.array_equal(_np(t), w) for t, w in zip((a, b, c), was))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_many_tensors_unaligned_and_resumed(bits):
    """More tensors than one launch takes, some at odd offsets of a shared buffer; a second optimiser
    that goes on from the first one's state takes the same step."""
    import torch
    from splatx_cuda.network import AdamW
    g = torch.Generator().manual_seed(1)
    flat, gflat = (torch.randn(60000, generator=g).cuda() for _ in range(2))
    cuts = np.sort(np.random.default_rng(0).choice(np.arange(1, 60000), 900, replace=False))
    edges = list(zip([0, *cuts], [*cuts, 60000]))
    params, grads = [flat[i:j] for i, j in edges], [gflat[i:j] for i, j in edges]
    opt = AdamW(params, state_bits=bits, **CFG)
    opt.step(grads)
    if bits == 32:
        zero = np.zeros(60000, F)
        want = _numpy_step(_np(torch.randn(60000, generator=torch.Generator().manual_seed(1))), _np(gflat), zero, zero, 1)[0]
        assert np.array_equal(_np(flat), want)
    copy = flat.clone()
    state = {k: v if k == "step" else [t.clone() for t in v] for k, v in opt.state().items()}
    other = AdamW([copy[i:j] for i, j in edges], state_bits=bits, state=state, **CFG)
    opt.step(grads)
    other.step(grads)
    assert torch.equal(flat, copy)
    for k, v in opt.state().items():
        assert v == other.state()[k] if k == "step" else all(
            torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(v, other.state()[k]))


def test_adamw8_long_tail_and_zeros():
    """Second moments over 12 decades in one run: none that is above zero becomes zero, and weights
    whose gradient stops go on moving by less than the learning rate. A run without gradients stays
    exactly as it is (no decay)."""
    import torch
    from splatx_cuda.network import AdamW
    p = torch.zeros(512, device="cuda")
    g = torch.zeros(512, device="cuda")
    g[:256] = 10.0 ** torch.linspace(-12, 0, 256)
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=8)
    opt.step([g])
    st = opt.state()
    assert bool((st["exp_avg_sq"][0].float()[:256] > 0).all())
    assert not p[256:].any() and float(st["exp_avg_scale"][0][1]) == 0.0
    for _ in range(20):
        was = p.clone()
        opt.step([torch.zeros_like(g)])
        assert float((p - was).abs().max()) <= 1e-2
    assert bool(torch.isfinite(p).all())


def test_adamw_follows_the_32_bit_moments():
    """A quadratic bowl: with 8-bit moments the loss falls as with 32-bit ones."""
    import torch
    from splatx_cuda.network import AdamW
    target = torch.randn(3000, generator=torch.Generator().manual_seed(0)).cuda()
    last = {}
    for bits in (32, 8):
        p = torch.zeros(3000, device="cuda")
        opt = AdamW([p], lr=2e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(300):
            opt.step([2 * (p - target)])
        last[bits] = float(((p - target) ** 2).mean())
    assert last[32] < 1e-2 and last[8] < 2e-2, last


def test_adamw_parameters_given_other_memory():
    """A parameter whose data moves between steps is updated where it is then; one that changes its
    size or type is refused."""
    import torch
    from splatx_cuda.network import AdamW
    p = torch.nn.Parameter(torch.randn(500, device="cuda"))
    g = torch.randn(500, device="cuda")
    opt = AdamW([p], **CFG)
    opt.step([g])
    was, old = _np(p), p.data
    kept = old.clone()
    p.data = old.clone()
    opt.step([g])
    assert torch.equal(old, kept) and not np.array_equal(_np(p), was)
    for bad in (torch.randn(499, device="cuda"), torch.randn(500, device="cuda").half(), torch.randn(500, 2, device="cuda")[:, 0]):
        p.data = bad
        with pytest.raises(ValueError):
            opt.step([torch.randn_like(bad).contiguous()])


def test_adamw_refusals():
    import ctypes as C
    import torch
    from splatx_cuda import _native as n
    from splatx_cuda.network import AdamW
    p = torch.zeros(8, 4, device="cuda")
    ok = AdamW([p])
    for f in (lambda: AdamW([]), lambda: AdamW([p.cpu()]), lambda: AdamW([p.t()]), lambda: AdamW([p.double()]),
              lambda: AdamW([p], state_bits=16), lambda: AdamW([p], state={"step": 1}),
              lambda: AdamW([p], state={"step": 0, "exp_avg": [p[0]], "exp_avg_sq": [p]}),
              lambda: ok.step([]), lambda: ok.step([p.view(-1)]), lambda: ok.step([p.cpu()]),
              lambda: ok.step([p.t().contiguous().t()]), lambda: ok.step([p.double()]),
              lambda: AdamW([p], betas=(1.0, 0.9)).step([p]), lambda: AdamW([p], eps=-1.0).step([p]),
              lambda: AdamW([p], lr=math.inf).step([p]), lambda: ok.step([p], grad_scale=math.nan)):
        with pytest.raises(ValueError):
            f()
    assert ok.state()["step"] == 0
    L = n.lib()
    cfg = n.SxAdamwConfig(0.9, 0.99, 1e-8, 1.0, 1, 32)
    t = n.SxAdamwTensor(p.data_ptr(), p.data_ptr(), p.data_ptr(), p.data_ptr(), None, None, 32, 0.0, 0.0, 0, 0)
    step = lambda cfg=cfg, t=t, k=1: L.sxcuda_adamw_step(C.byref(t) if t else None, k, C.byref(cfg) if cfg else None, None)  # noqa: E731
    def with_(s, **kw):
        c = type(s).from_buffer_copy(s)
        for k, v in kw.items():
            setattr(c, k, v)
        return c
    got = [step(cfg=None), step(t=None), step(k=-1), step(cfg=with_(cfg, step=0)), step(cfg=with_(cfg, state_bits=4)),
           step(cfg=with_(cfg, state_bits=8)), step(t=with_(t, n=-1)), step(t=with_(t, param=None)),
           step(t=with_(t, grad=p.data_ptr() + 2)), step(t=with_(t, grad_dtype=3)), step(t=with_(t, exp_avg=None))]
    assert got == [n.SXCUDA_EINVAL] * len(got), got
    assert L.sxcuda_adamw_step(None, 0, C.byref(cfg), None) == n.SXCUDA_OK
    torch.cuda.synchronize()
    assert not p.any()


def test_adamw_refuses_a_parameter_given_twice():
    import torch
    from splatx_cuda.network import AdamW
    p, empty = torch.zeros(8, device="cuda"), torch.zeros(0, device="cuda")
    with pytest.raises(ValueError):
        AdamW([p, p])
    with pytest.raises(ValueError):
        AdamW([{"params": [p]}, {"params": [p.view(2, 4)]}])
    AdamW([p, empty, empty])


def test_adamw_step_shows_to_autograd():
    """A graph that saved a parameter's value must not run backward on the updated one."""
    import torch
    from splatx_cuda.network import AdamW
    p, kept = (torch.ones(8, device="cuda", requires_grad=True) for _ in range(2))
    lost, fine = (p * p).sum(), (kept * kept).sum()
    AdamW([p, kept], **CFG).step([torch.ones_like(p), None])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lost.backward()
    fine.backward()
    assert kept.grad.eq(2).all()


def test_second_derivatives_are_refused():
    import torch
    from splatx_cuda import network
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(network.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    q = torch.randn(1, 4, 2, 16, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(network.attention(q, q, q).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
