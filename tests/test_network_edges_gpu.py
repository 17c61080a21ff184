"""Linear layers and the rotation where a call's plan, a value that is not finite or a caller's own list must not
decide the answer."""
import math

import pytest

pytestmark = pytest.mark.gpu


# one row and few rows; tiles that are cut along K; whole tiles; results that copies do not reach, cut and whole
PLANS = [(1, 64, 32), (4, 4096, 40), (5, 4096, 32), (300, 4096, 256), (300, 64, 256), (40, 64, 101), (40, 4096, 101),
         (5, 64, 32)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
def test_infinite_pre_activations_in_every_plan(act, dtype):
    """z of -inf gives the limit of relu and gelu and NaN of what is inf / inf, +inf and NaN stay, whichever kernel
    ends the call; the other columns are what they are without them."""
    import torch
    from splatx_cuda import network
    T = getattr(torch, dtype)
    below = {None: -math.inf, "relu": 0.0, "gelu": 0.0}.get(act, math.nan)
    for m, k, n in PLANS:
        gen = torch.Generator().manual_seed(m + k)
        x, w = torch.randn(m, k, generator=gen).to(T).cuda(), (torch.randn(n, k, generator=gen) * k ** -0.5).to(T).cuda()
        b = torch.zeros(n, device="cuda")
        want = network.linear_fwd(x, w, b, activation=act)[0]
        b[3], b[8], b[n - 1] = -math.inf, math.inf, math.nan
        y, pre = network.linear_fwd(x, w, b, activation=act, keep=True)
        assert bool((pre[:, 3] == -math.inf).all()) and bool((pre[:, 8] == math.inf).all()) and bool(pre[:, n - 1].isnan().all())
        assert bool(y[:, 3].isnan().all() if math.isnan(below) else (y[:, 3] == below).all()), (m, k, n)
        assert bool((y[:, 8] == math.inf).all()) and bool(y[:, n - 1].isnan().all()), (m, k, n)
        others = [i for i in range(n) if i not in (3, 8, n - 1)]
        assert torch.equal(y[:, others], want[:, others]), (m, k, n)


# the last values of a head are not rotated: 16-byte accesses of 8, 4 and 2 pairs, and value by value
@pytest.mark.parametrize("pairs", ["axis", "whole", "neighbours"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("dim, axes", [(64, (16, 16)), (64, (24, 16)), (48, (20, 20)), (40, (2, 4)), (37, (8, 6))])
def test_values_that_are_not_rotated_pass(dim, axes, dtype, pairs):
    """Without norm a NaN or an infinity among them is nobody else's, forward and backward; with norm an infinity makes
    the others 0 and itself NaN."""
    import torch
    from splatx_cuda import network
    T, rotated = getattr(torch, dtype), sum(axes)
    gen = torch.Generator().manual_seed(dim)
    x = torch.randn(2, 9, 3, dim, generator=gen).to(T).cuda()
    pos = (torch.rand(2, 9, 2, generator=gen) * 100).cuda()
    how = {"axes": axes, "pairs": pairs}
    turn = lambda t, **kw: network.qk_norm_rotary_fwd(t, None, pos, **how, **kw)[0]  # noqa: E731
    back = lambda t: network.qk_norm_rotary_bwd(t, None, x, None, pos, **how, norm=False)[0]  # noqa: E731
    for value in (math.nan, math.inf, -math.inf):
        for at in range(rotated, dim):
            bad = x.clone()
            bad[1, 4, 2, at] = value
            for f in (lambda t: turn(t, norm=False), back):
                got, want = f(bad), f(x)
                assert torch.equal(want[..., rotated:], x[..., rotated:])
                want[1, 4, 2, at] = value
                assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0)), (value, at)
            if value == math.inf:
                got, want = turn(bad), turn(x)
                want[1, 4, 2], want[1, 4, 2, at] = 0.0, math.nan
                assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), at


def test_gelu_in_float32_over_its_tail():
    """z Phi(z) relative to its value as far as that is a normal number. In units of 2^-24: the reciprocal and its
    argument 2, with the polynomial after them 2 more, CUDA's exponential 4 (2 ulp), the lost part of z^2, the three
    products and the fit 4.2, with z 1: 14 of 16. And Phi's own slope beside the largest and infinite z."""
    import torch
    from splatx_cuda import network
    z = torch.cat([torch.linspace(-12.9, 12.9, 200_001, dtype=torch.float64), -torch.logspace(-30, 1.1, 5000, dtype=torch.float64)])
    z = z.float().cuda()[:, None]
    one = torch.ones(1, 1, device="cuda")
    y, pre = network.linear_fwd(z, one, activation="gelu", keep=True)
    assert torch.equal(pre, z)
    want = z.double() * 0.5 * torch.special.erfc(-z.double() / math.sqrt(2))
    off = (y.double() - want).abs() / want.abs().clamp(min=2.0 ** -126)
    assert float(off.max()) <= 2.0 ** -20, (float(off.max()), float(z[off.argmax()]))
    far = torch.tensor([[14.0], [1e10], [3e38], [math.inf], [-20.0], [-1e10], [-3e38]], device="cuda").repeat(3, 1)  # more than a few rows
    y = network.linear_fwd(far, one, activation="gelu")[0]
    assert torch.equal(y, far.clamp(min=0.0))
    v_b = network.linear_bwd(torch.ones(1, 1, device="cuda"), far[:1], one, one[0], far[3:4], activation="gelu")[2]
    assert float(v_b) == 1.0


def test_far_positions():
    """An angle is off by 2^-28 of a turn and by the series and their roundings (2^-22), however far the position: up to
    2^76 turns. From 2^80 on it is 0, and what is not finite stays NaN."""
    import torch
    from decimal import Decimal, getcontext
    from splatx_cuda import network
    getcontext().prec = 100
    tau = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
    whole = [0, 1, -1, 7, 1 << 20, (1 << 30) - 1, -(1 << 33) + 5, (1 << 40) + 3, (1 << 46) + 1, -(1 << 48) + 1, (1 << 51) - 1,
             *[(1 << 52) + i for i in range(7)], 1 << 53, -(1 << 53) - 2, 1 << 60, -(1 << 62) - 4096]
    real = torch.tensor([0.3, 1e5 / 3, -2.0 ** 52 * 1.5, 2.0 ** 53 * 1.25, -2.0 ** 54, 1e20, -3e22]).tolist()  # as float32 has them
    freqs = [1.0, 0.1, 10000.0 ** -0.25, 3.7]
    for positions, dtype in ((whole, torch.int64), (real, torch.float32)):
        n = len(positions)
        x = torch.tensor([1.0, 0.0]).repeat(n, 4)[None, :, None].cuda()
        y = network.qk_norm_rotary_fwd(x, None, torch.tensor(positions, dtype=dtype)[:, None].cuda(), axes=(8,), freqs=freqs,
                                       pairs="neighbours", norm=False)[0]
        for p, row in zip(positions, y[0, :, 0].view(n, 4, 2).tolist()):
            for f, (c, s) in zip(freqs, row):
                turns = Decimal(p) * Decimal(f) / tau
                rest = 2 * math.pi * float(turns - turns.to_integral_value())
                bound = 2 * math.pi * 2.0 ** -28 + 2.0 ** -22
                assert abs(c - math.cos(rest)) <= bound and abs(s - math.sin(rest)) <= bound, (p, f, c, s)
    x = torch.randn(1, 4, 3, 8, generator=torch.Generator().manual_seed(1)).cuda()
    y = network.qk_norm_rotary_fwd(x, None, torch.tensor([[1e26], [-1e30], [3e38], [-2e38]], device="cuda"), axes=(8,),
                                   freqs=[1.0, 2.0, 1e100, 1e300], norm=False)[0]
    assert torch.equal(y, x)
    for p in (math.inf, -math.inf, math.nan):
        y = network.qk_norm_rotary_fwd(x, None, torch.full((4, 1), p, device="cuda"), axes=(4,), norm=False)[0]
        assert bool(y[..., :4].isnan().all()) and torch.equal(y[..., 4:], x[..., 4:])


@pytest.mark.parametrize("rows", [0, 1, 7, 300])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_one_row_may_have_any_stride(dtype, rows):
    """At the C entry: a weight and its gradient of one row, and x, v_y and their like of one, are not asked for a stride."""
    import ctypes as C
    import torch
    from splatx_cuda import _native as n, network
    k, o, code = 72, 1, {"bfloat16": 2, "float32": 0}[dtype]
    gen = torch.Generator().manual_seed(rows)
    x, w, g = (torch.randn(s, generator=gen).to(getattr(torch, dtype)).cuda() for s in ((rows, k), (o, k), (rows, o)))
    b = torch.ones(o, device="cuda")
    y, pre = network.linear_fwd(x, w, b, activation="silu", keep=True)
    want = (y, pre, *network.linear_bwd(g, x, w, b, pre, activation="silu"))
    got = [torch.full_like(t, 7.0) for t in want]
    y, pre, v_x, v_w, v_b = got
    x_stride, y_stride = (0, 0) if rows <= 1 else (k, o)
    ins = n.SxLinearInputs(x.data_ptr(), w.data_ptr(), b.data_ptr(), rows, k, o, x_stride, 0, code, 0, 2)
    stream = torch.cuda.current_stream().cuda_stream
    for entry, args in ((n.lib().sxcuda_linear_fwd, (n.SxLinearOutputs(None, 0, y.data_ptr(), y_stride, pre.data_ptr(), y_stride),)),
                        (n.lib().sxcuda_linear_bwd, (n.SxLinearGradsIn(g.data_ptr(), y_stride, want[1].data_ptr(), y_stride),
                                                     n.SxLinearGrads(v_x.data_ptr(), x_stride, v_w.data_ptr(), 0, v_b.data_ptr())))):
        nbytes, args = C.c_size_t(0), [C.byref(a) for a in (ins, *args)]
        n.check(entry(*args, None, C.byref(nbytes), None))
        ws = torch.empty(max(nbytes.value, 32), dtype=torch.uint8, device="cuda")
        n.check(entry(*args, ws.data_ptr(), C.byref(nbytes), stream))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [(300, 72, 101), (300, 4096, 101), (5, 72, 333), (131, 64, 3)], ids=lambda s: "x".join(map(str, s)))
def test_copies_end_with_the_row(size, dtype):
    """At the C entry: rows of an odd length on a start and a pitch that copies reach. They must end inside 16 bytes and
    leave what is behind the row, and read a residual as far as its row."""
    import ctypes as C
    import torch
    from splatx_cuda import _native as n, network
    m, k, o = size
    gen = torch.Generator().manual_seed(o)
    T, code = getattr(torch, dtype), {"float16": 1, "bfloat16": 2}[dtype]
    x, w, r = (torch.randn(s, generator=gen).to(T).cuda() for s in ((m, k), (o, k), (m, o)))
    b = torch.randn(o, generator=gen).cuda()
    pitch, first = (o + 15) // 8 * 8, 8
    for residual in (False, True):
        want, want_pre = network.linear_fwd(x, w, b, activation="gelu", residual=r if residual else None, keep=True)
        y, pre, add = (torch.full((m + 2, pitch), 7.0, dtype=T, device="cuda") for _ in range(3))
        inner = lambda t: torch.as_strided(t, (m, o), (pitch, 1), pitch + first)  # noqa: E731
        add.fill_(math.nan)
        inner(add).copy_(r)
        at = [t.data_ptr() + (pitch + first) * 2 for t in (y, pre, add)]
        assert not any(p % 16 for p in at)
        ins = n.SxLinearInputs(x.data_ptr(), w.data_ptr(), b.data_ptr(), m, k, o, k, k, code, 0, 3)
        outs = n.SxLinearOutputs(at[2] if residual else None, pitch, at[0], pitch, at[1], pitch)
        nbytes, entry = C.c_size_t(0), n.lib().sxcuda_linear_fwd
        n.check(entry(C.byref(ins), C.byref(outs), None, C.byref(nbytes), None))
        ws = torch.empty(max(nbytes.value, 32), dtype=torch.uint8, device="cuda")
        n.check(entry(C.byref(ins), C.byref(outs), ws.data_ptr(), C.byref(nbytes), torch.cuda.current_stream().cuda_stream))
        for t, v in ((y, want), (pre, want_pre)):
            assert torch.equal(inner(t), v)
            inner(t).fill_(7.0)
            assert bool((t == 7.0).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [(1, 101, 72), (300, 101, 1), (300, 101, 72), (4000, 333, 40)], ids=lambda s: "x".join(map(str, s)))
def test_gradient_copies_end_with_the_row(size, dtype):
    """The same of v_x and v_weight, one row of them among the cases, which any pitch is good for."""
    import ctypes as C
    import torch
    from splatx_cuda import _native as n, network
    m, k, o = size
    gen = torch.Generator().manual_seed(m + o)
    T, code = getattr(torch, dtype), {"float16": 1, "bfloat16": 2}[dtype]
    x, w, g = (torch.randn(s, generator=gen).to(T).cuda() for s in ((m, k), (o, k), (m, o)))
    want = network.linear_bwd(g, x, w)[:2]
    pitch = (k + 15) // 8 * 8
    got = [torch.full((rows + 2, pitch), 7.0, dtype=T, device="cuda") for rows in (m, o)]
    at = [t.data_ptr() + (pitch + 8) * 2 for t in got]
    ins = n.SxLinearInputs(x.data_ptr(), w.data_ptr(), None, m, k, o, k, k, code, 0, 0)
    gin, out = n.SxLinearGradsIn(g.data_ptr(), o, None, 0), n.SxLinearGrads(at[0], pitch, at[1], pitch, None)
    nbytes, entry = C.c_size_t(0), n.lib().sxcuda_linear_bwd
    n.check(entry(C.byref(ins), C.byref(gin), C.byref(out), None, C.byref(nbytes), None))
    ws = torch.empty(max(nbytes.value, 32), dtype=torch.uint8, device="cuda")
    n.check(entry(C.byref(ins), C.byref(gin), C.byref(out), ws.data_ptr(), C.byref(nbytes), torch.cuda.current_stream().cuda_stream))
    for t, v in zip(got, want):
        rows = torch.as_strided(t, v.shape, (pitch, 1), pitch + 8)
        assert torch.equal(rows, v)
        rows.fill_(7.0)
        assert bool((t == 7.0).all())
