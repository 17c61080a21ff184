"""What the linear layers and the norm and rotation of queries and keys refuse before they reach a device."""
import ctypes as C
import math

import pytest
import torch

from splatx_cuda import _native as n, network


def test_linear_refuses():
    x, w, b = torch.zeros(4, 16), torch.zeros(8, 16), torch.zeros(8)
    for f in (lambda: network.linear_fwd(x, w, activation="tanh"), lambda: network.linear_fwd(x, w[:, :8]),
              lambda: network.linear_fwd(x, w[0]), lambda: network.linear_fwd(x, w.half()), lambda: network.linear_fwd(x[:, :0], w[:, :0]),
              lambda: network.linear_fwd(x.double(), w.double()), lambda: network.linear_fwd(x, w, b[:5]),
              lambda: network.linear_fwd(x, w, b), lambda: network.linear_fwd(torch.zeros(()), w)):
        with pytest.raises(ValueError):
            f()


def test_rotary_refuses():
    q, k, pos = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16), torch.zeros(2, 5, 2)
    fwd = network.qk_norm_rotary_fwd
    for f in (lambda: fwd(q[0], k, pos, axes=(8, 8)), lambda: fwd(q, k[:, :4], pos, axes=(8, 8)), lambda: fwd(q, k.half(), pos, axes=(8, 8)),
              lambda: fwd(q, k[..., :8], pos, axes=(8, 8)), lambda: fwd(q, k, pos, axes=(8, 10)), lambda: fwd(q, k, pos, axes=(7, 8)),
              lambda: fwd(q, k, pos, axes=(8, -2)), lambda: fwd(q, k, pos, axes=()), lambda: fwd(q, k, pos, axes=(2, 2, 2, 2, 2)),
              lambda: fwd(q, k, pos, axes=(8,)), lambda: fwd(q, k, pos[:1], axes=(8, 8)), lambda: fwd(q, k, pos.double(), axes=(8, 8)),
              lambda: fwd(q, k, pos, axes=(8, 8), pairs="halves"), lambda: fwd(q, k, pos, axes=(8, 8), base=0.0),
              lambda: fwd(q, k, pos, axes=(8, 8), base=math.nan), lambda: fwd(q, k, pos, axes=(8, 8), freqs=[1.0]),
              lambda: fwd(q, None, pos, axes=(8, 8), k_weight=torch.ones(16)), lambda: fwd(q, k, pos, axes=(8, 8), q_weight=torch.ones(8)),
              lambda: fwd(q, k, pos, axes=(8, 8), norm=False, q_weight=torch.ones(16)),
              lambda: fwd(q, k, pos, axes=(8, 8), q_weight=torch.ones(16), k_weight=torch.ones(16).half()),
              lambda: fwd(q, k, pos, axes=(8, 8))):
        with pytest.raises(ValueError):
            f()


def _with(s, **kw):
    t = type(s).from_buffer_copy(s)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.fixture
def lib():
    if not n.library_path().exists():
        pytest.skip("library not built")
    return n.lib()


AT = 1 << 20  # an address that nothing reads: every call here is refused


def test_linear_entry_refuses(lib):
    ok = n.SxLinearInputs(AT, AT, AT, 4, 16, 8, 16, 16, 2, 0, 3)
    out = n.SxLinearOutputs(AT, 8, AT, 8, AT, 8)
    nbytes = C.c_size_t(1 << 30)
    fwd = lambda i=ok, o=out, ws=AT: lib.sxcuda_linear_fwd(C.byref(i) if i else None, C.byref(o) if o else None, ws, C.byref(nbytes), None)  # noqa: E731
    bad = [dict(x=None), dict(weight=None), dict(x=AT + 1), dict(weight=AT + 1), dict(bias=AT + 2), dict(rows=-1), dict(rows=1 << 30),
           dict(in_features=0), dict(out_features=0), dict(in_features=1 << 30), dict(x_stride=15), dict(weight_stride=15),
           dict(dtype=3), dict(bias_dtype=-1), dict(activation=5), dict(activation=-1)]
    assert [fwd(_with(ok, **b)) for b in bad] == [n.SXCUDA_EINVAL] * len(bad)
    assert fwd(None) == n.SXCUDA_EINVAL
    gin, gout = n.SxLinearGradsIn(AT, 8, AT, 8), n.SxLinearGrads(AT, 16, AT, 16, AT)
    bwd = lambda i=ok, g=gin, o=gout: lib.sxcuda_linear_bwd(C.byref(i), C.byref(g) if g else None, C.byref(o) if o else None, AT, C.byref(nbytes), None)  # noqa: E731
    got = [bwd(_with(ok, **b)) for b in bad]
    got += [bwd(g=None), bwd(o=None), bwd(g=_with(gin, v_y=None)), bwd(g=_with(gin, v_y_stride=7)), bwd(g=_with(gin, pre=None)),
            bwd(_with(ok, activation=0)), bwd(g=_with(gin, pre_stride=7)), bwd(o=_with(gout, v_x=AT + 1)),
            bwd(o=_with(gout, v_x_stride=15)), bwd(o=_with(gout, v_weight_stride=15)), bwd(o=_with(gout, v_bias=AT + 2))]
    assert got == [n.SXCUDA_EINVAL] * len(got), got
    assert lib.sxcuda_linear_status(None) == n.SXCUDA_EINVAL


def test_rotary_entry_refuses(lib):
    freqs = (C.c_double * 8)(*[1.0] * 8)
    view = n.SxAttentionView(AT, 5 * 64, 64, 16)
    ok = n.SxRotaryInputs(view, view, AT, 10, 2, 1, C.addressof(freqs), AT, AT, 2, 5, 4, 4, 16, 2, (C.c_int32 * 4)(8, 8), 0, 0, 0, 0, 1, 1e-6)
    nbytes = C.c_size_t(1 << 30)
    fwd = lambda i=ok, q=view, k=view: lib.sxcuda_qk_norm_rotary_fwd(C.byref(i) if i else None, C.byref(q) if q else None, C.byref(k) if k else None, None)  # noqa: E731
    bad_view = [_with(view, data=None), _with(view, data=AT + 2), _with(view, token_stride=-1)]
    overlap = [_with(view, head_stride=8), _with(view, token_stride=0), _with(view, batch_stride=0)]
    inf = (C.c_double * 8)(*[math.inf] * 8)
    bad = [dict(positions=None), dict(positions=AT + 2), dict(pos_token_stride=-1), dict(freqs=None), dict(freqs=C.addressof(inf)),
           dict(q_weight=AT + 2), dict(batch=-1), dict(tokens=-1), dict(q_heads=0), dict(k_heads=-1), dict(head_dim=0),
           dict(head_dim=257), dict(head_dim=15), dict(axes=0), dict(axes=5), dict(axis_dims=(C.c_int32 * 4)(7, 8)),
           dict(axis_dims=(C.c_int32 * 4)(-2, 8)), dict(pairs=3), dict(dtype=3), dict(param_dtype=3), dict(pos_dtype=3),
           dict(norm=2), dict(norm=0), dict(eps=-1.0), dict(eps=math.nan), *[dict(q=v) for v in bad_view], *[dict(k=v) for v in bad_view]]
    got = [fwd(_with(ok, **b)) for b in bad] + [fwd(None), fwd(q=None), fwd(k=None)]
    got += [fwd(q=v) for v in bad_view + overlap] + [fwd(k=v) for v in bad_view + overlap]
    assert got == [n.SXCUDA_EINVAL] * len(got), got
    grads = n.SxRotaryGrads(view, view, view, view, AT, AT)
    bwd = lambda i=ok, g=grads: lib.sxcuda_qk_norm_rotary_bwd(C.byref(i), C.byref(g) if g else None, AT, C.byref(nbytes), None)  # noqa: E731
    got = [bwd(_with(ok, **b)) for b in bad]
    assert got == [n.SXCUDA_EINVAL] * len(got), got
