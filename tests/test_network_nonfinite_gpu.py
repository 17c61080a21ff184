"""Attention where what a query sees is not finite.

softmax of scores among which one is NaN or +inf, or of which all are -inf, is NaN, and so is its
log-sum and every gradient that such a row takes part in. Only a query that sees no key has output 0
and log-sum -inf. A key that a query does not see has weight 0, whatever its finite value. Rows that see
only finite scores keep the definition's values, within the bounds of test_network_attention_gpu.
"""
import math

import pytest

from test_network_attention_gpu import ROUND, _check, _definition, _inputs, _seen

pytestmark = pytest.mark.gpu

NAN, INF = math.nan, math.inf
# columns of every kind that a tile of scores has: one batch entry for each
AT = [*range(0, 32), *range(64, 96)]
_name = lambda s: "x".join(map(str, s))  # noqa: E731


def _fwd_bwd(q, k, v, g, **how):
    from splatx_cuda import network
    out, lse = network.attention_fwd(q, k, v, **how)
    return out, lse, network.attention_bwd(g, q, k, v, out, lse, **how)


def _all_nan(**results):
    """Of each result every value, in every batch entry."""
    for name, t in results.items():
        assert bool(t.isnan().all()), (name, [b for b in range(len(t)) if not t[b].isnan().all()])


def _nan_queries(shape, causal, dtype):
    """Some queries are NaN: their rows are NaN and the others as they were."""
    from splatx_cuda import network
    q, k, v, g = _inputs(sum(shape), *shape, dtype)
    lq = shape[1]
    rows = sorted({0, lq // 3, lq - 1})
    clean = q.clone()
    q[:, rows] = NAN
    out, lse = network.attention_fwd(q, k, v, causal=causal)
    _all_nan(out=out[:, rows], lse=lse[:, :, rows])
    seen = _seen(shape[0], lq, shape[2], causal, None, None)
    want = _definition(clean, k, v, g, None, seen, shape[5] ** -0.5, ROUND[dtype])
    fine = [i for i in range(lq) if i not in rows]
    _check("out", out.transpose(1, 2)[:, :, fine], *(t[:, :, fine] for t in want["out"]))
    _check("lse", lse[:, :, fine], *(t[:, :, fine] for t in want["lse"]))


def _key_at_every_place(value, d, lk, dtype):
    """Batch entry i has `value` at key AT[i]: every row and every gradient is NaN. (The first value of
    each query is 1, so that with +inf the score is +inf.)"""
    q, k, v, g = _inputs(d + lk, len(AT), 40, lk, 2, 1, d, dtype)
    q[..., 0] = 1
    for b, at in enumerate(AT):
        k[b, at, :, 0] = value
    out, lse, (v_q, v_k, v_v) = _fwd_bwd(q, k, v, g)
    _all_nan(out=out, lse=lse, v_q=v_q, v_k=v_k, v_v=v_v)


def _query_in_the_keys_gradients(d, dtype):
    """Batch entry i has NaN at query AT[i]; the other queries' own gradients stay finite."""
    q, k, v, g = _inputs(d, len(AT), 96, 140, 2, 1, d, dtype)
    for b, at in enumerate(AT):
        q[b, at] = NAN
    _, _, (v_q, v_k, v_v) = _fwd_bwd(q, k, v, g)
    _all_nan(v_k=v_k, v_v=v_v)
    bad = v_q.isnan().flatten(2)
    for b, at in enumerate(AT):
        assert bool(bad[b, at].all()) and int(bad[b].any(1).sum()) == 1, at


# the kernels without tensor cores: 32 bits, and rows that are not in pieces of 16 bytes
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape,dtype", [((2, 96, 96, 2, 2, 64), "float32"), ((1, 300, 300, 2, 1, 128), "float32"),
                                         ((2, 1, 900, 4, 4, 128), "float32"), ((1, 90, 90, 2, 2, 36), "bfloat16"),
                                         ((1, 90, 90, 2, 2, 33), "float16")])
def test_cuda_core_kernels_keep_a_nan_query(shape, dtype, causal):
    _nan_queries(shape, causal, dtype)


@pytest.mark.parametrize("d,dtype", [(64, "float32"), (128, "float32"), (36, "bfloat16")])
def test_cuda_core_kernels_keep_what_is_not_finite_at_every_place(d, dtype):
    _key_at_every_place(NAN, d, 96, dtype)
    _key_at_every_place(INF, d, 300, dtype)
    _query_in_the_keys_gradients(d, dtype)


# tensor cores: the first key tile whole, partly behind the mask or the length; several tiles
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(2, 96, 96, 2, 2, 64), (2, 96, 96, 2, 2, 128), (40, 300, 300, 4, 2, 128),
                                   (40, 300, 300, 4, 2, 64), (1, 128, 128, 1, 1, 80)], ids=_name)
def test_a_nan_query_is_nan_and_alone(shape, causal, dtype):
    _nan_queries(shape, causal, dtype)


@pytest.mark.parametrize("dtype,large", [("bfloat16", 3e38), ("float16", 6e4), ("float32", 3e38)])
@pytest.mark.parametrize("d", [64, 128])
def test_an_unseen_key_has_weight_zero_at_every_place(d, dtype, large):
    """Batch entry i has large values at key AT[i]: the rows before it, which do not see it in the
    causal square, do not change by a bit."""
    import torch
    from splatx_cuda import network
    q, k, v, _ = _inputs(d, len(AT), 128, 128, 2, 1, d, dtype)
    out, lse = network.attention_fwd(q, k, v, causal=True)
    for b, at in enumerate(AT):
        v[b, at] = large
    again, lse2 = network.attention_fwd(q, k, v, causal=True)
    assert torch.equal(lse, lse2)
    for b, at in enumerate(AT):
        assert torch.equal(out[b, :at], again[b, :at]), at


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", [(2, 1, 8000, 4, 4, 128), (1, 1, 8000, 4, 4, 64), (2, 5, 3000, 8, 2, 128),
                                   (1, 300, 2000, 2, 2, 64)], ids=_name)
def test_a_nan_query_over_split_keys(shape, dtype):
    """Few queries: the keys are split over CTAs and the parts joined."""
    _nan_queries(shape, False, dtype)
    _nan_queries(shape, True, dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,h,hk", [(1, 4, 4), (3, 8, 2)])
def test_a_key_that_is_not_finite_among_split_keys(lq, h, hk, d, dtype):
    """One part of the keys is NaN, the others are not."""
    from splatx_cuda import network
    q, k, v, _ = _inputs(3, 1, lq, 8000, h, hk, d, dtype)
    k[:, 5000] = NAN
    out, lse = network.attention_fwd(q, k, v)
    _all_nan(out=out, lse=lse)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("lk", [96, 500])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [NAN, INF])
def test_a_key_that_is_not_finite_shows_at_every_place(value, d, lk, dtype):
    _key_at_every_place(value, d, lk, dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
def test_a_nan_query_shows_in_the_keys_gradients_at_every_place(d, dtype):
    _query_in_the_keys_gradients(d, dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 96, 96, 2, 2, 64), (1, 200, 300, 2, 1, 128), (1, 1, 8000, 4, 4, 128),
                                   (1, 5, 3000, 8, 2, 64)], ids=_name)
def test_scores_of_minus_infinity(shape, dtype):
    """A key whose score is -inf has weight 0 beside finite ones; where all are -inf the row is NaN
    (0 / 0), unlike a row that sees no key."""
    import torch
    from splatx_cuda import network
    b, lq, lk, h, hk, d = shape
    q, k, v, g = _inputs(d + lk, *shape, dtype)
    q[..., 0] = 1
    k[..., 0] = 0
    k[:, ::7, :, 0] = -INF
    out, lse = network.attention_fwd(q, k, v)
    keep = torch.ones(lk, dtype=torch.bool, device="cuda")
    keep[::7] = False
    seen = _seen(b, lq, int(keep.sum()), False, None, None)
    want = _definition(q, k[:, keep], v[:, keep], g, None, seen, d ** -0.5, ROUND[dtype])
    _check("out", out.transpose(1, 2), *want["out"])
    _check("lse", lse, *want["lse"])
    k[..., 0] = -INF
    out, lse, (v_q, v_k, v_v) = _fwd_bwd(q, k, v, g)
    _all_nan(out=out, lse=lse, v_q=v_q, v_k=v_k, v_v=v_v)
    none = torch.zeros(b, dtype=torch.int32, device="cuda")
    out, lse = network.attention_fwd(q, k, v, kv_lens=none)
    assert not out.any() and bool((lse == -INF).all())
    # the first tokens' queries before any key, the last one behind one of them
    few = torch.full((b,), 1, dtype=torch.int32, device="cuda")
    out, lse = network.attention_fwd(q, k, v, kv_lens=few, causal=True)
    assert not out[:, :-1].any() and bool((lse[:, :, :-1] == -INF).all())
    _all_nan(out=out[:, -1:], lse=lse[:, :, -1:])
