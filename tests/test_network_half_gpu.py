"""Attention in float16, which keeps its 11 bits only above 2^-14: gradients far below their largest, and
padding behind the lengths (the largest row norms, from which the backward takes its scale, are those below
them). Bounds and checks are those of test_network_attention_gpu."""
import math

import pytest

from test_network_attention_gpu import _inputs, _run

pytestmark = pytest.mark.gpu


# values three times as large as usual: keys that hardly any query looks at have gradients far below the
# largest, whose bits a scale from the values' largest magnitudes (several bits more cautious than one from
# the rows' norms) rounded away
@pytest.mark.parametrize("seed,shape,causal", [
    (1451, (1, 62, 555, 1, 1, 128), False), (1477, (3, 6, 99, 2, 2, 128), False),
    (1603, (3, 947, 947, 6, 3, 80), True), (1685, (2, 4, 1527, 4, 2, 128), False),
    (1756, (3, 56, 456, 3, 3, 128), True), (1940, (2, 167, 167, 3, 3, 64), True),
    (2035, (3, 2, 560, 3, 3, 32), True), (2372, (1, 71, 1269, 1, 1, 128), True)],
    ids=lambda x: "x".join(map(str, x)) if isinstance(x, tuple) else str(x))
def test_small_gradients_keep_their_bits(seed, shape, causal):
    _run(*_inputs(seed, *shape, "float16", spread=3.0), causal=causal)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128, 36])
def test_padded_batches_ignore_what_lies_beyond_the_lengths(d, causal):
    """Lengths of zero, one, inside and at tile edges, longer queries than keys; NaN and infinities in
    every padded row."""
    import torch
    from splatx_cuda import network
    q_lens = torch.tensor([300, 0, 1, 128, 129, 257, 300, 5], dtype=torch.int32, device="cuda")
    kv_lens = torch.tensor([290, 290, 1, 0, 128, 129, 64, 290], dtype=torch.int32, device="cuda")
    q, k, v, g = _inputs(7, 8, 300, 290, 2, 1, d, "float16")
    clean = [t.clone() for t in (q, k, v, g)]
    for b in range(8):
        for t, n in ((q, q_lens[b]), (g, q_lens[b]), (k, kv_lens[b]), (v, kv_lens[b])):
            t[b, int(n):] = math.nan
            t[b, int(n)::3] = math.inf
    how = dict(causal=causal, q_lens=q_lens, kv_lens=kv_lens)
    out, lse, grads = _run(*clean, **how)
    again = network.attention_fwd(q, k, v, **how)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    again = network.attention_bwd(g, q, k, v, *again, **how)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))
