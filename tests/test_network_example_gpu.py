"""The colour network's training path end to end: attention, layer norm and AdamW between the
executor's forward and backward."""
import pathlib
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_color_network_learns(bits):
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "splatx-metal_b200" / "examples"))
    import color_network
    from splatx_cuda import network
    losses = color_network.train(splats=1500, steps=60, state_bits=bits)
    assert np.all(np.isfinite(losses))
    assert np.mean(losses[-5:]) < 0.8 * losses[0], (losses[0], losses[-5:])
    assert network.attention_status() == 0
