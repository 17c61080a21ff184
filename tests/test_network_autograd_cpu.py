"""What the autograd forms of the network operators ask of the calls underneath, which are stood in for here."""
import pytest
import torch

from splatx_cuda import network


@pytest.fixture
def kept(monkeypatch):
    """The `keep` of every linear_fwd."""
    seen = []

    def linear_fwd(x, weight, bias=None, *, activation=None, residual=None, keep=False):
        seen.append(keep)
        z = x @ weight.T
        return torch.relu(z), z if keep else None

    monkeypatch.setattr(network, "linear_fwd", linear_fwd)
    return seen


@pytest.mark.parametrize("off", [torch.no_grad, torch.inference_mode])
def test_linear_keeps_nothing_without_gradients(kept, off):
    x, w = torch.randn(5, 4), torch.nn.Parameter(torch.randn(3, 4))
    with off():
        y = network.linear(x, w, activation="relu")
    assert kept == [False] and not y.requires_grad and torch.equal(y, torch.relu(x @ w.T))
    y = network.linear(x, w, activation="relu")
    assert kept[1:] == [True] and y.requires_grad
    with torch.no_grad(), torch.enable_grad():
        assert network.linear(x, w, activation="relu").requires_grad
    assert kept[2:] == [True]
    network.linear(x, w)
    network.linear(x, w.detach(), activation="relu")
    network.linear(x, w.detach(), activation="relu", residual=torch.zeros(5, 3, requires_grad=True))
    assert kept[3:] == [False] * 3


def test_rotary_gradients_are_of_the_axes_and_freqs_that_were_given(monkeypatch):
    """A caller's list may change, and an iterator end, between the forward and the backward."""
    seen = []

    def fwd(q, k, positions, **how):
        seen.append((tuple(how["axes"]), tuple(how["freqs"])))
        return q * 1.0, None

    def bwd(v_q_out, v_k_out, q, k, positions, **how):
        seen.append((tuple(how["axes"]), tuple(how["freqs"])))
        return v_q_out, None, None, None

    monkeypatch.setattr(network, "qk_norm_rotary_fwd", fwd)
    monkeypatch.setattr(network, "qk_norm_rotary_bwd", bwd)
    q = torch.randn(1, 2, 3, 8, requires_grad=True)
    axes, freqs = [4, 4], torch.tensor([1.0, 0.5, 0.25, 0.125])
    for a, f in ((axes, freqs), (iter((4, 4)), iter((1.0, 0.5, 0.25, 0.125)))):
        y, _ = network.qk_norm_rotary(q, None, torch.zeros(2, 2), axes=a, freqs=f)
        axes[0], freqs[0] = 2, 7.0
        y.sum().backward()
        axes[0], freqs[0] = 4, 1.0
    assert seen == [((4, 4), (1.0, 0.5, 0.25, 0.125))] * 4
