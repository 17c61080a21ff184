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
