"""Trains a small transformer that gives splats their base colours, through the rasteriser.

    python splatx-metal_b200/examples/color_network.py --steps 80 --state-bits 8

Every Gaussian is a token: the network sees its position, scales, rotation and opacity and answers
with its three degree-0 SH coefficients. A step writes them into the executor's resident arena,
renders one view with the executor's forward and backward (``step_accumulate``), takes the loss
gradient of the coefficients from the resident gradient buffers as the gradient of the network's
output, and updates the network's weights with ``AdamW``. Attention, layer norm and AdamW are
``splatx_cuda.network``'s; the matrix products of the layers are torch's. With ``--spatial`` the
products, with their gelu and residuals, are ``splatx_cuda.network``'s too, and queries and keys are
normalised and rotated by the Gaussians' places.
"""
from __future__ import annotations

import argparse
import contextlib
import pathlib
import sys

import numpy as np
import torch
import torch.nn.functional as F

if __name__ == "__main__":
    sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

from splatx_cuda import network
from splatx_cuda.executor import TrainStepExecutor
from splatx_cuda.parallel import device_tensor
from splatx_cuda.scene import small_scene

SH0 = 4  # the parameter group of the degree-0 coefficients


class ColorNetwork(torch.nn.Module):
    """[splats, features] -> [splats, 3]; 32-bit weights, bfloat16 activations. spatial: attention knows where
    the splats are, and ``forward`` takes their places, [splats, 3], from about -128 to 128."""

    def __init__(self, features: int, width: int = 128, heads: int = 2, layers: int = 2, spatial: bool = False):
        super().__init__()
        self.heads, self.layers = heads, layers
        sizes = {"embed": (width, features), "head": (3, width)}
        for i in range(layers):
            sizes |= {f"qkv{i}": (3 * width, width), f"proj{i}": (width, width),
                      f"up{i}": (4 * width, width), f"down{i}": (width, 4 * width)}
        self.w = torch.nn.ParameterDict(
            {k: torch.randn(s) * s[1] ** -0.5 for k, s in sizes.items()})
        norms = [f"{n}{i}" for i in range(layers) for n in ("attn", "mlp")] + ["last"]
        self.scale = torch.nn.ParameterDict({k: torch.ones(width) for k in norms})
        d = width // heads
        self.axes = (d - 2 * (d // 3 // 2 * 2), d // 3 // 2 * 2, d // 3 // 2 * 2) if spatial else None
        self.qk = torch.nn.ParameterDict({f"{n}{i}": torch.ones(d) for i in range(layers if spatial else 0) for n in "qk"})
        self.shift = torch.nn.ParameterDict({k: torch.zeros(width) for k in norms})

    def _linear(self, x, name):
        return F.linear(x, self.w[name].to(x.dtype))

    def _norm(self, x, name):
        return network.layer_norm(x, self.scale[name], self.shift[name])

    def forward(self, features, places=None):
        if self.axes is not None:
            return self._spatial(features.to(torch.bfloat16)[None], places[None])
        x = self._linear(features.to(torch.bfloat16)[None], "embed")
        for i in range(self.layers):
            qkv = self._linear(self._norm(x, f"attn{i}"), f"qkv{i}")
            q, k, v = qkv.unflatten(-1, (3, self.heads, -1)).unbind(2)  # views, not copies
            x = x + self._linear(network.attention(q, k, v).flatten(2), f"proj{i}")
            x = x + self._linear(F.gelu(self._linear(self._norm(x, f"mlp{i}"), f"up{i}")), f"down{i}")
        return self._linear(self._norm(x, "last"), "head")[0].float()

    def _spatial(self, x, places):
        def linear(x, name, **how):
            return network.linear(x, self.w[name].to(x.dtype), **how)

        x = linear(x, "embed")
        for i in range(self.layers):
            qkv = linear(self._norm(x, f"attn{i}"), f"qkv{i}")
            q, k, v = qkv.unflatten(-1, (3, self.heads, -1)).unbind(2)
            q, k = network.qk_norm_rotary(q, k, places, axes=self.axes, base=100.0, q_weight=self.qk[f"q{i}"],
                                          k_weight=self.qk[f"k{i}"])
            x = linear(network.attention(q, k, v).flatten(2), f"proj{i}", residual=x)
            x = linear(linear(self._norm(x, f"mlp{i}"), f"up{i}", activation="gelu"), f"down{i}", residual=x)
        return linear(self._norm(x, "last"), "head")[0].float()


class ResidentGroup:
    """A parameter group of the executor's arena as rows, and its gradients: the arena keeps tiles of
    32 Gaussians, in each the group's components as runs of 32 floats."""

    def __init__(self, ex: TrainStepExecutor, group: int, count: int, device: int):
        b = ex.resident_buffers()
        self.count, d, rows = count, b["dims"][group], b["padded_rows"]
        self.params, self.grads = (device_tensor(b[k][group], rows * d, device).view(rows // 32, d, 32)
                                   for k in ("params", "grads"))

    def write(self, rows: torch.Tensor):
        padded = F.pad(rows, (0, 0, 0, self.params.shape[0] * 32 - self.count))
        self.params.copy_(padded.view(-1, 32, rows.shape[1]).transpose(1, 2))

    def read_grads(self) -> torch.Tensor:
        return self.grads.transpose(1, 2).reshape(-1, self.grads.shape[1])[: self.count]


def train(splats: int = 2048, steps: int = 80, width: int = 128, state_bits: int = 32, seed: int = 0,
          lr: float = 2e-3, device: int = 0, spatial: bool = False) -> list[float]:
    """The loss of every step."""
    torch.manual_seed(seed)
    scene, cam = small_scene(seed=seed, n=splats)
    # colours that follow from where a splat is: what there is to learn
    colors = np.sin(2.0 * scene.means + np.array([0.0, 1.0, 2.0])).astype(np.float32)
    groups = [np.ascontiguousarray(g.reshape(splats, -1)) for g in scene.groups()]
    zeros = [np.zeros_like(g) for g in groups]
    with contextlib.closing(TrainStepExecutor(splats, 0, ssim_weight=0.2, device=device)) as ex:
        groups[SH0] = colors
        ex.upload_params(groups, zeros, zeros, splats)
        *_, target = ex.step(cam.viewmat, cam.K, cam.width, cam.height, None, splats, degrees_to_use=0,
                             forward_only=True, want_render=True)
        target = torch.from_numpy(np.ascontiguousarray(target)).to(f"cuda:{device}")
        features = np.concatenate([scene.means, scene.scales, scene.quats, scene.opacities[:, None]], 1)
        features = torch.from_numpy(features).to(target.device)
        features = (features - features.mean(0)) / features.std(0)
        net = ColorNetwork(features.shape[1], width, spatial=spatial).to(target.device)
        places = features[:, :3] * 32.0 if spatial else None
        opt = network.AdamW(net.parameters(), lr=lr, weight_decay=0.01, state_bits=state_bits)
        sh0 = ResidentGroup(ex, SH0, splats, device)
        torch.cuda.synchronize(device)
        losses = []
        # everything on the executor's stream: its steps and torch's kernels follow one another
        with torch.cuda.stream(torch.cuda.ExternalStream(ex.stream_handle(), device=device)):
            for _ in range(steps):
                out = net(features, places)
                sh0.write(out.detach())
                ex.clear_grads()
                ex.step_accumulate(cam.viewmat, cam.K, cam.width, cam.height, target.data_ptr(), splats)
                out.backward(sh0.read_grads())
                opt.step()
                net.zero_grad(set_to_none=True)
                losses.append(ex.last_result()[0])
        torch.cuda.synchronize(device)
    return losses


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--splats", type=int, default=2048)
    p.add_argument("--steps", type=int, default=80)
    p.add_argument("--width", type=int, default=128)
    p.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    p.add_argument("--lr", type=float, default=2e-3)
    p.add_argument("--spatial", action="store_true")
    a = p.parse_args()
    losses = train(a.splats, a.steps, a.width, a.state_bits, lr=a.lr, spatial=a.spatial)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.5f}")
    print(f"step {len(losses) - 1:4d}  loss {losses[-1]:.5f}")


if __name__ == "__main__":
    main()
