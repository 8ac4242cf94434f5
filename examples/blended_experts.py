"""Fits an image with one small decoder per tile, blended over the tiles' borders.

Each pixel's grid features, joined by the code of its own tile, go to the decoders of the four tiles whose
centres surround it, and the four colours come back weighted bilinearly: no seams where tiles meet.  It
runs the row operators as a training program uses them: the lookup of the codes, the sort by expert,
the experts' layers, the weighted return, every gradient, and FusedAdam on fp32 masters.

    python examples/blended_experts.py [steps]
"""
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch

from odie_amd import synth
from odie_amd.encoding import GridEncoding
from odie_amd.mixture import ExpertMixture
from odie_amd.optimizer import FusedAdam

ENCODING = dict(n_levels=16, n_features_per_level=2, log2_hashmap_size=12, base_resolution=4, per_level_scale=1.3)
LOSS_SCALE = 4096.0    # fp16 gradients of a mean over a batch


def surrounding_tiles(coords, regions_x, regions_y):
    """The four tiles whose centres surround each of coords [N, 2] in [0, 1]^2, and their bilinear weights:
    expert int32 [N, 4], -1 for a tile outside the image, and weights [N, 4] that sum to 1 over the others."""
    size = torch.tensor((regions_x, regions_y), device=coords.device)
    place = coords * size - 0.5
    low = place.floor()
    part = place - low
    experts, weights = [], []
    for dy in (0, 1):
        for dx in (0, 1):
            corner = low.long() + torch.tensor((dx, dy), device=coords.device)
            inside = ((corner >= 0) & (corner < size)).all(1)
            share = torch.stack((part[:, 0] if dx else 1 - part[:, 0], part[:, 1] if dy else 1 - part[:, 1]), 1).prod(1)
            experts.append(torch.where(inside, corner[:, 1] * regions_x + corner[:, 0], -1))
            weights.append(torch.where(inside, share, 0.0))
    weights = torch.stack(weights, 1)
    return torch.stack(experts, 1).to(torch.int32), weights / weights.sum(1, keepdim=True)


class BlendedFit:
    def __init__(self, image, regions_x, regions_y, *, hidden=64, codes=16, lr=2e-3, seed=0):
        self.height, self.width = image.shape[:2]
        self.regions = (regions_x, regions_y)
        self.rgb = image.reshape(-1, 3).float().cuda() / 255
        tiles = regions_x * regions_y
        self.encoding = GridEncoding(ENCODING, dtype=torch.float16)
        with torch.no_grad():
            self.encoding.params.copy_(torch.from_numpy(synth.table(seed, self.encoding.n_params)))
        self.mixture = ExpertMixture(tiles, self.encoding.n_output_dims, hidden, 3, codes=codes, vocab=tiles, seed=seed)
        # fp16 parameters with fp32 masters; the grid's parameters are fp32 themselves
        self.optimizers = [(p, FusedAdam(p.detach().float().flatten(), lr, half_copy=p.data))
                           for p in self.mixture.parameters()]
        self.optimizers.append((self.encoding.params, FusedAdam(self.encoding.params.data, 10 * lr)))

    def predict(self, ids):
        """RGB [N, 3] of pixel ids [N]."""
        x, y = ids % self.width, ids // self.width
        coords = torch.stack(((x + 0.5) / self.width, (y + 0.5) / self.height), 1).float()
        tile = (coords[:, 1] * self.regions[1]).long() * self.regions[0] + (coords[:, 0] * self.regions[0]).long()
        expert, weights = surrounding_tiles(coords, *self.regions)
        return self.mixture(self.encoding(coords), expert, weights, tile)

    def step(self, ids):
        """One training step on pixel ids [N]; returns the mean squared error as a tensor."""
        loss = (self.predict(ids).float() - self.rgb[ids]).square().mean()
        (loss * LOSS_SCALE).backward()
        for parameter, optimizer in self.optimizers:
            optimizer.step(parameter.grad.flatten(), loss_scale=LOSS_SCALE)
            parameter.grad = None
        return loss.detach()


def main(steps=200, height=768, width=1024, regions_x=8, regions_y=6, batch=65536):
    generator = torch.Generator(device='cuda').manual_seed(0)
    fit = BlendedFit(torch.from_numpy(synth.image(0, width, height)), regions_x, regions_y)
    losses = []
    for step in range(steps):
        losses.append(fit.step(torch.randint(0, height * width, (batch,), generator=generator, device='cuda')))
        if step % 20 == 0 or step == steps - 1:
            print('step %4d  mse %.5f' % (step, float(losses[-1])), flush=True)
    return torch.stack(losses)


if __name__ == '__main__':
    main(*map(int, sys.argv[1:2]))
