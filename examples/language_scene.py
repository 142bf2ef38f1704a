"""A scene whose Gaussians hold tokens: train the codebook behind them and the vocabulary that the
rendered features are scored against.

Each Gaussian of a fixed scene holds a token; its features are the token's row of a learned codebook
(``embed_tokens``).  They are rasterized, three channels at a time, into a feature image, and every
pixel that the scene covers is scored against every row of a learned vocabulary with the cross
entropy of its label (``linear_cross_entropy``); pixels that show background have no label.  The
gradient goes back through the rasterizer to the codebook.

The labels come from the same scene with a hidden codebook and vocabulary, so that they can be learned.

    python -m examples.language_scene --steps 60
"""

from __future__ import annotations

import argparse

import torch

from gswarp_amd import configs
from gswarp_amd.rasterizer import GaussianRasterizationSettings, GaussianRasterizer
from gswarp_amd.vocabulary import Vocabulary

IGNORED = -100
CHANNELS = 12  # of a Gaussian's features: four renderings of three


def feature_image(scene, features, settings):
    """((pixels, channels), (pixels,) alpha) of per-Gaussian features."""
    rendered = []
    for c in range(0, features.shape[1], 3):
        colour, _, meta = GaussianRasterizer(settings)(
            scene["means3D"], torch.zeros_like(scene["means3D"]), scene["opacities"],
            colors_precomp=features[:, c:c + 3].contiguous(), scales=scene["scales"], rotations=scene["rotations"])
        rendered.append(colour)
    return torch.cat(rendered).flatten(1).T, meta.alpha.detach().flatten()


def train(steps: int = 60, count: int = 20_000, size: int = 256, tokens: int = 64, classes: int = 40, seed: int = 0,
          device="cuda"):
    """The losses of `steps` steps."""
    torch.manual_seed(seed)
    device = torch.device(device)
    scene = configs.make_scene(1, count=count, width=size, height=size, device=device)
    settings = GaussianRasterizationSettings(
        image_height=size, image_width=size, tanfovx=scene["tanfovx"], tanfovy=scene["tanfovy"],
        bg=torch.zeros(3, device=device), scale_modifier=1.0, viewmatrix=scene["viewmatrix"],
        projmatrix=scene["projmatrix"], sh_degree=0, campos=scene["campos"], prefiltered=False)
    scene["scales"] = scene["scales"] * 2.0  # a closed surface rather than dust
    # a token for each region of space
    cell = ((scene["means3D"] - scene["means3D"].amin(0)) * 2.0).long()
    token = ((cell * torch.tensor([7, 31, 127], device=device)).sum(1) % tokens).int()

    def tables():
        return (Vocabulary(tokens, CHANNELS, scale=CHANNELS ** 0.5, device=device),
                Vocabulary(classes, CHANNELS, logit_scale=4.0, device=device))

    with torch.no_grad():
        codebook, vocabulary = tables()
        hidden, alpha = feature_image(scene, codebook(token), settings)
        labels = (hidden @ vocabulary.weight.T).argmax(1)
        labels[alpha < 0.5] = IGNORED

    codebook, vocabulary = tables()
    optimizer = torch.optim.Adam([*codebook.parameters(), *vocabulary.parameters()], lr=0.05)
    losses = []
    for _ in range(steps):
        image, _ = feature_image(scene, codebook(token), settings)
        loss = vocabulary.loss(image, labels, ignore_index=IGNORED)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=60)
    losses = train(parser.parse_args().steps)
    for i in range(0, len(losses), 10):
        print(f"step {i:3d}  loss {losses[i]:.4f}")
    print(f"last      loss {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
