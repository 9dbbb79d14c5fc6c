"""Fine-tunes q, k, v and o of a small synthetic DiT over frozen fp8 linears, with the Muon optimiser.

One step uses the three operators together: image tokens carry (row, column) positions that turn
their queries and keys, every frozen linear runs on fp8 codes in both directions, and the trained
projections take orthogonalised updates.

    python examples/fp8_muon_finetune.py --depth 4 --dim 1024 --steps 20
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

REPO = Path(__file__).resolve().parents[1]
if str(REPO) not in sys.path:
    sys.path.insert(0, str(REPO))

from moss_image_b200.dit import build_lora_model, flow_matching_loss  # noqa: E402
from moss_image_b200.muon import Muon  # noqa: E402
from moss_image_b200.rotary import rotary_frequencies, rotary_table  # noqa: E402


def image_positions(side: int, text_tokens: int, device: torch.device) -> torch.Tensor:
    """(row, column) of a side x side image's tokens, then the text tokens on the diagonal past it."""
    rows, columns = torch.meshgrid(torch.arange(side, device=device), torch.arange(side, device=device), indexing="ij")
    image = torch.stack((rows.flatten(), columns.flatten()), 1)
    text = (side + torch.arange(text_tokens, device=device))[:, None].expand(-1, 2)
    return torch.cat((image, text))


def finetune(*, depth: int, dim: int, heads: int, side: int, text_tokens: int, batch: int, steps: int, lr: float,
             device: torch.device, seed: int = 0) -> list[float]:
    """The losses of ``steps`` steps on one fixed synthetic batch."""
    model = build_lora_model(depth, device=device, dim=dim, heads=heads, mlp_dim=4 * dim, seed=seed, full_qkvo=True,
                             frozen="fp8").train()
    head = dim // heads
    axis = rotary_frequencies(head // 2, device=device)
    rotary = rotary_table(image_positions(side, text_tokens, device), (axis, axis))
    optimizer = Muon((p for p in model.parameters() if p.requires_grad), lr=lr)
    gen = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=gen, device=device).to(torch.bfloat16)

    latents, noise = randn(batch, side * side, dim), randn(batch, side * side, dim)
    text = randn(batch, text_tokens, dim)
    t = torch.rand(batch, generator=gen, device=device)
    losses = []
    for _ in range(steps):
        loss = flow_matching_loss(model, latents, text, t, noise, rotary)
        loss.backward()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        losses.append(float(loss.detach()))
    return losses


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--depth", type=int, default=4)
    parser.add_argument("--dim", type=int, default=1024)
    parser.add_argument("--heads", type=int, default=8)
    parser.add_argument("--side", type=int, default=32, help="image tokens per side")
    parser.add_argument("--text-tokens", type=int, default=128)
    parser.add_argument("--batch", type=int, default=2)
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--lr", type=float, default=2e-2)
    args = parser.parse_args()
    losses = finetune(depth=args.depth, dim=args.dim, heads=args.heads, side=args.side, text_tokens=args.text_tokens,
                      batch=args.batch, steps=args.steps, lr=args.lr, device=torch.device("cuda", 0))
    for step, loss in enumerate(losses):
        print(f"step {step:3d}  loss {loss:.4f}")


if __name__ == "__main__":
    main()
