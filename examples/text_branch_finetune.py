"""Trains text branches of a small synthetic DiT over frozen int8 linears, keeping 8-bit codes of activations.

One step uses the operators together: every block's image tokens pass a layer norm and look at a caption's
states (captions of several lengths, padded to one), the inputs of checkpointed blocks and of the trained
projections are kept as codes, and the weight gradients read them.

    python examples/text_branch_finetune.py --depth 4 --dim 1024 --steps 20
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


def finetune(*, depth: int, dim: int, heads: int, image_tokens: int, text_tokens: int, text_dim: int, batch: int, steps: int,
             lr: float, device: torch.device, seed: int = 0, coded: bool = True) -> list[float]:
    """The losses of ``steps`` steps on one fixed synthetic batch."""
    model = build_lora_model(depth, device=device, dim=dim, heads=heads, mlp_dim=4 * dim, rank=16, seed=seed,
                             text_dim=text_dim, coded=coded).train()
    optimizer = torch.optim.AdamW((p for p in model.parameters() if p.requires_grad), lr=lr)
    gen = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=gen, device=device).to(torch.bfloat16)

    latents, noise = randn(batch, image_tokens, dim), randn(batch, image_tokens, dim)
    none = randn(batch, 0, dim)  # no text tokens in the stream: the captions come through the branches
    context = randn(batch, text_tokens, text_dim)
    lengths = torch.linspace(text_tokens, 1, batch, device=device).long()
    mask = torch.arange(text_tokens, device=device)[None] < lengths[:, None]
    t = torch.rand(batch, generator=gen, device=device)
    losses = []
    for _ in range(steps):
        with torch.autocast("cuda", torch.bfloat16):
            loss = flow_matching_loss(model, latents, none, t, noise, context=context, context_mask=mask)
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
    parser.add_argument("--image-tokens", type=int, default=1024)
    parser.add_argument("--text-tokens", type=int, default=128)
    parser.add_argument("--text-dim", type=int, default=768)
    parser.add_argument("--batch", type=int, default=4)
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--lr", type=float, default=1e-4)
    parser.add_argument("--whole", action="store_true", help="keep whole activations instead of codes")
    args = parser.parse_args()
    losses = finetune(depth=args.depth, dim=args.dim, heads=args.heads, image_tokens=args.image_tokens,
                      text_tokens=args.text_tokens, text_dim=args.text_dim, batch=args.batch, steps=args.steps, lr=args.lr,
                      device=torch.device("cuda", 0), coded=not args.whole)
    for step, loss in enumerate(losses):
        print(f"step {step:3d}  loss {loss:.4f}")


if __name__ == "__main__":
    main()
