"""Synthetic DiT block and block stack that host the int8 hot path (benchmark harness).

The shapes follow the benchmark configuration of this path: width 3072, 24 heads x 128,
joint attention over image + text tokens, MLP 3072 -> 12288 -> 3072 with GELU, and a
per-block adaLN modulation linear 3072 -> 6 x 3072. The block mirrors the structure of the
reference ``Block._forward_impl`` (training/model.py:269-314): RMSNorm + scale/shift
modulation, q/k/v projections with per-head RMSNorm on q and k, joint attention, gated
residual, modulated MLP with a gated residual. Every linear is a
:class:`~moss_image_b200.quantization.FrozenInt8Linear`; q/k/v/o carry LoRA adapters.

The stack wraps its forward in :func:`activation_cpu_offload` and checkpoints each block
(non-reentrant), as the reference trainer does with ``grad_checkpointing: true``
(training/model.py:687-709), so the offloaded tensors are the block inputs. Blocks may be
swapped or streamed with :func:`~moss_image_b200.memory.place_model`, and
:meth:`SyntheticDiT.forward_packed` runs a heterogeneous batch as one packed stream.
Per-sample modulation and gates are applied by the native segment kernels on CUDA
(:mod:`moss_image_b200.packed`). Attention uses torch's scaled-dot-product attention (library
code; the jagged, variable-length form for packed streams). Queries and keys may be turned by
their positions (a table from :func:`~moss_image_b200.rotary.rotary_table`), and the frozen linears
may be held in block-scaled fp8 instead of int8.

A block may have a trained :class:`TextBranch`, in which its tokens look at a text encoder's states
(:mod:`moss_image_b200.cross_attention`), and what training keeps of activations may be 8-bit codes
(:mod:`moss_image_b200.activation_codes`): the inputs of checkpointed blocks (``coded_checkpoints`` of the
stack), swapped and streamed ones among them, and of the trained projections with 16-bit products (``coded_inputs`` of the
blocks), where nothing else keeps them anyway.
"""

from __future__ import annotations

import math
from contextlib import nullcontext

import torch
from torch import nn
from torch.nn import functional as F
from torch.utils.checkpoint import checkpoint

from .activation_codes import CodedActivation, coded_checkpoints, coded_linear, codes_serve, encode_activation
from .activation_offload import KEEP_RESIDENT, activation_cpu_offload
from .cross_attention import cross_attention, cross_attention_packed
from .fp8 import quantize_frozen_linears_fp8
from .lora import LoRALinear
from .memory import offloaded_block
from .norms import layer_norm, rms_norm
from .packed import (
    CHECKPOINT_CHECK,
    VARLEN_LOOP_MAX_SEQUENCES,
    batch_offsets,
    condition_for_tokens,
    cumulative_lengths,
    modulation_sample_indices,
    segment_gate,
    segment_modulate,
    sequence_lengths,
    varlen_attention,
)
from .quantization import quantize_frozen_linears
from .rotary import apply_rotary


class RMSNorm(nn.Module):
    """Root-mean-square norm with a learned gain (training/model.py:154-172 arithmetic:
    f32 statistics, cast to the input dtype, then times the gain). CUDA inputs run the
    native norm kernels."""

    def __init__(self, dim: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.is_cuda:
            return rms_norm(x, self.weight, self.eps)
        normalized = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + self.eps)
        return normalized.to(x.dtype) * self.weight


class LayerNorm(nn.Module):
    """Layer norm with a learned gain and offset; CUDA inputs run the native kernels."""

    def __init__(self, dim: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.is_cuda:
            return layer_norm(x, self.weight, self.bias, self.eps)
        return F.layer_norm(x.float(), x.shape[-1:], self.weight.float(), self.bias.float(), self.eps).to(x.dtype)


def keeps_codes(linear: nn.Module, tokens: torch.Tensor) -> bool:
    """Whether ``linear(tokens)`` would keep the tokens' codes in their place: a trained linear or adapter with 16-bit products."""
    if not torch.is_grad_enabled():
        return False
    if isinstance(linear, LoRALinear):
        return linear.keeps_codes(tokens)
    return isinstance(linear, nn.Linear) and linear.weight.requires_grad and codes_serve(tokens, linear.weight.dtype)


def project(linear: nn.Module, tokens: torch.Tensor, coded: CodedActivation | None) -> torch.Tensor:
    """``linear(tokens)``; where it can, it keeps the tokens' codes for its gradient if they are given."""
    if coded is None or not keeps_codes(linear, tokens):
        return linear(tokens)
    if isinstance(linear, LoRALinear):
        return linear(tokens, coded)
    return coded_linear(tokens, linear.weight, linear.bias, coded=coded)


class TextBranch(nn.Module):
    """``tokens + o(attention(q(norm(tokens)), k(context), v(context)))``: a trained residual branch in which image
    tokens look at a text encoder's states. ``o`` starts at zero, so a new branch changes nothing."""

    def __init__(self, dim: int, heads: int, text_dim: int, k_heads: int | None = None) -> None:
        super().__init__()
        self.head_dim = dim // heads
        shared = (heads if k_heads is None else k_heads) * self.head_dim
        self.norm = LayerNorm(dim)
        self.q = nn.Linear(dim, dim, bias=False)
        self.k = nn.Linear(text_dim, shared, bias=False)
        self.v = nn.Linear(text_dim, shared, bias=False)
        self.o = nn.Linear(dim, dim, bias=False)
        nn.init.zeros_(self.o.weight)
        self.coded_inputs = False

    def forward(self, tokens: torch.Tensor, context: torch.Tensor, keys: torch.Tensor | None = None,
                offsets: torch.Tensor | None = None) -> torch.Tensor:
        """``tokens`` ``[B, T, dim]`` and ``context`` ``[B, S, text_dim]`` with an optional bool mask ``keys`` ``[B, S]``; or, with
        the stream's boundaries ``offsets``, ``[1, total, dim]``, ``[1, states, text_dim]`` and the captions' boundaries ``keys``."""
        def heads(x: torch.Tensor) -> torch.Tensor:
            return x.unflatten(-1, (-1, self.head_dim))

        h = self.norm(tokens)
        coded = encode_activation(h) if self.coded_inputs and keeps_codes(self.q, h) else None
        # the rest of what is kept lives anyway: the context belongs to the caller, and the attention keeps its own output
        q, k, v = heads(project(self.q, h, coded)), heads(self.k(context)), heads(self.v(context))
        if offsets is None:
            attended = cross_attention(q, k, v, key_mask=keys).flatten(2)
        else:
            attended = cross_attention_packed(q[0], k[0], v[0], offsets, keys).flatten(1)[None]
        return tokens + self.o(attended)


class SyntheticBlock(nn.Module):
    """One joint attention + MLP block with its own adaLN modulation linear."""

    def __init__(self, dim: int = 3072, heads: int = 24, mlp_dim: int = 12288) -> None:
        super().__init__()
        self.dim = dim
        self.heads = heads
        self.norm1 = RMSNorm(dim)
        self.norm2 = RMSNorm(dim)
        self.q_norm = RMSNorm(dim // heads)
        self.k_norm = RMSNorm(dim // heads)
        self.proj = nn.ModuleDict({name: nn.Linear(dim, dim, bias=False) for name in ("q", "k", "v", "o")})
        self.mlp_up = nn.Linear(dim, mlp_dim, bias=True)
        self.mlp_down = nn.Linear(mlp_dim, dim, bias=True)
        self.adaln = nn.Linear(dim, 6 * dim, bias=True)
        self.text: TextBranch | None = None
        self.coded_inputs = False

    def forward(self, tokens: torch.Tensor, cond: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, context: torch.Tensor | None = None,
                keys: torch.Tensor | None = None) -> torch.Tensor:
        """tokens: [B, T, dim] with cond [B, dim] (timestep embedding per sample), or a packed
        [1, total, dim] stream with cu_seqlens (int64 [S + 1]) and cond [S, dim]. With ``cos`` and
        ``sin`` (float32 [T, half], one row per token) q and k are turned by their positions. ``context`` and ``keys``:
        what the text branch looks at (:meth:`TextBranch.forward`), between the attention and the MLP.

        The conditioning follows training/model.py:288-312: ``norm(x) * (1 + scale) + shift``
        and ``x + branch * gate`` per sample, each op rounded in the activation dtype. On CUDA
        the per-sample conditions are applied by the native segment kernels; attention is
        block-diagonal over the packed sequences.
        """
        batch, seq, dim = tokens.shape
        sequences = cond.shape[0]
        modulation = self.adaln(F.silu(cond)).view(sequences, 6, dim)
        shift_a, scale_a, gate_a, shift_f, scale_f, gate_f = modulation.unbind(1)
        offsets = batch_offsets(batch, seq, tokens.device) if cu_seqlens is None else cu_seqlens
        if tokens.is_cuda:
            def modulate(x, scale, shift):
                return segment_modulate(x, scale, shift, offsets)

            def gated(x, branch, gate):
                return segment_gate(x, branch, gate, offsets)
        else:  # the reference's expansion (training/model.py:752-772)
            index = modulation_sample_indices(modulation, tokens, cu_seqlens)

            def modulate(x, scale, shift):
                return x * (1 + condition_for_tokens(scale, index)) + condition_for_tokens(shift, index)

            def gated(x, branch, gate):
                return x + branch * condition_for_tokens(gate, index)

        h = modulate(self.norm1(tokens), scale_a, shift_a)
        coded = None
        if self.coded_inputs and any(keeps_codes(self.proj[name], h) for name in ("q", "k", "v")):
            coded = encode_activation(h)  # one set for the three
        q = self.q_norm(project(self.proj["q"], h, coded).unflatten(-1, (self.heads, -1)))
        k = self.k_norm(project(self.proj["k"], h, coded).unflatten(-1, (self.heads, -1)))
        v = project(self.proj["v"], h, coded).unflatten(-1, (self.heads, -1))
        if cos is not None:
            q, k = apply_rotary(q, k, cos, sin)
        if cu_seqlens is None:
            output = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2))
            attended = output.transpose(1, 2).flatten(2)
            copied = attended.data_ptr() != output.data_ptr()
            del output
        else:
            copied = len(sequence_lengths(cu_seqlens)) <= VARLEN_LOOP_MAX_SEQUENCES  # joined from one output for each
            attended = varlen_attention(q[0], k[0], v[0], offsets, sequence_lengths(cu_seqlens)).flatten(1)[None]
        # (the attention keeps its output for the backward pass: where this is a view of it, codes would come on top)
        coded = encode_activation(attended) if self.coded_inputs and copied and keeps_codes(self.proj["o"], attended) else None
        tokens = gated(tokens, project(self.proj["o"], attended, coded), gate_a)
        if self.text is not None and context is not None:
            tokens = self.text(tokens, context, keys, cu_seqlens)
        h = modulate(self.norm2(tokens), scale_f, shift_f)
        return gated(tokens, self.mlp_down(F.gelu(self.mlp_up(h), approximate="tanh")), gate_f)


class TimestepEmbedding(nn.Module):
    """Sinusoidal flow-matching time embedding followed by a small MLP (kept in fp32)."""

    def __init__(self, dim: int, freq_dim: int = 256) -> None:
        super().__init__()
        self.freq_dim = freq_dim
        self.mlp = nn.Sequential(nn.Linear(freq_dim, dim), nn.SiLU(), nn.Linear(dim, dim))

    def forward(self, t: torch.Tensor) -> torch.Tensor:
        half = self.freq_dim // 2
        freqs = torch.exp(-math.log(10000.0) * torch.arange(half, device=t.device, dtype=torch.float32) / half)
        phase = (1000.0 * t.float())[:, None] * freqs[None]
        emb = torch.cat((phase.cos(), phase.sin()), -1)
        return self.mlp(emb.to(self.mlp[0].weight.dtype))


class SyntheticDiT(nn.Module):
    """Stack of synthetic blocks with checkpointing and saved-activation offload."""

    def __init__(self, depth: int = 36, dim: int = 3072, heads: int = 24, mlp_dim: int = 12288,
                 gradient_checkpointing: bool = True) -> None:
        super().__init__()
        self.time_embedding = TimestepEmbedding(dim)
        self.layers = nn.ModuleList(SyntheticBlock(dim, heads, mlp_dim) for _ in range(depth))
        self.final_norm = RMSNorm(dim)
        self.gradient_checkpointing = gradient_checkpointing
        self.activation_offload = False
        self.coded_checkpoints = False

    def forward(self, tokens: torch.Tensor, timestep: torch.Tensor, skip_layers: tuple[int, ...] = (),
                rotary: tuple[torch.Tensor, torch.Tensor] | None = None, context: torch.Tensor | None = None,
                context_mask: torch.Tensor | None = None) -> torch.Tensor:
        """``rotary``: the (cos, sin) tables of the tokens' positions, shared by all blocks. ``context`` ``[B, S, text_dim]``
        and its bool mask ``[B, S]``: the states that the blocks' text branches look at."""
        scope = activation_cpu_offload(self, self.activation_offload, tokens.device)
        with scope:
            cond = self.time_embedding(timestep).to(tokens.dtype)
            tokens = self._run_layers(tokens, cond, frozenset(skip_layers), rotary=rotary, context=context,
                                      keys=context_mask, scope=scope)
            return self.final_norm(tokens)

    def forward_packed(self, samples: list[torch.Tensor], timestep: torch.Tensor,
                       rotary: tuple[torch.Tensor, torch.Tensor] | None = None,
                       context: list[torch.Tensor] | None = None) -> list[torch.Tensor]:
        """One traversal over a heterogeneous batch: ``samples[i]`` is ``[tokens_i, dim]``.

        Mirrors ``forward_packed`` (training/model.py:502-626): the samples are concatenated
        into one ``[1, total, dim]`` stream with cumulative boundaries, every linear runs once
        over all tokens, attention is isolated per sample, and each sample keeps its own
        timestep conditioning. ``rotary``: the (cos, sin) tables of the stream, one row per token, the
        samples' one after another. ``context[i]``: ``[states_i, text_dim]`` of sample i (none for an empty
        caption). Returns the per-sample outputs.
        """
        if not samples:
            raise ValueError("forward_packed requires at least one sample.")
        device = samples[0].device
        if any(sample.ndim != 2 or sample.shape[0] == 0 or sample.device != device for sample in samples):
            raise ValueError("Each packed sample must be a non-empty [tokens, dim] tensor on one device.")
        lengths = [sample.shape[0] for sample in samples]
        if rotary is not None and any(table.shape[0] != sum(lengths) for table in rotary):
            raise ValueError("The rotary tables of a packed stream have one row for each of its tokens.")
        times = torch.as_tensor(timestep, device=device).reshape(-1).expand(len(samples))
        cu_seqlens = cumulative_lengths(lengths, device)
        cu_seqlens.moss_lengths = tuple(lengths)  # known on the host: no device read per block
        setattr(cu_seqlens, KEEP_RESIDENT, True)  # the same boundaries tensor in every recomputation
        tokens = torch.cat(samples, 0).unsqueeze(0)
        states = keys = None
        if context is not None:
            if len(context) != len(samples):
                raise ValueError("A packed batch has one context for each of its samples.")
            states = torch.cat(context, 0).unsqueeze(0)
            keys = cumulative_lengths([c.shape[0] for c in context], device)
            setattr(keys, KEEP_RESIDENT, True)
        scope = activation_cpu_offload(self, self.activation_offload, device)
        with scope:
            cond = self.time_embedding(times).to(tokens.dtype)
            tokens = self._run_layers(tokens, cond, frozenset(), cu_seqlens, rotary, states, keys, scope)
            return list(self.final_norm(tokens)[0].split(lengths, 0))

    def _run_layers(self, tokens: torch.Tensor, cond: torch.Tensor, skipped: frozenset[int],
                    cu_seqlens: torch.Tensor | None = None,
                    rotary: tuple[torch.Tensor, torch.Tensor] | None = None, context: torch.Tensor | None = None,
                    keys: torch.Tensor | None = None, scope: object = None) -> torch.Tensor:
        """Resident, synchronously swapped or streamed blocks, as ``place_model`` left them.

        Mirrors training/model.py:672-709: blocks at or past ``len(layers) - blocks_to_swap``
        run through the streamer (prefetching the next streamed block in the direction of
        traversal, checkpointed whenever gradients are enabled) or, without a streamer,
        from their CPU masters; the others are checkpointed when training.
        """
        boundary = len(self.layers) - getattr(self, "blocks_to_swap", 0)
        manager = getattr(self, "block_swap_manager", None)
        streamed = [index for index in range(boundary, len(self.layers)) if index not in skipped]
        position = {index: slot for slot, index in enumerate(streamed)}
        if rotary is not None:  # the same dense table in every block, marked on tensors of the model's own
            rotary = tuple(table.contiguous().view_as(table) for table in rotary)
            for table in rotary:
                setattr(table, KEEP_RESIDENT, True)
        for index, layer in enumerate(self.layers):
            if index in skipped:
                continue
            inputs = (tokens, cond) if cu_seqlens is None else (tokens, cond, cu_seqlens)
            if rotary is not None:
                inputs = (tokens, cond, cu_seqlens, *rotary)
            if context is not None:
                inputs = (tokens, cond, cu_seqlens, *(rotary or (None, None)), context, keys)
            # every block that is checkpointed, wherever its parameters are
            kept = coded_checkpoints(tokens, scope) if self.coded_checkpoints and torch.is_grad_enabled() else nullcontext()
            if manager is not None and index >= boundary:
                at = position[index]
                with kept:
                    tokens = manager.block(
                        index, *inputs,
                        forward_prefetch=streamed[at + 1] if at + 1 < len(streamed) else None,
                        backward_prefetch=streamed[at - 1] if at else None,
                        checkpoint_block=torch.is_grad_enabled(),
                    )
            elif index >= boundary:
                with kept:
                    tokens = offloaded_block(layer, *inputs)
            elif self.gradient_checkpointing and self.training and torch.is_grad_enabled():
                with kept:
                    tokens = checkpoint(layer, *inputs, use_reentrant=False, determinism_check=CHECKPOINT_CHECK)
            else:
                tokens = layer(*inputs)
        return tokens


def inject_lora(model: nn.Module, rank: int, alpha: float, targets: tuple[str, ...] = ("q", "k", "v", "o"),
                a_std: float | None = 0.01) -> list[str]:
    """Wrap the named projections of every block in :class:`LoRALinear`.

    A ~ N(0, a_std) (the benchmark's adapter init; ``None`` keeps the reference's Kaiming
    init), B = 0. Returns the wrapped module paths.
    """
    names = []
    for index, layer in enumerate(model.layers):
        _inject_block(layer, rank, alpha, targets, a_std)
        names.extend(f"layers.{index}.proj.{name}" for name in targets)
    return names


def _inject_block(layer: SyntheticBlock, rank: int, alpha: float, targets: tuple[str, ...],
                  a_std: float | None) -> None:
    for name in targets:
        base = layer.proj[name]
        wrapped = LoRALinear(base, rank, alpha).to(device=base.weight.device)
        if a_std is not None:
            with torch.no_grad():
                wrapped.lora_A.normal_(0.0, a_std)
        layer.proj[name] = wrapped


def build_lora_model(depth: int, *, device: torch.device, dim: int = 3072, heads: int = 24, mlp_dim: int = 12288,
                     rank: int = 32, alpha: float | None = None, seed: int = 0,
                     dtype: torch.dtype = torch.bfloat16, full_qkvo: bool = False,
                     frozen: str = "int8", text_dim: int | None = None, coded: bool = False) -> SyntheticDiT:
    """Random-init stack (weights ~ N(0, 0.02)), int8 base, LoRA on q/k/v/o.

    Mirrors the trainer's order (training/train.py:577-589): build, cast, inject LoRA,
    quantise the frozen linears - done block by block on the device so that the
    full-precision weights of only one block exist at a time.

    With ``full_qkvo`` the q/k/v/o projections are trained in full instead (trainable
    ``dtype`` masters, no adapters) and every other linear is frozen int8: the hybrid that
    ``quantize_frozen_linears`` allows at module level (training/quantization.py:156-157;
    the reference trainer itself only pairs int8 bases with LoRA, training/train.py:543-545).
    ``frozen="fp8"`` holds the frozen linears as block-scaled fp8 (:mod:`moss_image_b200.fp8`). ``text_dim`` gives
    every block a trained :class:`TextBranch` over states of that width. ``coded`` keeps block inputs as 8-bit
    codes (``coded_checkpoints``), and the inputs of trained projections and adapters whose products are 16-bit
    (``coded_inputs``).
    """
    if frozen not in ("int8", "fp8"):
        raise ValueError("frozen linears are held as int8 or fp8.")
    quantize = quantize_frozen_linears if frozen == "int8" else quantize_frozen_linears_fp8
    torch.manual_seed(seed)
    alpha = float(rank if alpha is None else alpha)
    model = SyntheticDiT(depth=0, dim=dim, heads=heads, mlp_dim=mlp_dim)
    model.time_embedding.to(device=device, dtype=dtype)
    model.final_norm.to(device=device, dtype=dtype)
    model.requires_grad_(False)
    quantize(model.time_embedding)
    layers = []
    for _ in range(depth):
        block = SyntheticBlock(dim, heads, mlp_dim).to(device=device)
        with torch.no_grad():
            for module in block.modules():
                if isinstance(module, nn.Linear):
                    module.weight.normal_(0.0, 0.02)
                    if module.bias is not None:
                        module.bias.zero_()
        block.to(dtype=dtype)
        block.requires_grad_(False)
        if full_qkvo:
            for name in ("q", "k", "v", "o"):
                block.proj[name].requires_grad_(True)
        else:
            _inject_block(block, rank, alpha, ("q", "k", "v", "o"), 0.01)
        quantize(block)
        if text_dim is not None:
            block.text = TextBranch(dim, heads, text_dim)
            for linear in (block.text.q, block.text.k, block.text.v):
                nn.init.normal_(linear.weight, 0.0, 0.02)
            block.text.to(device=device, dtype=dtype).coded_inputs = coded
        block.coded_inputs = coded
        layers.append(block)
    model.layers = nn.ModuleList(layers)
    model.coded_checkpoints = coded
    return model


def packed_flow_matching_loss(model: SyntheticDiT, latents: list[torch.Tensor], text: list[torch.Tensor],
                              t: torch.Tensor, noise: list[torch.Tensor],
                              rotary: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
    """The flow-matching loss of a heterogeneous batch in one packed traversal.

    ``latents[i]``/``noise[i]``: ``[image_tokens_i, dim]``; ``text[i]``: ``[text_tokens_i, dim]``; ``rotary``: tables
    with a row for each token of the stream (each sample's image tokens, then its text tokens).
    Each sample's loss is its mean over its image tokens; the batch loss is their mean.
    """
    samples = []
    for latent, context, noise_i, sigma in zip(latents, text, noise, t):
        sigma = sigma.to(latent.dtype)
        samples.append(torch.cat(((1 - sigma) * latent + sigma * noise_i, context), 0))
    outputs = model.forward_packed(samples, t, rotary)
    losses = [F.mse_loss(out[: latent.shape[0]].float(), (noise_i - latent).float())
              for out, latent, noise_i in zip(outputs, latents, noise)]
    return torch.stack(losses).mean()


def flow_matching_loss(model: SyntheticDiT, latents: torch.Tensor, text: torch.Tensor, t: torch.Tensor,
                       noise: torch.Tensor, rotary: tuple[torch.Tensor, torch.Tensor] | None = None,
                       context: torch.Tensor | None = None, context_mask: torch.Tensor | None = None) -> torch.Tensor:
    """Rectified-flow velocity loss on the image tokens (text tokens are conditioning, and so is the text branches' ``context``)."""
    sigma = t.view(-1, 1, 1).to(latents.dtype)
    noisy = (1 - sigma) * latents + sigma * noise
    tokens = torch.cat((noisy, text), dim=1)
    pred = model(tokens, t, rotary=rotary, context=context, context_mask=context_mask)[:, : latents.shape[1]]
    target = noise - latents
    return F.mse_loss(pred.float(), target.float())
