"""Rotary positions, fp8 frozen linears and the Muon optimiser together, as the example runs them."""

from __future__ import annotations

import copy
import importlib.util
from pathlib import Path

import pytest
import torch

from moss_image_b200.dit import SyntheticBlock, build_lora_model
from moss_image_b200.fp8 import FrozenFp8Linear
from moss_image_b200.lora import LoRALinear
from moss_image_b200.memory import place_model
from moss_image_b200.rotary import rotary_frequencies, rotary_table

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "fp8_muon_finetune.py"


def _example():
    spec = importlib.util.spec_from_file_location("fp8_muon_finetune", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_learns_its_batch(cuda_device):
    losses = _example().finetune(depth=2, dim=256, heads=4, side=8, text_tokens=16, batch=2, steps=12, lr=4e-3,
                                 device=cuda_device)
    # small steps along descent directions lower the loss of the batch they were taken on
    assert all(loss == loss for loss in losses)
    assert sum(losses[-3:]) < sum(losses[:3])


def test_lora_over_fp8_with_positions_offload_and_checkpointing(cuda_device):
    """The same gradients with and without saved-activation offload, and a position that matters."""
    model = build_lora_model(2, device=cuda_device, dim=256, heads=4, mlp_dim=512, rank=8, seed=3, frozen="fp8").train()
    assert isinstance(model.layers[0].proj["q"], LoRALinear) and isinstance(model.layers[0].proj["q"].base, FrozenFp8Linear)
    for layer in model.layers:
        for name in ("q", "k", "v", "o"):
            torch.nn.init.normal_(layer.proj[name].lora_B, std=0.02)
    tokens = torch.randn(2, 40, 256, device=cuda_device, dtype=torch.bfloat16)
    t = torch.tensor([0.2, 0.7], device=cuda_device)
    rotary = rotary_table(torch.arange(40, device=cuda_device), rotary_frequencies(64, device=cuda_device))
    trained = [p for p in model.parameters() if p.requires_grad]
    grads = []
    for offload in (False, True):
        model.activation_offload = offload
        model(tokens, t, rotary=rotary).float().square().mean().backward()
        grads.append([p.grad.clone() for p in trained])
        for p in trained:
            p.grad = None
    assert all(torch.equal(a, b) and a.isfinite().all() for a, b in zip(*grads))
    model.activation_offload = False
    with torch.no_grad():
        still = model(tokens, t, rotary=(torch.ones_like(rotary[0]), torch.zeros_like(rotary[1])))
        plain = model(tokens, t)
        turned = model(tokens, t, rotary=rotary)
    assert torch.equal(still, plain) and not torch.equal(turned, plain)


def test_streamed_fp8_blocks_with_positions(cuda_device):
    """Blocks whose fp8 codes stream from pinned host memory give the resident model's gradients."""
    resident, streamed = (build_lora_model(3, device=cuda_device, dim=128, heads=2, mlp_dim=256, rank=4, seed=5,
                                           frozen="fp8").train() for _ in range(2))
    for model in (resident, streamed):
        gen = torch.Generator(device=cuda_device).manual_seed(6)
        for layer in model.layers:
            for name in ("q", "k", "v", "o"):
                layer.proj[name].lora_B.data.normal_(0.0, 0.03, generator=gen)
    place_model(resident, cuda_device, 0)
    place_model(streamed, cuda_device, 2, block_swap_mode="async")
    tokens = torch.randn(2, 24, 128, device=cuda_device, dtype=torch.bfloat16)
    t = torch.tensor([0.3, 0.6], device=cuda_device)
    rotary = rotary_table(torch.arange(24, device=cuda_device), rotary_frequencies(64, device=cuda_device))
    outputs = [model(tokens, t, rotary=rotary) for model in (resident, streamed)]
    assert torch.equal(*outputs)
    for output in outputs:
        output.float().square().mean().backward()
    for a, b in zip(resident.parameters(), streamed.parameters()):
        assert (a.grad is None) == (b.grad is None)
        if a.grad is not None:
            assert torch.equal(a.grad, b.grad.to(a.grad.device))
    streamed.block_swap_manager.close()


def test_frozen_format_is_checked(cuda_device):
    with pytest.raises(ValueError, match="int8 or fp8"):
        build_lora_model(1, device=cuda_device, dim=64, heads=1, mlp_dim=64, frozen="fp4")
    assert SyntheticBlock(64, 1, 128).heads == 1


@pytest.mark.parametrize("mode", ["sync", "async"])
def test_swapped_fp8_blocks_of_any_width(cuda_device, mode):
    """Input widths that are no multiple of 16 (codes with padded rows), on the CPU or in a pinned master."""
    resident, swapped = (build_lora_model(3, device=cuda_device, dim=104, heads=2, mlp_dim=200, rank=4, seed=7,
                                          frozen="fp8").train() for _ in range(2))
    for model in (resident, swapped):
        gen = torch.Generator(device=cuda_device).manual_seed(8)
        for layer in model.layers:
            for name in ("q", "k", "v", "o"):
                layer.proj[name].lora_B.data.normal_(0.0, 0.03, generator=gen)
    place_model(resident, cuda_device, 0)
    place_model(swapped, cuda_device, 2, block_swap_mode=mode)
    tokens = torch.randn(2, 24, 104, device=cuda_device, dtype=torch.bfloat16)
    t = torch.tensor([0.3, 0.6], device=cuda_device)
    rotary = rotary_table(torch.arange(24, device=cuda_device), rotary_frequencies(52, device=cuda_device))
    outputs = [model(tokens, t, rotary=rotary) for model in (resident, swapped)]
    assert torch.equal(*outputs)
    for output in outputs:
        output.float().square().mean().backward()
    for a, b in zip(resident.parameters(), swapped.parameters()):
        assert (a.grad is None) == (b.grad is None)
        if a.grad is not None:
            assert torch.equal(a.grad, b.grad.to(a.grad.device))
    if swapped.block_swap_manager is not None:
        swapped.block_swap_manager.close()


def test_fp8_codes_keep_their_rows_through_moves_and_checkpoints(cuda_device):
    torch.manual_seed(9)
    linear = torch.nn.Linear(100, 70, device=cuda_device, dtype=torch.bfloat16).requires_grad_(False)
    module = FrozenFp8Linear(linear)
    x = torch.randn(5, 100, device=cuda_device, dtype=torch.bfloat16)
    want = module(x)
    assert module.weight_fp8.shape == (70, 100)
    state = {name: value.detach().cpu().contiguous() for name, value in module.state_dict().items()}
    assert list(state) == ["weight_fp8", "weight_scale", "bias"] and state["weight_fp8"].shape == (70, 100)
    other = FrozenFp8Linear(torch.nn.Linear(100, 70, device=cuda_device, dtype=torch.bfloat16).requires_grad_(False))
    for assign in (False, True):
        on_device = {name: value.to(cuda_device) for name, value in state.items()}
        assert not any(other.load_state_dict(on_device if assign else state, assign=assign))
        assert torch.equal(other(x), want)
    with pytest.raises(RuntimeError, match="weight_fp8"):
        other.load_state_dict({name: value for name, value in state.items() if name != "weight_fp8"})
    with pytest.raises(RuntimeError, match="weight_fp8"):
        other.load_state_dict({**state, "weight_fp8": state["weight_fp8"][:, :96]})
    assert torch.equal(other.cpu().to(cuda_device)(x), want)
    assert torch.equal(copy.deepcopy(other)(x), want)
    again = FrozenFp8Linear.from_codes(state["weight_fp8"].to(cuda_device), state["weight_scale"].to(cuda_device),
                                       state["bias"].to(cuda_device))
    assert torch.equal(again(x), want)


@pytest.mark.parametrize("frozen", ["int8", "fp8"])
def test_positions_in_a_packed_batch(cuda_device, frozen):
    from moss_image_b200.dit import packed_flow_matching_loss

    model = build_lora_model(2, device=cuda_device, dim=256, heads=4, mlp_dim=512, rank=8, seed=3, frozen=frozen).eval()
    lengths = (37, 5, 64)
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    samples = [torch.randn(n, 256, generator=gen, device=cuda_device).bfloat16() for n in lengths]
    t = torch.tensor([0.1, 0.5, 0.9], device=cuda_device)
    frequencies = rotary_frequencies(64, device=cuda_device)
    places = [torch.arange(n, device=cuda_device) for n in lengths]
    rotary = rotary_table(torch.cat(places), frequencies)
    with torch.no_grad():
        packed = model.forward_packed(samples, t, rotary=rotary)
        for i, (sample, own) in enumerate(zip(samples, places)):
            alone = model(sample[None], t[i:i + 1], rotary=rotary_table(own, frequencies))[0]
            # the same arithmetic through other kernels: bfloat16 roundings of two blocks
            assert float((packed[i].float() - alone.float()).norm() / alone.float().norm()) < 2e-2
        still = model.forward_packed(samples, t, rotary=(torch.ones_like(rotary[0]), torch.zeros_like(rotary[1])))
        plain = model.forward_packed(samples, t)
        assert all(torch.equal(a, b) for a, b in zip(still, plain))
        assert not torch.equal(packed[0], plain[0])
        moved = rotary_table(torch.cat([places[0], places[1], 7 * places[2]]), frequencies)
        other = model.forward_packed(samples, t, rotary=moved)
        assert torch.equal(other[0], packed[0]) and torch.equal(other[1], packed[1]) and not torch.equal(other[2], packed[2])
    for wrong in ((rotary[0][:-1], rotary[1][:-1]), rotary_table(torch.arange(200, device=cuda_device), frequencies)):
        with pytest.raises(ValueError, match="packed"):
            model.forward_packed(samples, t, rotary=wrong)
    model.train()
    latents, text = [s[:-2] for s in samples], [s[-2:] for s in samples]
    noise = [torch.randn(*x.shape, generator=gen, device=cuda_device).bfloat16() for x in latents]
    loss = packed_flow_matching_loss(model, latents, text, t, noise, rotary=rotary)
    loss.backward()
    assert loss.isfinite() and not torch.equal(loss, packed_flow_matching_loss(model, latents, text, t, noise))


def test_the_callers_tables_are_not_marked_and_strided_ones_stay_resident(cuda_device):
    from moss_image_b200.activation_offload import KEEP_RESIDENT, offload_ring

    model = build_lora_model(2, device=cuda_device, dim=256, heads=4, mlp_dim=512, rank=8, seed=3, frozen="fp8").train()
    model.gradient_checkpointing = False
    model.activation_offload = True
    tokens = torch.randn(1, 40, 256, device=cuda_device, dtype=torch.bfloat16)
    t = torch.tensor([0.4], device=cuda_device)
    dense = rotary_table(torch.arange(40, device=cuda_device), rotary_frequencies(64, device=cuda_device))
    strided = tuple(table.t().contiguous().t() for table in dense)
    ring = offload_ring(cuda_device)
    sent = []
    for tables in (dense, strided):
        before = ring.stats()["d2h_bytes"]
        model(tokens, t, rotary=tables).float().square().mean().backward()
        sent.append(ring.stats()["d2h_bytes"] - before)
        assert not any(hasattr(table, KEEP_RESIDENT) for table in tables)
    assert sent[0] == sent[1] > 0


def test_calls_run_on_their_tensors_device_whatever_the_current_one(cuda_device, monkeypatch):
    """Every entry point of these operators switches to the device of its tensors where another is current."""
    from moss_image_b200 import _lib
    from moss_image_b200.fp8 import fp8_linear_backward, fp8_linear_forward, quantize_fp8_rows, quantize_fp8_weight
    from moss_image_b200.muon import orthogonalize
    from moss_image_b200.rotary import apply_rotary

    x = torch.randn(4, 128, device=cuda_device)
    cos = torch.zeros(4, 4, device=cuda_device)

    def everything():
        codes, scale = quantize_fp8_weight(x)
        quantize_fp8_rows(x)
        y = fp8_linear_forward(x, codes, scale)
        fp8_linear_backward(y, codes, scale)
        orthogonalize(x)
        apply_rotary(x.view(1, 4, 4, 32), x.view(1, 4, 4, 32), cos, cos)

    everything()
    entered = []
    index = cuda_device.index or 0
    current = [index]

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)
            current[0] = index

        def __exit__(self, *error):
            current[0] = index + 1
            return False

    monkeypatch.setattr(torch.cuda, "device", Guard)
    everything()
    assert not entered  # the right device is current: no switch
    monkeypatch.setattr(_lib, "current_device_index", lambda: current[0])
    current[0] = index + 1
    everything()
    assert len(entered) == 6 and all(torch.device(device) == cuda_device for device in entered)
