"""Layer norm, attention to a caption's states and coded activations together, as a model and the example run them."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch
from torch.nn import functional as F

from moss_image_b200 import _lib
from moss_image_b200.activation_codes import coded_weight_gradient, decode_activation, encode_activation
from moss_image_b200.dit import TextBranch, build_lora_model
from moss_image_b200.fp8 import FrozenFp8Linear
from moss_image_b200.lora import LoRALinear
from moss_image_b200.memory import place_model
from moss_image_b200.packed import cumulative_lengths
from moss_image_b200.quantization import FrozenInt8Linear

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "text_branch_finetune.py"
BF16 = torch.bfloat16


def _example():
    spec = importlib.util.spec_from_file_location("text_branch_finetune", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("coded", [True, False])
def test_the_example_runs(cuda_device, coded):
    losses = _example().finetune(depth=2, dim=256, heads=4, image_tokens=70, text_tokens=20, text_dim=96, batch=3, steps=3,
                                 lr=1e-4, device=cuda_device, coded=coded)
    assert len(losses) == 3 and all(math.isfinite(loss) for loss in losses)


def _branch(seed=0, dim=128, heads=4, text_dim=96, k_heads=2):
    torch.manual_seed(seed)
    branch = TextBranch(dim, heads, text_dim, k_heads)
    for linear in (branch.q, branch.k, branch.v, branch.o):
        torch.nn.init.normal_(linear.weight, 0.0, 0.1)
    torch.nn.init.normal_(branch.norm.weight, 1.0, 0.1)
    torch.nn.init.normal_(branch.norm.bias, 0.0, 0.1)
    return branch.to("cuda", BF16)


def _plain(branch, tokens, context, mask):
    """The branch in float64 torch."""
    w = {name: p.detach().double().requires_grad_() for name, p in branch.named_parameters()}
    heads, dim = branch.q.out_features // branch.head_dim, branch.head_dim
    h = F.layer_norm(tokens, tokens.shape[-1:], w["norm.weight"], w["norm.bias"], 1e-6)
    q = (h @ w["q.weight"].T).unflatten(-1, (-1, dim)).transpose(1, 2)
    k, v = ((context @ w[f"{n}.weight"].T).unflatten(-1, (-1, dim)).transpose(1, 2) for n in "kv")
    k, v = (t.repeat_interleave(heads // t.shape[1], 1) for t in (k, v))
    logits = (q @ k.mT * dim ** -0.5).masked_fill(~mask[:, None, None], -math.inf)
    p = torch.exp(logits - logits.amax(-1, keepdim=True).clamp_min(-1e300))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    return tokens + (p @ v).transpose(1, 2).flatten(2) @ w["o.weight"].T, w


@pytest.mark.parametrize("coded", [False, True])
def test_a_branch_against_float64(cuda_device, coded):
    branch = _branch()
    branch.coded_inputs = coded
    tokens = torch.randn(3, 150, 128, device="cuda").to(BF16).requires_grad_()
    context = torch.randn(3, 140, 96, device="cuda").to(BF16).requires_grad_()
    mask = torch.arange(140, device="cuda")[None] < torch.tensor([140, 33, 0], device="cuda")[:, None]
    dy = torch.randn(3, 150, 128, device="cuda").to(BF16)
    y = branch(tokens, context, mask)
    got = torch.autograd.grad(y, [tokens, context, *branch.parameters()], dy)
    exact_tokens, exact_context = (t.detach().double().requires_grad_() for t in (tokens, context))
    exact, w = _plain(branch, exact_tokens, exact_context, mask)
    expected = torch.autograd.grad(exact, [exact_tokens, exact_context, *w.values()], dy.double())
    # a chain of up to ten bf16 roundings, 2^-8 each in the worst place and a third of that in the 2-norm; the codes of an input
    # are within 1/127 of their block's largest value, a quarter of that in the 2-norm
    allowed = 10 / 3 * 2.0 ** -8 + (3 / 4 / 127 if coded else 0.0)
    assert (y.double() - exact).norm() <= allowed * exact.norm()
    for part, whole in zip(got, expected):
        assert (part.double() - whole).norm() <= allowed * whole.norm()


def test_packed_captions_agree_with_padded_ones(cuda_device):
    branch = _branch(1)
    lengths_q, lengths_k = [60, 40, 50], [30, 0, 77]
    stream = torch.randn(1, 150, 128, device="cuda").to(BF16)
    states = torch.randn(1, 107, 96, device="cuda").to(BF16)
    packed = branch(stream, states, cumulative_lengths(lengths_k, stream.device), cumulative_lengths(lengths_q, stream.device))
    at_q = at_k = 0
    for nq, nk in zip(lengths_q, lengths_k):
        one = branch(stream[:, at_q : at_q + nq], states[:, at_k : at_k + nk])
        assert (packed[:, at_q : at_q + nq] - one).abs().max() <= 2.0 ** -7 * one.abs().max()
        at_q, at_k = at_q + nq, at_k + nk


def test_adapters_keep_codes_of_their_input(cuda_device):
    torch.manual_seed(2)
    base = torch.nn.Linear(256, 192).to("cuda", BF16).requires_grad_(False)
    layer = LoRALinear(FrozenInt8Linear(base), 8, 16.0).to("cuda")
    torch.nn.init.normal_(layer.lora_B, std=0.05)
    x = torch.randn(2, 90, 256, device="cuda").to(BF16).requires_grad_()
    dy = torch.randn(2, 90, 192, device="cuda").to(BF16)
    coded = encode_activation(x)
    grads = []
    for codes in (None, coded):
        with torch.autocast("cuda", BF16):
            y = layer(x, codes)
        grads.append([y.detach(), *torch.autograd.grad(y, [x, layer.lora_B, layer.lora_A], dy)])
    assert all(torch.equal(a, b) for a, b in zip(grads[0][:3], grads[1][:3]))
    dyb = (dy.reshape(-1, 192) @ layer.lora_B.detach().to(BF16))
    assert torch.equal(grads[1][3], coded_weight_gradient(dyb, coded.codes, coded.exponents, torch.float32) * layer.scale)
    assert (grads[1][3] - grads[0][3]).norm() <= 0.02 * grads[0][3].norm()
    with pytest.raises(ValueError, match="not those"):
        layer(x, encode_activation(x[:1]))


def _gradients(model, tokens, t, **options):
    with torch.autocast("cuda", BF16):
        out = model(tokens, t, **options)
    out.float().square().mean().backward()
    grads = {name: p.grad.clone() for name, p in model.named_parameters() if p.grad is not None}
    model.zero_grad(set_to_none=True)
    return out.detach(), grads


def test_a_model_with_codes_checkpoints_and_offload(cuda_device):
    """The same gradients wherever the codes are kept; and near those of whole activations."""
    model = build_lora_model(2, device=cuda_device, dim=256, heads=4, mlp_dim=512, rank=8, seed=3, text_dim=96).train()
    for layer in model.layers:
        torch.nn.init.normal_(layer.text.o.weight, std=0.05)
        for name in ("q", "k", "v", "o"):
            torch.nn.init.normal_(layer.proj[name].lora_B, std=0.02)
    tokens = torch.randn(2, 40, 256, device="cuda").to(BF16)
    context = torch.randn(2, 24, 96, device="cuda").to(BF16)
    mask = torch.arange(24, device="cuda")[None] < torch.tensor([24, 5], device="cuda")[:, None]
    t = torch.tensor([0.2, 0.7], device="cuda")
    options = {"context": context, "context_mask": mask}
    whole_out, whole = _gradients(model, tokens, t, **options)
    without, _ = _gradients(model, tokens, t)
    assert not torch.equal(without, whole_out)  # the captions matter
    for layer in model.layers:
        layer.coded_inputs = layer.text.coded_inputs = True
    model.coded_checkpoints = True
    out, coded = _gradients(model, tokens, t, **options)
    assert torch.equal(out, whole_out) and coded.keys() == whole.keys()
    model.activation_offload = True
    out, offloaded = _gradients(model, tokens, t, **options)
    assert torch.equal(out, whole_out) and all(torch.equal(coded[name], offloaded[name]) for name in coded)
    # a coded input is within 0.6% (3/4 of 1/127, 2-norm), and a gradient of two blocks passes at most 16 of them
    for name, grad in whole.items():
        assert (coded[name].float() - grad.float()).norm() <= 0.1 * grad.float().norm() + 1e-12, name


def test_packed_model_with_captions(cuda_device):
    model = build_lora_model(2, device=cuda_device, dim=128, heads=2, mlp_dim=256, rank=4, seed=4, text_dim=64, coded=True).train()
    for layer in model.layers:
        torch.nn.init.normal_(layer.text.o.weight, std=0.05)
    samples = [torch.randn(n, 128, device="cuda").to(BF16) for n in (30, 50)]
    context = [torch.randn(n, 64, device="cuda").to(BF16) for n in (9, 0)]
    t = torch.tensor([0.4, 0.6], device="cuda")
    outs = model.forward_packed(samples, t, context=context)
    assert [o.shape[0] for o in outs] == [30, 50]
    sum(o.float().square().mean() for o in outs).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.layers[0].text.parameters())
    with pytest.raises(ValueError, match="one context"):
        model.forward_packed(samples, t, context=context[:1])


def test_decoded_checkpoint_input(cuda_device):
    """A checkpointed block's gradient is that of the block at the decoded input."""
    model = build_lora_model(1, device=cuda_device, dim=128, heads=2, mlp_dim=256, rank=4, seed=5).train()
    for name in ("q", "k", "v", "o"):
        torch.nn.init.normal_(model.layers[0].proj[name].lora_B, std=0.05)
    tokens = torch.randn(1, 24, 128, device="cuda").to(BF16)
    t = torch.tensor([0.5], device="cuda")
    leaf = tokens.clone().requires_grad_()
    model.coded_checkpoints = True
    with torch.autocast("cuda", BF16):
        out = model(leaf * 1.0, t)
    dy = torch.randn_like(out)
    got = torch.autograd.grad(out, leaf, dy)[0]
    model.coded_checkpoints = False
    near = decode_activation(encode_activation(tokens)).requires_grad_()
    with torch.autocast("cuda", BF16):
        block = model.layers[0](near, model.time_embedding(t).to(BF16))
        whole = model.layers[0](tokens, model.time_embedding(t).to(BF16)).detach().requires_grad_()
        normed = model.final_norm(whole)
    inner = torch.autograd.grad(normed, whole, dy)[0]
    assert torch.equal(got, torch.autograd.grad(block, near, inner)[0])


@pytest.mark.parametrize("mode,text_dim", [("sync", 96), ("async", None)])
def test_swapped_and_streamed_blocks_keep_codes_too(cuda_device, mode, text_dim):
    """The same gradients wherever a block's parameters are, its checkpointed input kept as codes, with a text branch in it."""
    tokens = torch.randn(2, 40, 128, device="cuda").to(BF16)
    options = {} if text_dim is None else {"context": torch.randn(2, 24, text_dim, device="cuda").to(BF16)}
    t = torch.tensor([0.2, 0.7], device="cuda")
    results = []
    for blocks in (0, 2):
        model = build_lora_model(2, device=cuda_device, dim=128, heads=2, mlp_dim=256, rank=4, seed=6, text_dim=text_dim).train()
        for layer in model.layers:
            for name in ("q", "k", "v", "o"):
                torch.nn.init.constant_(layer.proj[name].lora_B, 0.01)
            if text_dim is not None:
                torch.nn.init.constant_(layer.text.o.weight, 0.02)
        model.coded_checkpoints = True
        place_model(model, cuda_device, blocks, block_swap_mode=mode)
        before = _lib.launch_counts.get("codes", 0)
        out, grads = _gradients(model, tokens, t, **options)
        # an encode and a decode for each block whose input is looked at again
        results.append((out, {name: grad.to(cuda_device) for name, grad in grads.items()}, _lib.launch_counts.get("codes", 0) - before))
    resident, placed = results
    assert resident[2] == placed[2] >= 4 and torch.equal(resident[0], placed[0]) and resident[1].keys() == placed[1].keys()
    assert all(torch.equal(resident[1][name], placed[1][name]) for name in resident[1])


def _held(run) -> int:
    """Bytes that a forward pass leaves in use, its result among them (as asked for: the allocator rounds by a megabyte)."""
    run()  # (workspaces and lazily made buffers are there)
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    kept = run()
    after = torch.cuda.memory_stats()["requested_bytes.all.current"]
    del kept
    return after - before


@pytest.mark.parametrize("packed", [False, True])
def test_coded_inputs_hold_less(cuda_device, packed):
    """What a branch and a block keep for the backward pass is less with codes, by about half of each input that is coded."""
    tokens = torch.randn(1, 4096, 512, device="cuda").to(BF16).requires_grad_()
    context = torch.randn(1, 3000, 256, device="cuda").to(BF16)
    bounds = (cumulative_lengths([1000, 2000], tokens.device), cumulative_lengths([2000, 2096], tokens.device)) if packed else (None, None)
    branch = _branch(3, dim=512, heads=8, text_dim=256)
    branches = []
    for coded in (False, True):
        branch.coded_inputs = coded
        branches.append(_held(lambda: branch(tokens, context, *bounds)))
    saved = tokens.numel() * (2 - 33 / 32)
    assert abs(branches[0] - branches[1] - saved) < 0.02 * saved
    block = build_lora_model(1, device=cuda_device, dim=512, heads=8, mlp_dim=1024, rank=8, seed=7).train().layers[0]
    cond = torch.randn(2 if packed else 1, 512, device="cuda").to(BF16)
    blocks = []
    for coded in (False, True):
        block.coded_inputs = coded
        with torch.autocast("cuda", BF16):
            blocks.append(_held(lambda: block(tokens, cond, bounds[1])))
    copies = 2 if packed else 1  # q, k and v's input; and o's, where the attention's outputs are joined to one
    assert abs(blocks[0] - blocks[1] - copies * saved) < 0.02 * saved


def _kept(layer, x, codes):
    """What a call keeps of its tokens, by dtype, with its gradients."""
    kept = []

    def note(t):
        if t.numel() == x.numel():
            kept.append(t.dtype)
        return t

    with torch.autograd.graph.saved_tensors_hooks(note, lambda t: t):
        y = layer(x, codes)
    return set(kept), torch.autograd.grad(y.float().square().sum(), [x, layer.lora_A, layer.lora_B])


@pytest.mark.parametrize("base", ["int8", "fp8", "dense"])
def test_adapters_on_any_base_keep_codes_where_they_say_so(cuda_device, base):
    torch.manual_seed(8)
    linear = torch.nn.Linear(256, 192).to("cuda", BF16).requires_grad_(False)
    linear = {"int8": FrozenInt8Linear, "fp8": FrozenFp8Linear, "dense": lambda x: x}[base](linear)
    layer = LoRALinear(linear, 8, 16.0).to("cuda")
    layer.lora_A.data, layer.lora_B.data = layer.lora_A.data.float(), torch.randn(192, 8, device="cuda") * 0.05
    x = torch.randn(90, 256, device="cuda").to(BF16).requires_grad_()
    coded = encode_activation(x)
    with torch.autocast("cuda", BF16):
        assert layer.keeps_codes(x)
        kept, grads = _kept(layer, x, coded)
        whole_kept, whole = _kept(layer, x, None)
    assert kept == {torch.int8} and whole_kept == {BF16}
    assert torch.equal(grads[0], whole[0]) and torch.equal(grads[2], whole[2])
    # a decoded input is within 1/127 of its block's largest value, a quarter of that in the 2-norm; the gradient is linear in it
    assert 0 < (grads[1] - whole[1]).norm() <= 0.02 * whole[1].norm()
    # float32 products: the tokens are kept, and the codes not used
    assert not layer.keeps_codes(x)
    kept, grads = _kept(layer, x, coded)
    assert torch.int8 not in kept and torch.equal(grads[1], _kept(layer, x, None)[1][1])
    layer.lora_A.requires_grad_(False)
    with torch.autocast("cuda", BF16), torch.no_grad():
        assert not layer.keeps_codes(x)


@pytest.mark.parametrize("frozen,autocast,expected", [("int8", True, 2), ("fp8", True, 2), ("int8", False, 0), ("fp8", False, 0)])
def test_blocks_encode_only_what_a_projection_keeps(cuda_device, frozen, autocast, expected):
    model = build_lora_model(1, device=cuda_device, dim=256, heads=4, mlp_dim=512, rank=8, seed=9, frozen=frozen).train()
    block = model.layers[0]
    block.coded_inputs = True
    bounds = cumulative_lengths([30, 50], torch.device("cuda"))
    tokens, cond = torch.randn(1, 80, 256, device="cuda").to(BF16), torch.randn(2, 256, device="cuda").to(BF16)
    before = _lib.launch_counts.get("codes", 0)
    with torch.autocast("cuda", BF16, enabled=autocast):
        block(tokens, cond, bounds)
    assert _lib.launch_counts.get("codes", 0) - before == expected  # q, k and v's input, and o's


def test_a_branch_with_float32_masters_runs_without_codes(cuda_device):
    branch = _branch(5).float()
    tokens, context = (torch.randn(2, n, c, device="cuda").to(BF16).requires_grad_() for n, c in ((40, 128), (30, 96)))
    results = []
    for coded in (False, True):
        branch.coded_inputs = coded
        with torch.autocast("cuda", BF16):
            y = branch(tokens, context)
        results.append([y, *torch.autograd.grad(y.float().square().sum(), [tokens, *branch.parameters()])])
    assert all(torch.equal(a, b) for a, b in zip(*results))
