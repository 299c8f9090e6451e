"""Rotary positions against their formula in 64 bits, and together with cross attention in a layer."""

from __future__ import annotations

import math

import pytest
import torch

from deformops_b200 import NoBackendError
from deformops_b200.nn import RotaryCrossAttn
from deformops_b200.registry import Backend, rotary
from tests.test_cross_attention import TYPES, masks


def turned(x, positions, sections, base=10000.0, interleaved=False, joint=False, inverse=False):
    x, positions = x.double(), positions.double()
    if positions.dim() == 2:
        positions = positions.unsqueeze(0)
    total, done, out = sum(sections), 0, x.clone()
    for axis, count in enumerate(sections):
        for i in range(count):
            j = done + i
            angle = positions[:, :, axis, None] * (base ** (-j / total) if joint else base ** (-i / count))
            c, s = angle.cos(), angle.sin() * (-1 if inverse else 1)
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + total)
            out[..., a] = x[..., a] * c - x[..., b] * s
            out[..., b] = x[..., a] * s + x[..., b] * c
        done += count
    return out


def bound(x, want, sections, interleaved):
    """Half a step for the result; sine, cosine and the angle 2^-22 each, two products and a sum 2^-23."""
    u = torch.finfo(x.dtype).eps / 2
    size = x.double().abs()
    pairs = sum(sections)
    both = size.clone()
    if interleaved:
        both[..., :2 * pairs] = (size[..., 0:2 * pairs:2] + size[..., 1:2 * pairs:2]).repeat_interleave(2, -1)
    else:
        both[..., :2 * pairs] = (size[..., :pairs] + size[..., pairs:2 * pairs]).repeat(1, 1, 1, 2)
    return 1.01 * u * want.abs() + 4 * 2.0 ** -22 * both + torch.finfo(x.dtype).tiny


CASES = [  # B, N, G, D, sections, interleaved, joint
    (1, 1, 1, 2, (1,), False, False), (2, 7, 8, 32, (8, 8), False, False), (2, 333, 8, 32, (8, 8), True, False),
    (1, 50, 3, 128, (16, 24, 24), False, True), (3, 19, 4, 80, (10, 15, 15), True, False),
    (1, 65, 5, 26, (3, 5), False, False), (1, 65, 5, 27, (3, 5), True, False), (2, 9, 2, 40, (0, 16), False, False),
    (1, 4, 2, 256, (64, 64), False, False), (1, 2100, 1, 64, (32,), False, False), (2, 11, 2, 24, (0, 0), False, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_values_and_gradients(case, dtype):
    B, N, G, D, sections, interleaved, joint = case
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(B, N, G, D, generator=gen, device="cuda").to(dtype).requires_grad_()
    grad = torch.randn(B, N, G, D, generator=gen, device="cuda").to(dtype)
    for positions in (200 * torch.randn(B, N, len(sections), generator=gen, device="cuda"),
                      torch.randint(-5, 3000, (N, len(sections)), generator=gen, device="cuda"),
                      torch.randint(0, 1 << 20, (B, N, len(sections)), generator=gen, device="cuda").int(),
                      1e6 + torch.rand(N, len(sections), generator=gen, device="cuda").double()):
        options = {"sections": sections, "interleaved": interleaved, "joint": joint}
        out = rotary(x, positions, **options)
        want = turned(x.detach(), positions, sections, interleaved=interleaved, joint=joint)
        assert out.dtype == dtype and out.is_contiguous()
        assert ((out.double() - want).abs() <= bound(x.detach(), want, sections, interleaved)).all()
        (back,) = torch.autograd.grad(out, x, grad)
        want = turned(grad, positions, sections, interleaved=interleaved, joint=joint, inverse=True)
        assert ((back.double() - want).abs() <= bound(grad, want, sections, interleaved)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_alignment(dtype, interleaved):
    x = torch.randn(2, 30, 4, 32, device="cuda").to(dtype)
    positions = torch.rand(2, 30, 2, device="cuda") * 50
    want = rotary(x, positions, interleaved=interleaved)
    odd = torch.zeros(2, 30, 4, 35, dtype=dtype, device="cuda")
    odd[..., 1:33] = x
    shifted = torch.zeros(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape).copy_(x)
    wide = positions.repeat_interleave(2, 1)[:, ::2]
    for view in (odd[..., 1:33], x.transpose(1, 2).contiguous().transpose(1, 2), shifted,
                 x.transpose(1, 3).contiguous().transpose(1, 3)):
        assert torch.equal(rotary(view, wide, interleaved=interleaved), want)
    # one set of positions for all samples
    assert torch.equal(rotary(x, positions[0], interleaved=interleaved),
                       rotary(x, positions[:1].expand(2, -1, -1), interleaved=interleaved))


@pytest.mark.gpu
def test_far_positions():
    """At 2^31 an angle formed in 32 bits is wrong altogether; in 64 it is 2^-20 off."""
    x = torch.randn(1, 4, 2, 64, device="cuda")
    positions = torch.tensor([[2 ** 31 - 1], [2 ** 30 + 7], [-2 ** 31], [12345678901]], device="cuda")
    want = turned(x, positions, (32,))
    assert (rotary(x, positions).double() - want).abs().max() < 2e-5


@pytest.mark.gpu
def test_both_call_paths_agree_and_twice_differentiable():
    x = torch.randn(2, 30, 4, 32, device="cuda", requires_grad=True)
    positions = torch.rand(30, 2, device="cuda") * 50
    want = rotary(x, positions)
    plan = {"frequencies": [10000.0 ** (-i / 8) for i in range(8)] * 2, "axes": [0] * 8 + [1] * 8}
    got = torch.ops.deformops_b200.rotary_turn(x, positions, plan["frequencies"], plan["axes"], False, False)
    assert torch.equal(got, want)
    assert torch.equal(rotary(x, positions, backend=Backend.CUDA, sections=[8, 8]), want)
    compiled = torch.compile(lambda t: rotary(t, positions), backend="eager", fullgraph=True)
    assert torch.equal(compiled(x), want)
    for out in (want, got):
        weight = torch.randn_like(x, requires_grad=True)
        (first,) = torch.autograd.grad(out, x, weight, create_graph=True)
        (second,) = torch.autograd.grad(first, weight, torch.ones_like(first))
        assert torch.allclose(second, rotary(torch.ones_like(x), positions), atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 5, 2, 32), (2, 0, 2, 32)])
def test_empty(shape):
    x = torch.zeros(*shape, device="cuda", requires_grad=True)
    out = rotary(x, torch.zeros(shape[1], 2, device="cuda"))
    assert out.shape == shape
    assert torch.autograd.grad(out.sum(), x)[0].shape == shape


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x, p = torch.zeros(1, 3, 2, 32, device="cuda"), torch.zeros(3, 2, device="cuda")
    with pytest.raises(ValueError, match="one device"):
        rotary(x, p.cpu())
    with pytest.raises(ValueError, match="detach"):
        rotary(x, p.requires_grad_())
    with pytest.raises(NoBackendError, match="at most 128"):
        rotary(torch.zeros(1, 3, 2, 320, device="cuda"), p.detach(), sections=(80, 80))
    with pytest.raises(NoBackendError, match="float64"):
        rotary(x.double(), p.detach())


@pytest.mark.parametrize("x, positions, options, message", [
    ((3, 2, 32), (3, 2), {}, "x must have 4"),
    ((1, 3, 2, 32), (3,), {"sections": (16,)}, "positions must have"),
    ((1, 3, 2, 32), (4, 2), {}, "tokens of x"),
    ((2, 3, 2, 32), (1, 3, 2), {}, "batch of x"),
    ((1, 3, 2, 32), (3, 3), {}, "pass sections"),
    ((1, 3, 2, 32), (3, 2), {"sections": (16,)}, "one axis per section"),
    ((1, 3, 2, 32), (3, 2), {"sections": (9, 8)}, "at most 16"),
    ((1, 3, 2, 32), (3, 2), {"sections": (-1, 8)}, "negative"),
])
def test_refusals(x, positions, options, message):
    with pytest.raises(ValueError, match=message):
        rotary(torch.zeros(x), torch.zeros(positions), **options)


def test_refusals_without_a_gpu():
    x, p = torch.zeros(1, 3, 2, 32), torch.zeros(3, 2)
    with pytest.raises(NoBackendError, match="no CPU path"):
        rotary(x, p)
    with pytest.raises(NoBackendError, match="not part of this build"):
        rotary(x, p, backend=Backend.TRITON)
    with pytest.raises(ValueError, match="float32, float64"):
        rotary(x, p.half())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layer_is_its_parts(dtype):
    """Pixels of two levels and queries with places of their own, one step of training: the layer's result and
    gradients are those of rotation, attention and projections in 64 bits, within the attention's own bounds."""
    torch.manual_seed(0)
    layer = RotaryCrossAttn(64, 48, num_heads=4, num_kv_heads=2, sections=(4, 4)).cuda().to(dtype)
    B, Q, levels = 2, 37, [(12, 9), (6, 5)]
    S = sum(h * w for h, w in levels)
    places = torch.cat([torch.stack(torch.meshgrid(torch.arange(h, device="cuda") + 0.5, torch.arange(w, device="cuda") + 0.5,
                                                   indexing="ij"), -1).view(-1, 2) for h, w in levels])
    q = torch.randn(B, Q, 64, device="cuda").to(dtype).requires_grad_()
    memory = torch.randn(B, S, 48, device="cuda").to(dtype).requires_grad_()
    centres = torch.rand(B, Q, 2, device="cuda") * 12
    padding = masks("padding", B, Q, S, 4)["key_padding_mask"]
    out = layer(q, memory, centres, places, key_padding_mask=padding)
    do = torch.randn_like(out)
    grads = torch.autograd.grad(out, [q, memory, *layer.parameters()], do)
    wide = RotaryCrossAttn(64, 48, num_heads=4, num_kv_heads=2, sections=(4, 4)).cuda().double()
    wide.load_state_dict({n: t.double() for n, t in layer.state_dict().items()})
    q64, m64 = (t.detach().double().requires_grad_() for t in (q, memory))
    seen = {}
    for name in ("proj_query", "proj_key", "proj_value", "proj_output"):
        def keep(module, inputs, result, name=name):
            seen[name] = [inputs[0].detach().flatten(0, 1).abs()]
            result.register_hook(lambda g: seen[name].append(g.flatten(0, 1).abs()))
        getattr(wide, name).register_forward_hook(keep)
    rotate = lambda x, p: _turn_graph(x, p, (4, 4))  # noqa: E731
    query = rotate(wide.proj_query(q64).view(B, Q, 4, 16), centres)
    key = rotate(wide.proj_key(m64).view(B, S, 2, 16), places.expand(B, S, 2))
    value = wide.proj_value(m64).view(B, S, 2, 16)
    scores = torch.einsum("bqghd,bsgd->bghqs", query.view(B, Q, 2, 2, 16), key) / 4
    weights = torch.softmax(scores.masked_fill(padding.view(B, 1, 1, 1, S), -math.inf), -1)
    want = wide.proj_output(torch.einsum("bghqs,bsgd->bqghd", weights, value).reshape(B, Q, 64))
    grads64 = torch.autograd.grad(want, [q64, m64, *wide.parameters()], do.double())
    # each of about ten roundings along the way is half a step of values of the result's own size; a
    # parameter's gradient is a sum over tokens, off by that of what is summed
    limit = 10 * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2e-5
    sizes = [want, *grads64[:2]]
    for name, _ in wide.named_parameters():
        x, g = seen[name.split(".")[0]]
        sizes.append(g.T @ x if name.endswith("weight") else g.sum(0))
    for a, b, size in zip([out, *grads], [want, *grads64], sizes):
        assert (a.double() - b).norm() <= limit * size.norm()


def _turn_graph(x, positions, sections):
    pairs = sum(sections)
    angle = torch.cat([positions[..., a, None].double() * torch.pow(10000.0, -torch.arange(n, device=x.device).double() / n)
                       for a, n in enumerate(sections)], -1).unsqueeze(2)
    a, b = x[..., :pairs], x[..., pairs:2 * pairs]
    return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), x[..., 2 * pairs:]], -1)


def test_layer_refuses_sizes():
    for options in ({"num_heads": 5}, {"num_heads": 4, "num_kv_heads": 3}, {"num_heads": 0}):
        with pytest.raises(ValueError):
            RotaryCrossAttn(64, **options)



@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", [torch.float32, torch.float64], ids=str)
def test_far_float_positions(dtype, kind):
    """A product in 64 bits is 2^-53 of its turns off, and the frequency as much: pi 2^-51 of the largest position in all, and the
    reduced angle 2^-22 as near the origin."""
    x = torch.randn(1, 12, 2, 64, device="cuda").to(dtype)
    far = torch.tensor([3e5, 6.5e6, 6.6e6, 1e8, -2.5e8, 1e9, 2.0 ** 31, -1e10, 12345678901.0, 1e11, 1e12, -1e12], device="cuda", dtype=kind)
    want = turned(x, far.view(-1, 1), (32,))
    off = (rotary(x, far.view(-1, 1)).double() - want).abs()
    size = x.double().abs()
    size = (size[..., :32] + size[..., 32:]).repeat(1, 1, 1, 2)
    limit = bound(x, want, (32,), False) + size * (far.double().abs() * 2.0 ** -51 * 3.15).view(1, -1, 1, 1)
    assert (off <= limit).all()
    # whatever they are, the pairs keep their lengths
    huge = torch.tensor([1e15, -1e20, 3e38], device="cuda", dtype=kind).view(-1, 1)
    out = rotary(x[:, :3], huge).double()
    length = lambda t: (t[..., :32] ** 2 + t[..., 32:] ** 2).sqrt()  # noqa: E731
    assert ((length(out) / length(x[:, :3].double()) - 1).abs() <= 2 * torch.finfo(dtype).eps + 2.0 ** -20).all()
