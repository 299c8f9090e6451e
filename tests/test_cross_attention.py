"""Cross attention against its formula in 64 bits, with bounds that count the roundings."""

from __future__ import annotations

import math

import pytest
import torch

from deformops_b200 import NoBackendError
from deformops_b200.registry import Backend, cross_attention

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(B, Q, S, G, K, D, dtype, seed=0, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(seed)
    draw = lambda *s: torch.randn(*s, generator=gen, device=device).to(dtype)  # noqa: E731
    return draw(B, Q, G, D), draw(B, S, K, D), draw(B, S, K, D), draw(B, Q, G * D)


def hidden_of(B, Q, S, G, padding, mask, device):
    """(B, G, Q, S): true where a state may not be seen."""
    hidden = torch.zeros(B, G, Q, S, dtype=torch.bool, device=device)
    if padding is not None:
        hidden |= padding.view(B, 1, 1, S)
    if mask is not None:
        hidden |= mask if mask.dim() == 4 else mask.view(-1, 1, Q, S)
    return hidden


def formula(q, k, v, do, padding=None, mask=None, scale=None):
    """Outputs, gradients and how far each may be off, all (value, bound) in 64 bits.

    With u half a step of the type and w = 2^-24: scores are sums of D products (float32 operands go
    through two terms of 11 bits: 2^-21 of a product), weights and ds are rounded to the type (not for
    float32), sums over n terms are n w off at most, and every result is rounded once.
    """
    B, Q, G, D = q.shape
    S, K = k.shape[1:3]
    dtype = q.dtype
    u, w = torch.finfo(dtype).eps / 2, 2.0 ** -24
    wide = dtype == torch.float32
    product = 2.0 ** -21 if wide else 0.0
    inner = 0.0 if wide else u
    scale = D ** -0.5 if scale is None else scale
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    q, do = q.transpose(1, 2), do.view(B, Q, G, D).transpose(1, 2)
    k, v = (t.transpose(1, 2).repeat_interleave(G // K, 1) for t in (k, v))
    hidden = hidden_of(B, Q, S, G, padding, mask, q.device)
    # what nobody may see is never used
    unused = hidden.all(2).unsqueeze(-1)
    shared = unused.view(B, K, G // K, S, 1).all(2).repeat_interleave(G // K, 1)
    k, v = k.masked_fill(shared, 0.0), v.masked_fill(shared, 0.0)
    some = ~hidden.all(-1, keepdim=True)
    s = (q @ k.transpose(-1, -2)) * scale
    p = torch.softmax(s.masked_fill(hidden, -1e300), -1) * some
    p = p.masked_fill(hidden, 0.0)
    size = (q.abs() @ k.abs().transpose(-1, -2)) * scale
    # of a weight, relative: its score's error and those of the sum (both sides), 2^-21 for each exponential
    # (2 ulp, and the score's own rounding at its size), S w for the sum
    off = ((D + 4) * w + product) * size.masked_fill(hidden, 0.0).amax(-1, keepdim=True)
    off = 2 * (off + 2.0 ** -21) + (S + 8) * w
    o = p @ v
    pv = p @ v.abs()
    eo = u * o.abs() + (off + inner + product + (S + 8) * w) * pv
    dp = do @ v.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = ((D + 4) * w + product) * (do.abs() @ v.abs().transpose(-1, -2))
    e_delta = (do.abs() * eo).sum(-1, keepdim=True) + (D + 4) * w * (do.abs() * o.abs()).sum(-1, keepdim=True)
    e_ds = p * (e_dp + e_delta) + (off + inner + product) * ds.abs()
    n = Q * (G // K) + 8
    dq = ds @ k * scale
    dk = ds.transpose(-1, -2) @ q * scale
    dv = p.transpose(-1, -2) @ do
    e_dq = u * dq.abs() + ((e_ds + (S + 8) * w * ds.abs()) @ k.abs()) * scale
    e_dk = ((e_ds + n * w * ds.abs()).transpose(-1, -2) @ q.abs()) * scale
    e_dv = ((off + inner + product + n * w) * p).transpose(-1, -2) @ do.abs()

    def heads(t):
        return t.view(B, K, G // K, S, D).sum(2).transpose(1, 2)

    tiny = torch.finfo(dtype).tiny
    dk, dv, e_dk, e_dv = map(heads, (dk, dv, e_dk, e_dv))
    e_dk, e_dv = e_dk + u * dk.abs(), e_dv + u * dv.abs()
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    pairs = ((back(o).reshape(B, Q, G * D), back(eo).reshape(B, Q, G * D)), (back(dq), back(e_dq)), (dk, e_dk), (dv, e_dv))
    # (products below the smallest normal number of 16-bit types are off by its half step)
    return [(x, 1.02 * e + tiny) for x, e in pairs]


def check(got, want, names=("out", "grad_query", "grad_key", "grad_value")):
    for name, x, (y, bound) in zip(names, got, want):
        x = x.detach().double()
        assert x.shape == y.shape, name
        worst = ((x - y).abs() / bound).max().item() if x.numel() else 0.0
        assert worst <= 1.0, f"{name} is {worst:.2f} of its bound off"


def run(q, k, v, do, **options):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = cross_attention(q, k, v, **options)
    return [out, *torch.autograd.grad(out, [q, k, v], do)]


def masks(kind, B, Q, S, G, device="cuda", seed=1):
    gen = torch.Generator(device=device).manual_seed(seed)
    draw = lambda *s: torch.rand(*s, generator=gen, device=device)  # noqa: E731
    padding = mask = None
    if "padding" in kind:
        padding = draw(B, S) < 0.4
        padding[:, S // 2:] |= draw(B, 1) < 0.5
    if "shared" in kind:
        mask = draw(Q, S) < 0.5
    elif "heads" in kind:
        mask = draw(B, G, Q, S) < 0.6
        mask[:, 0] = True                                    # a head that sees nothing
    elif "queries" in kind:
        mask = draw(B, Q, S) < 0.7
        mask[:, Q // 2] = True                               # a query that sees nothing
    if "none" in kind:
        padding = torch.ones(B, S, dtype=torch.bool, device=device)
    return {"key_padding_mask": padding, "attention_mask": mask}


SIZES = [  # B, Q, S, G, K, D, masks
    (1, 1, 1, 1, 1, 8, ""), (1, 1, 77, 8, 8, 64, ""), (3, 1, 1500, 8, 2, 128, "padding"), (2, 5, 129, 4, 4, 32, "queries"),
    (2, 16, 64, 8, 8, 32, ""), (1, 17, 300, 6, 3, 40, "heads"), (2, 100, 1344, 8, 8, 32, "padding"),
    (2, 100, 1000, 8, 8, 32, "queries"), (1, 300, 2311, 8, 8, 32, "padding queries"), (1, 129, 65, 4, 1, 96, "shared"),
    (2, 1000, 16, 2, 2, 64, "heads"), (1, 257, 513, 4, 2, 128, "padding"), (2, 33, 127, 2, 2, 16, "none"),
    (1, 640, 640, 3, 3, 64, ""), (1, 200, 130, 16, 4, 128, "queries"), (1, 2, 5000, 2, 2, 32, "padding"),
    (10, 40, 1000, 16, 16, 128, ""), (3, 130, 700, 60, 60, 128, ""), (10, 40, 1000, 16, 16, 64, ""), (5, 128, 128, 1, 1, 128, ""), (1, 70, 4099, 1, 1, 56, "padding"),
    # shared heads that do not divide a tile, or fill more than one; lists of many tiles
    (1, 50, 200, 6, 2, 128, "heads"), (2, 45, 333, 12, 2, 32, "padding queries"), (1, 9, 150, 70, 1, 64, "queries"), (1, 2, 140, 130, 1, 128, ""),
    (1, 3, 4000, 4, 1, 128, "heads"), (1, 4, 3001, 2, 1, 64, "heads"), (1, 20, 70001, 1, 1, 16, "padding"), (2, 300, 2200, 2, 1, 72, "padding queries"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_outputs_and_gradients(size, dtype):
    B, Q, S, G, K, D, kind = size
    q, k, v, do = make(B, Q, S, G, K, D, dtype)
    options = masks(kind, B, Q, S, G)
    want = formula(q, k, v, do, options["key_padding_mask"], options["attention_mask"])
    got = run(q, k, v, do, **options)
    assert all(t.dtype == dtype for t in got)
    check(got, want)
    with torch.no_grad():
        assert torch.equal(cross_attention(q, k, v, **options), got[0])
    again = run(q, k, v, do, **options)
    assert all(torch.equal(a, b) for a, b in zip(got, again))        # the same bits on every run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("Q", [1, 20, 150])
def test_states_that_nobody_sees_may_hold_anything(dtype, Q, D):
    B, S, G, K = 2, 1900, 4, 2
    q, k, v, do = make(B, Q, S, G, K, D, dtype)
    padding = torch.zeros(B, S, dtype=torch.bool, device="cuda")
    padding[0, 100:300] = True
    padding[0, 1700:] = True
    padding[1, 700::3] = True                       # whole tiles first
    clean = run(q, k, v, do, key_padding_mask=padding)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max):
        kb, vb = (t.masked_fill(padding.view(B, S, 1, 1), bad) for t in (k, v))
        got = run(q, kb, vb, do, key_padding_mask=padding)
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
        # the same through a mask of every query
        wide = padding.view(B, 1, S).expand(B, Q, S)
        assert all(torch.equal(a, b) for a, b in zip(run(q, kb, vb, do, attention_mask=wide), clean))
    assert all(torch.isfinite(t).all() for t in clean)
    assert clean[2].masked_select(padding.view(B, S, 1, 1)).eq(0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_nothing_to_see_is_zero(dtype):
    q, k, v, do = make(2, 40, 90, 2, 2, 32, dtype)
    hidden = torch.ones(2, 90, dtype=torch.bool, device="cuda")
    assert all(t.eq(0).all() for t in run(q, k, v, do, key_padding_mask=hidden))
    for shape in ((2, 0, 90), (0, 40, 90), (2, 40, 0)):
        B, Q, S = shape
        q, k, v, do = make(B, Q, S, 2, 2, 32, dtype)
        got = run(q, k, v, do)
        assert got[0].shape == (B, Q, 64) and all(t.eq(0).all() for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_large_scores(dtype):
    """Scores of hundreds: the maximum moves by more than an exponential's range from tile to tile."""
    q, k, v, do = make(1, 150, 700, 2, 2, 64, dtype)
    k = (k * torch.linspace(0.05, 8.0, 700, device="cuda").view(1, -1, 1, 1)).to(dtype)
    check(run(q, k, v, do, scale=0.5), formula(q, k, v, do, scale=0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("Q", [3, 130])
def test_strides(dtype, Q):
    B, S, G, K, D = 2, 200, 8, 4, 32
    q, k, v, do = make(B, Q, S, G, K, D, dtype)
    mask = masks("queries", B, Q, S, G)["attention_mask"]
    want = run(q, k, v, do, attention_mask=mask)
    packed = torch.stack([k, v], 2)                                    # keys and values side by side
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(B, S, K, D + 1, dtype=dtype, device="cuda")
    odd[..., :D] = k
    shifted = torch.zeros(v.numel() + 3, dtype=dtype, device="cuda")[3:].view(v.shape).copy_(v)
    turned = mask.transpose(1, 2).contiguous().transpose(1, 2)
    for a, b, c, m in ((q, packed[:, :, 0], packed[:, :, 1], mask), (heads_first, odd[..., :D], v, turned),
                       (q, k, shifted, mask.view(B, 1, Q, S).expand(B, G, Q, S))):
        got = run(a, b, c, do, attention_mask=m)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    # broadcast states: their gradient is the sum over the samples
    one = run(q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1), do)
    full = run(q, k[:1].repeat(B, 1, 1, 1), v[:1].repeat(B, 1, 1, 1), do)
    assert all(torch.equal(x, y) for x, y in zip(one, full))
    leaf = k[:1].clone().requires_grad_()
    out = cross_attention(q, leaf.expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1))
    (grad,) = torch.autograd.grad(out, leaf, do)
    assert torch.allclose(grad.double(), full[2].double().sum(0, keepdim=True), atol=4 * torch.finfo(dtype).eps * full[2].abs().max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("Q", [2, 70])
def test_one_state_or_one_head_for_all(dtype, Q, D):
    """Expanded operands: their strides are 0, and their gradients sums."""
    q, k, v, do = make(2, Q, 200, 4, 4, D, dtype)
    for of in ((slice(None), slice(0, 1)), (slice(0, 1),), (slice(None), slice(None), slice(0, 1))):
        a, b = k[of].expand_as(k), v[of].expand_as(v)
        check(run(q, a, b, do), formula(q, a, b, do))
        c = q[of].expand_as(q)
        check(run(c, k, v, do), formula(c, k, v, do))


@pytest.mark.gpu
def test_gradient_against_differences():
    """float32, along random directions: central differences with a step of 2^-6 are off by its square."""
    q, k, v, do = make(1, 6, 40, 4, 2, 16, torch.float32, seed=5)
    mask = masks("queries", 1, 6, 40, 4)["attention_mask"]
    grads = run(q, k, v, do, attention_mask=mask)[1:]
    for i in range(3):
        step = torch.randn_like((q, k, v)[i]) * 2.0 ** -6
        ends = []
        for sign in (1, -1):
            args = [q, k, v]
            args[i] = args[i] + sign * step
            ends.append((cross_attention(*args, attention_mask=mask).double() * do.double()).sum().item())
        slope = (ends[0] - ends[1]) / 2
        # third derivatives of a softmax-weighted mean are of the first one's order here
        assert abs(slope - (grads[i].double() * step.double()).sum().item()) < 2e-3 * step.norm().item() * grads[i].norm().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_both_call_paths_agree(dtype):
    q, k, v, do = make(2, 70, 150, 4, 2, 32, dtype)
    options = masks("padding queries", 2, 70, 150, 4)
    want = run(q, k, v, do, **options)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = torch.ops.deformops_b200.cross_attention_forward(*leaves, options["key_padding_mask"], options["attention_mask"],
                                                           32 ** -0.5)[0]
    got = [out, *torch.autograd.grad(out, leaves, do)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(cross_attention(q, k, v, backend=Backend.CUDA, **options), want[0])
    compiled = torch.compile(lambda *a: cross_attention(*a, **options), backend="eager", fullgraph=True)
    assert torch.equal(compiled(q, k, v), want[0])


@pytest.mark.gpu
def test_captured_and_replayed():
    q, k, v, do = make(2, 300, 1111, 8, 8, 32, torch.bfloat16)
    options = masks("padding queries", 2, 300, 1111, 8)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        out = cross_attention(*leaves, **options)
        return [out, *torch.autograd.grad(out, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        for t in leaves:
            t.mul_(0.5)
        options["key_padding_mask"].logical_not_()
    graph.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float32, 96)], ids=str)
def test_a_captured_run_of_calls(dtype, D):
    """Rotations, a pass over many rows and one over single tokens, one behind the other in one graph."""
    from deformops_b200.registry import rotary

    q, k, v, do = make(2, 150, 700, 4, 2, D, dtype)
    padding = masks("padding", 2, 150, 700, 4)["key_padding_mask"]
    places = torch.rand(700, 2, device="cuda") * 50
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        turned = rotary(k, places)
        out = cross_attention(rotary(q, places[:150]), turned, v, key_padding_mask=padding)
        token = cross_attention(out.view(2, 150, 4, D)[:, :1], turned, v)
        return [out, token, *torch.autograd.grad([out, token], leaves, [do, do[:, :1]])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    with torch.no_grad():
        for t in leaves:
            t.mul_(-0.75)
    torch.cuda.synchronize()
    # the two, at once on two streams: no workspace is shared
    streams = [torch.cuda.Stream() for _ in graphs]
    for stream, (graph, _) in zip(streams, graphs):
        with torch.cuda.stream(stream):
            graph.replay(), graph.replay()
    torch.cuda.synchronize()
    want = step()
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("Q", [2, 40])
def test_offsets_past_32_bits(Q):
    """A cache whose tokens lie 2^20 elements apart: the last ones behind 2^31."""
    S, step = 2500, 1 << 20
    q, k, v, do = make(1, Q, S, 2, 1, 64, torch.bfloat16)
    cache = torch.empty(S * step, dtype=torch.bfloat16, device="cuda")
    far = [cache.as_strided((1, S, 1, 64), (0, step, 0, 1), at) for at in (0, 64)]
    for to, of in zip(far, (k, v)):
        to.copy_(of)
    check(run(q, *far, do), formula(q, k, v, do))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, D", [(torch.float16, 32), (torch.float16, 128), (torch.float32, 32), (torch.float32, 64),
                                      (torch.float32, 128)], ids=str)
@pytest.mark.parametrize("Q", [5, 200])
def test_rows_do_not_meet(dtype, D, Q):
    """A query that holds NaN has a result of NaN, and no other query has another result for it."""
    q, k, v, _ = make(2, Q, 150, 4, 2, D, dtype)
    want = cross_attention(q, k, v)
    q[1, 2, 3, 0] = math.nan
    got = cross_attention(q, k, v).view(2, Q, 4, D)
    assert got[1, 2, 3].isnan().all()
    got[1, 2, 3] = want.view_as(got)[1, 2, 3]
    assert torch.equal(got.view_as(want), want)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_long_sums_in_float32(D):
    """Sums on the tensor cores are cut off at every addition, by 2^-25.7 of the sum at most on average: 24 additions a
    tile, four tiles to a sum, are 1.8e-6 of the result; scores and products with terms add a third of that."""
    q, k, v, do = make(2, 700, 4096, 2, 2, D, torch.float32)
    got, want = run(q, k, v, do), formula(q, k, v, do)
    for x, (y, _) in zip(got, want):
        assert (x.detach().double() - y).norm() <= 2.5e-6 * y.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [-12, 8])
@pytest.mark.parametrize("heads, D", [((4, 4), 32), ((2, 1), 128), ((70, 1), 64)], ids=str)
def test_small_and_large_gradients_in_float16(heads, D, shift):
    """A weight times a gradient is often below 2^-14, where float16 loses bits.  Results are off by their own rounding, half of
    2^-24 at least, and by six half steps: dS, the weights, o (by way of delta) and what these add up to."""
    q, k, v, do = make(1, 40 if heads[0] == 70 else 150, 1000, *heads, D, torch.float16)
    do = (do * 2.0 ** shift).to(torch.float16)
    for x, (y, _) in zip(run(q, k, v, do), formula(q, k, v, do)):
        assert (x.double() - y).norm() <= y.numel() ** 0.5 * 2.0 ** -25 + 6 * 2.0 ** -11 * y.norm()


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    sets = [make(2, 64, 2000, 4, 4, 64, torch.float16, seed=s) for s in range(2)]
    want = [run(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(run(*s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    q, k, v, do = make(1, 4, 6, 2, 2, 32, torch.float16)
    with pytest.raises(NoBackendError, match="head dimension"):
        cross_attention(*make(1, 4, 6, 2, 2, 136, torch.float16)[:3])
    with pytest.raises(NoBackendError, match="head dimension"):
        cross_attention(*make(1, 4, 6, 2, 2, 12, torch.float16)[:3])
    with pytest.raises(NoBackendError, match="float64"):
        cross_attention(q.double(), k.double(), v.double())
    with pytest.raises(ValueError, match="one device"):
        cross_attention(q, k, v.cpu())
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            cross_attention(q, k, v, scale=scale)
    leaf = q.clone().requires_grad_()
    (grad,) = torch.autograd.grad(cross_attention(leaf, k, v), leaf, do.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


@pytest.mark.parametrize("change, message", [
    (lambda a: a.update(query=torch.zeros(2, 3, 64)), "query must have 4"),
    (lambda a: a.update(key=torch.zeros(2, 5, 2, 16)), "head dimension of query"),
    (lambda a: a.update(key=torch.zeros(1, 5, 2, 32)), "batch of query"),
    (lambda a: a.update(value=torch.zeros(2, 6, 2, 32)), "states of key"),
    (lambda a: a.update(key=torch.zeros(2, 5, 3, 32), value=torch.zeros(2, 5, 3, 32)), "multiple of the 3 heads"),
    (lambda a: a.update(key=torch.zeros(2, 5, 2, 32).half()), "common dtype"),
    (lambda a: a.update({n: a[n].long() for n in ("query", "key", "value")}), "floating-point"),
    (lambda a: a.update(key_padding_mask=torch.zeros(2, 5)), "bool tensor"),
    (lambda a: a.update(key_padding_mask=torch.zeros(2, 4, dtype=torch.bool)), "states of key"),
    (lambda a: a.update(attention_mask=torch.zeros(2, 3, 5)), "added to the scores"),
    (lambda a: a.update(attention_mask=torch.zeros(2, 3, 3, 5, dtype=torch.bool)), "1 or 4"),
    (lambda a: a.update(attention_mask=torch.zeros(4, 5, dtype=torch.bool)), "queries"),
    (lambda a: a.update(attention_mask=torch.zeros(1, 3, 5, dtype=torch.bool)), "batch of query"),
])
def test_refusals(change, message):
    args = {"query": torch.zeros(2, 3, 4, 32), "key": torch.zeros(2, 5, 2, 32), "value": torch.zeros(2, 5, 2, 32),
            "key_padding_mask": None, "attention_mask": None}
    change(args)
    with pytest.raises(ValueError, match=message):
        cross_attention(args.pop("query"), args.pop("key"), args.pop("value"), **args)


def test_refusals_without_a_gpu():
    q, k = torch.zeros(2, 3, 4, 32), torch.zeros(2, 5, 2, 32)
    with pytest.raises(NoBackendError, match="no CPU path"):
        cross_attention(q, k, k)
    with pytest.raises(NoBackendError, match="not part of this build"):
        cross_attention(q, k, k, backend=Backend.EAGER)
    with pytest.raises(TypeError, match="string"):
        cross_attention(q, k, k, backend="cuda")


def test_statuses_of_the_c_interface():
    import ctypes

    from deformops_b200._loader import AttentionCall, load_library

    shim = load_library()
    three = ctypes.c_int64 * 3

    def call(**changes):
        fields = {"batch": 1, "queries": 4, "states": 9, "heads": 4, "kv_heads": 2, "head_dim": 32,
                  "query_strides": three(512, 128, 32), "key_strides": three(576, 64, 32),
                  "value_strides": three(576, 64, 32), "mask": None, "mask_heads": 0, "dtype": 2, "scale": 0.1}
        fields.update(changes)
        c = AttentionCall(**fields)
        return shim.attention_forward(ctypes.byref(c), *[None] * 6, 0, -1, None)

    assert call() == -1 and "null" in shim.last_error()
    assert call(dtype=3) == -1 and "dtype" in shim.last_error()
    assert call(heads=3) == -1 and call(batch=-1) == -1 and call(scale=0.0) == -1 and call(mask_heads=3) == -1
    assert call(head_dim=36) == -2 and call(head_dim=136) == -2 and call(states=1 << 31) == -2
    assert call(query_strides=three(512, 127, 32)) == -1 and "strides" in shim.last_error()
    assert call(key_strides=three(-8, 64, 32)) == -1
    assert call(key_strides=three(576, 0, 32)) == -2 and call(query_strides=three(512, 128, 0)) == -2
    assert call(query_strides=three(512, 0, 32)) == -2 and "of their own" in shim.last_error()
    assert call(queries=0) == 0 and call(batch=0) == 0
    assert shim.attention_forward(None, *[None] * 6, 0, -1, None) == -1
    # 129 states: 8 words, lists of 3 and 2 tiles with their counts (in whole 16 bytes)
    assert shim.attention_mask_bytes(2, 5, 129, 2, 0) == 2 * (8 + 8) * 4
    assert shim.attention_mask_bytes(2, 5, 129, 2, 4) == 4 * 2 * (2 * 8 + 8 * (2 + 4 * 5))


def rows_within(got, want, steps=6):
    """Row by row (the last axis): half a step of 2^-24 for what is small, and so many half steps of the row's norm."""
    off, size = (got.double() - want).norm(dim=-1), want.norm(dim=-1)
    worst = (off / (want.shape[-1] ** 0.5 * 2.0 ** -25 + steps * 2.0 ** -11 * size)).max().item()
    assert worst <= 1.0, f"{worst:.2f} of the bound off"


@pytest.mark.gpu
@pytest.mark.parametrize("S", [1000, 4096])
@pytest.mark.parametrize("heads, D", [((4, 4), 32), ((4, 2), 64), ((2, 1), 128), ((70, 1), 64)], ids=str)
def test_rows_of_unlike_gradients_in_float16(heads, D, S):
    """Gradients 2^12 apart: between samples, heads and rows, and for states that only the small rows see.  Every row of
    dq, dk and dv is off by its own rounding and by that of dS, of the weights and of o: six half steps hold them, as where
    all rows are alike.  Small rows keep their bits: what is 2^-27 of the bound that dS is scaled by is normal, and theirs
    is 2^-12 of it, times 1 / S, times 2^-4 for a product of vectors that are not parallel (one bit short over 4096
    states, which makes one half step two)."""
    G, K = heads
    B, Q = 3, 40 if G == 70 else 150
    q, k, v, do = make(B, Q, S, G, K, D, torch.float16)
    by = torch.full((B, Q, G), 2.0 ** 9, device="cuda")
    by[0, ::2] *= 2.0 ** -12
    by[1] *= 2.0 ** -12
    by[2, :, : G // K] *= 2.0 ** -12                        # of one key head
    do = (do.view(B, Q, G, D) * by.unsqueeze(-1)).to(torch.float16).view(B, Q, G * D)
    mask = torch.zeros(B, Q, S, dtype=torch.bool, device="cuda")
    mask[0, 1::2, 3 * S // 4:] = True
    got = run(q, k, v, do, attention_mask=mask)[1:]
    for x, (y, _) in zip(got, formula(q, k, v, do, mask=mask)[1:]):
        rows_within(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(4, 2), (70, 1)], ids=str)
def test_gradients_of_other_samples_and_heads_do_not_matter(heads):
    G, K = heads
    q, k, v, do = make(3, 60, 500, G, K, 32, torch.float16)
    want = run(q, k, v, do)
    louder = do.view(3, 60, G, 32).clone()
    louder[1] *= 2.0 ** 10
    louder[2, :, : G // K] *= 2.0 ** 12
    louder[2, 5, 0, 3] = math.inf
    got = run(q, k, v, louder.view_as(do))
    for x, y in zip(got[1:], want[1:]):
        assert torch.equal(x[0], y[0])
        assert torch.equal(x[2, :, x.shape[2] // K:], y[2, :, y.shape[2] // K:])
    # of the head with the infinity: the other rows' dq
    finite = louder.clone()
    finite[2, 5, 0, 3] = 1.0
    dq = run(q, k, v, finite.view_as(do))[1]
    dq[2, 5, 0] = got[1][2, 5, 0]
    assert torch.equal(got[1].nan_to_num(), dq.nan_to_num()) and got[1][2, 5, 0].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("size, least, most", [(800.0, -10, -10), (8000.0, -14, -12), (1.0, -22, -20), (2.0 ** -12, 0, 8)], ids=str)
@pytest.mark.parametrize("heads", [(2, 2), (70, 1)], ids=str)
def test_values_of_any_size_in_float16(heads, size, least, most):
    """dS is as large as |do| |v|: states whose v is the same in all channels, and gradients that are too."""
    q, k, v, do = make(1, 30, 8, *heads, 128, torch.float16)
    v = (v[..., :1] * size).expand_as(v).contiguous()
    by = 2.0 ** torch.linspace(least, most, 30, device="cuda").round().view(1, 30, 1)
    do = by.expand_as(do).to(torch.float16).contiguous()
    got, want = run(q, k, v, do), formula(q, k, v, do)
    assert all(torch.isfinite(t).all() for t in got)
    check(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, Q", [((1, 1), 40), ((70, 1), 1)], ids=str)
def test_small_weights_in_float16(heads, Q):
    """Over 2^20 states a weight is 2^-20, where a step of float16 is 2^-24."""
    q, k, v, do = make(1, Q, 1 << 20, *heads, 16, torch.float16)
    do = do * 2.0 ** 12
    got, want = run(q, k, v, do), formula(q, k, v, do)
    for x, (y, _) in zip(got[1:], want[1:]):
        assert (x.double() - y).norm() <= y.numel() ** 0.5 * 2.0 ** -25 + 6 * 2.0 ** -11 * y.norm()


@pytest.mark.parametrize("Q, S", [(300, 17821), (640, 4096), (9000, 20000), (1 << 16, 1 << 16), (1 << 18, 1 << 18), (1 << 10, 1 << 22), (1 << 20, 1 << 12), (17, 1 << 24)])
@pytest.mark.parametrize("B, D", [(1, 32), (8, 16)])
def test_workspace_is_no_larger_than_the_tensors(Q, S, B, D):
    """float32, forward: three terms of 2 bytes of k and v (in vectors of eight channels), and parts: as many as eight CTAs
    of 256 rows (24 of 128) to each of 148 SMs have rows, and one more result.  Never a product of rows and states."""
    import ctypes

    from deformops_b200._loader import AttentionCall, load_library

    G = 8
    three = ctypes.c_int64 * 3
    states = three(S * G * D, G * D, D)
    call = AttentionCall(batch=B, queries=Q, states=S, heads=G, kv_heads=G, head_dim=D, query_strides=three(Q * G * D, G * D, D),
                         key_strides=states, value_strides=states, mask=None, mask_heads=0, dtype=0, scale=0.1)
    rows, terms = B * G * Q, 2 * 6 * B * S * G * D
    most = terms + 4 * (D + 1) * (rows + 148 * 24 * 128) + 64
    assert 0 < load_library().attention_workspace_bytes(ctypes.byref(call), 0) <= most


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(8, 640, 4096, 8, 8, 32), (8, 100, 17821, 8, 8, 32), (2, 300, 17821, 2, 1, 16), (1, 8192, 4096, 2, 2, 32), (1, 600, 4500, 6, 6, 32),
                                  (4, 2000, 512, 8, 8, 32), (2, 200, 1344, 8, 8, 24)], ids=str)
def test_long_sums_in_float32_up_to_32_channels(size):
    """As with more channels, 1.8e-6 for sums of four tiles and a third of that for scores and terms; small CTAs have sums of up to
    eight, 3.6e-6.  Gradients have sums of four."""
    q, k, v, do = make(*size, torch.float32)
    got, want = run(q, k, v, do), formula(q, k, v, do)
    for x, (y, _), most in zip(got, want, (4.2e-6, 2.5e-6, 2.5e-6, 2.5e-6)):
        assert (x.detach().double() - y).norm() <= most * y.norm()


def test_scales_that_overflow_are_refused():
    """Scores are formed in base 2: a scale whose product with log2(e) is no number any more would make NaN of them."""
    import ctypes

    from deformops_b200._loader import AttentionCall, load_library

    three = ctypes.c_int64 * 3
    for scale, bytes_needed in ((2.0 ** 127, True), (3e38, False), (math.inf, False)):
        call = AttentionCall(batch=1, queries=40, states=9, heads=1, kv_heads=1, head_dim=32, query_strides=three(1280, 32, 32),
                             key_strides=three(288, 32, 32), value_strides=three(288, 32, 32), mask=None, mask_heads=0, dtype=0,
                             scale=scale)
        assert (load_library().attention_workspace_bytes(ctypes.byref(call), 0) > 0) == bytes_needed


@pytest.mark.gpu
@pytest.mark.parametrize("B, Q, D, S", [(40, 1, 32, 30), (40, 12, 128, 14), (40, 1, 32, 20000), (40, 40, 32, 20000), (40, 300, 64, 20000), (20, 200, 128, 6000), (40, 200, 64, 60)], ids=str)
def test_one_large_score_among_small_ones_in_float16(B, Q, D, S):
    """Every row sees one state of weight 1 whose values are 0, and others whose weights, all alike, are 10 1/2 steps of 2^-24: what is
    left of the result is theirs.  Weights and result are rounded, half a step each; sums in 32 bits and the score another."""
    gap = -math.log(10.5 * 2.0 ** -24)
    q, k, v, _ = make(B, Q, S, 4, 4, D, torch.float16)
    q[:], k[:] = 0, 0
    q[..., 0] = 4.0
    k[:, 7, :, 0] = 4.0
    v[:, 7] = 0
    v = v.abs()
    out = cross_attention(q, k, v, scale=gap / 16)
    want = formula(q, k, v, out, scale=gap / 16)[0][0]
    assert (out.double() - want).norm() <= want.numel() ** 0.5 * 2.0 ** -25 + 3 * 2.0 ** -11 * want.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("Q, S", [(40000, 60), (200, 40000), (140000, 20)])
def test_bounds_of_long_axes_in_float16(Q, S):
    """The largest row or state is found wherever it is: were it not, the products with it would overflow."""
    q, k, v, do = make(2, Q, S, 2, 2, 32, torch.float16)
    for at in (0, Q // 2 + 3, Q - 1):
        do[1, at] *= 2.0 ** 11
    v[0, S - 1] *= 2.0 ** 11
    v[1, S // 3] *= 2.0 ** 11
    got, want = run(q, k, v, do), formula(q, k, v, do)
    # gradients past the largest number of the type (2^11 times 2^11 times the rest) are infinities, and nothing else is
    past = [(y.abs() - bound) > 65520 for y, bound in want]
    near = [(y.abs() + bound) > 65504 for y, bound in want]
    for x, over, may, (y, _) in zip(got, past, near, want):
        assert torch.equal(x[over].double(), y[over].sign() * math.inf) and torch.isfinite(x[~may]).all()
    check([x.masked_fill(may, 0.0) for x, may in zip(got, near)], [(y.masked_fill(may, 0.0), b) for (y, b), may in zip(want, near)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads, Q", [((2, 1), 70), ((70, 1), 3), ((2, 2), 5)], ids=str)
@pytest.mark.parametrize("size", [300.0, 600.0])
def test_scores_of_tens_of_millions(dtype, heads, Q, size):
    """Of 1.2 and 4.6 x 10^7, in base 2 times 1.44 and up to 2^26: their float32 is rounded by 4 at most, so weights say little in a
    backward pass, but nothing overflows, and results are means of the values."""
    q, k, v, do = make(1, Q, 200, *heads, 128, dtype)
    q, k = (t.sign() * size for t in (q, k))
    k[:, 3] = q[:, 0, :1]
    out, *grads = run(q, k, v, do, scale=1.0)
    assert torch.isfinite(out).all() and out.abs().max() <= 1.01 * v.abs().max()
    assert all(torch.isfinite(t).all() for t in grads)
