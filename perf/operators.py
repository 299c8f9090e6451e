"""Cross attention to an encoder's states and rotary positions of several axes, as cases that can be timed.

* ``cross``   ``registry.cross_attention``: queries that attend to all states of an encoder, which are
              of another length; the dense counterpart of the sampling in ``registry.msda``.
* ``rotary``  ``registry.rotary``: the rotation that gives queries and keys their place (row and
              column in an image, time as well in a video) before they meet.

``own`` chooses what ``run`` calls: the plain form, made of elementary torch operations in 32 bits (angles
in 64), or the operators of this package.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}

# Pyramids of the package's own configurations, flattened level after level
_PYRAMID_1024 = "128x128,64x64,32x32"
_PYRAMID_DETR = "100x134,50x67,25x34,13x17"
_PYRAMID_SMALL = "32x32,16x16,8x8"


def _cross(name, train, dtype, batch, queries, states, heads, kv_heads, head_dim, mask="none"):
    """``states``: a number of tokens or the levels of a pyramid.  ``mask``: ``padding`` (images or
    texts of several sizes in one batch, one mask for all queries) or ``queries`` (a mask for every
    query, the same for all heads; a few queries are left with nothing)."""
    return {"name": name, "entry": "cross", "train": train, "dtype": dtype, "batch": batch,
            "queries": queries, "states": states, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "mask": mask}


def _rotary(name, train, dtype, batch, tokens, heads, head_dim, sections, interleaved=False):
    """``tokens``: levels of a pyramid or ``frames x rows x columns``, whose pixels are the tokens."""
    return {"name": name, "entry": "rotary", "train": train, "dtype": dtype, "batch": batch,
            "tokens": tokens, "heads": heads, "head_dim": head_dim, "sections": sections,
            "interleaved": interleaved}


def listed():
    return [
        # a detection decoder's 300 object queries over the encoder's whole pyramid: training, and
        # the same in float32 when the images of a batch are scored
        _cross("objects_train_bf16", True, "bfloat16", 4, 300, _PYRAMID_DETR, 8, 8, 32, "padding"),
        _cross("objects_score_f32", False, "float32", 2, 300, _PYRAMID_DETR, 8, 8, 32, "padding"),
        # a segmentation decoder's 100 queries, each within the mask that it predicted one layer before
        _cross("masked_train_f16", True, "float16", 8, 100, "64x64", 8, 8, 32, "queries"),
        # pixels of a feature map attend to a short text
        _cross("text_bf16", False, "bfloat16", 4, 4096, "77", 8, 8, 64, "padding"),
        # a decoder with shared key heads over an encoder's long output: training
        _cross("long_train_bf16", True, "bfloat16", 2, 2048, "4096", 16, 4, 128),
        # serving: every sequence of the batch has one new token; the encoder's states stay
        _cross("token_bf16", False, "bfloat16", 16, 1, "1500", 32, 8, 128),
        # the smallest call: one token over one short text
        _cross("token_small_f16", False, "float16", 1, 1, "77", 8, 8, 64),
        # a layer of the CPU-sized configuration in float32, as a test or a small model trains it
        _cross("small_train_f32", True, "float32", 2, 100, _PYRAMID_SMALL, 8, 8, 32, "padding"),
        # keys of a pixel decoder's pyramid get their row and column
        _rotary("pyramid_bf16", False, "bfloat16", 4, _PYRAMID_1024, 8, 32, "8,8"),
        # a video's tokens: time, row and column; training
        _rotary("video_train_f16", True, "float16", 2, "16x32x32", 16, 128, "16,24,24"),
        # one new token of each sequence in a batch
        _rotary("token_rotary_bf16", False, "bfloat16", 16, "1x1x1", 32, 128, "16,24,24"),
        # float32 training on the detection pyramid, neighbouring channels as pairs
        _rotary("pyramid_train_f32", True, "float32", 2, _PYRAMID_DETR, 8, 32, "8,8", True),
    ]


def _levels(text):
    return [tuple(int(n) for n in part.split("x")) for part in text.split(",")]


def _tokens(text):
    return sum(math.prod(level) for level in _levels(text))


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cost(case):
    width = 4 if case["dtype"] == "float32" else 1
    if case["entry"] == "rotary":
        return (2 if case["train"] else 1) * width * case["batch"] * _tokens(case["tokens"]) * case["heads"] * case["head_dim"]
    return ((3 if case["train"] else 1) * width * case["batch"] * case["heads"] * case["queries"]
            * _tokens(case["states"]) * (case["head_dim"] + 32))


def draw(rng):
    entry = rng.choice(["cross", "cross", "cross", "rotary"])
    most = max(_cost(c) for c in listed() if c["entry"] == entry)
    while True:
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        train = rng.random() < 0.55
        batch = _log_uniform(rng, 1, 16)
        if entry == "rotary":
            heads, head_dim = rng.choice([(8, 32), (8, 32), (16, 64), (16, 128), (32, 128), (6, 80), (1, 64)])
            pairs = head_dim // 2
            if rng.random() < 0.5:
                height = _log_uniform(rng, 3, 140)
                width = max(3, int(height * rng.uniform(0.7, 1.5)))
                tokens = f"{height}x{width},{(height + 1) // 2}x{(width + 1) // 2}"
                sections = f"{pairs // 2},{pairs - pairs // 2}"
            else:
                tokens = f"{_log_uniform(rng, 1, 32)}x{_log_uniform(rng, 1, 40)}x{_log_uniform(rng, 1, 40)}"
                sections = f"{pairs // 4},{pairs * 3 // 8},{pairs * 3 // 8}"
            case = _rotary("", train, dtype, batch, tokens, heads, head_dim, sections, rng.random() < 0.4)
        else:
            heads, kv_heads, head_dim = rng.choice([(8, 8, 32), (8, 8, 32), (8, 8, 64), (16, 4, 128), (32, 8, 128),
                                                    (6, 6, 64), (8, 8, 16), (4, 4, 96), (12, 2, 40)])
            kind = rng.choice(["token", "objects", "objects", "pixels", "long"])
            if kind == "token":
                queries, states, train = rng.choice([1, 1, 1, 2, 5, 16]), _log_uniform(rng, 1, 20000), False
            elif kind == "objects":
                queries, states = _log_uniform(rng, 20, 900), _log_uniform(rng, 300, 20000)
            elif kind == "pixels":
                queries, states = _log_uniform(rng, 900, 9000), _log_uniform(rng, 16, 512)
            else:
                queries, states = _log_uniform(rng, 300, 2800), _log_uniform(rng, 300, 4500)
            case = _cross("", train, dtype, batch, queries, str(states), heads, kv_heads, head_dim,
                          rng.choice(["none", "padding", "queries"]))
        del case["name"]
        if _cost(case) <= most:
            return case


def _pyramid_padding(case, gen):
    """(B, S) true where an image, smaller than the batch's largest, has no pixels; a text no words."""
    B, levels = case["batch"], _levels(case["states"])
    part = 0.55 + 0.45 * torch.rand(B, 2, generator=gen, device="cuda")
    part[0] = 1.0
    rows = []
    for level in levels:
        h, w = level if len(level) == 2 else (1, level[0])
        y = torch.arange(h, device="cuda").view(1, h, 1) >= torch.ceil(part[:, 0] * h).view(B, 1, 1)
        x = torch.arange(w, device="cuda").view(1, 1, w) >= torch.ceil(part[:, 1] * w).view(B, 1, 1)
        rows.append((x if h == 1 else y | x).reshape(B, h * w))
    return torch.cat(rows, 1)


def _query_masks(case, gen):
    """(B, Q, S) true where a query may not look: all but a stretch of the states, or all of them."""
    B, Q, S = case["batch"], case["queries"], _tokens(case["states"])
    middle = torch.rand(B, Q, 1, generator=gen, device="cuda")
    reach = 0.05 + 0.3 * torch.rand(B, Q, 1, generator=gen, device="cuda")
    reach = torch.where(torch.rand(B, Q, 1, generator=gen, device="cuda") < 0.02, -1.0, reach)
    place = (torch.arange(S, device="cuda") + 0.5) / S
    near = (place - middle).abs() + 0.1 * torch.rand(B, Q, S, generator=gen, device="cuda")
    return near > reach


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]
    B, G, D = case["batch"], case["heads"], case["head_dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    state = {"entry": case["entry"], "train": case["train"]}
    if case["entry"] == "rotary":
        # pixel centres in units of pixels; frames count from somewhere within a long video
        places = []
        for level in _levels(case["tokens"]):
            axes = [torch.arange(n, device="cuda") + 0.5 for n in level[-2:]]
            if len(level) == 3:
                axes.insert(0, torch.arange(level[0], device="cuda") + 1000.0 * (seed % 7))
            places.append(torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, len(level)))
        positions = torch.cat(places)
        state["positions"] = positions.expand(B, *positions.shape).contiguous()
        state["sections"] = tuple(int(n) for n in case["sections"].split(","))
        state["interleaved"] = case["interleaved"]
        shape = (B, positions.shape[0], G, D)
        inputs, out_shape = [normal(*shape)], shape
    else:
        Q, S, K = case["queries"], _tokens(case["states"]), case["kv_heads"]
        state["padding"] = _pyramid_padding(case, gen) if case["mask"] == "padding" else None
        state["mask"] = _query_masks(case, gen) if case["mask"] == "queries" else None
        inputs, out_shape = [normal(B, Q, G, D), normal(B, S, K, D), normal(B, S, K, D)], (B, Q, G * D)
    state["inputs"] = [t.requires_grad_(case["train"]) for t in inputs]
    if case["train"]:
        state["grad"] = normal(*out_shape)
    return state


def _plain_cross(query, key, value, padding, mask):
    B, Q, G, D = query.shape
    S, K = key.shape[1:3]
    # (B, K, heads that share a key head, Q, D) with (B, K, 1, S, D)
    q = query.view(B, Q, K, G // K, D).permute(0, 2, 3, 1, 4)
    k = key.permute(0, 2, 1, 3).unsqueeze(2)
    v = value.permute(0, 2, 1, 3).unsqueeze(2)
    scores = torch.matmul(q * D ** -0.5, k.transpose(-1, -2))
    if padding is not None:
        scores = scores.masked_fill(padding.view(B, 1, 1, 1, S), -math.inf)
    if mask is not None:
        scores = scores.masked_fill(mask.view(B, 1, 1, Q, S), -math.inf)
    top = scores.detach().amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    # a query with nothing left to look at: zeros
    weights = weights * torch.where(total > 0, 1.0 / total.clamp_min(1e-30), 0.0)
    return torch.matmul(weights, v).permute(0, 3, 1, 2, 4).reshape(B, Q, G * D)


def _angles(positions, sections, base=10000.0):
    """(B, N, 1, pairs) in 64 bits: every axis has a geometric series of its own."""
    parts = []
    for axis, pairs in enumerate(sections):
        steps = torch.arange(pairs, dtype=torch.float64, device=positions.device) / max(pairs, 1)
        parts.append(positions[..., axis, None].double() * torch.pow(base, -steps))
    return torch.cat(parts, -1).unsqueeze(2)


def _plain_rotary(x, positions, sections, interleaved):
    angle = _angles(positions, sections)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    turned = 2 * sum(sections)
    head, rest = x[..., :turned], x[..., turned:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else head.chunk(2, -1)
    a, b = a * cos - b * sin, a * sin + b * cos
    head = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([head, rest], -1)


def _forward(state, inputs):
    if state["entry"] == "rotary":
        if own:
            from deformops_b200.registry import rotary

            return rotary(inputs[0], state["positions"], sections=state["sections"],
                          interleaved=state["interleaved"])
        return _plain_rotary(inputs[0], state["positions"], state["sections"], state["interleaved"])
    if own:
        from deformops_b200.registry import cross_attention

        return cross_attention(*inputs, key_padding_mask=state["padding"], attention_mask=state["mask"])
    return _plain_cross(*inputs, state["padding"], state["mask"])


def run(state):
    inputs = state["inputs"]
    dtype = inputs[0].dtype
    if not state["train"]:
        with torch.no_grad():
            return [_forward(state, inputs if own else [t.float() for t in inputs]).to(dtype)]
    if own:
        out = _forward(state, inputs)
        return [out.detach(), *torch.autograd.grad(out, inputs, state["grad"])]
    wide = [t.detach().float().requires_grad_() for t in inputs]
    out = _forward(state, wide)
    grads = torch.autograd.grad(out, wide, state["grad"].float())
    return [out.detach().to(dtype), *(g.to(dtype) for g in grads)]


def work(case):
    """Inputs read once, outputs written once; two matrix products forward, five backward (the weights
    are formed once more there), over all pairs of query and state, masked or not."""
    e = 4 if case["dtype"] == "float32" else 2
    B, G, D = case["batch"], case["heads"], case["head_dim"]
    if case["entry"] == "rotary":
        values, places = B * _tokens(case["tokens"]) * G * D, B * _tokens(case["tokens"]) * len(_levels(case["tokens"])[0]) * 4
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * values * e + places), "flops": passes * 3 * values}
    Q, S, K = case["queries"], _tokens(case["states"]), case["kv_heads"]
    rows, states = B * Q * G * D * e, 2 * B * S * K * D * e
    mask = B * S if case["mask"] == "padding" else B * Q * S if case["mask"] == "queries" else 0
    product = 2 * B * G * Q * S * D
    total = {"bytes": 2 * rows + states + mask, "flops": 2 * product}
    if case["train"]:
        total["bytes"] += 3 * rows + 2 * states + mask + rows
        total["flops"] += 5 * product
    return total


def exact(case, seed):
    """In 64 bits from the definitions, sample by sample and with the gradients' formulas written out."""
    state = prepare(case, seed)
    inputs = [t.detach().double() for t in state["inputs"]]
    grad = state["grad"].double() if case["train"] else None
    if case["entry"] == "rotary":
        return _exact_rotary(state, inputs[0], grad)
    q, k, v = inputs
    B, Q, G, D = q.shape
    S, K = k.shape[1:3]
    share = G // K
    out = torch.zeros(B, Q, G, D, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        allowed = torch.ones(Q, S, dtype=torch.bool, device=q.device)
        if state["padding"] is not None:
            allowed &= ~state["padding"][b]
        if state["mask"] is not None:
            allowed &= ~state["mask"][b]
        some = allowed.any(1)
        for g in range(G):
            h = g // share
            s = (q[b, :, g] @ k[b, :, h].T) / math.sqrt(D)
            p = torch.zeros_like(s)
            if some.any():
                p[some] = torch.softmax(s[some].masked_fill(~allowed[some], -math.inf), 1)
            out[b, :, g] = p @ v[b, :, h]
            if grad is None:
                continue
            do = grad.view(B, Q, G, D)[b, :, g]
            dp = do @ v[b, :, h].T
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(D)
            dq[b, :, g] = ds @ k[b, :, h]
            dk[b, :, h] += ds.T @ q[b, :, g]
            dv[b, :, h] += p.T @ do
    out = out.reshape(B, Q, G * D)
    return [out] if grad is None else [out, dq, dk, dv]


def _exact_rotary(state, x, grad):
    sections, positions = state["sections"], state["positions"].double()

    def turn(t, sign):
        t = t.clone()
        pairs, done = sum(sections), 0
        for axis, count in enumerate(sections):
            for i in range(count):
                angle = sign * positions[:, :, axis] * 10000.0 ** (-i / count)
                c, s = angle.cos().unsqueeze(-1), angle.sin().unsqueeze(-1)
                j = done + i
                first, second = (2 * j, 2 * j + 1) if state["interleaved"] else (j, j + pairs)
                a, b = t[..., first].clone(), t[..., second].clone()
                t[..., first], t[..., second] = a * c - b * s, a * s + b * c
            done += count
        return t

    return [turn(x, 1.0)] if grad is None else [turn(x, 1.0), turn(grad, -1.0)]
