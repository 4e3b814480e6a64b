"""The decoder-layer operators of inductor_x_amd.kernels as a set of measurable cases.

Each case names one call of one operator: the residual add + RMS norm with an 8-bit result
(`norm`), rotary positions over several axes (`rotary`), and attention with a sliding window and
first tokens that stay visible (`prefill`: forward, `train`: forward and gradients, `decode`: one
token per sequence against a cache).  With `own` false a call runs as elementary torch operations
in 32 bits, with `own` true as the calls a program makes of this package.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
NONE_VISIBLE = -1e30  # below every score: the reference point of a row that sees no key

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _norm(rows, cols, group, dtype):
    return {"op": "norm", "rows": rows, "cols": cols, "group": group, "dtype": dtype}


def _rotary(batch, length, heads, kv_heads, dim, rotary, axes, first, interleaved, inverse, dtype):
    return {"op": "rotary", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "axes": axes, "first": first, "interleaved": interleaved, "inverse": inverse, "dtype": dtype}


def _attention(op, batch, heads, kv_heads, queries, keys, dim, window, sinks, shortest, token_major, dtype):
    """shortest: the share of the padded length that the shortest sequence of the batch has (1.0: none is
    padded); token_major: heads beside tokens in memory, [batch, token, head, dim], as a projection leaves them."""
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries, "keys": keys, "dim": dim,
            "window": window, "sinks": sinks, "shortest": shortest, "token_major": token_major, "dtype": dtype}


def listed():
    return [
        # one token of four sequences between two projections: the smallest call there is, latency alone
        {"name": "norm of 4 tokens", **_norm(4, 4096, 0, "bf16")},
        # the benchmark's norm (8192 rows of 4096) at twice the rows, a scale for every 128 columns
        {"name": "norm of 16384 tokens", **_norm(16384, 4096, 128, "bf16")},
        # one new token for eight sequences, far into their texts
        {"name": "rotary of 8 tokens", **_rotary(8, 1, 32, 8, 128, 128, 1, 100000, False, False, "bf16")},
        # a training batch of image and text tokens: time, height and width
        {"name": "rotary forward", **_rotary(4, 4096, 32, 8, 128, 128, 3, 0, False, False, "bf16")},
        # its gradient for heads that are rotated in part, pairs side by side, an odd length
        {"name": "rotary gradient", **_rotary(3, 2047, 24, 24, 96, 64, 2, 5000, True, True, "fp16")},
        # a padded batch of short texts, heads and window of odd sizes
        {"name": "prefill of short texts", **_attention("prefill", 5, 12, 4, 333, 333, 64, 100, 3, 0.2, True, "fp16")},
        # a text of 8192 tokens at once
        {"name": "prefill of 8192", **_attention("prefill", 1, 32, 8, 8192, 8192, 128, 1024, 4, 1.0, True, "bf16")},
        # 4096 more tokens of a text whose first 28672 are in the cache, wide window
        {"name": "prefill over a cache", **_attention("prefill", 1, 32, 8, 4096, 32768, 128, 8192, 128, 1.0, False, "bf16")},
        # fine-tuning on short padded texts, every query head with a key head of its own
        {"name": "training on short texts", **_attention("train", 3, 8, 8, 777, 777, 96, 256, 8, 0.5, True, "fp16")},
        # the attention benchmark's batch of four texts of 4096 tokens, with shared key heads and a window
        {"name": "training on 4096", **_attention("train", 4, 32, 8, 4096, 4096, 128, 1024, 4, 1.0, True, "bf16")},
        # one conversation, one token
        {"name": "decode for 1 sequence", **_attention("decode", 1, 32, 8, 1, 8192, 128, 1024, 4, 1.0, False, "bf16")},
        # a serving batch, caches filled to different lengths
        {"name": "decode for 64 sequences", **_attention("decode", 64, 32, 8, 1, 16384, 128, 4096, 4, 0.02, True, "bf16")},
    ]


def _spread(rng, low, high):
    """A whole number, spread evenly over the logarithm of the range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("norm", "rotary", "prefill", "train", "decode"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "norm":
        cols = rng.choice((_spread(rng, 64, 16384), 8 * _spread(rng, 8, 2048), 128 * _spread(rng, 1, 128)))
        return _norm(_spread(rng, 1, max(1, 2**26 // cols)), cols, rng.choice((0, 128)), dtype)
    if op == "rotary":
        dim = rng.choice((64, 80, 96, 128, 128))
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
        batch = _spread(rng, 1, 16)
        length = _spread(rng, 1, max(1, 2**26 // (batch * dim * (heads + kv_heads))))
        return _rotary(batch, length, heads, kv_heads, dim, rng.choice((dim, dim, dim // 2 // 8 * 8)), rng.choice((1, 2, 3)),
                       _spread(rng, 1, 1000000) - 1, rng.random() < 0.3, rng.random() < 0.4, dtype)
    dim = rng.choice((64, 64, 80, 96, 128, 128, 128))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 5, 8))
    shortest = rng.choice((1.0, rng.uniform(0.01, 1.0)))
    token_major = rng.random() < 0.5
    sinks = rng.choice((0, 1, 4, 4, rng.randint(2, 100), 128))
    if op == "decode":
        batch = _spread(rng, 1, 64)
        keys = _spread(rng, 1, 32768 if batch <= 8 else 8192)
        return _attention(op, batch, heads, kv_heads, 1, keys, dim, _spread(rng, 1, 8192), sinks, shortest, token_major, dtype)
    batch = _spread(rng, 1, 4)
    most = int(math.sqrt(2**29 / (batch * heads)))  # the plain form keeps whole score matrices
    queries = _spread(rng, 1, min(8192, most))
    keys = queries if op == "train" or rng.random() < 0.6 else queries + _spread(rng, 1, 8192)
    return _attention(op, batch, heads, kv_heads, queries, keys, dim, _spread(rng, 1, 4096), sinks, shortest, token_major, dtype)


def _lengths(case):
    """Sequence lengths of the batch: the longest fills the padding, the others step down to the shortest."""
    most, batch = case["keys"], case["batch"]
    least = max(1, int(case["shortest"] * most))
    return [most - (most - least) * i // max(1, batch - 1) for i in range(batch)]


def _sections(case):
    """Rotated pairs per axis: the first axis takes what does not divide."""
    pairs, axes = case["rotary"] // 2, case["axes"]
    each = pairs // axes
    return [pairs - each * (axes - 1)] + [each] * (axes - 1)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, spread=1.0):
        return (torch.randn(*shape, device="cuda", dtype=torch.float32, generator=gen) * spread).to(t)

    state = {"case": case}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        state["h"] = normal(rows, cols)
        state["r"] = normal(rows, cols, spread=2.0)
        state["r"][:, :: max(1, cols // 5)] *= 20  # a few columns of a residual stream stand far above the others
        state["w"] = 1 + normal(cols, spread=0.1)
        return state
    if case["op"] == "rotary":
        batch, length, pairs = case["batch"], case["length"], case["rotary"] // 2
        state["q"] = normal(batch, length, case["heads"], case["dim"])
        state["k"] = normal(batch, length, case["kv_heads"], case["dim"])
        # the first axis counts on, the others run over the rows and columns of frames of 24 x 40 patches
        start = case["first"] + torch.randint(0, 1000, (batch, 1), device="cuda", generator=gen)
        at = start + torch.arange(length, device="cuda").view(1, length)
        state["positions"] = torch.stack([at, at % 960 // 40, at % 40][: case["axes"]]).to(torch.int32).contiguous()
        state["sections"] = _sections(case)
        state["inv_freq"] = (10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)).float()
        return state
    batch, queries, keys, dim = case["batch"], case["queries"], case["keys"], case["dim"]

    def heads_of(n, tokens):
        if case["token_major"]:
            return normal(batch, tokens, n, dim).transpose(1, 2)
        return normal(batch, n, tokens, dim)

    state["q"] = heads_of(case["heads"], queries)
    state["k"] = heads_of(case["kv_heads"], keys)
    state["v"] = heads_of(case["kv_heads"], keys)
    state["scale"] = 1.0 / math.sqrt(dim)
    padded = case["op"] == "decode" or case["shortest"] < 1.0
    state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if padded else None
    if case["op"] == "decode":
        state["q"] = state["q"][:, :, 0]
    if case["op"] == "train":
        state["dout"] = heads_of(case["heads"], queries)
        for name in ("q", "k", "v"):
            state[name].requires_grad_()
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        if case["op"] == "norm":
            return _plain_norm(state, case)
        if case["op"] == "rotary":
            return _plain_rotary(state, case)
        return _plain_attention(state, case)


def _run_own(state, case):
    from inductor_x_amd import decoder, kernels

    op = case["op"]
    if op == "norm":
        return kernels.add_rmsnorm_quant(state["h"], state["r"], state["w"], 1e-6, group=case["group"])
    if op == "rotary":
        return kernels.rotary_axes(state["q"], state["k"], state["positions"], state["inv_freq"], state["sections"],
                                   interleaved=case["interleaved"], inverse=case["inverse"])
    if op == "prefill":
        return kernels.window_attention(state["q"], state["k"], state["v"], state["scale"], case["window"], case["sinks"],
                                        lengths=state["lengths"])
    if op == "decode":
        return kernels.window_attention_decode(state["q"], state["k"], state["v"], state["lengths"], state["scale"],
                                               case["window"], case["sinks"])
    q, k, v = state["q"], state["k"], state["v"]
    out = decoder.window_attention(q, k, v, state["scale"], case["window"], case["sinks"], lengths=state["lengths"])
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), state["dout"]))


def _plain_norm(state, case):
    s = state["h"].float() + state["r"].float()
    y = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * state["w"].float()
    rows, cols = s.shape
    group = case["group"] or cols
    groups = -(-cols // group)
    y = torch.nn.functional.pad(y, (0, groups * group - cols)).view(rows, groups, group)
    largest = y.abs().amax(-1, keepdim=True)
    scales = torch.where(largest == 0, torch.ones_like(largest), largest / E4M3_MAX)
    q = (y / scales).view(rows, groups * group)[:, :cols].to(torch.float8_e4m3fn)
    return q, scales.view(rows, groups), s.to(state["h"].dtype)


def _angles(state, case):
    """[batch, length, pairs] in 64 bits: far positions lose their angle in 32."""
    axis = torch.repeat_interleave(torch.arange(case["axes"], device="cuda"),
                                   torch.tensor(state["sections"], device="cuda"), output_size=case["rotary"] // 2)
    return state["positions"].double()[axis].permute(1, 2, 0) * state["inv_freq"].double()


def _plain_rotary(state, case):
    angle = _angles(state, case).unsqueeze(2)
    cos, sin = angle.cos().float(), angle.sin().float()
    if case["inverse"]:
        sin = -sin

    def rotate(x):
        y = x.float()
        head = y[..., : case["rotary"]]
        if case["interleaved"]:
            a, b = head[..., 0::2], head[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = head.chunk(2, -1)
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned, y[..., case["rotary"]:]), -1).to(x.dtype)

    return rotate(state["q"]), rotate(state["k"])


def _visible(case, lengths, queries, keys):
    """[batch or 1, 1, 1, queries, keys]: what each query sees."""
    key = torch.arange(keys, device="cuda").view(1, 1, keys)
    if case["op"] == "decode":
        at = lengths.view(-1, 1, 1).long() - 1
        seen = (key <= at) & ((key > at - case["window"]) | (key < case["sinks"]))
    else:
        at = torch.arange(queries, device="cuda").view(1, queries, 1) + (keys - queries)
        seen = (key <= at) & ((key > at - case["window"]) | (key < case["sinks"]))
        if lengths is not None:
            seen = seen & (at < lengths.view(-1, 1, 1))
    return seen.view(seen.shape[0], 1, 1, seen.shape[1], keys)


def _plain_attention(state, case):
    q = state["q"].unsqueeze(2) if case["op"] == "decode" else state["q"]
    batch, heads, queries, dim = q.shape
    kv_heads, keys = state["k"].shape[1:3]
    share = (batch, kv_heads, heads // kv_heads, queries, dim)
    qf = q.float().reshape(share)
    kf, vf = state["k"].float().unsqueeze(2), state["v"].float().unsqueeze(2)
    seen = _visible(case, state["lengths"], queries, keys)
    p = torch.matmul(qf, kf.transpose(-1, -2))
    p.mul_(state["scale"]).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True).clamp_min(NONE_VISIBLE)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total.clamp_min(1e-30))
    out = torch.matmul(p, vf)
    shaped = out.reshape(q.shape).to(q.dtype)
    if case["op"] == "decode":
        return shaped[:, :, 0]
    if case["op"] == "prefill":
        return shaped, (top + total.log()).masked_fill(total == 0, -math.inf).reshape(batch, heads, queries)
    g = state["dout"].float().reshape(share)
    g = g * seen.any(-1, keepdim=True)
    dv = torch.matmul(p.transpose(-1, -2), g).sum(2)
    ds = torch.matmul(g, vf.transpose(-1, -2))
    ds.sub_((g * out).sum(-1, keepdim=True)).mul_(p).mul_(state["scale"])
    dq = torch.matmul(ds, kf).reshape(q.shape)
    dk = torch.matmul(ds.transpose(-1, -2), qf).sum(2)
    return shaped, dq.to(q.dtype), dk.to(q.dtype), dv.to(q.dtype)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def _pairs(case):
    """Visible (query, key) pairs of one head over the batch, and key rows that any query sees."""
    window, sinks = case["window"], case["sinks"]

    def upto(n):  # pairs of the queries at positions 0 .. n - 1
        first = min(n, window)
        total = first * (first + 1) // 2
        rest = n - first  # position window + j sees the window and min(sinks, j + 1) tokens before it
        total += rest * window
        ramp = min(rest, sinks)
        return total + ramp * (ramp + 1) // 2 + (rest - ramp) * sinks

    pairs = rows = 0
    for length in _lengths(case):
        if case["op"] == "decode":
            first = length - 1
        else:
            first = case["keys"] - case["queries"]
        if length <= first:
            continue
        pairs += upto(length) - upto(first)
        start = max(0, first + 1 - window)
        rows += length - start + min(sinks, start)
    return pairs, rows


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        groups = -(-case["cols"] // (case["group"] or case["cols"]))
        return {"bytes": n * (2 + 2 + 2 + 1) + 4 * case["rows"] * groups + 2 * case["cols"], "flops": 6 * n}
    if case["op"] == "rotary":
        tokens = case["batch"] * case["length"]
        n = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 4 * n + 4 * tokens * case["axes"], "flops": 3 * n}
    pairs, rows = _pairs(case)
    dim, heads, kv_heads = case["dim"], case["heads"], case["kv_heads"]
    q_bytes = 2 * case["batch"] * heads * case["queries"] * dim
    kv_bytes = 2 * 2 * rows * kv_heads * dim
    products = 2 * pairs * heads * dim
    if case["op"] == "train":  # two products forward, five backward; q, k, v, dout in, out and gradients back
        return {"bytes": 4 * q_bytes + 2 * kv_bytes, "flops": 7 * products}
    lse = 0 if case["op"] == "decode" else 4 * case["batch"] * heads * case["queries"]
    return {"bytes": 2 * q_bytes + kv_bytes + lse, "flops": 2 * products}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(state, case)
        if case["op"] == "rotary":
            return _exact_rotary(state, case)
        return _exact_attention(state, case)


def _exact_norm(state, case):
    s = state["h"].double().add(state["r"])
    length = torch.linalg.vector_norm(s, dim=-1, keepdim=True)
    y = s.mul(state["w"].double()).div((length.pow(2) / s.shape[1] + 1e-6).sqrt())
    pieces, scales = [], []
    for part in y.split(case["group"] or y.shape[1], dim=1):
        unit = torch.linalg.vector_norm(part, ord=math.inf, dim=1, keepdim=True) / E4M3_MAX
        unit = torch.where(unit == 0, 1.0, unit)
        pieces.append(part / unit)
        scales.append(unit)
    return torch.cat(pieces, 1), torch.cat(scales, 1), s


def _exact_rotary(state, case):
    """Each pair as a complex number times the unit number of its angle."""
    turns = []
    for axis, pairs in enumerate(state["sections"]):
        done = sum(state["sections"][:axis])
        f = state["inv_freq"][done : done + pairs].double()
        turns.append(torch.outer(state["positions"][axis].double().flatten(), f))
    angle = torch.cat(turns, 1)
    unit = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle).unsqueeze(1)

    def rotate(x):
        y = x.double().reshape(-1, x.shape[2], x.shape[3])
        head = y[..., : case["rotary"]]
        half = case["rotary"] // 2
        pair = head.unflatten(-1, (half, 2)) if case["interleaved"] else head.unflatten(-1, (2, half)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit)
        turned = turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2)
        y = y.clone()
        y[..., : case["rotary"]] = turned
        return y.view(x.shape)

    return rotate(state["q"]), rotate(state["k"])


def _exact_attention(state, case):
    """One sequence and one key head at a time, and only over the keys that exist."""
    op = case["op"]
    q = state["q"].detach()
    q = q.unsqueeze(2) if op == "decode" else q
    batch, heads, queries, dim = q.shape
    kv_heads = case["kv_heads"]
    each = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((batch, heads, queries), -math.inf, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out) if op == "train" else None
    dk = torch.zeros(state["k"].shape, dtype=torch.float64, device="cuda") if op == "train" else None
    dv = torch.zeros_like(dk) if op == "train" else None
    for b, length in enumerate(_lengths(case)):
        first = length - 1 if op == "decode" else case["keys"] - queries
        n = min(queries, length - first)  # queries of this sequence that exist
        if n <= 0:
            continue
        at = torch.arange(first, first + n, device="cuda").unsqueeze(1)
        key = torch.arange(length, device="cuda").unsqueeze(0)
        hidden = (key > at) | ((at - key >= case["window"]) & (key >= case["sinks"]))
        for h in range(kv_heads):
            rows = slice(h * each, (h + 1) * each)
            kd = state["k"][b, h, :length].detach().double()
            vd = state["v"][b, h, :length].detach().double()
            qd = q[b, rows, :n].double()
            score = (qd.reshape(-1, dim) @ kd.T).view(each, n, length) * state["scale"]
            score.masked_fill_(hidden, -math.inf)
            z = torch.logsumexp(score, -1)
            p = score.sub_(z.unsqueeze(-1)).exp_()
            o = (p.view(-1, length) @ vd).view(each, n, dim)
            out[b, rows, :n], lse[b, rows, :n] = o, z
            if op == "train":
                g = state["dout"][b, rows, :n].double()
                dv[b, h, :length] = p.reshape(-1, length).T @ g.reshape(-1, dim)
                slope = (g.reshape(-1, dim) @ vd.T).view(each, n, length)
                slope = (slope - (g * o).sum(-1, keepdim=True)).mul_(p)
                dq[b, rows, :n] = (slope.reshape(-1, length) @ kd).view(each, n, dim) * state["scale"]
                dk[b, h, :length] = slope.reshape(-1, length).T @ qd.reshape(-1, dim) * state["scale"]
    if op == "decode":
        return out[:, :, 0]
    if op == "prefill":
        return out, lse
    return out, dq, dk, dv
