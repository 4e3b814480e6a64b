"""Decoder-layer operators against their plain forms in 64 bits: residual norm with an 8-bit result, rotary
positions over several axes, attention with a sliding window and visible first tokens.

Tolerances are error bounds derived from the roundings each kernel makes (half a step of the type per rounding, the
fp32 accumulation bounds beside it); tests/decoder_reference.py holds those of attention."""
import math

import pytest
import torch

from tests import decoder_reference as R
from tests.helpers import announce

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def K():
    from inductor_x_amd import kernels

    return kernels


def within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} against {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() - bound).amax() if got.numel() else torch.tensor(-1.0)
    assert over <= 0, f"{what}: {over.item():.3g} over the bound"


# ------------------------------------------------------------------------------------ norm
def norm_operands(rows, cols, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    h = torch.randn(rows, cols, generator=gen).to(dtype)
    r = (2 * torch.randn(rows, cols, generator=gen)).to(dtype)
    r[:, :: max(1, cols // 5)] *= 20
    w = (1 + 0.1 * torch.randn(cols, generator=gen)).to(dtype)
    return h, r, w


def check_norm(got, h, r, w, eps, group):
    q, scales, s = got
    x, unit, total = R.norm_quant(h, r, w, eps, group)
    assert q.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32 and s.dtype == h.dtype
    within(s.reshape(total.shape), total, total.abs() * R.half_step(h.dtype) + 2.0**-25, "s")
    # the sum of squares: at most 32 terms in a row per thread and ten folding steps, halved by the square root,
    # and a handful of single roundings: below 4e-6
    within(scales.reshape(unit.shape), unit, unit * 4e-6, "scales")
    # e4m3: half a step of the value, half the smallest step near zero, and 8e-6 from y and the scale
    within(q.reshape(x.shape), x, x.abs() * (2.0**-4 + 8e-6) + 2.0**-10, "q")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (70, 88), (5, 128), (2, 129), (66, 130), (37, 255), (19, 256), (9, 257), (7, 512),
                                       (9, 1000), (4, 1024), (6, 2048), (3, 2051), (33, 4096), (2, 5120), (2, 8192), (2, 16384), (1, 20001), (1, 32768)])
def test_norm_quant(K, rows, cols, group, dtype):
    announce(f"add_rmsnorm_quant rows={rows} cols={cols} group={group} {dtype}")
    h, r, w = norm_operands(rows, cols, dtype)
    check_norm(K.add_rmsnorm_quant(h.to(DEV), r.to(DEV), w.to(DEV), 1e-6, group=group), h, r, w, 1e-6, group)


def test_norm_quant_strides_and_axes(K):
    announce("add_rmsnorm_quant strides")
    h, r, w = norm_operands(24, 384, BF)
    wide = torch.zeros(24, 1024, dtype=BF, device=DEV)
    wide[:, 128:512] = h.to(DEV)
    odd = torch.zeros(24 * 384 + 1, dtype=BF, device=DEV)[1:].view(24, 384)  # rows off the 16-byte grid
    odd.copy_(r)
    got = K.add_rmsnorm_quant(wide[:, 128:512], odd, w.to(DEV), 1e-6, group=128)
    check_norm(got, h, r, w, 1e-6, 128)
    got3 = K.add_rmsnorm_quant(h.to(DEV).view(2, 12, 384), r.to(DEV).view(2, 12, 384), w.to(DEV), 1e-6, group=128)
    assert got3[0].shape == (2, 12, 384) and got3[1].shape == (2, 12, 3) and got3[2].shape == (2, 12, 384)
    check_norm(got3, h, r, w, 1e-6, 128)


def test_norm_quant_empty_zero_and_nonfinite(K):
    announce("add_rmsnorm_quant edge values")
    w = torch.ones(256, dtype=BF, device=DEV)
    q, scales, s = K.add_rmsnorm_quant(torch.empty(0, 256, dtype=BF, device=DEV), torch.empty(0, 256, dtype=BF, device=DEV), w)
    assert q.shape == (0, 256) and scales.shape == (0, 1) and s.shape == (0, 256)
    h = torch.randn(4, 256).to(BF)
    h[0] = 0
    h[1, 3] = float("nan")
    h[2, 200] = float("inf")
    z = torch.zeros(4, 256, dtype=BF, device=DEV)
    q, scales, s = (t.float().cpu() for t in K.add_rmsnorm_quant(h.to(DEV), z, w, 1e-6, group=128))
    assert (q[0] == 0).all() and (scales[0] == 1).all()
    assert torch.isnan(q[1]).all() and torch.isnan(scales[1]).all()
    # an infinity: its own 128 columns become NaN, the others zero, as inf * 0 and x * 0 say
    assert torch.isnan(scales[2, 1]) and scales[2, 0] == 1 and (q[2, :128] == 0).all()
    assert torch.isfinite(q[3]).all() and scales[3].min() > 0
    assert torch.equal(s.isnan(), h.float().isnan())
    # the smallest numbers of the type: no division by a scale that underflowed
    tiny = torch.full((2, 256), 2.0**-133).to(BF)
    q, scales, _ = K.add_rmsnorm_quant(tiny.to(DEV), torch.zeros_like(tiny).to(DEV), w, 1e-6)
    assert torch.isfinite(q.float()).all() and (scales > 0).all()


# ------------------------------------------------------------------------------------ rotary
def check_rotary(got, x, positions, inv_freq, sections, interleaved, inverse):
    want = R.rotary(x, positions, inv_freq, sections, interleaved, inverse)
    # a rounding of the result, and in fp32: sine and cosine off by 4e-7 (angle 2e-7, function 2 ulp), two products
    # and a sum of numbers no larger than the pair, 2e-7
    size = x.double().abs().amax(-1, keepdim=True).expand_as(want)
    within(got, want, want.abs() * R.half_step(x.dtype) + 1.5e-6 * size + 2.0**-25, "rotary")


@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,N,Nk,D,pairs,sections,first", [
    (1, 1, 1, 1, 2, 1, [1], 0),
    (2, 5, 4, 2, 64, 32, [32], 0),
    (1, 7, 3, 1, 80, 20, [12, 8], 1000000),
    (3, 33, 8, 2, 128, 64, [16, 24, 24], 123456),
    (2, 3, 2, 2, 96, 48, [1, 46, 0, 1], 50),
    (1, 4, 5, 5, 22, 7, [3, 4], 9),
    (1, 515, 16, 4, 128, 64, [64], 0),
])
def test_rotary(K, B, S, N, Nk, D, pairs, sections, first, interleaved, dtype):
    announce(f"rotary_axes {B, S, N, Nk, D, pairs, sections, first, interleaved} {dtype}")
    gen = torch.Generator().manual_seed(1)
    q, k = torch.randn(B, S, N, D, generator=gen).to(dtype), torch.randn(B, S, Nk, D, generator=gen).to(dtype)
    positions = first + torch.randint(0, 5000, (len(sections), B, S), generator=gen)
    inv_freq = (10000.0 ** (-torch.arange(pairs).double() / pairs)).float()
    for inverse in (False, True):
        got = K.rotary_axes(q.to(DEV), k.to(DEV), positions.to(torch.int32).to(DEV), inv_freq.to(DEV), sections, interleaved, inverse)
        for x, y in zip((q, k), got):
            check_rotary(y, x, positions, inv_freq, sections, interleaved, inverse)


def test_rotary_forms_of_operands(K):
    announce("rotary_axes strides, int64 far positions, fp64 frequencies, one axis without its dimension, empty")
    gen = torch.Generator().manual_seed(2)
    qkv = torch.randn(2, 9, 3, 4, 64, generator=gen).to(BF)  # [B, S, (q, k, v), N, D] as one projection leaves it
    dev = qkv.to(DEV)
    positions = torch.randint(2**33, 2**33 + 10, (2, 9), generator=gen)
    inv_freq = 10000.0 ** (-torch.arange(32).double() / 32)
    got = K.rotary_axes(dev[:, :, 0], dev[:, :, 1], positions.to(DEV), inv_freq.to(DEV))
    for x, y in zip((qkv[:, :, 0], qkv[:, :, 1]), got):
        # 2^33 positions at frequency 1: 1.4e9 turns in 64 bits, 2e-7 of a turn off, 1.3e-6 of the angle
        want = R.rotary(x, positions.unsqueeze(0), inv_freq, [32], False, False)
        within(y, want, want.abs() * R.half_step(BF) + 1e-5 * x.double().abs().amax(), "far")
    heads_first = torch.randn(2, 4, 9, 64, generator=gen).to(BF)
    t = heads_first.to(DEV).transpose(1, 2)
    y, _ = K.rotary_axes(t, t, torch.zeros(2, 9, dtype=torch.int32, device=DEV), inv_freq.to(DEV))
    assert torch.equal(y.cpu(), heads_first.transpose(1, 2)) and y.stride() == t.stride()  # position 0 turns nothing
    e, _ = K.rotary_axes(t[:, :0], t[:, :0], torch.zeros(2, 0, dtype=torch.int32, device=DEV), inv_freq.to(DEV))
    assert e.shape == (2, 0, 4, 64)


# ------------------------------------------------------------------------------------ decode
def caches(B, Nk, capacity, D, dtype, token_major, gen):
    shape = (B, capacity, Nk, D) if token_major else (B, Nk, capacity, D)
    c = torch.randn(*shape, generator=gen).to(dtype)
    return c.transpose(1, 2) if token_major else c


def same_memory(t):
    """The tensor on the GPU with its strides."""
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV)
    return out.copy_(t)


def decode_reference(q, k, v, lengths, scale, window, sinks):
    B, N, D = q.shape
    out, weight = torch.zeros(B, N, D, dtype=torch.float64), torch.zeros(B, N, D, dtype=torch.float64)
    for b, n in enumerate(lengths):
        n = min(max(n, 0), k.shape[2])
        if n:
            r = R.attention(q[b : b + 1].unsqueeze(2), k[b : b + 1, :, :n], v[b : b + 1, :, :n], scale, window, sinks)
            out[b], weight[b] = r["out"][0, :, 0], r["weight"][0, :, 0]
    return out, weight


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("B,N,Nk,D,capacity,window,sinks,lengths", [
    (1, 1, 1, 8, 1, 1, 0, [1]),
    (3, 4, 2, 64, 40, 16, 3, [0, 17, 40]),
    (2, 8, 1, 128, 300, 64, 4, [300, 66]),
    (1, 40, 2, 96, 200, 1000, 0, [199]),           # 20 query heads on a key head: two workgroups' worth
    (5, 6, 3, 80, 129, 33, 64, [1, 2, 98, 129, 97]),
    (1, 8, 2, 128, 5000, 4096, 4, [4999]),           # many splits
    (2, 3, 1, 56, 700, 512, 100, [611, 700]),
    (4, 2, 2, 64, 65, 2**31 - 1, 2**31 - 1, [65, 1, 0, 64]),
])
def test_decode(K, B, N, Nk, D, capacity, window, sinks, lengths, token_major, dtype):
    announce(f"window_attention_decode {B, N, Nk, D, capacity, window, sinks, lengths, token_major} {dtype}")
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(B, N, D, generator=gen).to(dtype)
    k, v = (caches(B, Nk, capacity, D, dtype, token_major, gen) for _ in range(2))
    want, weight = decode_reference(q, k, v, lengths, D**-0.5, window, sinks)
    # what lies behind a sequence's length, or between its first tokens and its window, must not matter
    for b, n in enumerate(lengths):
        for c in (k, v):
            c[b, :, n:] = float("nan")
            c[b, :, min(sinks, n) : max(0, n - window)] = float("inf")
    got = K.window_attention_decode(q.to(DEV), same_memory(k), same_memory(v), torch.tensor(lengths, dtype=torch.int32, device=DEV),
                                    D**-0.5, window, sinks)
    assert got.dtype == dtype
    within(got, want, R.attention_bound(want, weight, dtype), "decode")


def test_decode_lengths_beyond_the_cache(K):
    announce("window_attention_decode lengths beyond the capacity and below zero")
    gen = torch.Generator().manual_seed(4)
    q = torch.randn(3, 4, 64, generator=gen).to(BF)
    k, v = (caches(3, 2, 50, 64, BF, False, gen) for _ in range(2))
    want, weight = decode_reference(q, k, v, [50, 0, 50], 0.125, 20, 2)
    got = K.window_attention_decode(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor([51, -3, 2**31 - 1], dtype=torch.int32, device=DEV),
                                    0.125, 20, 2)
    within(got, want, R.attention_bound(want, weight, BF), "clamped")


def test_decode_offsets_past_32_bits(K):
    announce("window_attention_decode in a cache whose byte offsets pass 2^32")
    # two sequences of 8 heads: rows 2 KiB apart, 1.2 million tokens: 2.4 GB a sequence, the window at its end
    capacity, n = 1_200_000, 1_199_990
    gen = torch.Generator().manual_seed(5)
    cache = torch.zeros(2, capacity, 8, 128, dtype=BF, device=DEV)
    near = torch.randn(2, 64, 8, 128, generator=gen).to(BF)
    cache[:, n - 64 : n] = near.to(DEV)
    q = torch.randn(2, 8, 128, generator=gen).to(BF)
    view = cache.transpose(1, 2)
    got = K.window_attention_decode(q.to(DEV), view, view, torch.tensor([n, n], dtype=torch.int32, device=DEV), 0.1, 64, 0)
    small = near.transpose(1, 2)
    want, weight = decode_reference(q, small, small, [64, 64], 0.1, 64, 0)
    within(got, want, R.attention_bound(want, weight, BF), "far")


def test_decode_captured_and_on_another_stream(K):
    announce("window_attention_decode captured in a graph, on a side stream")
    gen = torch.Generator().manual_seed(6)
    q = torch.randn(2, 8, 128, generator=gen).to(BF).to(DEV)
    k, v = (caches(2, 2, 2000, 128, BF, False, gen).to(DEV) for _ in range(2))
    lengths = torch.tensor([2000, 700], dtype=torch.int32, device=DEV)
    call = lambda: K.window_attention_decode(q, k, v, lengths, 0.09, 1500, 4)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for step in range(4):
        q.copy_(torch.randn(2, 8, 128, generator=gen).to(BF))
        lengths.copy_(torch.tensor([1 + 400 * step, 2000 - 300 * step], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, call()), f"replay {step}"
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, call())


# ------------------------------------------------------------------------------------ prefill and training
WINDOW_CASES = [
    # B, N, Nk, Sq, Sk, D, window, sinks, lengths
    (1, 1, 1, 1, 1, 8, 1, 0, None),
    (2, 2, 1, 5, 5, 64, 3, 0, None),
    (1, 2, 2, 64, 64, 128, 64, 0, None),
    (2, 3, 1, 65, 65, 128, 1, 1, None),                # every query sees itself and the first key
    (1, 8, 1, 130, 130, 64, 40, 4, None),              # eight heads in a workgroup
    (2, 4, 2, 333, 333, 80, 100, 3, [333, 41]),
    (3, 6, 2, 200, 200, 128, 64, 70, [1, 200, 130]),   # more first keys than a window
    (1, 5, 1, 300, 300, 96, 2**31 - 1, 0, None),       # plain causal, an odd group
    (1, 4, 1, 1, 700, 128, 256, 4, None),              # one query over a cache
    (2, 8, 2, 37, 612, 128, 129, 33, [612, 590]),
    (2, 2, 1, 100, 900, 64, 70, 4, [850, 700]),        # in the second sequence no query exists
    (1, 4, 4, 700, 700, 128, 200, 2, None),
    (1, 4, 2, 517, 1030, 128, 64, 128, None),
    (1, 2, 1, 900, 900, 128, 300, 900, None),          # everything is a first key
    (1, 2, 1, 900, 900, 64, 100, 701, None),           # first keys over eleven tiles
    # gradients of the first keys from queries far beyond their window, a kernel of their own
    (2, 8, 2, 777, 777, 128, 64, 4, [777, 300]),
    (2, 5, 1, 400, 400, 64, 33, 2, [400, 30]),         # the second sequence ends inside the first window
    (1, 6, 3, 600, 1500, 80, 100, 33, [1400]),
    (1, 1, 1, 1200, 1200, 96, 200, 1, None),
    (1, 2, 1, 900, 900, 64, 100, 200, None),           # seven blocks of first keys
    # rows that see a few keys in blocks of three and more tiles
    (2, 3, 1, 300, 300, 128, 3, 1, [300, 150]),
    (1, 1, 1, 777, 777, 64, 2, 0, None),
    (2, 2, 2, 200, 500, 128, 5, 3, [433, 500]),
]


def window_operands(B, N, Nk, Sq, Sk, D, dtype, token_major, seed=7):
    gen = torch.Generator().manual_seed(seed)
    q, dout = (caches(B, N, Sq, D, dtype, token_major, gen) for _ in range(2))
    k, v = (caches(B, Nk, Sk, D, dtype, token_major, gen) for _ in range(2))
    return q, k, v, dout


def device_lengths(lengths):
    return None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)


def poison(t, first, lengths):
    """NaN in every row that does not exist (row i of a sequence sits at position first + i)."""
    for b, n in enumerate(lengths or []):
        t[b, :, max(0, n - first):] = float("nan")


def lse_bound(want):
    # each term of the sum carries the error of its score, 6.2e-5 (attention_bound); log and exp add a few 2^-24
    return 1e-4 + 4e-7 * want.abs()


def check_window(K, case, dtype, token_major):
    B, N, Nk, Sq, Sk, D, window, sinks, lengths = case
    q, k, v, dout = window_operands(B, N, Nk, Sq, Sk, D, dtype, token_major)
    want = R.attention(q, k, v, D**-0.5, window, sinks, lengths, dout)
    poison(q, Sk - Sq, lengths), poison(dout, Sk - Sq, lengths), poison(k, 0, lengths), poison(v, 0, lengths)
    dq_, k_, v_, do_ = (same_memory(t) for t in (q, k, v, dout))
    ln = device_lengths(lengths)
    out, lse = K.window_attention(dq_, k_, v_, D**-0.5, window, sinks, ln)
    assert out.stride() == dq_.stride() and out.dtype == dtype and lse.dtype == torch.float32
    within(out, want["out"], R.attention_bound(want["out"], want["weight"], dtype), "out")
    none = torch.isinf(want["lse"])
    assert torch.equal(torch.isinf(lse.cpu()), none) and (out.cpu()[none] == 0).all()
    live = ~none
    within(lse.cpu()[live], want["lse"][live], lse_bound(want["lse"][live]), "lse")
    grads = K.window_attention_backward(dq_, k_, v_, out, do_, lse, D**-0.5, window, sinks, ln)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert got.dtype == dtype
        within(got, want[name], R.attention_bound(want[name], want[name + "_weight"], dtype), name)
    same, lse2, low = K.window_attention(dq_, k_, v_, D**-0.5, window, sinks, ln, keep_low=True)
    assert torch.equal(same, out) and torch.equal(lse2, lse)
    # out and its remainder together carry the roundings of the probabilities, and of the remainder: a step's step
    h = R.half_step(dtype)
    within(same.double().cpu() + low.double().cpu(), want["out"],
           want["out"].abs() * h * h + want["weight"] * (h + 2e-4) + 1e-5, "out + low")
    finer = K.window_attention_backward(dq_, k_, v_, out, do_, lse, D**-0.5, window, sinks, ln, low)
    for name, got in zip(("dq", "dk", "dv"), finer):
        within(got, want[name], R.attention_bound(want[name], want[name + "_weight"], dtype), name)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("case", WINDOW_CASES, ids=str)
def test_window_attention(K, case, token_major, dtype):
    announce(f"window_attention {case} token_major={token_major} {dtype}")
    check_window(K, case, dtype, token_major)


def test_window_gradients_through_autograd():
    announce("decoder.window_attention through autograd, strided gradient, against torch's own gradients in fp64")
    from inductor_x_amd import decoder

    B, N, Nk, S, D, window, sinks = 2, 4, 2, 150, 64, 40, 3
    q, k, v, _ = window_operands(B, N, Nk, S, S, D, BF, True)
    leaves = [same_memory(t).requires_grad_() for t in (q, k, v)]
    out = decoder.window_attention(*leaves, 0.125, window, sinks)
    out.sum().backward()  # a gradient of stride zero
    want = R.attention(q, k, v, 0.125, window, sinks, None, torch.ones_like(q))
    for leaf, name in zip(leaves, ("dq", "dk", "dv")):
        within(leaf.grad, want[name], R.attention_bound(want[name], want[name + "_weight"], BF), name)
    ref = [t.double().requires_grad_() for t in (q, k, v)]
    see = R.visible(0, S, S, window, sinks, S)
    s = (ref[0] @ ref[1].repeat_interleave(2, 1).transpose(-1, -2) * 0.125).masked_fill(~see, -math.inf)
    (s.softmax(-1) @ ref[2].repeat_interleave(2, 1)).sum().backward()
    for t, name in zip(ref, ("dq", "dk", "dv")):
        assert (t.grad - want[name]).abs().max() < 1e-12


@pytest.mark.parametrize("wanted", [0, 1, 2])
def test_window_gradient_of_one_operand(wanted):
    announce(f"decoder.window_attention, a gradient of operand {wanted} alone")
    from inductor_x_amd import decoder

    q, k, v, dout = window_operands(2, 4, 2, 90, 90, 64, BF, False, seed=16)
    want = R.attention(q, k, v, 0.125, 30, 2, [90, 20], dout)
    operands = [t.to(DEV) for t in (q, k, v)]
    operands[wanted].requires_grad_()
    decoder.window_attention(*operands, 0.125, 30, 2, device_lengths([90, 20])).backward(dout.to(DEV))
    for i, (t, name) in enumerate(zip(operands, ("dq", "dk", "dv"))):
        if i == wanted:
            within(t.grad, want[name], R.attention_bound(want[name], want[name + "_weight"], BF), name)
        else:
            assert t.grad is None


def test_rotary_gradients_through_autograd():
    announce("decoder.rotary_axes through autograd")
    from inductor_x_amd import decoder

    gen = torch.Generator().manual_seed(8)
    q, k = torch.randn(2, 5, 3, 32, generator=gen), torch.randn(2, 5, 1, 32, generator=gen)
    positions = torch.randint(0, 50, (2, 2, 5), generator=gen)
    inv_freq = 100.0 ** (-torch.arange(12).double() / 12)
    dq, dk = torch.randn(2, 5, 3, 32, generator=gen), torch.randn(2, 5, 1, 32, generator=gen)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k)]
    outs = decoder.rotary_axes(*leaves, positions.to(DEV), inv_freq.to(DEV), [5, 7])
    torch.autograd.backward(outs, [dq.to(DEV), dk.to(DEV)])
    for x, g, leaf in ((q, dq, leaves[0]), (k, dk, leaves[1])):
        ref = x.double().requires_grad_()
        y = ref.clone()
        angle = torch.cat([positions[0].double().unsqueeze(-1) * inv_freq[:5], positions[1].double().unsqueeze(-1) * inv_freq[5:]], -1).unsqueeze(2)
        a, b = ref[..., :12], ref[..., 12:24]
        y = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), ref[..., 24:]), -1)
        y.backward(g.double())
        within(leaf.grad, ref.grad, 1e-5 + 1e-6 * ref.grad.abs(), "rotary gradient")


# ------------------------------------------------------------------------------------ calls of other kinds
def test_window_attention_on_slices_and_broadcasts():
    announce("window_attention on slices of one projection, on keys expanded over the batch")
    from inductor_x_amd import decoder, kernels as K

    B, S, N, Nk, D, window, sinks = 2, 190, 6, 2, 64, 50, 2
    gen = torch.Generator().manual_seed(9)
    qkv = torch.randn(B, S, N + 2 * Nk, D, generator=gen).to(BF)
    dev = qkv.to(DEV).requires_grad_()
    parts = lambda t: (t[:, :, :N].transpose(1, 2), t[:, :, N : N + Nk].transpose(1, 2), t[:, :, N + Nk :].transpose(1, 2))  # noqa: E731
    dout = torch.randn(B, N, S, D, generator=gen).to(BF)
    want = R.attention(*parts(qkv), 0.125, window, sinks, None, dout)
    out = decoder.window_attention(*parts(dev), 0.125, window, sinks)
    within(out, want["out"], R.attention_bound(want["out"], want["weight"], BF), "out")
    out.backward(dout.to(DEV))
    for got, name in zip(parts(dev.grad), ("dq", "dk", "dv")):
        within(got, want[name], R.attention_bound(want[name], want[name + "_weight"], BF), name)
    # one set of keys for the whole batch
    q, k, v, dout = window_operands(3, 4, 2, 70, 70, D, BF, False)
    k1, v1 = k[:1], v[:1]
    want = R.attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), 0.125, 20, 1, None, dout)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k1, v1)]
    out = decoder.window_attention(leaves[0], leaves[1].expand(3, -1, -1, -1), leaves[2].expand(3, -1, -1, -1), 0.125, 20, 1)
    within(out, want["out"], R.attention_bound(want["out"], want["weight"], BF), "out, shared keys")
    out.backward(dout.to(DEV))
    for leaf, name in zip(leaves[1:], ("dk", "dv")):
        # three gradients of 16 bits, added by autograd in 16 bits: two more roundings
        total, size = want[name].sum(0, keepdim=True), want[name].abs().sum(0, keepdim=True)
        bound = R.attention_bound(want[name], want[name + "_weight"], BF).sum(0, keepdim=True) + 2 * R.half_step(BF) * 1.02 * size
        within(leaf.grad, total, bound, name + ", shared keys")


def test_window_attention_far_rows():
    announce("window_attention with keys whose byte offsets pass 2^31, forward and gradients")
    from inductor_x_amd import kernels as K

    Sk, Sq, window, sinks, D, heads = 1_150_000, 70, 100, 5, 128, 8
    gen = torch.Generator().manual_seed(10)
    base = torch.zeros(1, Sk, heads, D, dtype=BF, device=DEV)
    head, tail = torch.randn(1, 8, heads, D, generator=gen).to(BF), torch.randn(1, 200, heads, D, generator=gen).to(BF)
    base[:, :8], base[:, Sk - 200 :] = head.to(DEV), tail.to(DEV)
    kv = base.transpose(1, 2)
    q, dout = (torch.randn(1, heads, Sq, D, generator=gen).to(BF) for _ in range(2))
    out, lse, low = K.window_attention(q.to(DEV), kv, kv, 0.09, window, sinks, keep_low=True)
    # the same positions with the unseen middle cut out: 8 + 200 keys, the window never reaches the first
    near = torch.cat((head, tail), 1).transpose(1, 2)
    want = R.attention(q, near, near, 0.09, window, sinks, None, dout)
    within(out, want["out"], R.attention_bound(want["out"], want["weight"], BF), "out")
    dq, dk, dv = K.window_attention_backward(q.to(DEV), kv, kv, out, dout.to(DEV), lse, 0.09, window, sinks, None, low)
    within(dq, want["dq"], R.attention_bound(want["dq"], want["dq_weight"], BF), "dq")
    for got, name in ((dk, "dk"), (dv, "dv")):
        assert not got[:, :, 8 : Sk - 200].any()
        got = torch.cat((got[:, :, :8], got[:, :, Sk - 200 :]), 2)
        within(got, want[name], R.attention_bound(want[name], want[name + "_weight"], BF), name)


def test_many_small_sequences():
    announce("70000 sequences of three tokens, 70000 caches")
    from inductor_x_amd import kernels as K

    gen = torch.Generator().manual_seed(11)
    q, k, v, dout = window_operands(70000, 1, 1, 3, 3, 8, BF, False, seed=11)
    d = [t.to(DEV) for t in (q, k, v, dout)]
    out, lse, low = K.window_attention(*d[:3], 0.3, 2, 0, keep_low=True)
    grads = K.window_attention_backward(*d[:3], out, d[3], lse, 0.3, 2, 0, None, low)
    last = slice(69990, 70000)
    want = R.attention(*(t[last] for t in (q, k, v)), 0.3, 2, 0, None, dout[last])
    within(out[last], want["out"], R.attention_bound(want["out"], want["weight"], BF), "out")
    for got, name in zip(grads, ("dq", "dk", "dv")):
        within(got[last], want[name], R.attention_bound(want[name], want[name + "_weight"], BF), name)
    got = K.window_attention_decode(q.to(DEV)[:, :, 2], d[1], d[2], torch.full((70000,), 3, dtype=torch.int32, device=DEV), 0.3, 2, 0)
    within(got[last], want["out"][:, :, 2], R.attention_bound(want["out"], want["weight"], BF)[:, :, 2], "decode")


def training_call(K, q, k, v, dout, window, sinks, lengths):
    out, lse, low = K.window_attention(q, k, v, 0.1, window, sinks, lengths, True)
    return (out, lse, *K.window_attention_backward(q, k, v, out, dout, lse, 0.1, window, sinks, lengths, low))


def test_window_attention_repeats_captures_and_streams(K):
    announce("window_attention: equal bits on every run, in a replayed graph, and on two streams at once")
    gen = torch.Generator().manual_seed(12)
    q, k, v, dout = (t.to(DEV) for t in window_operands(2, 8, 2, 500, 500, 128, BF, False, seed=12))
    lengths = torch.tensor([500, 301], dtype=torch.int32, device=DEV)
    call = lambda: training_call(K, q, k, v, dout, 90, 4, lengths)  # noqa: E731
    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]  # two graphs with workspaces of their own
    held = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(call())
    for step in range(3):
        q.copy_(torch.randn(q.shape, generator=gen).to(BF))
        lengths.copy_(torch.tensor([500 - 100 * step, 37 + step], dtype=torch.int32))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = call()
        for got in held:
            assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {step}"
    other = [t.to(DEV) for t in window_operands(2, 8, 2, 500, 500, 128, BF, False, seed=13)]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = []
    for side, operands in zip(sides, ((q, k, v, dout), other)):
        with torch.cuda.stream(side):
            results.append([training_call(K, *operands, 90, 4, lengths) for _ in range(4)])
    torch.cuda.synchronize()
    for runs, operands in zip(results, ((q, k, v, dout), other)):
        want = training_call(K, *operands, 90, 4, lengths)
        for got in runs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_training_step_captured():
    announce("rotary and window attention with their gradients in a replayed graph")
    from inductor_x_amd import decoder

    gen = torch.Generator().manual_seed(21)
    B, S, N, Nk, D = 2, 300, 4, 2, 64
    leaves = [torch.randn(B, S, n, D, generator=gen).to(BF).to(DEV).requires_grad_() for n in (N, Nk, Nk)]
    dout = torch.randn(B, N, S, D, generator=gen).to(BF).to(DEV)
    positions = torch.arange(S, device=DEV).expand(B, S).contiguous()
    inv_freq = 100.0 ** (-torch.arange(D // 2, device=DEV).double() / D)
    lengths = torch.tensor([300, 111], dtype=torch.int32, device=DEV)

    def step():
        q, k = decoder.rotary_axes(leaves[0], leaves[1], positions, inv_freq)
        out = decoder.window_attention(q.transpose(1, 2), k.transpose(1, 2), leaves[2].transpose(1, 2), 0.125, 70, 3, lengths)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # loads the code; its graph of gradients is gone when it returns
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            for t in (*leaves, dout):
                t.copy_(torch.randn(t.shape, generator=gen).to(BF))
        lengths.copy_(torch.tensor([300 - 90 * i, 1 + i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), f"replay {i}"


def test_launches_are_logged(K):
    announce("the symbols of a call's launches, with gradients too")
    from inductor_x_amd import decoder, launcher

    q, k, v, dout = (t.to(DEV) for t in window_operands(1, 4, 2, 450, 450, 64, BF, False, seed=14))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    launcher.launch_log = []
    try:
        decoder.window_attention(*leaves, 0.1, 64, 4).backward(dout)
        K.window_attention_decode(q.detach()[:, :, 0], k.detach(), v.detach(), torch.full((1,), 450, dtype=torch.int32, device=DEV), 0.1, 64)
    finally:
        log, launcher.launch_log = launcher.launch_log, None
    kinds = ["fwd", "bwd_dq", "bwd_dkv", "bwd_sinks", "bwd_join"]
    assert log == [f"window_attention_{x}_bf16_d64" for x in kinds] + ["window_decode_bf16_d64"]


def test_norm_and_rotary_captured(K):
    announce("norm and rotary in one replayed graph")
    gen = torch.Generator().manual_seed(14)
    h, r, w = (t.to(DEV) for t in norm_operands(40, 512, BF))
    at = torch.zeros(1, 40, dtype=torch.int32, device=DEV)
    inv_freq = (100.0 ** (-torch.arange(32).float() / 32)).to(DEV)
    call = lambda: (*K.add_rmsnorm_quant(h, r, w, group=128), *K.rotary_axes(h.view(1, 40, 8, 64), r.view(1, 40, 8, 64), at, inv_freq))  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for step in range(3):
        h.copy_(torch.randn(40, 512, generator=gen).to(BF))
        at.copy_(torch.randint(0, 10000, (1, 40), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(held, call())), f"replay {step}"


def test_plans_do_not_outlive_their_shapes(K):
    announce("the same storage under other shapes, strides, types and alignments")
    gen = torch.Generator().manual_seed(15)
    raw = torch.randn(4096 * 3, generator=gen).to(BF).to(DEV)
    w = torch.ones(4096, dtype=BF, device=DEV)
    for rows, cols, offset in ((2, 512, 0), (4, 256, 0), (2, 512, 1), (2, 512, 8), (1, 1024, 0), (8, 128, 3)):
        h = raw[offset : offset + rows * cols].view(rows, cols)
        check_norm(K.add_rmsnorm_quant(h, h, w[:cols]), h.cpu(), h.cpu(), w[:cols].cpu(), 1e-6, 0)
    part, whole = raw[:2048].view(2, 1024)[:, :512], raw[:1024].view(2, 512)
    check_norm(K.add_rmsnorm_quant(part, whole, w[:512]), part.cpu(), whole.cpu(), w[:512].cpu(), 1e-6, 0)


def test_one_token_with_any_stride(K):
    announce("single tokens whose stride is no multiple of anything")
    gen = torch.Generator().manual_seed(18)
    raw = torch.randn(4, 2 * 2 * 64 + 64, generator=gen).to(BF).to(DEV)
    odd = lambda t: t[: 2 * 2 * 64].as_strided((2, 2, 1, 64), (128, 64, 7, 1))  # noqa: E731
    q, k, v, dout = (odd(t) for t in raw)
    want = R.attention(q.cpu(), k.cpu(), v.cpu(), 0.125, 5, 2, None, dout.cpu())
    out, lse, low = K.window_attention(q, k, v, 0.125, 5, 2, keep_low=True)
    within(out, want["out"], R.attention_bound(want["out"], want["weight"], BF), "out")
    for got, name in zip(K.window_attention_backward(q, k, v, out, dout, lse, 0.125, 5, 2, None, low), ("dq", "dk", "dv")):
        within(got, want[name], R.attention_bound(want[name], want[name + "_weight"], BF), name)
    got = K.window_attention_decode(q[:, :, 0], k, v, torch.ones(2, dtype=torch.int32, device=DEV), 0.125, 5, 2)
    within(got, want["out"][:, :, 0], R.attention_bound(want["out"], want["weight"], BF)[:, :, 0], "decode")


def test_second_gradients():
    announce("a gradient of the rotary gradient; window attention refuses one")
    from inductor_x_amd import decoder

    x = torch.randn(1, 3, 2, 8, device=DEV, requires_grad=True)
    at, freq = torch.arange(3, dtype=torch.int32, device=DEV).view(1, 3), torch.tensor([1.0, 0.1], device=DEV)
    y, _ = decoder.rotary_axes(x, x.detach(), at, freq)
    g = torch.autograd.grad(y.square().sum() / 2, x, create_graph=True)[0]
    # y is a rotation of x, so half its square sum has the gradient x, and x^3 summed over it the gradient 3 x^2
    assert torch.allclose(torch.autograd.grad((g**3).sum(), x)[0], 3 * x.detach() ** 2, rtol=1e-4, atol=1e-5)
    q = torch.randn(1, 2, 4, 8, dtype=BF, device=DEV, requires_grad=True)
    out = decoder.window_attention(q, q, q, 0.3, 2)
    first = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.float().square().sum().backward()


# ------------------------------------------------------------------------------------ used together
class Layer(torch.nn.Module):
    """The attention half of a decoder layer on these operators: norm with an 8-bit result, projections from it, rotary
    positions over three axes, window attention, output projection."""

    def __init__(self, width, heads, kv_heads, dim, window, sinks, gen):
        super().__init__()
        self.register_buffer("norm", torch.ones(width, dtype=BF, device=DEV))
        w = torch.randn((heads + 2 * kv_heads) * dim, width, generator=gen) / math.sqrt(width)
        scale = w.abs().amax(1, keepdim=True) / 448
        self.register_buffer("wqkv", (w / scale).to(torch.float8_e4m3fn).to(DEV).t())
        self.register_buffer("wqkv_scale", scale.t().contiguous().to(DEV))
        self.register_buffer("wo", (torch.randn(heads * dim, width, generator=gen) / math.sqrt(heads * dim)).to(BF).to(DEV))
        self.heads, self.kv_heads, self.dim, self.window, self.sinks = heads, kv_heads, dim, window, sinks
        self.register_buffer("inv_freq", (10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).float().to(DEV))

    def projections(self, h, r, positions):
        from inductor_x_amd import decoder

        q8, scales, s = decoder.add_rmsnorm_quant(h, r, self.norm)
        x = torch._scaled_mm(q8.flatten(0, 1), self.wqkv, scales.flatten(0, 1), self.wqkv_scale, out_dtype=BF)
        q, k, v = x.view(*h.shape[:2], -1, self.dim).split([self.heads, self.kv_heads, self.kv_heads], 2)
        q, k = decoder.rotary_axes(q, k, positions, self.inv_freq, [self.dim // 2 - 20, 10, 10])
        return s, q, k, v

    def forward(self, h, r, positions):
        from inductor_x_amd import decoder

        s, q, k, v = self.projections(h, r, positions)
        out = decoder.window_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), self.dim**-0.5, self.window, self.sinks)
        return s, torch.matmul(out.transpose(1, 2).flatten(-2), self.wo), k, v

    def step(self, h, r, positions, k_cache, v_cache, lengths):
        from inductor_x_amd import decoder

        s, q, k, v = self.projections(h, r, positions)
        at = (lengths - 1).long()
        rows = torch.arange(h.shape[0], device=DEV)
        k_cache[rows, at], v_cache[rows, at] = k[:, 0], v[:, 0]
        out = decoder.window_attention_decode(q[:, 0], k_cache.transpose(1, 2), v_cache.transpose(1, 2), lengths, self.dim**-0.5,
                                              self.window, self.sinks)
        return s, torch.matmul(out.flatten(-2), self.wo)


def layer_and_texts(B=2, S=75, width=256, window=20, sinks=3):
    gen = torch.Generator().manual_seed(16)
    layer = Layer(width, 8, 2, 64, window, sinks, gen)
    h, r = (torch.randn(B, S, width, generator=gen).to(BF).to(DEV) for _ in range(2))
    at = torch.arange(S).view(1, S).expand(B, S)
    positions = torch.stack((at + 1000, at // 10, at % 10)).to(torch.int32).contiguous().to(DEV)
    return layer, h, r, positions


def test_decoding_follows_the_prefill():
    announce("a layer's prefill against the same tokens decoded one by one over a cache")
    layer, h, r, positions = layer_and_texts()
    B, S = h.shape[:2]
    s, out, k, v = layer(h, r, positions)
    k_cache, v_cache = (torch.full((B, S + 30, 2, 64), float("nan"), dtype=BF, device=DEV) for _ in range(2))
    for t in range(S):
        lengths = torch.full((B,), t + 1, dtype=torch.int32, device=DEV)
        s1, o1 = layer.step(h[:, t : t + 1], r[:, t : t + 1], positions[:, :, t : t + 1].contiguous(), k_cache, v_cache, lengths)
        assert torch.equal(s1[:, 0], s[:, t])
        # both attention outputs are within two roundings of the same value (probabilities, result) times the weight,
        # below 1 for a mean of unit normals; the products then add 512 such errors over sqrt(512) weights of 1 / sqrt(512):
        # at most 2 * 2 * 2^-8 * sqrt(512) = 0.35 if all had one sign, 0.016 * 3 as independent errors; their own
        # roundings to 16 bits (inputs to and outputs of the projections in another order) are of the same size
        assert (o1.float() - out[:, t].float()).abs().max() <= 0.35
        assert (o1.float() - out[:, t].float()).norm() <= 0.03 * out[:, t].float().norm()
    keep = torch.equal(k_cache[:, :S].isnan(), torch.zeros_like(k_cache[:, :S], dtype=torch.bool))
    assert keep and k_cache[:, S:].isnan().all()  # rows behind the last token are left alone


def test_layer_compiles_into_one_graph():
    announce("a layer under torch.compile without a break, forward and decode, against its eager run")
    import inductor_x_amd  # noqa: F401

    layer, h, r, positions = layer_and_texts()
    want = layer(h, r, positions)
    got = torch.compile(layer, fullgraph=True)(h, r, positions)
    for a, b in zip(got, want):
        # the same kernels between products that the compiler may fuse with a conversion: rounding steps of bf16
        assert a.shape == b.shape and (a.float() - b.float()).norm() <= 0.02 * b.float().norm()


def test_gradients_compile():
    announce("rotary and window attention with gradients under torch.compile")
    from inductor_x_amd import decoder

    B, S, N, Nk, D = 2, 60, 4, 2, 64
    gen = torch.Generator().manual_seed(17)
    q, k, v = (torch.randn(B, S, n, D, generator=gen).to(BF) for n in (N, Nk, Nk))
    positions = torch.arange(S, dtype=torch.int32).view(1, 1, S).expand(1, B, S).contiguous().to(DEV)
    inv_freq = (100.0 ** (-torch.arange(D // 2).float() / (D // 2))).to(DEV)
    dout = torch.randn(B, N, S, D, generator=gen).to(BF).to(DEV)

    def f(q, k, v):
        q, k = decoder.rotary_axes(q, k, positions, inv_freq)
        return decoder.window_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), 0.125, 16, 2)

    results = []
    for fn in (f, torch.compile(f, fullgraph=True)):
        leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
        out = fn(*leaves)
        out.backward(dout)
        results.append([out.detach(), *(t.grad for t in leaves)])
    for a, b in zip(*results):
        assert torch.equal(a, b)  # the same kernels on the same operands


def test_recorded_calls_replay():
    announce("graphs recorded by make_fx and torch.jit.trace, replayed on other operands")
    from torch.fx.experimental.proxy_tensor import make_fx

    from inductor_x_amd import decoder, kernels as K

    gen = torch.Generator().manual_seed(22)
    B, S, N, Nk, D = 2, 60, 4, 2, 64
    draw = lambda: [torch.randn(B, S, n, D, generator=gen).to(BF).to(DEV) for n in (N, Nk, Nk)]  # noqa: E731
    positions = torch.arange(S, dtype=torch.int32, device=DEV).expand(B, S).contiguous()
    inv_freq = (100.0 ** (-torch.arange(D // 2).float() / (D // 2))).to(DEV)
    lengths = torch.tensor([60, 31], dtype=torch.int32, device=DEV)
    w = torch.ones(D, dtype=BF, device=DEV)

    def f(q, k, v):
        q, k = decoder.rotary_axes(q, k, positions, inv_freq)
        out = decoder.window_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), 0.125, 16, 2, lengths)
        last = K.window_attention_decode(q[:, -1], k.transpose(1, 2), v.transpose(1, 2), lengths, 0.125, 16, 2)
        return out, *(t.float() for t in decoder.add_rmsnorm_quant(last, last, w))

    def step(q, k, v):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        return torch.autograd.grad(f(q, k, v)[0].float().square().sum(), (q, k, v))

    first, second = draw(), draw()
    for replay in (make_fx(f)(*first), torch.jit.trace(f, tuple(first), check_trace=False)):
        for args in (first, second):
            for a, b in zip(replay(*args), f(*args)):
                assert torch.equal(a, b)
    replay = make_fx(step)(*first)
    for args in (first, second):
        for a, b in zip(replay(*args), step(*args)):
            assert torch.equal(a, b)


def test_rotary_tangents():
    announce("decoder.rotary_axes in forward mode: the tangent turns as the operand does")
    from torch.autograd import forward_ad as fw

    from inductor_x_amd import decoder

    gen = torch.Generator().manual_seed(23)
    q, tq = torch.randn(2, 2, 5, 3, 32, generator=gen)
    k, tk = torch.randn(2, 2, 5, 1, 32, generator=gen)
    positions = torch.randint(0, 50, (1, 2, 5), generator=gen)
    inv_freq = 100.0 ** (-torch.arange(12).double() / 12)
    place = lambda t: t.to(DEV)  # noqa: E731
    for grad in (False, True):
        for tangent in (place(tq), torch.ones(1, device=DEV).expand(2, 5, 3, 32)):  # of any layout
            with fw.dual_level():
                x = fw.make_dual(place(q).requires_grad_(grad), tangent)
                y, z = decoder.rotary_axes(x, fw.make_dual(place(k), place(tk)), place(positions), place(inv_freq), None, True)
                y, z = fw.unpack_dual(y), fw.unpack_dual(z)
            for got, x in ((y.primal, q), (y.tangent, tangent.cpu()), (z.primal, k), (z.tangent, tk)):
                check_rotary(got, x, positions, inv_freq, [12], True, False)
    with fw.dual_level():
        y, z = decoder.rotary_axes(fw.make_dual(place(q), place(tq)), place(k), place(positions), place(inv_freq))
        check_rotary(fw.unpack_dual(y).tangent, tq, positions, inv_freq, [12], False, False)
        t = fw.unpack_dual(z).tangent
        assert t is None or not t.any()


def test_gradients_arrive_anywhere():
    announce("window attention's gradient from outputs' gradients off the 16-byte grid: eager, the op, compiled")
    from inductor_x_amd import decoder

    q, k, v, dout = window_operands(2, 4, 2, 50, 50, 64, BF, False, seed=24)
    want = R.attention(q, k, v, 0.125, 16, 2, None, dout)
    flat = torch.empty(dout.numel() + 1, dtype=BF, device=DEV)
    odd = flat[1:].view(dout.shape).copy_(dout.to(DEV))
    wide = torch.empty(2, 4, 50, 68, dtype=BF, device=DEV)[..., :64].copy_(dout.to(DEV))
    f = lambda q, k, v: decoder.window_attention(q, k, v, 0.125, 16, 2)  # noqa: E731
    op = lambda q, k, v: torch.ops.npu_graph.window_attention(q, k, v, 0.125, 16, 2, None, True)[0]  # noqa: E731
    for fn in (f, op, torch.compile(f, fullgraph=True), torch.compile(f, fullgraph=True, backend="aot_eager")):
        for arriving in (odd, wide):
            leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
            fn(*leaves).backward(arriving)
            for leaf, name in zip(leaves, ("dq", "dk", "dv")):
                within(leaf.grad, want[name], R.attention_bound(want[name], want[name + "_weight"], BF), name)


# ------------------------------------------------------------------------------------ NaN and infinities in existing rows
def without(t, rows, columns):
    """t with the named elements (b, head, row, column) zero."""
    t = t.clone()
    for (b, h, r), c in zip(rows, columns):
        t[b, h, r, c] = 0
    return t


# B, N, Nk, Sq, Sk, D, window, sinks, lengths, rows of keys that hold something else than numbers
HIDDEN_CASES = [
    (1, 1, 1, 512, 512, 64, 64, 4, None, [65, 300]),          # a tile of first keys and window, read by four wavefronts
    (1, 6, 2, 512, 512, 128, 64, 4, None, [65, 130, 511]),    # an odd share of the heads
    (2, 8, 2, 700, 700, 128, 200, 2, [700, 333], [1, 320, 0]),
    (1, 4, 2, 200, 900, 128, 100, 40, None, [10, 790, 650]),  # over a cache; one row that nobody sees
    (1, 2, 1, 300, 300, 96, 2**31 - 1, 0, None, [150]),       # causal alone
    (1, 3, 1, 300, 300, 128, 3, 1, None, [100, 0]),           # D added up from P and dP over many tiles
    (2, 3, 1, 60, 60, 64, 5, 0, [60, 41], [20, 40]),          # and in one
    (1, 2, 1, 900, 900, 64, 100, 200, None, [70, 150, 500]),  # first keys with a kernel of their own
    (1, 8, 1, 2048, 2048, 128, 2048, 0, None, [1000]),        # a walk shared by workgroups
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("source", ["k", "v", "q", "dout"])
@pytest.mark.parametrize("case", HIDDEN_CASES, ids=str)
def test_hidden_pairs_do_not_count(K, case, source, dtype):
    """A NaN or an infinity reaches what sees it, as the formulas say, and nothing else."""
    announce(f"window_attention {case} with NaN and infinities in rows of {source} {dtype}")
    B, N, Nk, Sq, Sk, D, window, sinks, lengths, bad = case
    q, k, v, dout = window_operands(B, N, Nk, Sq, Sk, D, dtype, False, seed=25)
    t = {"q": q, "k": k, "v": v, "dout": dout}
    first = Sk - Sq
    if source in ("q", "dout"):
        bad = [max(0, r - first) for r in bad]
    rows = [(i % B, i % t[source].shape[1], r) for i, r in enumerate(bad)]
    columns = [[3], [D - 1], [0, 5]]
    clean = dict(t)
    clean[source] = without(t[source], rows, columns)
    for i, ((b, h, r), c) in enumerate(zip(rows, columns)):
        # an infinity in a score may mean a probability of zero, by its sign: NaN there
        t[source][b, h, r, c] = float("inf") if i == 1 and source in ("v", "dout") else float("nan")
    want = R.attention(*(clean[x] for x in "qkv"), D**-0.5, window, sinks, lengths, clean["dout"])
    # what an element that is no number reaches: rows [B, N, Sq], keys [B, Nk, Sk], and where it is by columns, those
    G = N // Nk
    lost = {x: torch.zeros_like(want[x], dtype=torch.bool) for x in ("out", "lse", "dq", "dk", "dv")}
    for (b, h, r), c in zip(rows, columns):
        see = R.visible(first, Sq, Sk, window, sinks, Sk if lengths is None else lengths[b])
        if source in "kv":
            heads = range(h * G, h * G + G)
            hit = see[:, r].nonzero()[:, 0]
            for n in heads:
                if source == "k":  # the score is lost
                    lost["out"][b, n, hit], lost["lse"][b, n, hit] = True, True
                else:
                    lost["out"][b, n, hit.unsqueeze(1), torch.tensor(c)] = True
                lost["dq"][b, n, hit] = True
            touched = see[hit].any(0).nonzero()[:, 0]  # keys that a lost row sees
            lost["dk"][b, h, touched] = True
            if source == "k":
                lost["dv"][b, h, touched] = True
        elif see[r].any():
            touched = see[r].nonzero()[:, 0]
            if source == "q":
                lost["out"][b, h, r], lost["lse"][b, h, r], lost["dv"][b, h // G, touched] = True, True, True
            else:
                lost["dv"][b, h // G, touched.unsqueeze(1), torch.tensor(c)] = True
            lost["dq"][b, h, r], lost["dk"][b, h // G, touched] = True, True
    ln = device_lengths(lengths)
    d = {x: y.to(DEV) for x, y in t.items()}
    out, lse, low = K.window_attention(d["q"], d["k"], d["v"], D**-0.5, window, sinks, ln, keep_low=True)
    got = {"out": out, "lse": lse}
    for kept in (None, low):
        got["dq"], got["dk"], got["dv"] = K.window_attention_backward(d["q"], d["k"], d["v"], out, d["dout"], lse, D**-0.5, window, sinks, ln, kept)
        for name, x in got.items():
            x = x.double().cpu()
            none = torch.isneginf(want[name])  # lse of rows that do not exist
            fine = ~lost[name] & ~none
            bound = lse_bound(want[name]) if name == "lse" else R.attention_bound(want[name], want["weight" if name == "out" else name + "_weight"], dtype)
            assert torch.isfinite(x[fine]).all(), f"{name}: {(~torch.isfinite(x[fine])).sum()} elements lost that see nothing of it"
            if fine.any():
                over = ((x - want[name]).abs() - bound)[fine].amax()
                assert over <= 0, f"{name}: {over:.3g} over the bound"
            assert not torch.isfinite(x[lost[name]]).any(), f"{name}: a number where there is none"
        if source == "v":  # an infinity keeps its sign
            for i, ((b, h, r), c) in enumerate(zip(rows, columns)):
                one = out[b, h * G : h * G + G][..., c].float().cpu()[lost["out"][b, h * G : h * G + G][..., c]]
                only = sum(x[:2] == (b, h) for x in rows) == 1
                assert not only or (torch.isposinf(one) if i == 1 else torch.isnan(one)).all()


# ------------------------------------------------------------------------------------ sizes of fp16 gradients
@pytest.mark.parametrize("size_do,size_v,scale", [
    (1.0, 1.0, 0.1), (1e-3, 1.0, 0.1), (1e-4, 1.0, 0.1), (1.0, 1e-3, 0.1), (1e-2, 1e-2, 0.1), ("mixed", 1.0, 0.1),
    (1000.0, 1.0, 0.1), (10.0, 1000.0, 0.1),  # |dP| past 2^8 max |dO|
    (30.0, 1000.0, 0.01),                     # dS past 65504
])
@pytest.mark.parametrize("N,Nk,Sq,Sk,window,sinks", [
    (2, 1, 2000, 2000, 2000, 0),   # probabilities of 2^-15 and less, a walk of keys shared by workgroups
    (2, 1, 2000, 2000, 128, 4),    # first keys with a kernel of their own
    (2, 2, 333, 900, 100, 300),    # many of them
    (3, 1, 250, 250, 3, 1),        # D from P and dP
])
def test_fp16_gradients_of_any_size(K, N, Nk, Sq, Sk, window, sinks, size_do, size_v, scale):
    announce(f"window_attention_backward fp16 {N, Nk, Sq, Sk, window, sinks} dout x {size_do} v x {size_v} scale {scale}")
    gen = torch.Generator().manual_seed(26)
    q, dout = (torch.randn(1, N, Sq, 64, generator=gen) for _ in range(2))
    k, v = (torch.randn(1, Nk, Sk, 64, generator=gen) for _ in range(2))
    if size_do == "mixed":
        dout = dout * 10.0 ** (-4 * torch.rand(1, N, Sq, 1, generator=gen))
    else:
        dout = dout * size_do
    q, k, v, dout = (t.to(HF) for t in (q, k, v * size_v, dout))
    want, bound, spread = R.fp16_gradient_bounds(q, k, v, scale, window, sinks, dout)
    d = [t.to(DEV) for t in (q, k, v, dout)]
    out, lse, low = K.window_attention(*d[:3], scale, window, sinks, keep_low=True)
    got = K.window_attention_backward(*d[:3], out, d[3], lse, scale, window, sinks, None, low)
    for name, x in zip(("dq", "dk", "dv"), got):
        # the gradient itself may be past the largest fp16 number (the first key of every row: 102468 in one case here)
        fits = want[name].abs() + bound[name] < 65504
        assert not torch.isfinite(x.cpu()[want[name].abs() - bound[name] > 65520]).any()
        x, want[name] = (torch.where(fits, t.double(), torch.zeros_like(want[name])) for t in (x.cpu(), want[name]))
        within(x, want[name], bound[name], name)
        if name in spread:
            # root mean square over all elements: the spread of dS's and the result's rounding, and as much again for P's in the
            # forward, which D carries (over few keys as large as dS's), rounded up to twice
            error = (x.double().cpu() - want[name]).square().mean().sqrt()
            assert error <= 2 * spread[name].square().mean().sqrt(), f"{name}: {error / spread[name].square().mean().sqrt():.2f} spreads"


# ------------------------------------------------------------------------------------ wide scores
def scored(kind, B, N, Nk, Sq, Sk, D, dtype, seed=27):
    """Operands whose scores, in units of the softmax's exponent, spread over hundreds: `rising` by 13 from a tile of 64 keys to
    the next (a new maximum in each), `creeping` by 3 (a maximum that stays behind for two), `falling` (the first stays),
    `wide` at random."""
    gen = torch.Generator().manual_seed(seed)
    q, dout = (torch.randn(B, N, Sq, D, generator=gen) for _ in range(2))
    k, v = (torch.randn(B, Nk, Sk, D, generator=gen) for _ in range(2))
    if kind == "wide":
        return *(t.to(dtype) for t in (q * 6, k * 2, v, dout)), D**-0.5
    slope = {"rising": 13.0, "creeping": 3.0, "falling": -13.0}[kind] * math.log(2) / 64
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[..., 0] += slope * D**0.5 / 8 * (torch.arange(Sk) - Sk / 2)
    return *(t.to(dtype) for t in (q, k, v, dout)), D**-0.5


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", ["rising", "creeping", "falling", "wide"])
@pytest.mark.parametrize("B,N,Nk,Sq,Sk,D,window,sinks,lengths", [
    (1, 2, 2, 700, 700, 128, 2**31 - 1, 0, None),
    (2, 6, 2, 700, 700, 64, 300, 5, [700, 333]),
    (1, 4, 1, 130, 1000, 96, 400, 70, None),
    (1, 2, 1, 900, 900, 64, 100, 200, None),     # first keys' gradients in a kernel of their own
    (1, 8, 1, 1500, 1500, 64, 1500, 0, None),    # a walk of keys shared by workgroups
    (1, 3, 1, 300, 300, 128, 4, 2, None),        # D from P and dP
])
def test_window_attention_of_wide_scores(K, B, N, Nk, Sq, Sk, D, window, sinks, lengths, kind, dtype):
    announce(f"window_attention {B, N, Nk, Sq, Sk, D, window, sinks, lengths} {kind} scores {dtype}")
    q, k, v, dout, scale = scored(kind, B, N, Nk, Sq, Sk, D, dtype)
    want, bound = R.wide_attention(q, k, v, scale, window, sinks, lengths, dout, dtype)
    d = [t.to(DEV) for t in (q, k, v, dout)]
    ln = device_lengths(lengths)
    out, lse, low = K.window_attention(*d[:3], scale, window, sinks, ln, True)
    within(out, want["out"], bound["out"], "out")
    live = ~torch.isinf(want["lse"])
    within(lse.cpu()[live], want["lse"][live], bound["lse"][live], "lse")
    for kept in (None, low):
        got = K.window_attention_backward(*d[:3], out, d[3], lse, scale, window, sinks, ln, kept)
        for name, x in zip(("dq", "dk", "dv"), got):
            within(x, want[name], bound[name], name)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", ["rising", "creeping", "falling", "wide"])
@pytest.mark.parametrize("B,N,Nk,capacity,D,window,sinks,lengths", [
    (2, 8, 2, 700, 128, 700, 0, [700, 333]),
    (1, 40, 2, 5000, 64, 4096, 70, [4999]),   # many shares
])
def test_decode_of_wide_scores(K, B, N, Nk, capacity, D, window, sinks, lengths, kind, dtype):
    announce(f"window_attention_decode {B, N, Nk, capacity, D, window, sinks, lengths} {kind} scores {dtype}")
    q, k, v, dout, scale = scored(kind, B, N, Nk, 1, capacity, D, dtype, seed=28)
    got = K.window_attention_decode(q.to(DEV)[:, :, 0], k.to(DEV), v.to(DEV), device_lengths(lengths), scale, window, sinks)
    for b, n in enumerate(lengths):
        want, bound = R.wide_attention(*(t[b : b + 1] for t in (q, k[:, :, :n], v[:, :, :n])), scale, window, sinks, None, dout[b : b + 1], dtype)
        within(got[b : b + 1], want["out"][:, :, 0], bound["out"][:, :, 0], "decode")


def test_graphs_are_released():
    announce("a forward pass whose gradient is never asked for keeps nothing")
    from inductor_x_amd import decoder

    q, k, v, dout = (t.to(DEV) for t in window_operands(2, 8, 2, 600, 600, 128, BF, False, seed=29))
    at, freq = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8).expand(2, 8).contiguous(), torch.ones(64, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    held = []
    for i in range(6):
        out = decoder.window_attention(*leaves, 0.1, 100, 4)
        turned = decoder.rotary_axes(leaves[0][:, :, :8].transpose(1, 2), leaves[1][:, :, :8].transpose(1, 2), at, freq)
        if i % 3 == 0:
            out.backward(dout)
        del out, turned
        for t in leaves:
            t.grad = None
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_allocated())
    assert len(set(held[1:])) == 1, held


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", [
    (1, 6, 3, 63, 149, 128, 2, 55, None, [141, 64]),
    (1, 2, 1, 130, 500, 64, 30, 4, None, [200]),
    (1, 8, 1, 300, 1600, 128, 1000, 0, None, [100, 299]),    # shared by workgroups
    (1, 2, 1, 900, 1200, 64, 100, 150, None, [199, 160]),    # first keys with a kernel of their own
    (2, 2, 1, 90, 90, 64, 20, 2, [0, 50], [10, 70]),         # a sequence without a position, a row that does not exist
], ids=str)
@pytest.mark.parametrize("source", ["k", "v"])
def test_rows_that_nobody_sees(K, case, source, dtype):
    """Their gradients are zero, whatever they hold."""
    test_hidden_pairs_do_not_count(K, case, source, dtype)


@pytest.mark.parametrize("source", ["k", "v", "q", "dout"])
def test_hidden_pairs_in_narrow_heads(K, source):
    announce(f"NaN in rows of {source}: heads of 80 columns beside tokens, repeated calls, other sequences of the batch")
    B, N, Nk, S, D, window, sinks = 3, 4, 2, 300, 80, 60, 3
    t = dict(zip(("q", "k", "v", "dout"), window_operands(B, N, Nk, S, S, D, BF, True, seed=30)))
    lengths = [300, 300, 177]
    want = R.attention(t["q"], t["k"], t["v"], 0.1, window, sinks, lengths, t["dout"])
    t[source][1] = float("nan")  # a whole sequence
    d = {x: same_memory(y) for x, y in t.items()}
    ln = device_lengths(lengths)
    first = None
    for _ in range(2):
        out, lse, low = K.window_attention(d["q"], d["k"], d["v"], 0.1, window, sinks, ln, True)
        got = (out, *K.window_attention_backward(d["q"], d["k"], d["v"], out, d["dout"], lse, 0.1, window, sinks, ln, low))
        for name, x in zip(("out", "dq", "dk", "dv"), got):
            bound = R.attention_bound(want[name], want["weight" if name == "out" else name + "_weight"], BF)
            within(x[::2], want[name][::2], bound[::2], name)
            lost = {"out": source != "dout", "dq": True, "dk": True, "dv": source != "v"}[name]
            assert torch.isnan(x[1]).all() if lost else torch.isfinite(x[1]).all(), name
        assert first is None or all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(first, got))
        first = got


@pytest.mark.parametrize("dtype", [BF, HF])
def test_replays_see_what_is_no_number(K, dtype):
    announce(f"a captured forward and backward pass replayed with NaN, infinities and numbers again {dtype}")
    gen = torch.Generator().manual_seed(31)
    q, k, v, dout = (t.to(DEV) for t in window_operands(2, 4, 2, 400, 400, 128, dtype, False, seed=31))
    lengths = torch.tensor([400, 290], dtype=torch.int32, device=DEV)
    call = lambda: training_call(K, q, k, v, dout, 64, 4, lengths)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for step in range(5):
        for t in (q, k, v, dout):
            t.copy_(torch.randn(t.shape, generator=gen).to(dtype))
        if step == 1:
            k[0, 1, 130], v[1, 0, 77, 5], dout[0, 2, 300, 8] = float("nan"), float("inf"), float("-inf")
        if step == 2:
            v *= 2000
        if step == 3:
            dout *= 1e-4
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        lost = [x.isnan().sum().item() for x in want]
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.equal(a.isnan(), b.isnan()) for a, b in zip(held, want)), f"replay {step}"
        assert (max(lost) > 0) == (step == 1), (step, lost)
