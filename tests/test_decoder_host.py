"""Argument checks and shape functions of the decoder-layer operators, without a GPU: the device check and the binding of a
launch are replaced, everything between them is the product's."""
import numpy as np
import pytest
import torch

from inductor_x_amd import decoder, kernels as K

BF = torch.bfloat16


class Launched(Exception):
    pass


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch):
    def bound(l, symbol, constants, grid):
        raise Launched(symbol)

    monkeypatch.setattr(K, "_check_cuda", lambda *t: None)
    monkeypatch.setattr(K, "_check_here", lambda *t: None)
    monkeypatch.setattr(K, "_bind", bound)
    K._operators().forget()
    yield
    K._operators().forget()


def test_tensors_on_the_host_are_refused(monkeypatch):
    monkeypatch.undo()
    x = torch.zeros(2, 64, dtype=BF)
    with pytest.raises(ValueError, match="GPU"):
        K.add_rmsnorm_quant(x, x, x[0])
    with pytest.raises(ValueError, match="GPU"):
        K.rotary_axes(x.view(1, 1, 2, 64), x.view(1, 1, 2, 64), torch.zeros(1, 1, dtype=torch.int32), torch.ones(4))
    with pytest.raises(ValueError, match="GPU"):
        K.window_attention_decode(x.view(1, 2, 64), x.view(1, 1, 2, 64), x.view(1, 1, 2, 64), torch.ones(1, dtype=torch.int32), 1.0, 1)


def test_norm_quant_refusals():
    h, w = torch.zeros(4, 256, dtype=BF), torch.ones(256, dtype=BF)
    with pytest.raises(Launched):
        K.add_rmsnorm_quant(h, h, w, group=128)
    for args, kw, text in [
        ((h, h.half(), w), {}, "share bf16 or fp16"),
        ((h.float(), h.float(), w.float()), {}, "share bf16 or fp16"),
        ((h, h[:2], w), {}, "same shape"),
        ((h, h, w[:128]), {}, "vector of the row length"),
        ((h, h, torch.ones(512, dtype=BF)[::2]), {}, "contiguous vector"),
        ((h, h, w), {"group": 64}, "group"),
        ((h[:, :0], h[:, :0], w[:0]), {}, "1..32768"),
        ((torch.zeros(1, 40000, dtype=BF),) * 2 + (torch.zeros(40000, dtype=BF),), {}, "1..32768"),
        ((torch.zeros(256, 4, dtype=BF).t(), h, w), {}, "columns must be contiguous"),
        ((torch.zeros(4, 3, 256, dtype=BF)[:, :2], torch.zeros(4, 2, 256, dtype=BF), w), {}, "evenly spaced"),
    ]:
        with pytest.raises(ValueError, match=text):
            K.add_rmsnorm_quant(*args, **kw)


def test_rotary_refusals():
    q, k = torch.zeros(2, 3, 4, 64, dtype=BF), torch.zeros(2, 3, 2, 64, dtype=BF)
    at, f = torch.zeros(2, 2, 3, dtype=torch.int32), torch.ones(32)
    with pytest.raises(Launched):
        K.rotary_axes(q, k, at, f, [20, 12])
    with pytest.raises(Launched):
        K.rotary_axes(q, k, at[0], f)
    for args, text in [
        ((q, k.half(), at, f, [20, 12]), "share"),
        ((q.double(), k.double(), at, f, [20, 12]), "share"),
        ((q[0], k[0], at, f, [20, 12]), r"\[B, S, N, D\]"),
        ((q, k[:, :2], at, f, [20, 12]), "share batch"),
        ((q.transpose(2, 3).contiguous().transpose(2, 3), k, at, f, [20, 12]), "contiguous"),
        ((q, k, at[:, :1], f, [20, 12]), "positions"),
        ((q, k, torch.zeros(5, 2, 3, dtype=torch.int32), f, [10, 10, 10, 1, 1]), "positions"),
        ((q, k, at.float(), f, [20, 12]), "positions"),
        ((q, k, at.transpose(1, 2).contiguous().transpose(1, 2), f, [20, 12]), "positions"),
        ((q, k, at, f.half(), [20, 12]), "inv_freq"),
        ((q, k, at, torch.ones(33), [20, 13]), "inv_freq"),
        ((q, k, at, torch.ones(0), [0, 0]), "inv_freq"),
        ((q, k, at, f, None), "sections"),
        ((q, k, at, f, [20, 13]), "sections"),
        ((q, k, at, f, [33, -1]), "sections"),
    ]:
        with pytest.raises(ValueError, match=text):
            K.rotary_axes(*args)


def decode_operands(B=2, N=4, Nk=2, capacity=16, D=64):
    return (torch.zeros(B, N, D, dtype=BF), torch.zeros(B, Nk, capacity, D, dtype=BF), torch.zeros(B, Nk, capacity, D, dtype=BF),
            torch.ones(B, dtype=torch.int32))


def test_decode_refusals():
    q, k, v, n = decode_operands()
    with pytest.raises(Launched):
        K.window_attention_decode(q, k, v, n, 0.1, 4, 1)
    for args, text in [
        ((q.unsqueeze(2), k, v, n, 0.1, 4, 1), r"\[B, N, D\]"),
        ((q, k, v[:, :, :8], n, 0.1, 4, 1), "share one"),
        ((q.half(), k, v, n, 0.1, 4, 1), "share bf16"),
        ((q[:, :3], k, v, n, 0.1, 4, 1), "multiple of the key heads"),
        ((q[..., :60], k[..., :60], v[..., :60], n, 0.1, 4, 1), "multiple of 8"),
        ((*decode_operands(D=136), 0.1, 4, 1), "multiple of 8"),
        ((q, k, v, n.long(), 0.1, 4, 1), "int32"),
        ((q, k, v, n[:1], 0.1, 4, 1), "one value per sequence"),
        ((q, k, v, n, 0.0, 4, 1), "scale"),
        ((q, k, v, n, float("nan"), 4, 1), "scale"),
        ((q, k, v, n, 0.1, 0, 1), "window"),
        ((q, k, v, n, 0.1, 4, -1), "sinks"),
        ((q, torch.zeros(2, 2, 16, 68, dtype=BF)[..., :64], v, n, 0.1, 4, 1), "16-byte aligned"),
        ((q, torch.zeros(2, 2, 64, 16, dtype=BF).transpose(2, 3), v, n, 0.1, 4, 1), "contiguous"),
        ((q, k.new_empty(1).expand(2, 2, 16, 64), v, n, 0.1, 4, 1), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=text):
            K.window_attention_decode(*args)
    assert K.window_attention_decode(q[:0], k[:0], v[:0], n[:0], 0.1, 4).shape == (0, 4, 64)
    assert (K.window_attention_decode(q, k[:, :, :0], v[:, :, :0], n, 0.1, 4) == 0).all()


def test_shape_functions():
    m = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    ops = torch.ops.npu_graph
    q, scales, s = ops.add_rmsnorm_quant(m(3, 5, 300), m(3, 5, 300), m(300), 1e-6, 128)
    assert q.dtype == torch.float8_e4m3fn and q.shape == s.shape == (3, 5, 300) and scales.shape == (3, 5, 3)
    a, b = ops.rotary_axes(m(2, 3, 4, 64), m(2, 3, 1, 64), m(1, 2, 3, dtype=torch.int32), m(32, dtype=torch.float32))
    assert a.shape == (2, 3, 4, 64) and b.shape == (2, 3, 1, 64)
    assert ops.window_attention_decode(m(2, 4, 64), m(2, 2, 9, 64), m(2, 2, 9, 64), m(2, dtype=torch.int32), 0.1, 4).shape == (2, 4, 64)
    q4, kv = m(2, 9, 4, 64).transpose(1, 2), m(2, 2, 11, 64)
    for keep in (False, True):
        out, lse, low = ops.window_attention(q4, kv, kv, 0.1, 4, 1, None, keep)
        assert out.shape == q4.shape and out.stride() == q4.stride() and lse.shape == (2, 4, 9) and lse.dtype == torch.float32
        assert low.shape == (q4.shape if keep else (0,))
    assert [t.shape for t in ops.window_attention_backward(q4, kv, kv, out, out, lse, 0.1, 4, 1, None, low)] == [q4.shape, kv.shape, kv.shape]


def window_operands(B=2, N=4, Nk=2, Sq=8, Sk=16, D=64):
    return torch.zeros(B, N, Sq, D, dtype=BF), torch.zeros(B, Nk, Sk, D, dtype=BF), torch.zeros(B, Nk, Sk, D, dtype=BF)


def test_window_refusals():
    q, k, v = window_operands()
    n = torch.ones(2, dtype=torch.int32)
    lse = torch.zeros(2, 4, 8)
    with pytest.raises(Launched):
        K.window_attention(q, k, v, 0.1, 4, 1, n)
    with pytest.raises(Launched):
        K.window_attention_backward(q, k, v, q, q, lse, 0.1, 4, 1, n)
    for args, text in [
        ((q[:, :, 0], k, v, 0.1, 4, 1), r"\[B, N, Sq, D\]"),
        ((q, k, v[:, :, :8], 0.1, 4, 1), "share one"),
        ((q, k.half(), v, 0.1, 4, 1), "share bf16"),
        ((q.float(), k.float(), v.float(), 0.1, 4, 1), "share bf16"),
        ((q[:, :3], k, v, 0.1, 4, 1), "multiple of the key heads"),
        ((q[:, :0], k, v, 0.1, 4, 1), "multiple of the key heads"),
        ((*window_operands(D=136), 0.1, 4, 1), "multiple of 8"),
        ((*window_operands(D=60), 0.1, 4, 1), "multiple of 8"),
        ((*window_operands(Sq=17), 0.1, 4, 1), "more queries than keys"),
        ((q[:1], k, v, 0.1, 4, 1), "share batch"),
        ((q, k, v, 0.1, 4, 1, n.long()), "int32"),
        ((q, k, v, 0.1, 4, 1, n[:1]), "one value per sequence"),
        ((q, k, v, float("inf"), 4, 1), "scale"),
        ((q, k, v, -1.0, 4, 1), "scale"),
        ((q, k, v, 0.1, 0, 1), "window"),
        ((q, k, v, 0.1, 4, -1), "sinks"),
        ((q, k, torch.zeros(2, 2, 16, 68, dtype=BF)[..., :64], 0.1, 4, 1), "16-byte aligned"),
        ((torch.zeros(2 * 4 * 8 * 64 + 1, dtype=BF)[1:].view(2, 4, 8, 64), k, v, 0.1, 4, 1), "16-byte aligned"),
        ((q, k.new_empty(1).expand(2, 2, 16, 64), v, 0.1, 4, 1), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=text):
            K.window_attention(*args)
    for args, text in [
        ((q, k, v, q, q.half(), lse, 0.1, 4, 1), "match q"),
        ((q, k, v, q[:, :, :4], q, lse, 0.1, 4, 1), "match q"),
        ((q, k, v, q, q.new_empty(1).expand(2, 4, 8, 64), lse, 0.1, 4, 1), "contiguous"),
        ((q, k, v, q, q, lse.half(), 0.1, 4, 1), "lse"),
        ((q, k, v, q, q, lse[:, :, :4], 0.1, 4, 1), "lse"),
        ((q, k, v, q, q, lse, 0.1, 4, 1, None, q[:1]), "low"),
    ]:
        with pytest.raises(ValueError, match=text):
            K.window_attention_backward(*args)
    out, lse = K.window_attention(q[:0], k[:0], v[:0], 0.1, 4)
    assert out.shape == (0, 4, 8, 64) and lse.shape == (0, 4, 8)
    out, lse = K.window_attention(q[:, :, :0], k, v, 0.1, 4)
    assert out.shape == (2, 4, 0, 64)
    grads = K.window_attention_backward(q[:, :, :0], k, v, out, out, lse, 0.1, 4)
    assert (grads[1] == 0).all() and (grads[2] == 0).all() and grads[1].shape == k.shape


def test_plain_arguments_are_no_tensors():
    """A plan is found by its arguments: a tensor among them could change its value behind the plan's back."""
    q, k, v = window_operands()
    n = torch.ones(2, dtype=torch.int32)
    h, w = torch.zeros(4, 256, dtype=BF), torch.ones(256, dtype=BF)
    turn = torch.zeros(2, 3, 4, 64, dtype=BF), torch.zeros(2, 3, 2, 64, dtype=BF), torch.zeros(2, 2, 3, dtype=torch.int32), torch.ones(32)
    for call in (lambda: K.window_attention(q, k, v, torch.tensor(0.1), 4),
                 lambda: K.window_attention(q, k, v, 0.1, torch.tensor(4)),
                 lambda: K.window_attention_backward(q, k, v, q, q, torch.zeros(2, 4, 8), 0.1, 4, torch.tensor(1)),
                 lambda: K.window_attention_decode(q[:, :, 0].contiguous(), k, v, n, torch.tensor(0.1), 4),
                 lambda: K.add_rmsnorm_quant(h, h, w, torch.tensor(1e-6)),
                 lambda: K.rotary_axes(*turn, torch.tensor([20, 12]))):
        with pytest.raises(ValueError, match="plain numbers"):
            call()


def test_arguments_of_other_kinds():
    q, k, v = window_operands()
    for scale in (np.float32(0.1), np.float64(0.1), 1):
        with pytest.raises(Launched):
            K.window_attention(q, k, v, scale, np.int64(4), True)
    for call in (lambda: K.window_attention(q, k, v, "0.1", 4), lambda: K.window_attention(q, k, v, None, 4),
                 lambda: K.window_attention_with_gradients(q, k, v, "0.1", 4), lambda: K.window_attention_with_gradients(q, k, None, 0.1, 4),
                 lambda: K.window_attention_with_gradients(q, k, v, 0.1, 4, 1, [8, 8])):
        with pytest.raises((TypeError, ValueError)):
            call()
    with pytest.raises(ValueError, match="plain numbers"):
        K.window_attention_with_gradients(q, k, v, torch.tensor(0.1), 4)
    with pytest.raises(ValueError, match="scale"):  # a refusal passes through the native side unchanged
        K.window_attention_with_gradients(q, k, v, -1.0, 4)
    with pytest.raises(Launched):
        K.window_attention_with_gradients(q, k, v, 0.1, 4)


def test_more_shapes_than_plans_are_kept():
    q = torch.empty(0, 4, 1, 64, dtype=BF)
    for n in range(1, 4200):  # no sequences: results and no launch
        kv = torch.empty(0, 2, n, 64, dtype=BF)
        out, lse = K.window_attention(q, kv, kv, 0.1, n)
        assert out.shape == q.shape and lse.shape == q.shape[:3]


def test_first_keys_have_a_kernel_of_their_own_or_not(monkeypatch):
    """Which kernels a backward pass consists of."""
    bound = []
    monkeypatch.setattr(K, "_bind", lambda l, symbol, constants, grid: bound.append(symbol) or (0, (1,) * 6 + (0,), b"", symbol))

    def kernels(B, N, Nk, Sq, Sk, window, sinks):
        del bound[:]
        q, k, v = window_operands(B, N, Nk, Sq, Sk)
        with pytest.raises(ValueError, match="current GPU"):  # nothing is enqueued for tensors of the host
            K.window_attention_backward(q, k, v, q, q, torch.zeros(B, N, Sq), 0.1, window, sinks)
        return len(bound)

    assert kernels(1, 4, 4, 832, 832, 256, 4) == 2     # 7 tiles of queries more than a window's
    assert kernels(1, 4, 4, 897, 897, 256, 4) == 4     # 9
    assert kernels(4, 16, 4, 897, 897, 576, 4) == 3    # 4 of four heads, shared by two workgroups: and a join
    assert kernels(16, 16, 4, 897, 897, 576, 4) == 4   # the same in enough sequences to need no shares
    assert kernels(1, 4, 4, 897, 897, 256, 0) == 2     # no first keys
    assert kernels(1, 4, 4, 897, 897, 256, 225) == 2   # a quarter of the keys
    assert kernels(1, 4, 1, 256, 5000, 64, 4) == 3     # shared by three workgroups
    assert kernels(1, 4, 4, 897, 897, 897, 4) == 3     # none beyond the window, shared by three workgroups
    assert kernels(16, 4, 4, 897, 897, 897, 4) == 2


def test_heads_of_a_workgroup():
    assert [K._largest_share(g) for g in (1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 24, 40)] == [0, 1, 0, 2, 0, 1, 0, 2, 2, 2, 2, 2]
    for units in (1, 8, 64, 1000):
        for blocks in (1, 4):
            for tiles in (1, 15, 100, 10000):
                n = K._sink_splits(units, blocks, tiles)
                assert n >= 1 and (n == 1 or tiles // n >= 4)


def test_shares_of_a_block_of_keys():
    for blocks in (1, 7, 64, 200, 257, 5000):
        for walk in (0, 1, 7, 40, 1000, 100000):
            for growing in (False, True):
                n = K._dkv_shares(blocks, walk, growing)
                assert n == 1 or (walk // n >= 4 and n * blocks <= 384 and n <= 16)


def test_splits_of_a_decode():
    for units in (1, 7, 64, 512, 5000):
        for tiles in (1, 3, 33, 129, 40000):
            n = K._decode_splits(units, tiles)
            assert 1 <= n <= 64 and (n == 1 or (tiles // n >= 4 and n <= 1 + 256 // units))


def test_gradient_formulas_against_differences():
    """The fp64 gradients that the kernels are held to, against central differences of the fp64 forward."""
    from tests import decoder_reference as R

    gen = torch.Generator().manual_seed(0)
    q, k, v, dout = (torch.randn(2, n, s, 8, generator=gen, dtype=torch.float64) for n, s in ((4, 6), (2, 9), (2, 9), (4, 6)))
    form = (0.4, 3, 2, [9, 7])
    grads = R.attention(q, k, v, *form, dout)
    loss = lambda: (R.attention(q, k, v, *form)["out"] * dout).sum().item()  # noqa: E731
    for t, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        flat = t.view(-1)
        for i in range(0, flat.numel(), 7):
            at, step = flat[i].item(), 1e-5
            flat[i] = at + step
            up = loss()
            flat[i] = at - step
            down = loss()
            flat[i] = at
            # truncation of order step^2, cancellation of order 1e-16 / step
            assert abs((up - down) / (2 * step) - grads[name].view(-1)[i].item()) < 1e-7, (name, i)
    x = torch.randn(1, 3, 2, 12, generator=gen, dtype=torch.float64)
    y = torch.randn(1, 3, 2, 12, generator=gen, dtype=torch.float64)
    at, freq = torch.randint(0, 50, (2, 1, 3), generator=gen), torch.rand(5, generator=gen, dtype=torch.float64)
    for beside in (False, True):
        turned = R.rotary(x, at, freq, [2, 3], beside, False)
        back = R.rotary(y, at, freq, [2, 3], beside, True)
        assert abs((turned * y).sum() - (x * back).sum()) < 1e-12  # a linear map and its transpose


def test_more_than_a_launch_takes():
    """Refused with the other operands: the runtime counts the threads of a launch in 32 bits."""
    def norm(rows, cols):
        h = torch.zeros(1, cols, dtype=BF).expand(rows, cols)
        return lambda: K.add_rmsnorm_quant(h, h, h[0])

    def rotary(tokens, pairs):
        x = torch.zeros(1, 1, 1, 2 * pairs, dtype=BF).expand(tokens, 1, 1, 2 * pairs)
        return lambda: K.rotary_axes(x, x, torch.empty(tokens, 1, dtype=torch.int32), torch.ones(pairs))

    def window(B):
        q = torch.zeros(1, 1, 1, 8, dtype=BF).expand(B, 1, 1, 8)
        return lambda: K.window_attention(q, q, q, 0.1, 1)

    def backward(B, Sk=1):
        q, k = (torch.zeros(1, 1, 1, 8, dtype=BF).expand(B, 1, s, 8) for s in (1, Sk))
        return lambda: K.window_attention_backward(q, k, k, q, q, torch.empty(B, 1, 1), 0.1, 1)

    def decode(B, N=1):
        q, k = torch.zeros(1, 1, 8, dtype=BF).expand(B, N, 8), torch.zeros(1, 1, 1, 8, dtype=BF).expand(B, 1, 1, 8)
        return lambda: K.window_attention_decode(q, k, k, torch.empty(B, dtype=torch.int32), 0.1, 1)

    for fits, too_many in ((norm(2**28 - 16, 128), norm(2**28, 128)), (norm(2**24 - 1, 2000), norm(2**24, 2000)),
                           (rotary(2**24 - 1, 128), rotary(2**24, 128)), (window(2**24 - 8), window(2**24)),
                           (decode(2**24 - 1), decode(2**24)), (decode(2**24 - 1, 16), decode(2**24, 16))):
        with pytest.raises(Launched):
            fits()
        with pytest.raises(ValueError, match="one launch"):
            too_many()
    with pytest.raises(ValueError, match="one launch"):
        backward(2**24)()


def test_each_kernel_of_a_backward_pass_fits(monkeypatch):
    bound = []
    monkeypatch.setattr(K, "_bind", lambda l, symbol, constants, grid: bound.append(symbol) or (0, (1,) * 6 + (0,), b"", symbol))
    q = torch.zeros(1, 1, 1, 8, dtype=BF).expand(2**23, 1, 1, 8)
    with pytest.raises(ValueError, match="one launch"):  # dK and dV have workgroups of 512
        K.window_attention_backward(q, q, q, q, q, torch.empty(2**23, 1, 1), 0.1, 1)
    assert ["dq" in x for x in bound] == [True]


def test_plans_take_no_memory():
    """What a plan needs to know of its results are strides: making it allocates none of them (these would be terabytes)."""
    x = torch.zeros(1, 1, 1, 64, dtype=BF).as_strided((2**6, 2**12, 2**10, 64), (0, 0, 0, 1))
    y = torch.zeros(1, 1, 1, 64, dtype=BF).as_strided((1, 2**10, 2**19, 64), (0, 0, 0, 1))
    with pytest.raises(Launched):
        K.rotary_axes(x, x, torch.empty(2**6, 2**12, dtype=torch.int32), torch.ones(32))
    with pytest.raises(Launched):
        K.window_attention(y, y, y, 0.1, 100)
    for shape, strides in (((2, 3, 5, 8), (120, 40, 8, 1)), ((2, 3, 5, 8), (120, 8, 24, 1)), ((2, 3, 5, 8), (0, 8, 24, 1)), ((2, 3, 5, 8), (240, 16, 48, 2)),
                           ((1, 3, 1, 8), (7, 8, 3, 1)), ((2, 0, 5, 8), (120, 40, 8, 1)), ((2, 3, 5, 8), (400, 16, 80, 1))):
        t = torch.zeros(2000, dtype=BF).as_strided(shape, strides)
        assert K._output_like(t)[1] == torch.empty_like(t).stride()


def test_elements_of_a_rotary_workgroup(monkeypatch):
    """A workgroup counts the elements of its tokens' heads in 32 bits."""
    def call(tokens, N, D):
        x = torch.zeros(1, 1, 1, D, dtype=BF).expand(1, tokens, N, D)
        q = x.as_strided((1, tokens, N, D), (0, 0, 0, 1))
        return lambda: K.rotary_axes(q, q[:, :, :1], torch.empty(1, tokens, dtype=torch.int32), torch.ones(1))

    for fits in (call(1, 2**14 - 2, 2**17), call(2**15, 128, 2**9)):
        with pytest.raises(Launched):
            fits()
    with pytest.raises(ValueError, match="one workgroup"):
        call(1, 2**14, 2**17)()
    counted = []
    monkeypatch.setattr(K, "_bind", lambda l, symbol, constants, grid: counted.append(constants[-2]) or (0, (1,) * 6 + (0,), b"", symbol))
    with pytest.raises(ValueError, match="current GPU"):
        call(2**16, 2**10, 2**15)()
    assert counted[0] * (2**10 + 1) * 2**15 < 2**31 - 256 <= (counted[0] + 1) * (2**10 + 1) * 2**15


def test_plans_are_kept_and_start_over(monkeypatch):
    """A key's plan is made once; after 4096 keys of an operator the table starts over, and an early key is planned again."""
    made, check = [], K._window_check
    monkeypatch.setattr(K, "_window_check", lambda *a: made.append(a[4]) or check(*a))
    q = torch.empty(0, 4, 1, 64, dtype=BF)

    def call(n):
        kv = torch.empty(0, 2, n, 64, dtype=BF)
        out, lse = K.window_attention(q, kv, kv, 0.1, n)
        assert out.shape == q.shape and lse.shape == q.shape[:3]
        return len(made)

    assert [call(1), call(1), call(2), call(1), call(2)] == [1, 1, 2, 2, 2]
    for n in range(3, 4097):
        assert call(n) == n
    assert call(1) == 4096 and call(4096) == 4096     # all of them still there
    assert call(4097) == 4097                         # the table is full: this key starts a new one
    assert call(4097) == 4097 and call(1) == 4098 and call(1) == 4098 and call(4096) == 4099
    h = torch.empty(0, 8, dtype=BF)
    K.add_rmsnorm_quant(h, h, torch.empty(8, dtype=BF))  # another operator's plans are its own
    assert call(4097) == 4099


def test_scales_that_32_bits_do_not_hold():
    """The kernels take the scale, and its inverse, in 32 bits."""
    q, k, v = window_operands()
    n, lse = torch.ones(2, dtype=torch.int32), torch.zeros(2, 4, 8)
    for scale in (1e-46, 1e-39, 1e-31, 1e31, 1e39, 1e300):
        for call in (lambda: K.window_attention(q, k, v, scale, 4), lambda: K.window_attention_backward(q, k, v, q, q, lse, scale, 4),
                     lambda: K.window_attention_decode(q[:, :, 0].contiguous(), k, v, n, scale, 4),
                     lambda: K.window_attention_with_gradients(q, k, v, scale, 4)):
            with pytest.raises(ValueError, match="scale"):
                call()
    for scale in (1e-30, 1e30):
        with pytest.raises(Launched):
            K.window_attention(q, k, v, scale, 4)


def test_other_operators_keep_their_scales(monkeypatch):
    monkeypatch.setattr(K, "_find", lambda l, symbol: (_ for _ in ()).throw(Launched(symbol)))
    monkeypatch.setattr(K.codecache, "aot_source", lambda name: "")
    q = torch.zeros(1, 1, 64, 128, dtype=BF)
    for scale in (1e-31, 1e31):
        with pytest.raises(Exception) as e:
            K.fused_attention(q, q, q, scale, False)
        assert "scale" not in str(e.value)
    with pytest.raises(ValueError, match="scale must be positive and finite$"):
        K.fused_attention(q, q, q, -1.0, False)
