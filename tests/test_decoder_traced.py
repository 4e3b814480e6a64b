"""Calls of the decoder-layer operators that somebody rides along with: tracers, dispatch modes, functorch transforms and
tensor subclasses have to see the registered op, not the allocations of its results.

Without a GPU: the operands are empty, so the product's host side runs whole and launches nothing, and the ops get the GPU
implementation for the CPU too."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils._pytree import tree_map

from inductor_x_amd import decoder, kernels as K

BF = torch.bfloat16
OPS = torch.ops.npu_graph


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch):
    monkeypatch.setattr(K, "_check_cuda", lambda *t: None)
    monkeypatch.setattr(K, "_check_here", lambda *t: None)
    K._operators().forget()
    lib = torch.library.Library("npu_graph", "IMPL", "CPU")
    for name, implementation in decoder.IMPLEMENTATIONS.items():
        lib.impl(name, implementation)
    yield
    lib._destroy()
    K._operators().forget()


def operands():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)  # noqa: E731
    q, kv = z(0, 4, 8, 64), z(0, 2, 16, 64)
    n = z(0, dtype=torch.int32)
    turn = (z(0, 3, 4, 64), z(0, 3, 2, 64), z(2, 0, 3, dtype=torch.int32), z(32, dtype=torch.float32))
    return q, kv, n, turn, (z(0, 256), z(0, 256), z(256))


Q, KV, N, TURN, NORM = operands()
LSE = torch.zeros(0, 4, 8)
CALLS = {
    "decoder norm": (lambda h, r, w: decoder.add_rmsnorm_quant(h, r, w, group=128)[2], NORM, "add_rmsnorm_quant"),
    "decoder rotary": (lambda *t: decoder.rotary_axes(*t, [20, 12])[0], TURN, "rotary_axes"),
    "decoder window": (lambda q, k, v, n: decoder.window_attention(q, k, v, 0.1, 4, 1, n), (Q, KV, KV, N), "window_attention"),
    "decoder decode": (lambda q, k, v, n: decoder.window_attention_decode(q, k, v, n, 0.1, 4, 1), (Q[:, :, 0], KV, KV, N), "window_attention_decode"),
    "kernels norm": (lambda h, r, w: K.add_rmsnorm_quant(h, r, w, 1e-6, 128)[2], NORM, "add_rmsnorm_quant"),
    "kernels rotary": (lambda *t: K.rotary_axes(*t, [20, 12], True, True)[1], TURN, "rotary_axes"),
    "kernels window": (lambda q, k, v, n: K.window_attention(q, k, v, 0.1, 4, 1, n)[0], (Q, KV, KV, N), "window_attention"),
    "kernels window, low": (lambda q, k, v, n: K.window_attention(q, k, v, 0.1, 4, 1, n, True)[2], (Q, KV, KV, N), "window_attention"),
    "kernels backward": (lambda q, k, v, lse: K.window_attention_backward(q, k, v, q, q, lse, 0.1, 4, 1)[1], (Q, KV, KV, LSE), "window_attention_backward"),
    "kernels decode": (lambda q, k, v, n: K.window_attention_decode(q, k, v, n, 0.1, 4, 1), (Q[:, :, 0], KV, KV, N), "window_attention_decode"),
}
each_call = pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())
        return func(*args, **(kwargs or {}))


@each_call
def test_make_fx_records_the_op(call):
    fn, args, name = call
    for mode in ("real", "fake"):
        graph = make_fx(fn, tracing_mode=mode)(*args).graph
        assert [n.target for n in graph.nodes if n.op == "call_function" and "npu_graph" in str(n.target)] == [getattr(OPS, name).default]
        last = next(n for n in graph.nodes if n.op == "output").args[0]
        assert "empty" not in str(last.target)


@each_call
def test_jit_trace_records_the_op(call):
    fn, args, name = call
    traced = torch.jit.trace(fn, args, check_trace=False)
    assert f"npu_graph::{name}(" in str(traced.inlined_graph)
    assert traced(*args).shape == fn(*args).shape


@each_call
def test_dispatch_modes_see_the_op(call):
    fn, args, name = call
    with Seen() as outer, Seen() as inner:
        fn(*args)
    assert f"npu_graph::{name}" in inner.names and f"npu_graph::{name}" in outer.names


@each_call
def test_fake_tensors_stay_fake(call):
    fn, args, _ = call
    mode = FakeTensorMode()
    want = fn(*args)
    got = fn(*(mode.from_tensor(t) for t in args))
    assert isinstance(got, FakeTensor) and got.shape == want.shape and got.dtype == want.dtype


class Dispatching(torch.Tensor):
    """A wrapper that counts the ops that reach it."""

    seen = []

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, strides=inner.stride(), dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        cls.seen.append(func.name())
        unwrap = lambda x: x.inner if isinstance(x, cls) else x  # noqa: E731
        return tree_map(lambda x: cls(x) if isinstance(x, torch.Tensor) else x, func(*tree_map(unwrap, args), **tree_map(unwrap, kwargs or {})))


class Tagged(torch.Tensor):
    """A subclass in name only: results of its operators are of it too."""


@each_call
def test_subclasses_see_the_op(call):
    fn, args, name = call
    del Dispatching.seen[:]
    assert isinstance(fn(*(Dispatching(t) for t in args)), Dispatching)
    assert f"npu_graph::{name}" in Dispatching.seen
    assert isinstance(fn(args[0].as_subclass(Tagged), *args[1:]), Tagged)


def test_parameters_are_no_subclass():
    with torch.no_grad():
        assert not K.watched(torch.nn.Parameter(Q), KV, None)
    assert K.watched(Q.as_subclass(Tagged)) and not K.watched(Q)


def test_gradients_are_seen():
    q, k = Q.clone().requires_grad_(), KV.clone().requires_grad_()
    with Seen() as seen:
        out = decoder.window_attention(q, k, k, 0.1, 4, 1)
        out.backward(torch.ones_like(out))
    assert "npu_graph::window_attention" in seen.names and "npu_graph::window_attention_backward" in seen.names
    out = decoder.window_attention(q, k, k, 0.1, 4, 1)
    with Seen() as seen:  # a forward pass that nobody watched, its gradient watched
        out.backward(torch.ones_like(out))
    assert "npu_graph::window_attention_backward" in seen.names
    x = TURN[0].clone().requires_grad_()
    y, _ = decoder.rotary_axes(x, *TURN[1:], [20, 12])
    with Seen() as seen:
        y.backward(torch.ones_like(y))
    assert "npu_graph::rotary_axes" in seen.names

    def step(q, k, v, dout):
        return torch.autograd.grad(decoder.window_attention(q, k, v, 0.1, 4, 1), (q, k, v), dout)

    graph = make_fx(step)(*(t.clone().requires_grad_() for t in (Q, KV, KV)), torch.zeros_like(Q)).graph
    assert sum("window_attention_backward" in str(n.target) for n in graph.nodes) == 1


def test_functorch_never_gets_uninitialised_memory():
    """A transform runs the op through a rule or raises."""
    with Seen() as seen:
        try:
            torch.vmap(lambda w: decoder.add_rmsnorm_quant(NORM[0], NORM[1], w)[2])(torch.ones(3, 256, dtype=BF))
        except RuntimeError:
            return
    assert "npu_graph::add_rmsnorm_quant" in seen.names


def test_a_view_with_its_sign_in_the_metadata():
    """The imaginary part of a conjugate is stored with the other sign."""
    freq = torch.complex(torch.zeros(32), torch.ones(32)).conj().imag
    assert freq.is_neg() and K.watched(freq)
    assert K.rotary_axes(*TURN[:3], torch.ones(33)[:32], [20, 12])[0].shape == TURN[0].shape


def test_forward_mode_is_refused_or_right():
    """A result that lost its tangent would read as a constant."""
    from torch.autograd import forward_ad as fw

    for name, (fn, args, _) in CALLS.items():
        if name == "decoder rotary":
            continue
        for grad in (False, True):
            with fw.dual_level(), pytest.raises((NotImplementedError, RuntimeError), match="forward|jvp"):
                x = args[0].clone().requires_grad_(grad)
                fn(fw.make_dual(x, torch.zeros_like(x)), *args[1:])
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda x: fn(x, *args[1:]), (args[0],), (args[0],))
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda x: torch.vmap(lambda y: fn(y, *args[1:]))(x.unsqueeze(0)), (args[0],), (args[0],))
    q, k, positions, freq = TURN
    with fw.dual_level():
        y, z = decoder.rotary_axes(fw.make_dual(q, q.clone()), k, positions, freq, [20, 12])
        assert fw.unpack_dual(y).tangent is not None
        with pytest.raises(NotImplementedError, match="frequencies"):
            decoder.rotary_axes(q, k, positions, fw.make_dual(freq, freq.clone()), [20, 12])
        with torch.no_grad():
            y, _ = decoder.rotary_axes(fw.make_dual(q, q.clone()), k, positions, freq, [20, 12])
        assert fw.unpack_dual(y).tangent is not None
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda x: decoder.rotary_axes(x, *TURN[1:], [20, 12])[0], (q,), (q,))
    assert fw.unpack_dual(decoder.rotary_axes(*TURN, [20, 12])[0]).tangent is None


def arrivals(shape):
    """Gradients of a shape [B, N, S, D] in layouts and at addresses that the kernels do not take."""
    n = torch.Size(shape).numel()
    yield torch.ones(n + 1, dtype=BF)[1:].view(shape)                                              # contiguous, off the 16-byte grid
    yield torch.ones(1, dtype=BF).expand(shape)                                                    # a sum's
    yield torch.ones(*shape[:3], shape[3] + 4, dtype=BF)[..., : shape[3]]                          # rows off the grid
    yield torch.ones(*shape[:2], shape[3], shape[2], dtype=BF).transpose(2, 3)                     # columns apart


def test_gradients_arrive_anywhere(monkeypatch):
    """The address that reaches the kernels, through the op and through the native function."""
    ready = []

    def plan(q, k, v, out, dout, lse, *rest):
        ready.append(dout.data_ptr() % 16 == 0 and dout.stride(3) == 1 and all(s % 8 == 0 for s in dout.stride()[:3]))
        return (), tuple((tuple(t.shape), t.contiguous().stride(), t.dtype, True) for t in (q, k, v)), 3

    ops = K._operators()
    number = ops.operator(plan, (0, 1, 2, 3, 4, 5, 9, 10), lambda *a: None)
    monkeypatch.setattr(K, "_WINDOW_BACKWARD", number)
    q, kv, lse = torch.zeros(2, 4, 8, 64, dtype=BF), torch.zeros(2, 2, 16, 64, dtype=BF), torch.zeros(2, 4, 8)
    for dout in arrivals(q.shape):
        before = dout.clone()
        OPS.window_attention_backward(q, kv, kv, q, dout, lse, 0.1, 4)
        assert ready.pop() and torch.equal(dout, before)
        ops.forget()
    empty = torch.zeros(0, 4, 8, 64, dtype=BF)
    for dout in arrivals(q.shape):
        again = K.placed(dout)
        assert torch.equal(again, dout) and again.data_ptr() % 16 == 0 and again.is_contiguous()
    aligned = torch.ones(q.shape, dtype=BF).transpose(1, 2)
    assert K.placed(aligned).data_ptr() == aligned.data_ptr() and K.placed(empty).data_ptr() == empty.data_ptr()


def test_sums_of_empty_batches():
    """Their gradient has strides of zero, and contiguous() leaves an empty tensor as it is."""
    for watched in (False, True):
        q, k, x = (t.clone().requires_grad_() for t in (Q, KV, TURN[0]))
        with (Seen() if watched else torch.enable_grad()):
            decoder.window_attention(q, k, k, 0.1, 4, 1).sum().backward()
            decoder.rotary_axes(x, *TURN[1:], [20, 12])[0].sum().backward()
        assert q.grad.shape == q.shape and k.grad.shape == k.shape and x.grad.shape == x.shape
