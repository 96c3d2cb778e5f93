"""The calls around autograd.linear, optim.orthogonalize and FusedMuon: what records or watches them, which views, graphs, hooks and arguments they take, and
what they refuse."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils._pytree import tree_map

import speech2lip_amd as s2l
from speech2lip_amd import _abi, autograd, optim


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


class Watching(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


class Wrapped(torch.Tensor):
    """A subclass that dispatches for itself: it holds a tensor and unwraps it for every operator."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, strides=t.stride(), dtype=t.dtype, device=t.device)

    def __init__(self, t):
        self.inner = t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        inner = lambda t: t.inner if isinstance(t, Wrapped) else t  # noqa: E731
        wrap = lambda t: Wrapped(t) if isinstance(t, torch.Tensor) else t  # noqa: E731
        return tree_map(wrap, func(*tree_map(inner, args), **tree_map(inner, kwargs or {})))


def _refused_under_jit_trace(x, w, p):
    """The recorded program would hold the allocation of the result and not the launch that writes it."""
    for f in (lambda t: autograd.linear(t, w), lambda t: optim.orthogonalize(t), lambda t: optim.orthogonalize([t, t])[0]):
        with pytest.raises(NotImplementedError):
            torch.jit.trace(f, x, check_trace=False)
    p.grad = torch.zeros_like(p)
    opt = s2l.FusedMuon([p])
    with FakeTensorMode(), pytest.raises(NotImplementedError):
        opt.step()


def test_recording_without_a_gpu():
    x, w = torch.zeros(2, 3), torch.zeros(4, 3)
    _refused_under_jit_trace(x, w, torch.nn.Parameter(torch.zeros(4, 3)))
    for f in (lambda t: autograd.linear(t, w), lambda t: optim.orthogonalize(t)):      # other recorders: as any call without a GPU
        for call in (lambda: make_fx(f)(x), lambda: f(Wrapped(x))):
            with pytest.raises(RuntimeError, match="GPU"):
                call()
        with Watching(), pytest.raises(RuntimeError, match="GPU"):
            f(x)


@pytest.mark.gpu
def test_jit_trace_is_refused(dev):
    _refused_under_jit_trace(torch.randn(2, 3, device=dev), torch.randn(4, 3, device=dev), torch.nn.Parameter(torch.zeros(4, 3, device=dev)))


def _both_passes(act):
    def f(x, w, b, r, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = autograd.linear(*leaves, act)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    return f


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ("real", "fake"))
def test_make_fx_records_the_operators(mode, dev):
    """The recorded program, run on other values, gives the eager call's bits."""
    values, dy = _layer(dev, 1)
    fresh, fdy = _layer(dev, 2)
    for act in ("none", "relu", "gelu"):
        f = _both_passes(act)
        program = make_fx(f, tracing_mode=mode)(*values, dy)
        assert {"speech2lip_amd.linear_forward.default", "speech2lip_amd.linear_backward.default"} <= {str(n.target) for n in program.graph.nodes}
        assert all(torch.equal(a, b) for a, b in zip(f(*fresh, fdy), program(*fresh, fdy)))
    g = lambda t: optim.orthogonalize([t[0], t[1, :9]])  # noqa: E731
    one, other = torch.randn(2, 20, 30, device=dev), torch.randn(2, 20, 30, device=dev)
    program = make_fx(g, tracing_mode=mode)(one)
    assert all(torch.equal(a, b) for a, b in zip(g(other), program(other)))


@pytest.mark.gpu
def test_modes_subclasses_counters_and_selective_checkpoints(dev):
    from functools import partial
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
    from torch.utils.flop_counter import FlopCounterMode
    values, dy = _layer(dev, 3)
    g = torch.randn(20, 30, device=dev)
    for act in ("none", "leaky_relu", "silu"):
        f = _both_passes(act)
        want = f(*values, dy)
        for mode in (Watching(), FlopCounterMode(display=False)):
            with mode:
                got, orth = f(*values, dy), optim.orthogonalize(g)
            assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(orth, optim.orthogonalize(g))
            if isinstance(mode, Watching):
                assert sum("linear_forward" in n for n in mode.seen) == 1 and sum("linear_backward" in n for n in mode.seen) == 1
                assert sum("orthogonalize" in n for n in mode.seen) == 1
        leaves = [v.clone().requires_grad_() for v in values]
        y = autograd.linear(*leaves, act)      # an eager forward pass, its backward pass under a mode
        with Watching():
            assert all(torch.equal(a, b) for a, b in zip(want[1:], torch.autograd.grad(y, leaves, dy)))
        wrapped = autograd.linear(*(Wrapped(v) for v in values), act)
        assert isinstance(wrapped, Wrapped) and torch.equal(wrapped.inner, want[0])
        for saving in (True, False):
            policy = lambda ctx, op, *a, **k: CheckpointPolicy.MUST_SAVE if saving else CheckpointPolicy.PREFER_RECOMPUTE  # noqa: E731
            y = checkpoint(lambda *t: autograd.linear(*t, act).square(), *leaves, use_reentrant=False, context_fn=partial(create_selective_checkpoint_contexts, policy))
            plain = autograd.linear(*leaves, act).square()
            assert torch.equal(y, plain)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(plain, leaves, dy)))
    wrapped = optim.orthogonalize(Wrapped(g))
    assert isinstance(wrapped, Wrapped) and torch.equal(wrapped.inner, optim.orthogonalize(g))


@pytest.mark.gpu
def test_the_operators_check_what_they_are_given(dev):
    ops = torch.ops.speech2lip_amd
    autograd._linear_ops()
    (x, w, b, r), dy = _layer(dev, 4)
    y, kept = ops.linear_forward(x, w, b, r, 3, 0.0, True)
    assert torch.equal(y, autograd.linear(x, w, b, r, "gelu")) and kept.numel() == y.numel() * 4
    back = lambda **k: ops.linear_backward(*{**dict(dy=dy, x=x, w=w, kept=kept, xs=x.shape, ws=w.shape, act=3, slope=0.0, nx=True, nw=True, nb=True), **k}.values())  # noqa: E731
    assert [t.shape for t in back()] == [x.shape, w.shape, b.shape] and [t.numel() for t in back(nw=False, nb=False)] == [x.numel(), 0, 0]
    for bad in ((x, w.mT, b, r, 0), (x, w, x, r, 0), (x, w, b, b, 0), (x, w.half(), b, r, 0), (x, w, b, r, 5), (x, w, b, r, -1), (x.cpu(), w, b, r, 0)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.linear_forward(*bad, 0.0, True)
    for bad in (dict(dy=dy[1:]), dict(x=x[1:]), dict(x=None), dict(w=w.mT), dict(w=None), dict(kept=None), dict(kept=kept[1:]), dict(kept=kept.view(torch.float32)), dict(xs=w.shape),
                dict(ws=x.shape), dict(ws=(41,)), dict(xs=()), dict(act=7), dict(nx=False, nw=False), dict(nw=False), dict(dy=dy.half())):
        with pytest.raises((ValueError, RuntimeError)):
            back(**bad)
    for bad in ([x[0]], [x, w.half()], [x.long()]):
        with pytest.raises((ValueError, RuntimeError)):
            ops.orthogonalize(bad, 5, 3.4445, -4.7750, 2.0315, 1e-7)
    with pytest.raises(ValueError):
        ops.orthogonalize([x], 0, 3.4445, -4.7750, 2.0315, 1e-7)
    torch.library.opcheck(ops.linear_forward.default, (x, w, b, r, 3, 0.0, True), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(ops.linear_forward.default, (x, w, None, None, 0, 0.0, False), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(ops.linear_backward.default, (dy, x, w, kept, x.shape, w.shape, 3, 0.0, True, True, False), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(ops.orthogonalize.default, ([x, w], 5, 3.4445, -4.7750, 2.0315, 1e-7), test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_compiled_callers_break_their_graph_and_stay_right(dev):
    def f(x, w, b):
        return autograd.linear(x * 2, w, b, activation="silu").square().sum()
    leaves = [torch.randn(s, device=dev, requires_grad=True) for s in ((70, 33), (41, 33), (41,))]
    want = f(*leaves)
    grads = torch.autograd.grad(want, leaves)
    got = torch.compile(f, backend="eager")(*leaves)
    assert torch.equal(want, got) and all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(got, leaves)))
    g = torch.randn(30, 50, device=dev)
    assert torch.equal(torch.compile(lambda t: optim.orthogonalize(t + 0), backend="eager")(g), optim.orthogonalize(g))


@pytest.mark.gpu
def test_lazily_negated_tensors(dev):
    """A view whose memory holds the negated values (what `.conj().imag` of a complex tensor is) counts as the values that it shows."""
    torch.manual_seed(3)
    neg = lambda *s: torch._neg_view(torch.randn(*s, device=dev))  # noqa: E731
    held = {"x": neg(20, 30), "weight": neg(12, 30), "bias": neg(12), "residual": neg(20, 12)}
    assert all(t.is_neg() for t in held.values())
    dy = neg(20, 12)
    for act in ("none", "leaky_relu", "silu"):
        results = []
        for make in (lambda t: t.detach(), lambda t: t.detach().resolve_neg()):
            leaves = [make(t).requires_grad_() for t in held.values()]
            y = autograd.linear(*leaves, activation=act)
            results.append([y, *torch.autograd.grad(y, leaves, make(dy))])
        assert all(torch.equal(a, b) for a, b in zip(*results)), act
    column = torch.randn(20, 1, dtype=torch.complex64, device=dev).conj().imag      # one column: its stride says nothing
    assert column.is_neg() and torch.equal(autograd.linear(column, held["weight"][:, :1]), autograd.linear(column.clone().resolve_neg(), held["weight"][:, :1].resolve_neg()))
    assert torch.equal(optim.orthogonalize(held["x"]), optim.orthogonalize(held["x"].resolve_neg()))
    for opt in (s2l.FusedMuon, s2l.FusedAdam):
        ends = []
        for grad in (held["weight"], held["weight"].resolve_neg()):
            p = torch.nn.Parameter(torch.ones(12, 30, device=dev))
            p.grad = grad
            opt([p], lr=0.1).step()
            ends.append(p.detach())
        assert torch.equal(*ends)
        p = torch.nn.Parameter(neg(4, 5))
        p.grad = torch.ones(4, 5, device=dev)
        with pytest.raises(RuntimeError):
            opt([p]).step()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (6, 10241))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16), ids=str)
def test_the_tail_of_gelu(dtype, rows, dev):
    """gelu and its derivative on z in -10 .. 0 against 64 bits, relative to their own terms: one rounding at the store beside the evaluation's error.

    z = x * 1 is exact.  fp32: erfc's argument is off by two roundings, which its value amplifies (1 + z^2)-fold; exp's by one, z^2 / 2-fold; the functions
    and the remaining products take 10 units of 2^-24.  16-bit types: the formula's 4.8e-5, and 2^-24 (4 z^2 + 16) of its own arithmetic."""
    x = torch.linspace(-10, 0, rows, device=dev).to(dtype)[:, None].requires_grad_()
    w = torch.ones(1, 1, dtype=dtype, device=dev)
    y = autograd.linear(x, w, activation="gelu")
    (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    z = x.detach().double()
    phi, density = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5), torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
    e = 2.0 ** -24 * (4 * z * z + 16) + (0 if dtype == torch.float32 else 4.8e-5)
    info = torch.finfo(dtype)
    u, grid = info.eps / 2, info.tiny * info.eps / 2      # below the normal range: half a step of the grid
    for got, want, size in ((y, z * phi, (z * phi).abs()), (gx, phi + z * density, phi + (z * density).abs())):
        bound = u * want.abs() + (1 + u) * e * size + grid
        far = (got.detach().double() - want).abs() / bound.clamp_min(1e-300)
        assert float(far.max()) <= 1, (float(far.max()), float(z[far.argmax()]))


def _layer(dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(s, generator=g, device=dev) for s in ((70, 33), (41, 33), (41,), (70, 41))], torch.randn(70, 41, generator=g, device=dev)


@pytest.mark.gpu
def test_a_captured_backward_pass_of_leaves_that_an_eager_graph_holds_is_refused(dev):
    import gc
    values, dy = _layer(dev, 0)
    leaves = [v.requires_grad_() for v in values]
    alive = autograd.linear(*leaves, "gelu")      # say, a loss that is kept for a log
    for backward in (lambda y: torch.autograd.grad(y, leaves, dy), lambda y: y.backward(dy)):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="held by a graph made outside"):
            with torch.cuda.graph(graph):
                backward(autograd.linear(*leaves, "gelu"))
        torch.cuda.synchronize()
    want = torch.autograd.grad(alive, leaves, dy)      # the process, the eager graph and the device go on
    again = torch.autograd.grad(autograd.linear(*leaves, "gelu"), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    del alive
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(autograd.linear(*leaves, "gelu"), leaves, dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.gpu
def test_a_captured_backward_call_fills_the_gradients(dev):
    """loss.backward() under capture: two layers, one weight in both; replayed on new values."""
    def step(leaves, up):
        x, w, b, r = leaves
        y = autograd.linear(autograd.linear(x, w, b, residual=r, activation="silu"), w.mT, activation="relu")
        y.backward(up)
    values, _ = _layer(dev, 0)
    static = [v.clone().requires_grad_() for v in values]
    up = torch.zeros(70, 33, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, up)
    torch.cuda.current_stream().wait_stream(side)
    for v in static:
        v.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(static, up)
    for seed in (1, 2, 3):
        values, _ = _layer(dev, seed)
        with torch.no_grad():
            for s, v in zip(static, values):
                s.copy_(v)
            up.copy_(values[0] * 0.5)
        graph.replay()
        torch.cuda.synchronize()
        fresh = [v.clone().requires_grad_() for v in values]
        step(fresh, up)
        assert all(torch.equal(s.grad, f.grad) for s, f in zip(static, fresh)), seed


@pytest.mark.gpu
@pytest.mark.parametrize("opt", (s2l.FusedMuon, s2l.FusedAdam))
def test_a_captured_optimizer_step_is_refused(opt, dev):
    """Its report goes to pinned memory that the next step gives back to torch's host allocator: a replay would write into somebody else's."""
    p, q = (torch.nn.Parameter(torch.ones(12, 30, device=dev)) for _ in range(2))
    p.grad, q.grad = torch.full_like(p, 0.5), torch.full_like(p, 0.5)
    one, other = opt([p], lr=0.1), opt([q], lr=0.1)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(graph):
            p.grad.add_(0)
            one.step()
    torch.cuda.synchronize()
    assert bool((p == 1).all()) and not one.state[p]
    one.step()
    other.step()
    assert torch.equal(p, q) and not bool((p == 1).any())
    assert not any(bad for _, bad in one.nan_report())


def test_a_captured_optimizer_step_is_refused_on_the_host(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capture"):
        optim._refuse_capture("FusedMuon", torch.device("cuda:0"))
    optim._refuse_capture("FusedMuon", torch.device("cpu"))


def test_arguments_that_are_no_tensors():
    w = torch.zeros(4, 3)
    for bad in (([1.0], w), (None, w), (w, None), (w, w, 1.0), (w, w, None, "r"), (w.numpy(), w)):
        with pytest.raises(TypeError, match="are tensors"):
            autograd.linear(*bad)
    with pytest.raises(ValueError):
        autograd.linear(w, w, negative_slope="steep")


@pytest.mark.gpu
def test_an_error_of_a_saved_tensor_hook_is_the_callers(dev):
    x, w = torch.randn(5, 3, device=dev), torch.randn(4, 3, device=dev, requires_grad=True)

    def pack(t):
        raise TypeError("my own")
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t), pytest.raises(TypeError, match="my own"):
        autograd.linear(x, w)
    assert torch.equal(autograd.linear(x, w.detach()), autograd.linear(x, w))


def test_an_iteration_that_passed_vouches_for_no_other():
    """steps = 2.0 equals 2 and hashes as it does."""
    g = torch.zeros(3, 4)
    for steps in (2, 1):
        with pytest.raises(RuntimeError, match="GPU"):
            optim.orthogonalize(g, steps=steps)
    for bad in (2.0, True):
        with pytest.raises(ValueError, match="steps"):
            optim.orthogonalize(g, steps=bad)
    for k in range(200):
        with pytest.raises(RuntimeError, match="GPU"):
            optim.orthogonalize(g, steps=1, eps=1e-7 + k * 1e-9)
    assert optim._check_iteration.cache_info().currsize <= 64
    for bad in ((1.0, 2.0), (float("inf"), 0.0, 0.0), "abc"):
        with pytest.raises(ValueError):
            optim.orthogonalize(g, coefficients=bad)
    with pytest.raises(RuntimeError, match="GPU"):
        optim.orthogonalize(g, coefficients=torch.tensor([1.5, -0.5, 0.0]))


@pytest.mark.gpu
def test_the_backward_pass_again(dev):
    """Under retain_graph the same bits as often as asked; without it an error, unless nothing was kept (the residual's gradient is dy)."""
    values, dy = _layer(dev, 5)
    for act in ("none", "relu", "gelu"):
        leaves = [v.clone().requires_grad_() for v in values]
        y = autograd.linear(*leaves, act)
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        for keep in (True, False):
            assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, dy, retain_graph=keep)))
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, leaves, dy)
        residual = values[3].clone().requires_grad_()
        y = autograd.linear(*values[:3], residual, act)
        for _ in range(2):
            assert torch.equal(torch.autograd.grad(y, residual, dy)[0], dy)
        leaves = [v.clone().requires_grad_() for v in values]
        y = autograd.linear(*leaves, act)
        with torch.no_grad():      # an operand changed in between: refused, as torch's own layers do
            leaves[1].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, dy)


def test_calls_beyond_a_launch_are_refused_on_the_host():
    """2^32 threads or more: 2^26 outputs of a few rows, four to a workgroup of 256; 2^24 tiles of 128 x 128."""
    lib, p, most = _abi.load(), 4096, (1 << 31) - 1
    fwd = lambda rows, k, n, act=0, saved=0: lib.s2l_linear_forward(0, p, k, p, k, 0, 0, n, p, n, saved, p, rows, k, n, act, 0.0, 0)  # noqa: E731
    assert fwd(1, 1, 1 << 26) == -2 and fwd(8, 1, most) == -2
    assert fwd(most, 33, 1) == -2 and fwd(1 << 30, 32, 129) == -2 and fwd(8, 32, most, act=1, saved=p) == -2
    bwd = lambda rows, k, n: lib.s2l_linear_backward(0, p, n, p, k, p, k, p, p, k, 0, 0, p, rows, k, n, 0, 0.0, 0)  # noqa: E731
    assert bwd(most, 5, 4) == -2 and bwd(8, most, 4) == -2 and bwd(1 << 30, 129, 32) == -2


@pytest.mark.gpu
def test_the_librarys_refusals_are_the_packages_errors(dev):
    with pytest.raises(_abi.S2LError, match="bad size"):
        autograd.linear(torch.zeros(1, 1, device=dev), torch.zeros(1 << 26, 1, device=dev))
    with Watching(), pytest.raises(RuntimeError, match="bad size"):
        autograd.linear(torch.zeros(1, 1, device=dev), torch.zeros(1 << 26, 1, device=dev))


@pytest.mark.gpu
def test_calls_from_several_threads(dev):
    """Each thread on a stream of its own, forward, backward and orthogonalisation at once: the bits of the calls alone."""
    import threading
    sizes = ((70, 33, 41, "gelu"), (4160, 192, 4120, "relu"), (9, 256, 64, "none"), (4128, 520, 288, "silu"))
    jobs = []
    for i, (rows, k, n, act) in enumerate(sizes):
        g = torch.Generator(device=dev).manual_seed(i)
        dtype = torch.bfloat16 if i % 2 else torch.float32
        values = [torch.randn(s, generator=g, device=dev).to(dtype) for s in ((rows, k), (n, k), (n,), (rows, n))]
        dy, update = torch.randn(rows, n, generator=g, device=dev).to(dtype), torch.randn(3, 40 + i, 600, generator=g, device=dev)
        jobs.append((values, dy, act, update))

    def run(values, dy, act, update):
        return (*_both_passes(act)(*values, dy), optim.orthogonalize(update))
    want = [run(*j) for j in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = run(*jobs[i])
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(want[i], got)):
                        wrong.append(i)
        except Exception as e:      # noqa: BLE001 (reported below)
            wrong.append((i, e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and not any(t.is_alive() for t in threads), wrong
