"""optim.orthogonalize and FusedMuon (csrc/orthogonalize.hip) against their formulas in 64 bits.

Tolerances, derived.  p(s) = a s + b s^3 + c s^5 has |p(s) / s| <= 3.45 and |p'| <= 3.9 on [0, 1.2], so a perturbation of X (in the Frobenius norm) grows
at most 3.9-fold in each later step.  fp32 (two halves): every value is held to 2^-22 relative where fp32 holds 2^-24, sums are fp32's: the error is
held to 4 times that of the same iteration in fp32 torch products, plus one rounding.  16-bit types: the same up to the last two steps; each of
those rounds X, A and B to a half (u = 2^-11):  e = u (3.9 ||X||_F + ||B||_F ||X||_2 + (|b| + 2 |c| ||A||_2) ||A||_F ||X||_2), the last but one's
grown 3.9-fold; the result is rounded once."""
import copy
import math

import pytest
import torch

import speech2lip_amd as s2l
from speech2lip_amd import _abi, autograd, optim
from tests.test_gpu_callers import _cfg, _g11_device, _late_model, syncnet  # noqa: F401  (the fixture)

ABC = (3.4445, -4.7750, 2.0315)
TYPES = (torch.float32, torch.bfloat16, torch.float16)
SHAPES = [(1, 1), (1, 9), (9, 1), (3, 2), (16, 16), (63, 65), (64, 64), (65, 63), (20, 256), (256, 42), (64, 576), (129, 300), (333, 1000), (1000, 333), (257, 257)]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def iterate(g, steps=5, abc=ABC, eps=1e-7, dtype=torch.float64, states=None):
    """The iteration from the left, of the shorter side, in `dtype`; the norm in 64 bits."""
    tall = g.shape[-2] > g.shape[-1]
    x = g.double().mT if tall else g.double()
    norm = x.square().sum((-2, -1), keepdim=True).sqrt()
    x = (x / norm.clamp_min(eps)).to(dtype).contiguous()
    a, b, c = abc
    for _ in range(steps):
        gram = x @ x.mT.contiguous()
        poly = b * gram + c * (gram @ gram) + a * torch.eye(gram.shape[-1], dtype=dtype, device=g.device)
        if states is not None:
            states.append((x, gram, poly))
        x = poly @ x
    return x.mT if tall else x


def matrix(rows, cols, kind, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + rows * 31 + cols)
    n = torch.randn(rows, cols, generator=g, device=dev, dtype=torch.float64)
    if kind == "plain":
        return 1e-3 * n
    m = min(rows, cols)
    q = torch.linalg.qr(n.mT if rows < cols else n)[0]
    w = torch.linalg.qr(torch.randn(m, m, generator=g, device=dev, dtype=torch.float64))[0]
    i = torch.arange(1, m + 1, device=dev, dtype=torch.float64)
    s = {"falling": i ** -1.0, "steep": i ** -2.0, "deficient": (i <= max(1, m // 8)).double()}[kind]
    u = (q * s) @ w.mT
    return u.mT if rows < cols else u


def bound(g, dtype, steps=5, abc=ABC, eps=1e-7):
    """Largest allowed Frobenius error of a result of type `dtype` from the (rounded) input g."""
    states = []
    want = iterate(g, steps, abc, eps, states=states)
    single = iterate(g, steps, abc, eps, dtype=torch.float32)
    u = torch.finfo(dtype).eps / 2
    limit = 4 * float((single.double() - want).norm()) + (2 * u + 2.0 ** -22) * float(want.norm())
    if dtype != torch.float32:
        e, half = 0.0, 2.0 ** -11
        for x, gram, poly in states[-2:]:
            x2 = float(torch.linalg.matrix_norm(x, 2))
            a2 = x2 * x2
            e = 3.9 * e + half * (3.9 * float(x.norm()) + float(poly.norm()) * x2 + (abs(abc[1]) + 2 * abs(abc[2]) * a2) * float(gram.norm()) * x2)
        limit += e + torch.finfo(dtype).tiny * u * math.sqrt(want.numel())
    return want, limit


def hold(got, g, what, steps=5, abc=ABC, eps=1e-7):
    want, limit = bound(g, got.dtype, steps, abc, eps)
    off = float((got.double() - want).norm())
    assert got.shape == want.shape and off <= limit, (what, off, limit, float(want.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_against_the_formula(rows, cols, dtype, dev):
    for kind in ("plain", "falling", "steep", "deficient"):
        g = matrix(rows, cols, kind, dev).to(dtype)
        got = optim.orthogonalize(g)
        assert got.dtype == dtype and got.shape == g.shape
        hold(got, g, (rows, cols, kind))
        assert torch.equal(got, optim.orthogonalize(g))


@pytest.mark.gpu
def test_large_and_wide_tiles(dev):
    """Sizes whose launches take the 128-wide tiles, also of an odd number of 64s; long thin ones."""
    for dtype in TYPES:
        for rows, cols in ((2113, 2200), (1100, 4100), (4096, 20), (17, 5000)):
            g = matrix(rows, cols, "plain", dev).to(dtype)
            hold(optim.orthogonalize(g), g, (rows, cols))
    g = torch.stack([matrix(704, 832, "falling", dev, seed=s) for s in range(9)]).bfloat16()
    got = optim.orthogonalize(g)
    for k in range(9):
        hold(got[k], g[k], k)


@pytest.mark.gpu
def test_long_gram_products_in_pieces(dev):
    """Lists whose 128-wide tiles are enough for the part, with matrices so long that their Gram products are cut along k: uneven pieces, sides of
    an odd number of 64s, more than sixteen pieces' worth of length, matrices beside them that stay whole; a workspace of NaN, guarded ends."""
    lib = _abi.load()
    lists = [[(1024, 1024)] * 2 + [(1000, 4100), (4096, 1024), (1100, 1090), (963, 4099)], [(640, 5000)] * 9, [(130, 30000)] + [(900, 1030)] * 5]
    for dt, dtype in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
        for shapes in lists:
            gs = [matrix(*s, "plain", dev, seed=i).to(dtype) for i, s in enumerate(shapes)]
            outs = [torch.full((g.numel() + 80,), 7.0, dtype=dtype, device=dev) for g in gs]
            size = outs[0].element_size()
            table = optim._matrix_table([(g.data_ptr(), o.data_ptr() + 40 * size, 0, *g.shape, 0.0) for g, o in zip(gs, outs)])
            need = lib.s2l_orthogonalize_work_bytes(table, len(gs))
            work = torch.full((need + 256,), 255, dtype=torch.uint8, device=dev)
            for again in range(2):
                _abi.check(lib.s2l_orthogonalize(dt, table, len(gs), *ABC, 1e-7, 5, work.data_ptr(), torch.cuda.current_stream().cuda_stream), "orth")
                now = [o[40:-40].reshape(g.shape).clone() for o, g in zip(outs, gs)]
                assert again == 0 or all(torch.equal(a, b) for a, b in zip(first, now))
                first = now
            assert all(bool((o[:40] == 7).all()) and bool((o[-40:] == 7).all()) for o in outs) and bool((work[need:] == 255).all())
            for i in {s: i for i, s in enumerate(shapes)}.values():
                hold(first[i], gs[i], shapes[i])


@pytest.mark.gpu
def test_single_launches_of_few_workgroups(dev):
    """128-wide tiles of at most one workgroup to a CU: two groups of waves share k."""
    for dtype in TYPES:
        for shape in ((4, 1024, 1024), (1, 1990, 2050), (5, 700, 1000)):
            g = torch.stack([matrix(*shape[1:], "falling", dev, seed=s) for s in range(shape[0])]).to(dtype)
            got = optim.orthogonalize(g)
            assert torch.equal(got, optim.orthogonalize(g))
            for k in (0, shape[0] - 1):
                hold(got[k], g[k], (shape, k))


@pytest.mark.gpu
def test_singular_values_against_the_polynomial(dev):
    """U p(...p(s)) V^T from the singular value decomposition, in 64 bits: the result's definition without the iteration."""
    for rows, cols in ((40, 70), (130, 96)):
        g = matrix(rows, cols, "falling", dev).float()
        u, s, vh = torch.linalg.svd(g.double(), full_matrices=False)
        s = s / s.norm()
        for steps in (1, 2, 5, 8):
            t = s.clone()
            for _ in range(steps):
                t = ABC[0] * t + ABC[1] * t ** 3 + ABC[2] * t ** 5
            got = optim.orthogonalize(g, steps=steps)
            _, limit = bound(g, torch.float32, steps)
            assert float((got.double() - (u * t) @ vh).norm()) <= limit + 1e-12


@pytest.mark.gpu
def test_other_coefficients_and_step_counts(dev):
    cubic = (1.5, -0.5, 0.0)
    for dtype in TYPES:
        for steps, abc in ((1, ABC), (2, ABC), (3, cubic), (12, cubic), (20, (2.0, -1.5, 0.5))):
            g = matrix(70, 90, "plain", dev).to(dtype)
            hold(optim.orthogonalize(g, steps=steps, coefficients=abc), g, (steps, abc), steps, abc)


@pytest.mark.gpu
def test_batches_lists_and_strides(dev):
    for dtype in TYPES:
        g = torch.stack([matrix(33, 47, "plain", dev, seed=s) for s in range(6)]).reshape(2, 3, 33, 47).to(dtype)
        got = optim.orthogonalize(g)
        assert got.shape == g.shape
        one = torch.stack([optim.orthogonalize(g[i, j]) for i in range(2) for j in range(3)]).reshape(g.shape)
        assert torch.equal(got, one)      # a matrix's result does not depend on its company
        t = g.mT
        assert torch.equal(optim.orthogonalize(t), optim.orthogonalize(t.contiguous()))
        assert torch.equal(optim.orthogonalize(g[:, ::2, 1:, 3:]), optim.orthogonalize(g[:, ::2, 1:, 3:].contiguous()))
        assert torch.equal(optim.orthogonalize(g[0, 0].expand(4, 33, 47))[3], one[0, 0])
        sizes = [(5, 9), (300, 40), (64, 64), (1, 1), (257, 130)]
        several = [matrix(*s, "plain", dev).to(dtype) for s in sizes]
        for x, y in zip(optim.orthogonalize(several), several):
            hold(x, y, tuple(y.shape))
    many = [matrix(8 + k % 5, 6 + k % 7, "plain", dev, seed=k).float() for k in range(130)]      # more than one set of launches holds
    for x, y in zip(optim.orthogonalize(many), many):
        hold(x, y, tuple(y.shape))
    assert optim.orthogonalize([]) == []
    empty = optim.orthogonalize(torch.zeros(0, 3, 4, device=dev))
    assert empty.shape == (0, 3, 4)
    assert optim.orthogonalize(torch.zeros(3, 0, device=dev)).shape == (3, 0)


@pytest.mark.gpu
def test_zeros_nans_and_extreme_norms(dev):
    for dtype in TYPES:
        good = matrix(70, 50, "plain", dev).to(dtype)
        nan, inf = good.clone(), good.clone()
        nan[3, 4], inf[69, 49] = float("nan"), float("-inf")
        out = optim.orthogonalize([nan, good, inf, torch.zeros_like(good), good])
        assert bool(torch.isnan(out[0]).all()) and bool(torch.isnan(out[2]).all())
        assert bool((out[3] == 0).all()) and torch.equal(out[1], out[4]) and torch.equal(out[1], optim.orthogonalize(good))
        one = torch.full((1, 1), float("nan"), dtype=dtype, device=dev)
        assert bool(torch.isnan(optim.orthogonalize(one)).all())
    g = matrix(70, 50, "plain", dev)
    for scale in (1e-20, 1e30, 3e37):      # squares that fp32 cannot hold; the result is the same matrix's
        x = (g * 1e3 * scale).float()
        hold(optim.orthogonalize(x, eps=1e-30), x, scale, eps=1e-30)
    big = torch.full((200, 300), 3e38, device=dev)      # a norm beyond fp32's range
    hold(optim.orthogonalize(big), big, "norm beyond fp32")
    tiny = (g / g.norm() * 1e-9).float()      # below eps: scaled by eps, in steps of 2^-36
    got = optim.orthogonalize(tiny, eps=1e-7)
    want = iterate(tiny, eps=1e-7)
    assert float((got.double() - want).abs().max()) <= 485 * 2.0 ** -35 + 1e-5 * float(want.abs().max())


@pytest.mark.gpu
def test_workspace_need_not_be_clean_and_nothing_is_written_behind_the_results(dev):
    lib = _abi.load()
    for dt, dtype in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
        shapes = [(65, 63), (130, 7), (300, 200)]
        gs = [matrix(*s, "plain", dev).to(dtype) for s in shapes]
        want = [optim.orthogonalize(g) for g in gs]
        outs = [torch.full((g.numel() + 80,), 7.0, dtype=dtype, device=dev) for g in gs]
        size = outs[0].element_size()
        table = optim._matrix_table([(g.data_ptr(), o.data_ptr() + 40 * size, 0, *g.shape, 0.0) for g, o in zip(gs, outs)])
        need = lib.s2l_orthogonalize_work_bytes(table, 3)
        for byte in (0, 255, 0x7e):
            work = torch.full((need + 256,), byte, dtype=torch.uint8, device=dev)
            _abi.check(lib.s2l_orthogonalize(dt, table, 3, *ABC, 1e-7, 5, work.data_ptr(), torch.cuda.current_stream().cuda_stream), "orth")
            for o, w in zip(outs, want):
                assert torch.equal(o[40:-40].reshape(w.shape), w) and bool((o[:40] == 7).all()) and bool((o[-40:] == 7).all())
            assert bool((work[need:] == byte).all())


@pytest.mark.gpu
def test_streams_and_graphs(dev):
    """On a side stream, and captured and replayed on new values between eager work: the bits of the eager call."""
    for dtype, shape in ((torch.float32, (3, 100, 130)), (torch.bfloat16, (1, 700, 900))):
        g = torch.stack([matrix(*shape[1:], "plain", dev, seed=s) for s in range(shape[0])]).to(dtype)
        want = optim.orthogonalize(g)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = optim.orthogonalize(g)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(want, got)
        static = g.clone()
        graphs, outs = [], []
        for _ in range(2):      # two graphs: each has its own workspace
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(optim.orthogonalize(static))
            graphs.append(graph)
        for seed in (5, 6, 7):
            fresh = torch.stack([matrix(*shape[1:], "plain", dev, seed=seed + s) for s in range(shape[0])]).to(dtype)
            static.copy_(fresh)
            for graph in graphs:
                graph.replay()
            torch.cuda.synchronize()
            want = optim.orthogonalize(fresh)
            assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def _muon_reference(p, m, g, lr, wd, mu, nesterov, mode, steps=5, abc=ABC, eps=1e-7):
    m = m + (1 - mu) * (g - m)
    u = g + mu * (m - g) if nesterov else m
    rows, cols = u.shape[0], u.numel() // u.shape[0]
    scale = 0.2 * math.sqrt(max(rows, cols)) if mode == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))
    o = iterate(u.reshape(rows, cols), steps, abc, eps).reshape(p.shape)
    return p * (1 - lr * wd) - lr * scale * o, m


@pytest.mark.gpu
def test_fused_muon_against_the_formula(dev):
    """Several steps over ragged matrices and convolutions: parameters and momentum against 64 bits.  The update's direction is held as `bound` holds it
    (the momentum, rounded to fp32, feeds it: one more 2^-23 of its norm, grown 485-fold at most); p takes two roundings a step."""
    shapes = [(256, 256), (256, 512), (20, 7), (64, 3, 3, 3), (7, 130), (1, 5), (300, 64)]
    for nesterov, mode, wd, mu in ((True, None, 0.1, 0.95), (False, "original", 0.0, 0.9), (True, "match_rms_adamw", 0.01, 0.0)):
        gen = torch.Generator(device=dev).manual_seed(4)
        ps = [torch.nn.Parameter(torch.randn(s, generator=gen, device=dev) / 16) for s in shapes]
        opt = s2l.FusedMuon(ps, lr=0.02, weight_decay=wd, momentum=mu, nesterov=nesterov, adjust_lr_fn=mode)
        ref = [(p.detach().double(), torch.zeros_like(p, dtype=torch.float64)) for p in ps]
        slack = [0.0] * len(ps)
        for step in range(3):
            grads = [torch.randn(s, generator=gen, device=dev) * (0.3 if step % 2 else 4.0) for s in shapes]
            for p, g in zip(ps, grads):
                p.grad = g.clone()
            versions = [p._version for p in ps]
            opt.step()
            assert all(p._version > v for p, v in zip(ps, versions))
            for k, (p, g) in enumerate(zip(ps, grads)):
                old_m = ref[k][1]
                new_p, new_m = _muon_reference(*ref[k], g.double(), 0.02, wd, mu, nesterov, mode)
                ref[k] = (new_p, new_m)
                m = opt.state[p]["momentum_buffer"]
                size = new_m.abs() + old_m.abs() + g.double().abs()
                assert bool(((m.double() - new_m).abs() <= 2.0 ** -22 * (step + 1) * size.max()).all())
                rows, cols = p.shape[0], p.numel() // p.shape[0]
                scale = 0.2 * math.sqrt(max(rows, cols)) if mode == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))
                u = (g.double() + mu * (new_m - g.double()) if nesterov else new_m).reshape(rows, cols)
                want, limit = bound(u.float(), torch.float32)
                slack[k] += 0.02 * scale * (limit + 485 * 2.0 ** -22) + 2.0 ** -23 * float(new_p.norm())
                assert float((p.detach().double() - new_p).norm()) <= slack[k], (step, k)
        assert not any(bad for _, bad in opt.nan_report()) and len(opt.nan_report()) == len(ps)


@pytest.mark.gpu
def test_state_dicts_are_torchs(dev):
    """torch.optim.Muon's state loads into FusedMuon and back; one further step of both agrees within torch's bf16 iteration (its products round to
    2^-8: up to 3.9 * 3.9 * ... of them; held to a twentieth of the step's norm on a well-conditioned update)."""
    gen = torch.Generator(device=dev).manual_seed(4)
    shapes = [(64, 96), (130, 50)]
    pa = [torch.nn.Parameter(torch.randn(s, generator=gen, device=dev)) for s in shapes]
    pb = [torch.nn.Parameter(p.detach().clone()) for p in pa]
    oa, ob = torch.optim.Muon(pa, lr=0.1, weight_decay=0.1), s2l.FusedMuon(pb, lr=0.1, weight_decay=0.1)
    for step in range(3):
        for p, q in zip(pa, pb):
            with torch.no_grad():
                q.copy_(p)
            p.grad = torch.randn(p.shape, generator=gen, device=dev)
            q.grad = p.grad.clone()
        before = [p.detach().clone() for p in pa]
        oa.step()
        ob.step()
        for p, q, old in zip(pa, pb, before):
            assert float((oa.state[p]["momentum_buffer"] - ob.state[q]["momentum_buffer"]).abs().max()) <= 1e-6
            assert float((p - q).detach().norm()) <= 0.05 * float((p - 0.99 * old).detach().norm())
    sa, sb = oa.state_dict(), ob.state_dict()
    assert set(sa["state"][0]) == set(sb["state"][0]) == {"momentum_buffer"} and sb["param_groups"][0].keys() >= sa["param_groups"][0].keys()
    oc = s2l.FusedMuon(pb, lr=0.5)
    oc.load_state_dict(copy.deepcopy(sa))      # (loading shares the tensors)
    torch.optim.Muon(pa, lr=0.5).load_state_dict({"state": sb["state"], "param_groups": sa["param_groups"]})
    want = [p.detach().clone() for p in pb]
    for q in pb:
        q.grad = torch.ones_like(q) + torch.randn(q.shape, generator=gen, device=dev)
    keep = [q.grad.clone() for q in pb]
    ob.load_state_dict(copy.deepcopy(sa | {"param_groups": sb["param_groups"]}))
    ob.step()
    first = [q.detach().clone() for q in pb]
    with torch.no_grad():
        for q, w, g in zip(pb, want, keep):
            q.copy_(w)
            q.grad = g
    oc.step()
    assert all(torch.equal(a, b.detach()) for a, b in zip(first, pb))


@pytest.mark.gpu
def test_adam_groups_and_the_nan_report(dev):
    gen = torch.Generator(device=dev).manual_seed(9)
    w = [torch.nn.Parameter(torch.randn(40, 30, generator=gen, device=dev)) for _ in range(2)]
    v = [torch.nn.Parameter(torch.randn(30, generator=gen, device=dev)) for _ in range(2)]
    v2 = [torch.nn.Parameter(p.detach().clone()) for p in v]
    opt = s2l.FusedMuon([{"params": w, "lr": 0.1}, {"params": v, "algorithm": "adam", "lr": 0.01}])
    alone = s2l.FusedAdam(v2, lr=0.01)
    for _ in range(3):
        for p in w + v:
            p.grad = torch.randn(p.shape, generator=gen, device=dev)
        for p, q in zip(v, v2):
            q.grad = p.grad.clone()
        opt.step()
        alone.step()
    assert all(torch.equal(p, q) for p, q in zip(v, v2))
    w[1].data[3, 4] = float("nan")
    v[0].data[2] = float("nan")
    for p in w + v:
        p.grad = torch.ones_like(p)
    assert opt.covers() == {id(p) for p in w + v}
    opt.step()
    bad = {id(p) for p, b in opt.nan_report() if b}
    assert bad == {id(w[1]), id(v[0])} and len(opt.nan_report()) == 4
    w[0].grad = None      # a parameter without a gradient is left alone
    old = w[0].detach().clone()
    opt.step()
    assert torch.equal(old, w[0].detach()) and len(opt.nan_report()) == 3


@pytest.mark.gpu
def test_a_residual_network_of_linear_layers_trains_with_muon(dev):
    """The operators as they are used together: a stack of residual layers (autograd.linear), its gradients against 64-bit autograd, stepped by FusedMuon
    with an Adam for biases and the output layer; the step is the formula's."""
    torch.manual_seed(0)
    width, rows = 96, 500

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.inner = torch.nn.ModuleList([torch.nn.Linear(42, width), torch.nn.Linear(width, width), torch.nn.Linear(width, width)])
            self.output_linear = torch.nn.Linear(width, 3)

        def forward(self, x):
            h = autograd.linear(x, self.inner[0].weight, self.inner[0].bias, activation="silu")
            for lay in self.inner[1:]:
                h = autograd.linear(h, lay.weight, lay.bias, residual=h, activation="gelu")
            return autograd.linear(h, self.output_linear.weight, self.output_linear.bias)

    net = Net().to(dev)
    x, y = torch.randn(rows, 42, device=dev), torch.rand(rows, 3, device=dev)
    groups = optim.muon_groups(net, muon=dict(lr=0.02, weight_decay=0.0), adam=dict(lr=1e-3))
    assert [len(g["params"]) for g in groups] == [3, 5] and groups[1]["params"][-2] is net.output_linear.weight
    opt = s2l.FusedMuon(groups)
    autograd.mse(net(x), y).backward()
    d = {k: p.detach().double().requires_grad_() for k, p in net.named_parameters()}
    f = torch.nn.functional
    h = f.silu(f.linear(x.double(), d["inner.0.weight"], d["inner.0.bias"]))
    for k in (1, 2):
        h = h + f.gelu(f.linear(h, d[f"inner.{k}.weight"], d[f"inner.{k}.bias"]))
    ((f.linear(h, d["output_linear.weight"], d["output_linear.bias"]) - y.double()) ** 2).mean().backward()
    for k, p in net.named_parameters():      # seven products deep, each within (n + 8) 2^-24 of its magnitudes: 1e-4 of the gradient's norm is ample
        assert float((p.grad.double() - d[k].grad).norm()) <= 1e-4 * float(d[k].grad.norm()), k
    before = {k: p.detach().clone() for k, p in net.named_parameters()}
    opt.step()
    for k in range(3):
        w = net.inner[k].weight
        want, _ = _muon_reference(before[f"inner.{k}.weight"].double(), torch.zeros_like(w, dtype=torch.float64), w.grad.double(), 0.02, 0.0, 0.95, True, None)
        assert float((w.detach().double() - want).norm()) <= 1e-3 * float((want - before[f"inner.{k}.weight"].double()).norm())
    for _ in range(3):
        opt.zero_grad()
        autograd.mse(net(x), y).backward()
        opt.step()
    assert all(bool(torch.isfinite(p).all()) for p in net.parameters())


@pytest.mark.gpu
def test_the_trainer_steps_fused_muon(golden, syncnet, dev):  # noqa: F811
    """Trainer.train_steps with FusedMuon over the lip model: the parameters move, its NaN flags reach the check_weights warnings under the state-dict's names."""
    import logging
    _, data, _, _, _ = _g11_device(golden, dev)
    frames = [dict(data, index=int(data["index"]) + k) for k in range(2)]
    m = _late_model(dev)
    opt = s2l.FusedMuon(optim.muon_groups(m, muon=dict(lr=1e-3, weight_decay=0.0), adam=dict(lr=1e-3)))
    tr = s2l.Trainer(m, opt, cfg=_cfg(m), syncnet=syncnet, use_syncloss=True, precision="bf16", hole_noise="device")
    old = {k: p.detach().clone() for k, p in m.named_parameters() if p.requires_grad}
    _, loss = tr.train_steps(frames, it=100001)
    assert bool(torch.isfinite(torch.as_tensor(float(loss["loss"]))))
    moved = {k for k, p in m.named_parameters() if k in old and not torch.equal(old[k], p.detach())}
    assert {"pts_linears.0.weight", "pts_linears.5.weight", "fc_uv.weight", "encoder_conv.0.weight", "output_linear.weight", "fc_time.bias"} <= moved
    m.pts_linears[2].weight.data[3, 3] = float("nan")
    records = []

    class Catch(logging.Handler):
        def emit(self, rec):
            records.append(rec.getMessage())
    log = logging.getLogger("speech2lip_amd.training")
    h = Catch()
    log.addHandler(h)
    try:
        tr.train_steps(frames, it=100002)
    finally:
        log.removeHandler(h)
    assert any("pts_linears.2.weight" in r for r in records), records


def test_refusals_need_no_gpu():
    z = torch.zeros
    with pytest.raises(_abi.S2LError):
        optim.orthogonalize(z(3, 4))
    for bad in (dict(update=z(3)), dict(update=z(3, 4).double()), dict(update=[z(3, 4), z(3, 4).bfloat16()]), dict(update=z(3, 4), steps=0), dict(update=z(3, 4), steps=101),
                dict(update=z(3, 4), steps=2.0), dict(update=z(3, 4), eps=0.0), dict(update=z(3, 4), coefficients=(1.0, 2.0)),
                dict(update=z(3, 4), coefficients=(float("nan"), 0.0, 0.0)), dict(update=z(3, 4), coefficients=(3.0, 3.0, 3.0)), dict(update=z(1, 131073))):
        with pytest.raises(ValueError):
            optim.orthogonalize(**bad)
    with pytest.raises(TypeError):
        optim.orthogonalize([[1.0]])
    p = lambda *s: torch.nn.Parameter(z(*s))  # noqa: E731
    for bad in (dict(lr=-1.0), dict(weight_decay=-1.0), dict(momentum=1.5), dict(adjust_lr_fn="x"), dict(ns_steps=0), dict(eps=0.0), dict(ns_coefficients=(9.0, 9.0, 9.0))):
        with pytest.raises(ValueError):
            s2l.FusedMuon([p(3, 4)], **bad)
    for bad in ([p(3)], [{"params": [p(3, 4)], "algorithm": "sgd"}], [{"params": [p(3)], "algorithm": "adam", "lr": -1.0}], [p(0, 4)], [p(1, 131073)]):
        with pytest.raises(ValueError):
            s2l.FusedMuon(bad)
    with pytest.raises(NotImplementedError):
        s2l.FusedMuon([{"params": [p(3)], "algorithm": "adam", "amsgrad": True}])
    q = p(3, 4)
    q.grad = z(3, 4)
    with pytest.raises(_abi.S2LError):
        s2l.FusedMuon([q]).step()


def test_c_entry_refusals_need_no_gpu():
    lib = _abi.load()
    table = lambda **k: optim._matrix_table([tuple({"src": 4096, "out": 4096, "momentum": 4096, "rows": 3, "cols": 4, "step": 0.1, **k}.values())])  # noqa: E731
    orth = lambda t, n=1, dt=0, abc=ABC, eps=1e-7, steps=5, work=4096: lib.s2l_orthogonalize(dt, t, n, *abc, eps, steps, work, 0)  # noqa: E731
    assert orth(table(), n=0) == 0 and orth(0, n=0) == 0 and orth(0, n=1) == -1
    assert orth(table(), dt=5) == -5 and orth(table(), n=-1) == -2
    assert orth(table(rows=0)) == -2 and orth(table(cols=-1)) == -2 and orth(table(rows=131073)) == -2
    assert orth(table(src=0)) == -1 and orth(table(out=0)) == -1 and orth(table(), work=0) == -1
    assert orth(table(src=4098)) == -3 and orth(table(out=4097), dt=1) == -3 and orth(table(), work=4104) == -3
    assert orth(table(), steps=0) == -2 and orth(table(), steps=101) == -2 and orth(table(), eps=0.0) == -2 and orth(table(), abc=(9.0, 9.0, 9.0)) == -2
    assert orth(table(), abc=(float("nan"), 0.0, 0.0)) == -2
    muon = lambda t, n=1, steps=5, work=4096: lib.s2l_muon_step(t, n, 0.9, 1, 1.0, *ABC, 1e-7, steps, 0, work, 0)  # noqa: E731
    assert muon(table(), n=0) == 0 and muon(table(momentum=0)) == -1 and muon(table(momentum=4098)) == -3 and muon(table(), steps=0) == -2 and muon(table(), work=0) == -1
    assert lib.s2l_orthogonalize_work_bytes(0, 3) == 0 and lib.s2l_orthogonalize_work_bytes(table(rows=0), 1) == 0
    assert lib.s2l_orthogonalize_work_bytes(table(), 1) == 4096 + 512 + 2 * (4 * 64 * 64 + 4 * 64 * 64)


def test_groups_of_a_model():
    net = torch.nn.Module()
    net.fc = torch.nn.Linear(4, 5)
    net.conv = torch.nn.Conv2d(3, 4, 3)
    net.output_linear = torch.nn.Linear(5, 3)
    net.frozen = torch.nn.Parameter(torch.zeros(3, 3), requires_grad=False)
    g = optim.muon_groups(net, muon=dict(lr=0.5), adam=dict(lr=0.25))
    assert [id(p) for p in g[0]["params"]] == [id(net.fc.weight), id(net.conv.weight)] and len(g[1]["params"]) == 4
    opt = s2l.FusedMuon(g)
    assert [x["lr"] for x in opt.param_groups] == [0.5, 0.25] and opt.param_groups[1]["eps"] == 1e-8 and opt.param_groups[0]["eps"] == 1e-7
