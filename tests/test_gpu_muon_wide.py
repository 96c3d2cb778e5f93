"""s2l_muon_step at the sizes that take the 128- and 64-wide tiles, two groups of waves, Gram products in pieces and more than one set of launches:
parameters, momentum and the NaN report against the formula in 64 bits, between guard bands.  Bounds as derived in test_gpu_muon.py."""
import math

import pytest
import torch

from speech2lip_amd import _abi, optim
from tests.test_gpu_muon import ABC, _muon_reference, bound

LR, SHRINK, MU = 0.02, 0.998, 0.95
SETS = {
    "64-wide": [(256, 256)] * 12 + [(320, 200), (64, 500), (200, 321)],
    "128-wide, one workgroup to a CU": [(1990, 2000)],
    "128-wide": [(1100, 1024)] * 5 + [(700, 1000), (1000, 700)],
    "in pieces": [(1024, 1024)] * 2 + [(1000, 4100), (4096, 1024), (1100, 1090)],
    "two sets of launches": [(40 + k % 7, 30 + k % 5) for k in range(60)],
}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", (1, 0))
@pytest.mark.parametrize("name", SETS)
def test_a_step_between_guard_bands(name, nesterov, dev):
    lib, shapes = _abi.load(), SETS[name]
    print(name, flush=True)
    gen = torch.Generator(device=dev).manual_seed(len(shapes))
    normal = lambda s, by: torch.randn(s, generator=gen, device=dev) * by  # noqa: E731
    ps, ms, gs = ([normal(s, by) for s in shapes] for by in (0.05, 0.3, 1.0))
    sick = {0: (0, 0), len(shapes) - 1: (shapes[-1][0] - 1, shapes[-1][1] - 1)}      # NaNs in two parameters: reported, and nowhere else
    for i, at in sick.items():
        ps[i][at] = float("nan")

    def banded(tensors):
        out = [torch.full((t.numel() + 80,), 7.0, device=dev) for t in tensors]
        for o, t in zip(out, tensors):
            o[40:-40].copy_(t.flatten())
        return out
    scales = [math.sqrt(max(1.0, r / c)) for r, c in shapes]
    runs = []
    for _ in range(2):
        pb, mb = banded(ps), banded(ms)
        table = optim._matrix_table([(g.data_ptr(), p.data_ptr() + 160, m.data_ptr() + 160, *g.shape, LR * s) for g, p, m, s in zip(gs, pb, mb, scales)])
        need = lib.s2l_orthogonalize_work_bytes(table, len(gs))
        work = torch.full((need + 256,), 255, dtype=torch.uint8, device=dev)
        flags = torch.zeros(len(gs) + 2, dtype=torch.int32, device=dev)
        _abi.check(lib.s2l_muon_step(table, len(gs), MU, nesterov, SHRINK, *ABC, 1e-7, 5, flags.data_ptr() + 4, work.data_ptr(),
                                     torch.cuda.current_stream().cuda_stream), "step")
        torch.cuda.synchronize()
        assert flags.tolist() == [0] + [int(i in sick) for i in range(len(gs))] + [0]
        assert all(bool((v[:40] == 7).all()) and bool((v[-40:] == 7).all()) for v in pb + mb) and bool((work[need:] == 255).all())
        runs.append([v[40:-40].reshape(s).clone() for vs in (pb, mb) for v, s in zip(vs, shapes * 2)])
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(*runs))
    for i, (r, c) in enumerate(shapes if len(shapes) < 20 else shapes[:3] + shapes[54:]):
        i = i if len(shapes) < 20 or i < 3 else 54 + i - 3
        p, m = runs[0][i], runs[0][len(shapes) + i]
        wd = (1 - SHRINK) / LR
        new_p, new_m = _muon_reference(ps[i].double(), ms[i].double(), gs[i].double(), LR, wd, MU, bool(nesterov), None)
        size = new_m.abs() + ms[i].double().abs() + gs[i].double().abs()
        assert bool(((m.double() - new_m).abs() <= 2.0 ** -22 * size.max()).all())
        u = gs[i].double() + MU * (new_m - gs[i].double()) if nesterov else new_m
        _, limit = bound(u.float(), torch.float32)
        where = torch.isnan(ps[i])
        assert torch.equal(torch.isnan(p), where) and int(where.sum()) == int(i in sick)
        off = (p.double() - new_p)[~where].norm()
        # the parameter: one rounding of shrink as a float, two of the update
        assert float(off) <= LR * scales[i] * (limit + 485 * 2.0 ** -22) + 3 * 2.0 ** -24 * float(new_p[~where].norm()), (name, i, float(off))
