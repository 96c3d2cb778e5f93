"""The dense layer at the sizes whose kernels the small ones do not reach: 128- and 256-wide tiles by either path, long contractions in pieces, dx and
dW in one launch, the passes that form dz.  Each case names the kernels that it is there for, as the library itself states them
(s2l_debug_linear_routes), and a last test that every kernel has a case.  Rows and columns leave remainders of the tiles; all goes through the C entries, with
guard bands around every output, against the formula in 64 bits with the bounds derived in test_gpu_linear.py."""
import ctypes

import pytest
import torch

from speech2lip_amd import _abi
from tests.test_gpu_linear import formula, hold, make

F32, BF16, F16 = 0, 1, 2
TYPES = (torch.float32, torch.bfloat16, torch.float16)
REGISTERS, DMA, TOGETHER = 2, 3, 4
ALL, DX, DW = 3, 1, 2
# (type, activation, rows, in, out, gradients): [forward path, tile, pieces], [dx ...], [dW ...], what forms dz; None: not asked for
CASES = {
    (BF16, "gelu", 4160, 192, 4120, ALL): ([DMA, 256, 1], [REGISTERS, 128, 4], [DMA, 128, 4], 16),
    (F16, "none", 4160, 4120, 192, ALL): ([REGISTERS, 128, 4], [DMA, 256, 1], [DMA, 128, 4], 0),
    (BF16, "silu", 4160, 4160, 4160, ALL): ([DMA, 256, 1], [DMA, 256, 1], [DMA, 128, 1], 16),
    (BF16, "relu", 16448, 1024, 1088, ALL): ([DMA, 256, 1], [DMA, 256, 1], [DMA, 64, 1], 1),
    (F32, "silu", 4136, 96, 4120, ALL): ([DMA, 128, 1], [REGISTERS, 64, 2], [REGISTERS, 64, 2], 16),
    (F16, "relu", 2112, 1024, 2056, ALL): ([DMA, 128, 1], [REGISTERS, 64, 1], [REGISTERS, 64, 1], 0),
    (BF16, "none", 2112, 1088, 2048, ALL): ([DMA, 128, 1], [TOGETHER, 64, 1], [TOGETHER, 64, 1], 0),
    (F32, "silu", 4128, 520, 288, ALL): ([REGISTERS, 64, 1], [TOGETHER, 64, 1], [TOGETHER, 128, 26], 2),
    (F32, "gelu", 4128, 512, 288, DW): ([DMA, 64, 1], None, [DMA, 128, 26], 2),
    (BF16, "relu", 36864, 256, 256, DW): ([DMA, 64, 1], None, [DMA, 128, 116], 1),
    (BF16, "relu", 36864, 256, 256, ALL): ([DMA, 64, 1], [TOGETHER, 64, 1], [TOGETHER, 128, 116], 1),
    (F16, "leaky_relu", 20032, 200, 192, ALL): ([REGISTERS, 64, 1], [TOGETHER, 64, 1], [TOGETHER, 128, 63], 1),
    (F32, "none", 65568, 264, 64, ALL): ([REGISTERS, 64, 1], [TOGETHER, 128, 1], [TOGETHER, 64, 52], 0),
    (BF16, "gelu", 2112, 2056, 1024, ALL): ([REGISTERS, 64, 1], [TOGETHER, 128, 1], [TOGETHER, 64, 1], 2),
    (F16, "gelu", 4800, 904, 1024, ALL): ([REGISTERS, 64, 1], [TOGETHER, 128, 1], [TOGETHER, 128, 4], 4),
    (F32, "relu", 4736, 904, 512, ALL): ([REGISTERS, 64, 1], [TOGETHER, 128, 1], [TOGETHER, 128, 15], 1),
    (F32, "leaky_relu", 544, 2056, 2080, ALL): ([REGISTERS, 64, 1], [TOGETHER, 64, 1], [TOGETHER, 128, 1], 1),
    (BF16, "none", 2112, 2056, 1024, DX): ([REGISTERS, 64, 1], [DMA, 128, 1], None, 0),
    (F32, "gelu", 65568, 264, 64, DX): ([REGISTERS, 64, 1], [DMA, 128, 1], None, 4),
    (BF16, "none", 192, 200, 8192, ALL): ([REGISTERS, 64, 1], [DMA, 128, 32], [DMA, 64, 1], 0),
    (F32, "gelu", 96, 136, 4096, ALL): ([REGISTERS, 64, 1], [DMA, 64, 32], [DMA, 64, 1], 1),
    (F16, "silu", 300, 256, 128, ALL): ([DMA, 64, 1], [DMA, 64, 1], [REGISTERS, 64, 1], 1),
    (F32, "none", 65568, 264, 64, DW): ([REGISTERS, 64, 1], None, [DMA, 64, 52], 0),
    (BF16, "leaky_relu", 4136, 75, 4121, ALL): ([REGISTERS, 128, 1], [REGISTERS, 64, 2], [REGISTERS, 64, 2], 0),
    (F32, "relu", 4136, 4121, 75, ALL): ([REGISTERS, 64, 2], [REGISTERS, 128, 1], [REGISTERS, 64, 2], 0),
    (F16, "relu", 4136, 4121, 75, ALL): ([REGISTERS, 64, 2], [REGISTERS, 128, 1], [REGISTERS, 64, 2], 0),
    (F16, "none", 200, 8192, 200, ALL): ([DMA, 128, 32], [REGISTERS, 64, 1], [REGISTERS, 64, 1], 0),
    (BF16, "relu", 200, 9000, 150, ALL): ([REGISTERS, 128, 29], [REGISTERS, 64, 1], [REGISTERS, 64, 1], 0),
    (F16, "relu", 20001, 136, 150, ALL): ([REGISTERS, 64, 1], [REGISTERS, 64, 1], [REGISTERS, 128, 63], 0),
    (F32, "none", 20001, 136, 150, ALL): ([REGISTERS, 64, 1], [REGISTERS, 64, 1], [REGISTERS, 128, 126], 0),
    (BF16, "silu", 16448, 64, 4104, ALL): ([DMA, 256, 1], [REGISTERS, 64, 1], [DMA, 64, 4], 32),
}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def routes(dt, act, rows, k, n, grads):
    out = (ctypes.c_int * 10)()
    assert _abi.load().s2l_debug_linear_routes(dt, _abi.S2L_ACT[act], 1, grads, rows, k, n, out) == 0
    out = list(out)
    return out[:3], out[3:6] if grads & DX else None, out[6:9] if grads & DW else None, out[9]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_the_cases_reach_what_they_are_there_for(case):
    assert routes(*case) == CASES[case]


def test_every_kernel_has_a_case():
    """By width and direction; fp32 has no 256-wide tiles, dW none either."""
    held = {"forward": set(), "dx": set(), "dW": set()}
    for (dt, act, *_), (y, dx, dw, dz) in CASES.items():
        gated = act.endswith("relu") and not dz
        for name, r in (("forward", y), ("dx", dx), ("dW", dw)):
            if r:
                held[name].add((r[0], r[1], r[2] > 1))
                if r[0] == TOGETHER and name == "dx":
                    held[name].add((dt == F32, r[1], dw[1]))
                if r[0] == REGISTERS and name != "forward":
                    held[name].add((r[1], gated))
    assert {(DMA, 64, False), (DMA, 128, False), (DMA, 256, False), (DMA, 128, True), (REGISTERS, 64, False), (REGISTERS, 128, False), (REGISTERS, 64, True),
            (REGISTERS, 128, True)} <= held["forward"]
    assert {(DMA, 64, False), (DMA, 128, False), (DMA, 256, False), (DMA, 64, True), (DMA, 128, True), (REGISTERS, 64, False), (REGISTERS, 128, False),
            (REGISTERS, 128, True), (64, True), (64, False), (128, True), (128, False)} <= held["dx"]
    assert {(f, a, b) for f in (True, False) for a in (64, 128) for b in (64, 128)} - held["dx"] == {(True, 64, 64)}      # that one: 64 x 64 x 64 in test_gpu_linear
    assert {(DMA, 64, False), (DMA, 64, True), (DMA, 128, False), (DMA, 128, True), (REGISTERS, 64, False), (REGISTERS, 64, True), (REGISTERS, 128, True),
            (TOGETHER, 64, False), (TOGETHER, 64, True), (TOGETHER, 128, False), (TOGETHER, 128, True), (64, True), (64, False), (128, True), (128, False)} <= held["dW"]
    assert {d for *_, d in CASES.values()} >= {0, 1, 2, 4, 16, 32}


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_formula_between_guard_bands(case, dev):
    dt, act, rows, k, n, grads = case
    lib, dtype, code = _abi.load(), TYPES[dt], _abi.S2L_ACT[act]
    print(case, flush=True)
    t, dy = make(rows, k, n, dtype, act, dev)
    want = formula(t, dy, act)
    d = {a: b.detach() for a, b in t.items()}
    size, s = d["x"].element_size(), torch.cuda.current_stream().cuda_stream
    band = lambda *shape: torch.full(shape, 7.0, dtype=dtype, device=dev)  # noqa: E731
    raw = lambda count: torch.full((count + 64,), 85, dtype=torch.uint8, device=dev)  # noqa: E731
    saved = raw(lib.s2l_linear_saved_bytes(dt, code, rows, n))
    work = raw(lib.s2l_linear_forward_work_bytes(dt, code, 1, rows, k, n))
    bwork = raw(lib.s2l_linear_backward_work_bytes(dt, code, rows, k, n))
    ldo = n + 5
    out, dx, dw, db = band(rows + 2, ldo), band(rows + 2, k + 3), band(n + 2, k), band(n + 2)

    def call():
        _abi.check(lib.s2l_linear_forward(dt, d["x"].data_ptr(), k, d["weight"].data_ptr(), k, d["bias"].data_ptr(), d["residual"].data_ptr(), n,
                                          out.data_ptr() + (ldo + 2) * size, ldo, saved.data_ptr(), work.data_ptr(), rows, k, n, code, 0.02, s), "forward")
        _abi.check(lib.s2l_linear_backward(dt, dy.data_ptr(), n, d["x"].data_ptr(), k, d["weight"].data_ptr(), k, saved.data_ptr(),
                                           dx.data_ptr() + (k + 3) * size if grads & DX else 0, k + 3, dw.data_ptr() + k * size if grads & DW else 0,
                                           db.data_ptr() + size if grads & DW else 0, bwork.data_ptr(), rows, k, n, code, 0.02, s), "backward")
        torch.cuda.synchronize()
        return [v.clone() for v in (out, dx, dw, db)]
    first = call()
    got = {"y": out[1:-1, 2:2 + n], **({"dx": dx[1:-1, :k]} if grads & DX else {}), **({"dweight": dw[1:-1], "dbias": db[1:-1]} if grads & DW else {})}
    for name, v in got.items():
        hold(v, want[name], (name, case))
    assert all(torch.equal(a, b) for a, b in zip(first, call()))      # the same bits again
    for v in got.values():
        v.fill_(7)
    assert all(bool((v == 7).all()) for v in (out, dx, dw, db))
    assert all(bool((v[-64:] == 85).all()) for v in (saved, work, bwork))


def test_refusals_need_no_gpu():
    lib, out = _abi.load(), (ctypes.c_int * 10)()
    ask = lambda dt=0, act=1, rows=3, k=8, n=6, to=out: lib.s2l_debug_linear_routes(dt, act, 1, 3, rows, k, n, to)  # noqa: E731
    assert ask() == 0 and ask(dt=3) == -5 and ask(act=5) == -5 and ask(rows=0) == -2 and ask(k=0) == -2 and ask(n=1 << 31) == -2 and ask(to=None) == -1
