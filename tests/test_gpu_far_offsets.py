"""The dense layer and the orthogonalisation where an element's offset passes 32 bits, and row strides on both sides of what the LDS-DMA path takes."""
import pytest
import torch

from speech2lip_amd import autograd, optim
from tests.test_gpu_linear import formula, hold, make


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    yield torch.device("cuda:0")
    torch.cuda.empty_cache()


ROWS, STEP = 2200000, 100000


@pytest.mark.gpu
@pytest.mark.parametrize("act,k,n", (("relu", 1024, 24), ("relu", 24, 1024), ("none", 1000, 17)))
def test_more_than_two_to_the_31_elements(act, k, n, dev):
    """2.2e9 elements of x, or of y and dy.  Whole numbers from -1 to 1: every sum is below 2^24 and exact, so that each result is the whole number, rounded."""
    gen = torch.Generator(device=dev).manual_seed(k)
    whole = lambda *s: torch.randint(-1, 2, s, generator=gen, device=dev, dtype=torch.int8).bfloat16()  # noqa: E731
    leaves = [whole(ROWS, k).requires_grad_(), whole(n, k).requires_grad_(), whole(n).requires_grad_()]
    dy = whole(ROWS, n)
    y = autograd.linear(*leaves, activation=act)
    gx, gw, gb = torch.autograd.grad(y, leaves, dy)
    x, w, b = (v.detach() for v in leaves)
    w, b, sum_w, sum_b = w.double(), b.double(), 0, 0
    for at in range(0, ROWS, STEP):
        xs, dys = x[at:at + STEP].double(), dy[at:at + STEP].double()
        z = xs @ w.t() + b
        dz = dys * (z > 0) if act == "relu" else dys
        assert torch.equal(y.detach()[at:at + STEP], (z.clamp(min=0) if act == "relu" else z).bfloat16()), at
        assert torch.equal(gx[at:at + STEP], (dz @ w).bfloat16()), at
        sum_w, sum_b = sum_w + dz.t() @ xs, sum_b + dz.sum(0)
    assert float(sum_w.abs().max()) < 2 ** 24 and torch.equal(gw, sum_w.bfloat16()) and torch.equal(gb, sum_b.bfloat16())


@pytest.mark.gpu
def test_more_than_two_to_the_31_values_kept(dev):
    """z of gelu, dz behind it: y and dx of all rows."""
    t, dy = make(ROWS, 24, 1024, torch.bfloat16, "gelu", dev, residual=False)
    y = autograd.linear(t["x"], t["weight"], t["bias"], activation="gelu")
    (gx,) = torch.autograd.grad(y, t["x"], dy)
    for at in range(0, ROWS, STEP):
        want = formula({**t, "x": t["x"].detach()[at:at + STEP]}, dy[at:at + STEP], "gelu")
        hold(y.detach()[at:at + STEP], want["y"], ("y", at))
        hold(gx[at:at + STEP], want["dx"], ("dx", at))


@pytest.mark.gpu
@pytest.mark.parametrize("ld", ((1 << 22) - 8, 1 << 22))
def test_rows_far_apart(ld, dev):
    """x as rows of a buffer of 35 GB: at the widest stride that 32-bit offsets within a tile of 256 rows hold, and one beyond; W's rows far apart too."""
    rows, k, n = 4160, 192, 4120
    t, dy = make(rows, k, n, torch.bfloat16, "silu", dev)
    x = torch.empty(rows, ld, dtype=torch.bfloat16, device=dev)[:, :k]
    x.copy_(t["x"].detach())
    x.requires_grad_()
    want = formula(t, dy, "silu")
    leaves = (x, t["weight"], t["bias"], t["residual"])
    y = autograd.linear(*leaves, "silu")
    for got, name in zip((y.detach(), *torch.autograd.grad(y, leaves, dy)), ("y", "dx", "dweight", "dbias", "dresidual")):
        hold(got, want[name], name)
    del x, leaves, y
    t, dy = make(300, 192, 256, torch.bfloat16, "none", dev)
    w = torch.empty(256, ld, dtype=torch.bfloat16, device=dev)[:, :192]
    w.copy_(t["weight"].detach())
    w.requires_grad_()
    want = formula(t, dy, "none")
    y = autograd.linear(t["x"], w, t["bias"], residual=t["residual"])
    for got, name in zip((y.detach(), *torch.autograd.grad(y, (t["x"], w), dy)), ("y", "dx", "dweight")):
        hold(got, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=str)
def test_a_matrix_of_more_than_two_to_the_31_elements(dtype, dev):
    """One entry of +-1 in each row, each in a column of its own: every singular value is the same, and the result that matrix times what the
    iteration makes of 1 / sqrt(rows).  Each value is a sum of one product and zeros; it passes 15 products of 22 bits (the last two steps of
    bfloat16: 11), whose errors |p'| <= 3.9 of the scalar iteration grows: 2^-18 and 2^-6 are generous, and any misplaced entry is off by 0.7."""
    rows, cols = 16640, 131072
    gen = torch.Generator(device=dev).manual_seed(1)
    middle = 1 + torch.randperm(cols - 2, generator=gen, device=dev)[:rows - 2]
    at = torch.cat((middle.new_tensor([cols - 1]), middle, middle.new_tensor([0])))
    sign = torch.randint(0, 2, (rows,), generator=gen, device=dev) * 2 - 1
    g = torch.zeros(rows, cols, dtype=dtype, device=dev)
    g[torch.arange(rows, device=dev), at] = sign.to(dtype)
    s = rows ** -0.5
    for _ in range(5):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    got = optim.orthogonalize(g)
    got[torch.arange(rows, device=dev), at] -= (s * sign).to(dtype)
    limit = 2.0 ** (-18 if dtype == torch.float32 else -6)
    assert float(got.abs().max()) <= limit, float(got.abs().max())
