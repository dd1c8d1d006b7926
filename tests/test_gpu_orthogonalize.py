"""Newton-Schulz orthogonalisation against the iteration in 64 bits.

Tolerance, derived, in the Frobenius norm.  Values are held to 22 bits and every product adds roundings of at most
e = 2^-21 relative to its terms; taken as independent, a product of X and Y is off by at most e |X|_F |Y|_F.  In one step of
norm r = |X|_F, with |P|_2 <= 1.6: Q is off by (|b| + 2 |c| 1.6) e r^2, times |X|_2 <= 1.3, and a X + Q X itself by e (|a| r +
|Q|_2 r) -- together below D e (r^2 + r) with D = 1.3 (|b| + 3.2 |c|) + |a| + 6.  Later steps multiply an error by at most
J = max |p'| on [0, 1.3], p(s) = a s + b s^3 + c s^5.  The result is rounded once: u |Y|_F.
"""
import ctypes as C

import pytest
import torch

from face_recognition_amd import _lib, projection

pytestmark = pytest.mark.gpu

USUAL = (3.4445, -4.7750, 2.0315)
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def iterate(g, steps, coefficients, dtype=torch.float64):
    """(result, |X|_F before every step) of one matrix on the CPU."""
    x = g.detach().cpu().to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / torch.linalg.matrix_norm(x)
    a, b, c = coefficients
    norms = []
    for _ in range(steps):
        norms.append(torch.linalg.matrix_norm(x).item())
        p = x @ x.t()
        x = a * x + (b * p + c * (p @ p)) @ x
    return (x.t() if tall else x), norms


def allowed(norms, want, coefficients, dt):
    a, b, c = coefficients
    s = torch.linspace(0, 1.3, 200, dtype=torch.float64)
    grow = (a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max().item()
    d = 1.3 * (abs(b) + 3.2 * abs(c)) + abs(a) + 6
    err = 0.0
    for r in norms:
        err = grow * err + d * 2.0 ** -21 * (r * r + r)
    return err + torch.finfo(dt).eps / 2 * torch.linalg.matrix_norm(want).item()


def check(got, g, steps, coefficients):
    assert got.shape == g.shape and got.dtype == g.dtype and got.is_contiguous()
    flat, src = got.reshape(-1, *g.shape[-2:]), g.reshape(-1, *g.shape[-2:])
    for y, one in zip(flat, src):
        want, norms = iterate(one, steps, coefficients)
        err = torch.linalg.matrix_norm(y.cpu().double() - want).item()
        lim = allowed(norms, want, coefficients, g.dtype)
        assert err <= lim, f"error {err:.3g}, {err / lim:.3g} of its bound"


def matrix(shape, dt, device, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen).to(dt).to(device)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 5), (5, 1), (3, 3), (8, 300), (300, 8), (64, 64), (100, 100), (129, 70), (65, 66), (257, 513),
                                   (520, 264), (2, 3, 40, 60), (5, 130, 72), (3, 1, 1)], ids=str)
def test_against_64_bits(device, shape, dt):
    g = matrix(shape, dt, device, sum(shape))
    check(projection.orthogonalize(g), g, 5, USUAL)


@pytest.mark.parametrize("n", [64, 200, 512])
def test_fp32_results_are_as_good_as_fp32_products(device, n):
    """Operands of 22 bits against 24: at most four times the error of the same iteration with every product in fp32, doubled
    for the luck of single roundings."""
    g = matrix((n, n), torch.float32, device, n)
    want, _ = iterate(g, 5, USUAL)
    plain, _ = iterate(g, 5, USUAL, torch.float32)
    mine = torch.linalg.matrix_norm(projection.orthogonalize(g).cpu().double() - want)
    assert mine <= 8 * torch.linalg.matrix_norm(plain.double() - want)


@pytest.mark.parametrize("coefficients,steps", [((1.5, -0.5, 0.0), 40), ((1.875, -1.25, 0.375), 30), (USUAL, 1), ((2.0, -1.5, 0.5), 3)])
def test_other_coefficients(device, coefficients, steps):
    g = matrix((48, 96), torch.float32, device, 5)
    y = projection.orthogonalize(g, steps=steps, coefficients=coefficients)
    check(y, g, steps, coefficients)
    if steps >= 30:                                                  # converged: p' vanishes at one, the last step's error is left
        d = 1.3 * (abs(coefficients[1]) + 3.2 * abs(coefficients[2])) + abs(coefficients[0]) + 6
        gram = (y.double() @ y.double().t()).cpu() - torch.eye(48, dtype=torch.float64)
        assert torch.linalg.matrix_norm(gram) <= 2 * 1.1 * d * 2.0 ** -21 * (48 + 48 ** 0.5)


def test_scale_zeros_and_not_a_number(device):
    g = matrix((40, 56), torch.float32, device, 9)
    base = projection.orthogonalize(g)
    for e in (-100, -40, 60, 120):                                   # squares leave the range of fp32
        assert torch.equal(projection.orthogonalize(g * 2.0 ** e), base)
    zero = torch.zeros(3, 40, 56, device=device)
    assert not projection.orthogonalize(zero).any()
    zero[1] = g
    zero[2, 3, 4] = float("nan")
    y = projection.orthogonalize(zero)
    assert not y[0].any() and torch.equal(y[1], base) and y[2].isnan().any()
    low = torch.outer(g[:, 0], g[0])                                 # rank one: one singular value, the rest stay zero
    check(projection.orthogonalize(low), low, 5, USUAL)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_views(device, dt):
    g = matrix((4, 90, 70), dt, device, 13)
    base = projection.orthogonalize(g)
    wide = torch.full((4, 95, 83), float("nan"), dtype=dt, device=device)
    wide[:, 2:92, 5:75] = g
    assert torch.equal(projection.orthogonalize(wide[:, 2:92, 5:75]), base)
    assert torch.equal(projection.orthogonalize(g.transpose(1, 2).contiguous().transpose(1, 2)), base)
    assert torch.equal(projection.orthogonalize(g[2].expand(3, 90, 70)), base[2].expand(3, 90, 70))
    for i in range(4):
        assert torch.equal(projection.orthogonalize(g[i]), base[i])
    assert projection.orthogonalize(g[:0]).shape == (0, 90, 70)


def test_captured_and_replayed(device):
    g = matrix((3, 130, 70), torch.bfloat16, device, 17)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        projection.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = projection.orthogonalize(g)
    for seed in (18, 19, 20):
        g.copy_(matrix((3, 130, 70), torch.bfloat16, device, seed))
        graph.replay()
        got = y.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, projection.orthogonalize(g))


def test_nothing_is_written_beside_the_output(device):
    lib = _lib.load()
    for rows, cols in ((33, 47), (70, 9), (128, 128)):
        g = matrix((rows, cols), torch.float16, device, 21)
        out = torch.full((rows * cols + 128,), 7.0, dtype=torch.float16, device=device)
        need = C.c_size_t()
        _lib.check(lib.fra_orthogonalize_workspace_bytes(1, rows, cols, C.byref(need)), "bytes")
        ws = torch.full((need.value + 256,), 9, dtype=torch.uint8, device=device)
        _lib.check(lib.fra_orthogonalize(_lib.FRA_F16, g.data_ptr(), cols, 0, 1, rows, cols, 5, *USUAL, out.data_ptr() + 128, ws.data_ptr(),
                                         need.value, _lib.current_stream_ptr(device)), "fra_orthogonalize")
        assert torch.equal(out[64:-64].view(rows, cols), projection.orthogonalize(g))
        assert (out[:64] == 7).all() and (out[-64:] == 7).all() and (ws[need.value:] == 9).all()


def test_a_training_step_of_grouped_projections(device):
    """The operators together: rows sorted by source, one projection each, a head over all of them, gradients, and the
    projections' updates made orthogonal -- against the same step in 64 bits."""
    m, d, groups = 600, 64, 3
    gen = torch.Generator().manual_seed(3)
    x = torch.nn.functional.normalize(torch.randn(m, d, generator=gen)).to(device)
    ids = torch.randint(-1, groups, (m,), generator=gen).to(device)
    w = (0.1 * torch.randn(groups, d, d, generator=gen)).to(device).requires_grad_(True)
    head = torch.randn(40, d, generator=gen).to(device).requires_grad_(True)
    target = torch.randn(m, 40, generator=gen).to(device)
    rg = projection.group_rows(ids, groups)
    y = projection.linear(projection.grouped_linear(x, w, rg, activation="silu", residual=x), head)
    dw, dh = torch.autograd.grad(((y - target) ** 2).mean(), [w, head])
    step = projection.orthogonalize(dw)

    x64, w64, h64 = x.cpu().double(), w.detach().cpu().double().requires_grad_(True), head.detach().cpu().double().requires_grad_(True)
    mid = [x64[i] + (torch.nn.functional.silu(w64[g] @ x64[i]) if g >= 0 else 0) for i, g in enumerate(ids.tolist())]
    y64 = torch.stack(mid) @ h64.t()
    dw64, dh64 = torch.autograd.grad(((y64 - target.cpu().double()) ** 2).mean(), [w64, h64])
    # fp32 chains of at most 600 terms: 2^-24 (600 + ...) of the terms' magnitudes, which are below 8 times the results' norms
    for got, want in ((y, y64), (dw, dw64), (dh, dh64)):
        assert (got.detach().cpu().double() - want.detach()).norm() <= 8 * 700 * 2.0 ** -24 * want.norm()
    check(step, dw, 5, USUAL)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 4090, 4100), (60, 500, 505), (60, 505, 500), (9, 1050, 1010)], ids=str)
def test_large_batches(device, shape, dt):
    """Enough tiles for the products' widest kinds (256 x 256, forward and turned, and 128 x 128), none of the sides a multiple of a tile, both ways
    round.  One step, in 64 bits on the device: the bound of the first step."""
    g = matrix(shape, dt, device, 3)
    a, b, c = USUAL
    y = projection.orthogonalize(g, steps=1)
    for i in (0, shape[0] - 1):
        x = g[i].double()
        x = x / torch.linalg.matrix_norm(x)
        tall = x.shape[0] > x.shape[1]
        x = x.mT if tall else x
        p = x @ x.mT
        want = a * x + (b * p + c * (p @ p)) @ x
        want = want.mT if tall else want
        err = torch.linalg.matrix_norm(y[i].double() - want).item()
        assert err <= allowed([1.0], want, USUAL, dt)
        assert (y[i].double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()       # no value out of place


@pytest.mark.parametrize("shape", [(4, 700, 700), (24, 510, 512), (3, 900, 910), (1, 1500, 1530)], ids=str)
def test_products_by_the_lower_triangle_in_small_tiles(device, shape):
    test_products_by_the_lower_triangle(device, shape)


# X X^T and P P by the lower triangle: whole tiles with quarters of others behind them (some past the last row), whole tiles only,
# several rounds; every matrix of the batch
@pytest.mark.parametrize("shape", [(8, 1024, 1024), (20, 520, 600), (20, 600, 520), (9, 1000, 1100), (60, 321, 330), (2, 2048, 2100), (3, 1930, 1930)], ids=str)
def test_products_by_the_lower_triangle(device, shape):
    g = matrix(shape, torch.float32, device, 4)
    a, b, c = USUAL
    y = projection.orthogonalize(g, steps=1)
    for i in range(shape[0]):
        x = g[i].double()
        x = x / torch.linalg.matrix_norm(x)
        tall = x.shape[0] > x.shape[1]
        x = x.mT if tall else x
        p = x @ x.mT
        want = a * x + (b * p + c * (p @ p)) @ x
        want = want.mT if tall else want
        assert torch.linalg.matrix_norm(y[i].double() - want).item() <= allowed([1.0], want, USUAL, torch.float32)
        assert (y[i].double() - want).abs().max() <= 2.0 ** -12 * want.abs().max()      # no value out of place


def test_a_derivative_is_refused_not_lost(device):
    w = matrix((24, 40), torch.float32, device, 23).requires_grad_(True)
    want = projection.orthogonalize(w.detach())
    assert not want.requires_grad
    y = projection.orthogonalize(w)
    assert torch.equal(y, want)
    with pytest.raises(RuntimeError, match="not differentiable"):
        (y.sum() + w.sum()).backward()                               # w's own path alone would be a wrong gradient
    assert w.grad is None
    with torch.no_grad():
        assert torch.equal(projection.orthogonalize(w), want) and not projection.orthogonalize(w).requires_grad
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w.detach(), torch.ones_like(w))
        with pytest.raises(NotImplementedError, match="jvp"):
            projection.orthogonalize(dual)
        assert torch.equal(projection.orthogonalize(w.detach()), want)      # no tangent, nothing to lose
    with torch.inference_mode():
        assert torch.equal(projection.orthogonalize(w), want)
