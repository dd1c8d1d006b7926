"""The products behind the embeddings on the kinds of tiles, and at the sizes, that the other tests do not reach."""
import pytest
import torch

from face_recognition_amd import projection
from test_gpu_orthogonalize import USUAL, allowed, matrix
from test_gpu_projection import TYPES, call, check, make, reference, run

pytestmark = pytest.mark.gpu


# narrow heads over many rows: dW's tiles mostly empty and cut into many shares, thousands of partial sums for bias and slope
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n,act", [(20001, 512, 40, "prelu"), (100001, 24, 40, "prelu"), (33000, 136, 130, "silu"), (12000, 1030, 7, None)])
def test_narrow_heads_over_many_rows(device, m, k, n, act, dt):
    t = make(m, k, n, dt, device, m + n, act=act, residual=False)
    check(run(t, act), reference(t, act))


@pytest.mark.parametrize("dt", TYPES[1:], ids=str)
@pytest.mark.parametrize("k,shift", [(135, 0), (136, 1)])
def test_largest_tiles_of_unaligned_operands(device, k, shift, dt):
    """512 tiles of 256 x 256 whose operands have no aligned rows (an odd K; a start one element behind an aligned one)."""
    m, n = 131000, 250
    t = make(m, k, n, dt, device, 96 + shift, act="silu")
    if shift:
        buf = torch.full((m * k + 1,), float("nan"), dtype=dt, device=device)
        buf[1:] = t["x"].view(-1)
        t["x"] = buf[1:].view(m, k)
    y = call(t, "silu")
    for rows in (slice(0, 300), slice(65000, 65300), slice(m - 300, m)):
        check({"y": y[rows]}, reference({name: v[rows] if name in ("x", "r", "dy") else v for name, v in t.items()}, "silu"))
    for rows in (slice(300, 500), slice(m - 65, m)):                  # and the bits of smaller tiles
        assert torch.equal(call(dict(t, x=t["x"][rows], r=t["r"][rows]), "silu"), y[rows])


# the product Q X of a step that is not the last, on tiles of 64, 128 and 256, wide and tall; batches of many small matrices
@pytest.mark.parametrize("steps", [2, 5])
@pytest.mark.parametrize("shape", [(4, 700, 720), (4, 720, 700), (9, 1010, 1050), (9, 1050, 1010), (60, 500, 505), (60, 505, 500), (8, 1024, 2048),
                                   (256, 64, 64), (250, 90, 100), (250, 100, 90)], ids=str)
def test_steps_on_every_kind_of_tile(device, shape, steps):
    """In 64 bits on the device, the bound of all steps.  A misplaced piece of eight values shows after two: they are about
    2^-6 each there, the bound is about 2^-11."""
    g = matrix(shape, torch.float32, device, 6)
    a, b, c = USUAL
    y = projection.orthogonalize(g, steps=steps)
    for i in range(shape[0]):
        x = g[i].double()
        tall = x.shape[0] > x.shape[1]
        x = (x.mT if tall else x) / torch.linalg.matrix_norm(x)
        norms = []
        for _ in range(steps):
            norms.append(torch.linalg.matrix_norm(x).item())
            p = x @ x.mT
            x = a * x + (b * p + c * (p @ p)) @ x
        want = x.mT if tall else x
        err, lim = torch.linalg.matrix_norm(y[i].double() - want).item(), allowed(norms, want, USUAL, torch.float32)
        assert err <= lim, f"matrix {i}: error {err:.3g}, {err / lim:.3g} of its bound"
