"""Products behind the embeddings against the same formulas in 64 bits.

Tolerances, derived.  u = eps / 2 is the half step of one rounding to the type, s = 2^-24 that of fp32.
  z      an fp32 sum of K products (exact for 16-bit types, rounded once for fp32) and a bias, in any order:
         |dz64| <= (K + 4) s (sum_k |x_k w_k| + |b|).
  y      the activation (1.13-Lipschitz at most) in fp32, good to 2^-20 (|z| + 1); then one rounding, u |y|.
  dz     z is kept in the type (u |z|), |act''| <= 1.2, |act'| <= 1.13 evaluated to 2^-20, the product rounded (u |dz|):
         |dy| ((1 + |z|) (2.4 u + 2^-20) + 1.2 (K + 4) s (sum + |b|)); relu and prelu jump at z = 0, so a z within its own error of
         zero may take either side: |dy| more there.  Without activation dz = dy.
  sums   of L terms t with errors e: sum e + (L + 4) s sum |t|, then u |result|.
Half a subnormal step of the type is added wherever a value is rounded to it.
"""
import ctypes as C
import math

import pytest
import torch

from face_recognition_amd import _lib, projection

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
S = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def half_sub(dt):
    return torch.finfo(dt).tiny * torch.finfo(dt).eps / 2


def act64(act, z, s):
    if act == "relu":
        return torch.relu(z)
    if act == "prelu":
        return torch.where(z > 0, z, z * s)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(z, approximate="tanh")
    return z


def make(m, k, n, dt, device, seed, lead=(), act=None, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=g).to(dt).to(device)

    t = {"x": r(m, k), "w": (torch.randn(*lead, n, k, generator=g) / math.sqrt(k)).to(dt).to(device), "dy": r(m, n)}
    t["b"] = r(*lead, n) if bias else None
    t["s"] = (0.25 + 0.1 * torch.randn(*lead, n, generator=g)).to(dt).to(device) if act == "prelu" else None
    t["r"] = r(m, n) if residual else None
    return t


def reference(t, act, ids=None):
    """name -> (value in 64 bits, largest allowed error), on the CPU."""
    dt = t["x"].dtype
    u, sub = half_step(dt), half_sub(dt)
    d = {n: v.detach().cpu().double() if v is not None else None for n, v in t.items()}
    ids = ids.cpu() if ids is not None else None
    m, k = d["x"].shape
    n = d["dy"].shape[1]
    ref = {"y": d["r"].clone() if d["r"] is not None else torch.zeros(m, n, dtype=torch.float64)}
    lim = {"y": u * ref["y"].abs() + sub}
    for name, src in (("dx", "x"), ("dw", "w"), ("db", "b"), ("ds", "s")):
        if d[src] is not None:
            ref[name], lim[name] = torch.zeros_like(d[src]), torch.zeros_like(d[src])
    for g in range(1 if ids is None else d["w"].shape[0]):
        rows = torch.arange(m) if ids is None else torch.nonzero(ids == g)[:, 0]
        par = (lambda v: v) if ids is None else (lambda v: v[g])
        x, w, dy = d["x"][rows], par(d["w"]), d["dy"][rows]
        s = par(d["s"]) if d["s"] is not None else None
        b = par(d["b"]) if d["b"] is not None else torch.zeros(n, dtype=torch.float64)
        z = (x @ w.t() + b).requires_grad_(True)
        zerr = (k + 4) * S * (x.abs() @ w.abs().t() + b.abs())
        a = act64(act, z, s)
        dz = torch.autograd.grad(a, z, dy)[0] if act else dy
        z, a = z.detach(), a.detach()
        y = a + (d["r"][rows] if d["r"] is not None else 0)
        ref["y"][rows] = y
        lim["y"][rows] = u * y.abs() + 1.13 * zerr + (2.0 ** -20 * (z.abs() + 1) if act else 2 * S * (z.abs() + y.abs())) + sub
        dzerr = torch.zeros_like(dz)
        if act:
            dzerr = dy.abs() * ((1 + z.abs()) * (2.4 * u + 2.0 ** -20) + 1.2 * zerr + sub) + sub
            if act in ("relu", "prelu"):
                dzerr += dy.abs() * 1.3 * (z.abs() <= zerr + sub)

        def put(name, v, err):
            at = slice(None) if ids is None else g
            ref[name][at], lim[name][at] = v, u * v.abs() + err + sub

        ref["dx"][rows] = dz @ w
        lim["dx"][rows] = u * (dz @ w).abs() + dzerr @ w.abs() + (n + 4) * S * (dz.abs() @ w.abs()) + sub
        rm = len(rows)
        put("dw", dz.t() @ x, dzerr.t() @ x.abs() + (rm + 4) * S * (dz.abs().t() @ x.abs()))
        if d["b"] is not None:
            put("db", dz.sum(0), dzerr.sum(0) + (rm + 4) * S * dz.abs().sum(0))
        if s is not None:
            neg = dy * torch.clamp(z, max=0)
            put("ds", neg.sum(0), (dy.abs() * (u * z.abs() + zerr + sub)).sum(0) + (rm + 4) * S * neg.abs().sum(0))
    return {name: (ref[name], lim[name]) for name in ref}


def check(out, ref):
    for name, v in out.items():
        want, lim = ref[name]
        assert v.shape == want.shape, name
        err = (v.detach().cpu().double() - want).abs()
        if err.numel():
            assert (err <= lim).all(), f"{name}: error {err.max():.3g}, {(err / lim).max():.3g} of its bound"


def call(t, act, groups=None, **over):
    kw = dict(bias=t["b"], activation=act, slope=t["s"], residual=t["r"])
    kw.update(over)
    if groups is None:
        return projection.linear(t["x"], t["w"], **kw)
    return projection.grouped_linear(t["x"], t["w"], groups, **kw)


def run(t, act, groups=None):
    leaves = {n: t[n].detach().clone().requires_grad_(True) for n in ("x", "w", "b", "s", "r") if t[n] is not None}
    y = call(dict(t, **leaves), act, groups)
    out = {"y": y}
    for name, v in zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["dy"])):
        if name == "r":
            assert torch.equal(v, t["dy"])
        else:
            out["d" + name] = v
    return out


# one value; below one tile; a few rows; odd on every side; just past tile and step borders; long contraction; many tiles
SHAPES = [(1, 1, 1, None), (1, 512, 512, "prelu"), (3, 7, 5, "silu"), (16, 64, 40, "relu"), (17, 72, 41, "gelu_tanh"),
          (50, 512, 333, "relu"), (64, 128, 64, None), (65, 129, 66, "prelu"), (129, 65, 257, "silu"), (2, 4099, 3, None),
          (200, 500, 301, "prelu"), (1000, 96, 136, "gelu_tanh"), (2100, 520, 1032, "silu"), (5000, 33, 2, "relu")]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n,act", SHAPES)
def test_linear_and_gradients(device, m, k, n, act, dt):
    t = make(m, k, n, dt, device, 1000 * m + k, act=act, bias=m % 2 == 1 or n % 2 == 1, residual=m % 3 != 0)
    check(run(t, act), reference(t, act))


GROUPED = [(1, 8, 8, 1, None), (9, 512, 512, 12, None), (64, 64, 64, 3, "relu"), (130, 40, 72, 2, "prelu"), (700, 129, 67, 7, "silu"),
           (3000, 64, 130, 5, "gelu_tanh"), (4100, 96, 40, 33, "prelu"), (30, 16, 9, 300, "silu")]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n,groups,act", GROUPED)
def test_grouped_linear_and_gradients(device, m, k, n, groups, act, dt):
    g = torch.Generator().manual_seed(m + groups)
    # skewed shares, some groups empty, some rows of no group on either side of the range
    ids = (torch.rand(m, generator=g) ** 2 * (groups + 1)).long() - (torch.rand(m, generator=g) < 0.1).long() * (groups + 2)
    t = make(m, k, n, dt, device, 7 * m + k, lead=(groups,), act=act, bias=m % 2 == 0, residual=m % 4 != 0)
    rg = projection.group_rows(ids.to(device), groups)
    check(run(t, act, rg), reference(t, act, torch.where((ids >= 0) & (ids < groups), ids, torch.full_like(ids, -1))))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shares", [(0, 5000, 0, 300, 129, 128, 1, 2000), (3000,), (0, 0, 6000), (257, 255, 256, 1024, 1)], ids=str)
def test_groups_of_very_different_sizes(device, shares, dt):
    """A group's rows come in pieces whose sums are joined; groups of one piece or none are written at once."""
    k, n, groups = 72, 40, len(shares)
    ids = torch.repeat_interleave(torch.arange(groups), torch.tensor(shares))
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(1))]
    t = make(len(ids), k, n, dt, device, 17, lead=(groups,), act="silu")
    check(run(t, "silu", projection.group_rows(ids.to(device), groups)), reference(t, "silu", ids))


# the gradients' products on tiles of one side in one launch (with as many shares as fill a round, and without), of different sides
# apart, dx on the largest tiles and on the smallest
@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n,act", [(4096, 1024, 600, "gelu_tanh"), (4100, 1020, 130, None), (2000, 1024, 520, "silu"), (1000, 100, 5000, "relu"),
                                       (16384, 2048, 24, None)])
def test_gradients_of_many_tiles(device, m, k, n, act, dt):
    t = make(m, k, n, dt, device, k + n, act=act, residual=False)
    check(run(t, act), reference(t, act))


# 38401 rows in 300 equal pieces of 129 leave the last two empty; 192 rows are one piece, 193 two
@pytest.mark.parametrize("shares", [(38401, 11599), (192, 193, 191, 1, 500)], ids=str)
def test_pieces_of_a_group(device, shares):
    ids = torch.repeat_interleave(torch.arange(len(shares)), torch.tensor(shares))
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(2))]
    t = make(len(ids), 24, 16, torch.float16, device, 18, lead=(len(shares),))
    check(run(t, None, projection.group_rows(ids.to(device), len(shares))), reference(t, None, ids))


@pytest.mark.parametrize("kind", ["all_one", "none", "last_only"])
def test_grouped_extremes(device, kind):
    m, k, n, groups = 333, 48, 56, 6
    ids = {"all_one": torch.full((m,), 2), "none": torch.full((m,), -5), "last_only": torch.full((m,), groups - 1)}[kind]
    t = make(m, k, n, torch.bfloat16, device, 5, lead=(groups,), act="silu", residual=kind != "last_only")
    out = run(t, "silu", projection.group_rows(ids.to(device).int(), groups))
    check(out, reference(t, "silu", ids))
    for g in range(groups):
        if not (ids == g).any():
            assert not out["dw"][g].any() and not out["db"][g].any()
    if kind == "none":
        assert torch.equal(out["y"].detach(), t["r"]) and not out["dx"].any()


@pytest.mark.parametrize("m", [0, 1, 63, 64, 65, 1000, 1025, 4095, 4096, 4097, 8192, 8193, 20000, 300001])
@pytest.mark.parametrize("groups", [1, 2, 37, 4096])
@pytest.mark.parametrize("it", [torch.int32, torch.int64], ids=str)
def test_group_rows_is_a_stable_sort(device, m, groups, it):
    g = torch.Generator().manual_seed(m + groups)
    ids = torch.randint(-1, groups + 1, (m,), generator=g).to(it)
    if it == torch.int64 and m > 2:
        ids[0], ids[1] = 2 ** 40, -2 ** 40          # no 32-bit truncation: 2^40 & 0xffffffff = 0 is a valid group
    rg = projection.group_rows(ids.to(device), groups)
    key = torch.where((ids >= 0) & (ids < groups), ids.long(), torch.full((m,), groups))
    assert torch.equal(rg.order.cpu().long(), torch.argsort(key, stable=True))
    want = torch.zeros(groups + 1, dtype=torch.long)
    want[1:] = torch.bincount(key, minlength=groups + 1)[:groups].cumsum(0)
    assert torch.equal(rg.offsets.cpu().long(), want)
    assert rg.order.dtype == rg.offsets.dtype == torch.int32


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_no_rows(device, dt):
    t = make(0, 24, 40, dt, device, 3, act="prelu")
    out = run(t, "prelu")
    assert out["y"].shape == (0, 40) and out["dx"].shape == (0, 24)
    assert not out["dw"].any() and not out["db"].any() and not out["ds"].any()
    t = make(0, 24, 40, dt, device, 3, lead=(3,), act="prelu")
    out = run(t, "prelu", projection.group_rows(torch.empty(0, dtype=torch.int64, device=device), 3))
    assert out["y"].shape == (0, 40) and out["dw"].shape == (3, 40, 24)
    assert not out["dw"].any() and not out["db"].any() and not out["ds"].any()


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_strides_and_alignment(device, dt):
    """Views instead of contiguous tensors give the very bits of their contiguous copies, and memory between the rows (NaN
    here) never enters a result."""
    m, k, n = 150, 88, 96
    for act, grouped in (("silu", False), ("prelu", True)):
        lead = (4,) if grouped else ()
        t = make(m, k, n, dt, device, 11, lead=lead, act=act)
        rg = projection.group_rows(torch.arange(m, device=device) % 5, 4) if grouped else None
        base = run(t, act, rg)
        for shift in (0, 1, 3):
            def wide(v, pad):
                buf = torch.full((*v.shape[:-1], v.shape[-1] + pad), float("nan"), dtype=dt, device=device)
                buf[..., shift:shift + v.shape[-1]] = v
                return buf[..., shift:shift + v.shape[-1]]
            views = {name: wide(t[name], 8) for name in ("x", "w", "dy", "r")}
            leaves = {name: v.detach().requires_grad_(True) for name, v in views.items() if name != "dy"}
            leaves["b"], leaves["s"] = (v.detach().clone().requires_grad_(True) if v is not None else None for v in (t["b"], t["s"]))
            y = call(dict(t, **leaves), act, rg)
            assert torch.equal(y, base["y"])
            names = [name for name, v in leaves.items() if v is not None and name != "r"]
            for name, v in zip(names, torch.autograd.grad(y, [leaves[x] for x in names], views["dy"])):
                assert torch.equal(v, base["d" + name]), name
    # transposed operands, a transposed and an expanded gradient, more leading axes
    t = make(m, k, n, dt, device, 12)
    base = run(t, "silu")
    assert torch.equal(call(dict(t, x=t["x"].t().contiguous().t(), w=t["w"].t().contiguous().t()), "silu"), base["y"])
    x3 = t["x"].reshape(5, 30, k).clone().requires_grad_(True)
    y = projection.linear(x3, t["w"], t["b"], "silu", residual=t["r"].reshape(5, 30, n))
    assert torch.equal(y.reshape(m, n), base["y"])
    assert torch.equal(torch.autograd.grad(y, x3, t["dy"].t().contiguous().t().reshape(5, 30, n))[0].reshape(m, k), base["dx"])
    x = t["x"].clone().requires_grad_(True)
    ones = torch.autograd.grad(projection.linear(x, t["w"], t["b"], "silu"), x, torch.ones(m, n, dtype=dt, device=device))[0]
    assert torch.equal(torch.autograd.grad(projection.linear(x, t["w"], t["b"], "silu").sum(), x)[0], ones)
    v = t["x"][0].clone()
    assert projection.linear(v, t["w"], t["b"]).shape == (n,)
    # a row repeated by expand, a matrix shared by groups through expand: its gradient is the sum over them
    assert torch.equal(projection.linear(v.expand(7, k), t["w"]), projection.linear(v.repeat(7, 1), t["w"]))
    w = t["w"].clone().requires_grad_(True)
    rg = projection.group_rows(torch.arange(m, device=device) % 3, 3)
    y = projection.grouped_linear(t["x"], w.expand(3, n, k), rg)
    assert torch.equal(y, projection.linear(t["x"], t["w"]))
    dw, = torch.autograd.grad(y, w, t["dy"])
    each = run(dict(t, w=t["w"].repeat(3, 1, 1), b=None, r=None), None, rg)["dw"]
    assert torch.equal(dw, each.sum(0))


@pytest.mark.parametrize("m,k,n", [(5, 70, 50), (300, 70, 200)])
@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_nan_and_infinity_stay_in_their_rows(device, m, k, n, dt):
    t = make(m, k, n, dt, device, 21, residual=False)
    clean = call(t, "relu")
    x = t["x"].clone()
    x[1, k - 1], x[3, 0] = float("nan"), float("inf")
    y = projection.linear(x, t["w"], t["b"], "relu")
    keep = torch.ones(m, dtype=torch.bool, device=device)
    keep[1] = keep[3] = False
    assert torch.equal(y[keep], clean[keep])
    assert y[1].isnan().all()                                        # a NaN goes through the activation
    pos = t["w"][:, 0] > 0
    assert (y[3][pos] == float("inf")).all() and (y[3][t["w"][:, 0] < 0] == 0).all()
    # a group whose rows hold a NaN leaves the other groups' gradients alone
    ids = torch.arange(m, device=device) % 2
    w2 = t["w"].repeat(2, 1, 1).requires_grad_(True)
    rg = projection.group_rows(ids, 2)
    good = torch.autograd.grad(projection.grouped_linear(t["x"], w2, rg), w2, t["dy"])[0]
    x = t["x"].clone()
    x[1] = float("nan")
    bad = torch.autograd.grad(projection.grouped_linear(x, w2, rg), w2, t["dy"])[0]
    assert torch.equal(bad[0], good[0]) and bad[1].isnan().all()


@pytest.mark.parametrize("act", [None, "silu", "gelu_tanh", "prelu"])
def test_gradients_against_differences(device, act):
    """L = sum dy y along a direction of x, W and b together, by central differences of fp32 results: with step h the kernel's
    rounding leaves 2 sum |dy| (error of y) / 2h, the third derivative h^2 / 6 sum |dy| |act'''| |dz|^3 and the path's curvature
    (z is quadratic along it) is even in h but for h^2 |act''| |dz| |dz2|.  |act'''| <= 2.5, |act''| <= 1.2."""
    m, k, n, h = 40, 24, 33, 2.0 ** -7
    t = make(m, k, n, torch.float32, device, 31, act=act, residual=False)
    if act == "prelu":                                               # piecewise linear: stay on one side of the kink
        t["x"], t["w"], t["b"] = t["x"].abs(), t["w"].abs(), -t["b"].abs() - 60
    out = run(t, act)
    g = torch.Generator().manual_seed(2)
    d = {name: torch.randn(t[name].shape, generator=g).to(device) for name in ("x", "w", "b")}
    want = sum((out["d" + name].double() * d[name].double()).sum().item() for name in d)
    value, err = [], []
    for sign in (1, -1):
        moved = dict(t, **{name: t[name] + sign * h * d[name] for name in d})
        value.append((call(moved, act).double() * t["dy"].double()).sum().item())
        zm = moved["x"].double().abs() @ moved["w"].double().abs().t() + moved["b"].double().abs()
        err.append((t["dy"].double().abs() * ((k + 8) * S * zm * 1.13 + 2.0 ** -20 * (zm + 1))).sum().item())
    x, w = t["x"].double(), t["w"].double()
    dz = d["x"].double() @ w.t() + x @ d["w"].double().t() + d["b"].double()
    dz2 = d["x"].double() @ d["w"].double().t()
    curve = 0.0
    if act in ("silu", "gelu_tanh"):
        curve = h * h * (t["dy"].double().abs() * (2.5 / 6 * dz.abs() ** 3 + 1.2 * dz.abs() * dz2.abs())).sum().item()
    # the fp32 gradients and the moved inputs are rounded as well: far below 2^-16 of the terms
    grad_err = 2.0 ** -16 * sum((out["d" + name].double().abs() * d[name].double().abs()).sum().item() for name in d)
    got = (value[0] - value[1]) / (2 * h)
    assert abs(got - want) <= sum(err) / (2 * h) + curve + grad_err


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_a_row_does_not_depend_on_the_rows_beside_it(device, dt):
    """Beyond the kernel for few rows a value is the same sum in the same order whatever tiles the batch's size asks for: the rows
    of a large ragged batch (512 tiles of 256 rows) equal those of its parts, forward and back."""
    m, k, n = 130900, 136, 250
    t = make(m, k, n, dt, device, 91, act="silu")

    def y_dx(rows):
        x = t["x"][rows].clone().requires_grad_(True)
        y = projection.linear(x, t["w"], t["b"], "silu", residual=t["r"][rows])
        return y.detach(), torch.autograd.grad(y, x, t["dy"][rows])[0]

    y, dx = y_dx(slice(None))
    for rows in (slice(0, 100), slice(50000, 57000), slice(m - 65, m)):
        part_y, part_dx = y_dx(rows)
        assert torch.equal(part_y, y[rows]) and torch.equal(part_dx, dx[rows])
    rows = slice(m - 300, m)
    check({"y": y[rows], "dx": dx[rows]}, reference({name: v[rows] if name in ("x", "r", "dy") else v for name, v in t.items()}, "silu"))


def test_repeated_runs_are_the_same_bits(device):
    t = make(3000, 130, 200, torch.bfloat16, device, 41, lead=(7,), act="prelu")
    rg = projection.group_rows(torch.arange(3000, device=device) * 7919 % 8, 7)
    first = run(t, "prelu", rg)
    for _ in range(3):
        for name, v in run(t, "prelu", rg).items():
            assert torch.equal(v, first[name]), name


def test_parameters_in_fp32_and_partial_gradients(device):
    t = make(77, 64, 48, torch.float16, device, 51, act="prelu")
    b, s = t["b"].float().requires_grad_(True), t["s"].float().requires_grad_(True)
    y = projection.linear(t["x"], t["w"], b, "prelu", s, t["r"])
    assert torch.equal(y, call(t, "prelu"))
    db, ds = torch.autograd.grad(y, [b, s], t["dy"])
    full = run(t, "prelu")
    assert db.dtype == ds.dtype == torch.float32
    assert torch.equal(db.half(), full["db"]) and torch.equal(ds.half(), full["ds"])
    for name in ("x", "w", "r"):
        leaf = t[name].clone().requires_grad_(True)
        d, = torch.autograd.grad(call(dict(t, **{name: leaf}), "prelu"), leaf, t["dy"])
        assert torch.equal(d, t["dy"] if name == "r" else full["d" + name])
    with torch.no_grad():
        assert not call(t, "prelu").requires_grad


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_far_outside_the_activation_bends(device, act, dt):
    # one product per value: z = 300 x is far below or above, in f16 past the type's range (where what is kept of z is an infinity)
    far = torch.tensor([1e3, 60000.0] if dt == torch.float16 else [1e3, 1e17, 1e25], dtype=dt)
    x = torch.cat([-far, far, torch.tensor([float("nan")], dtype=dt)])[:, None].to(device).requires_grad_(True)
    w = torch.full((1, 1), 300.0, dtype=dt, device=device)
    y = projection.linear(x, w, activation=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    k = len(far)
    assert torch.equal(y[:k], torch.zeros_like(y[:k])) and torch.equal(dx[:k], torch.zeros_like(y[:k]))
    assert torch.equal(y[k:2 * k], (300.0 * x[k:2 * k].float()).to(dt)) and torch.equal(dx[k:2 * k], torch.full_like(y[:k], 300.0))
    assert y[2 * k].isnan() and dx[2 * k].isnan()


def test_once_differentiable_and_saved_tensor_hooks(device):
    t = make(50, 24, 40, torch.float32, device, 55, act="prelu")
    full = run(t, "prelu")
    x = t["x"].clone().requires_grad_(True)
    dx, = torch.autograd.grad(call(dict(t, x=x), "prelu").pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()
    # what was saved comes back from elsewhere, and laid out differently
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), lambda v: v.to(device).t().contiguous().t() if v.dim() == 2 else v.to(device)):
        out = run(t, "prelu")
    for name, v in full.items():
        assert torch.equal(out[name], v), name
    # an input changed between the passes is noticed
    w = t["w"].clone().requires_grad_(True)
    y = call(dict(t, w=w), "prelu")
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, w, t["dy"])


def test_forward_mode_is_refused(device):
    t = make(5, 8, 6, torch.float32, device, 57)
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(t["x"], torch.ones_like(t["x"]))
        with pytest.raises(NotImplementedError, match="jvp"):
            call(dict(t, x=x), None)
        assert torch.equal(call(t, None), call(t, None))            # no tangent, nothing to lose


def test_saved_tensors_back_at_their_address_in_another_layout(device):
    # an allocator may hand the address of a freed view out again, to the packed copy that a hook brings back
    m, k, n = 48, 40, 56
    t = make(m, k, n, torch.float16, device, 56, bias=False, residual=False)
    memory = torch.zeros(m, 2 * k, dtype=torch.float16, device=device)
    x = memory[:, :k].copy_(t["x"])
    want = run(t, None)["dw"]

    def unpack(v):
        if v.shape != (m, k):
            return v.to(device)
        return memory.view(-1)[:m * k].view(m, k).copy_(v)

    w = t["w"].clone().requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), unpack):
        y = projection.linear(x, w)
    assert torch.equal(torch.autograd.grad(y, w, t["dy"])[0], want)


def test_captured_and_replayed(device):
    m, k, n, groups = 500, 136, 72, 5
    t = make(m, k, n, torch.bfloat16, device, 61, lead=(groups,), act="prelu")
    ids = torch.arange(m, device=device) * 31 % (groups + 1)
    static = {name: v.clone() for name, v in t.items()}
    leaves = {name: static[name].requires_grad_(True) for name in ("x", "w", "b", "s")}

    def step():
        rg = projection.group_rows(ids, groups)
        y = projection.grouped_linear(leaves["x"], leaves["w"], rg, leaves["b"], "prelu", leaves["s"], static["r"])
        z = projection.linear(y.detach(), leaves["w"][0, :, :n].detach())
        return [rg.order, y.detach(), z, *torch.autograd.grad(y, list(leaves.values()), static["dy"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (62, 63, 64):
        fresh = make(m, k, n, torch.bfloat16, device, seed, lead=(groups,), act="prelu")
        with torch.no_grad():
            for name, v in fresh.items():
                static[name].copy_(v)
            ids.copy_((ids + seed) % (groups + 2))
        graph.replay()
        got = [v.clone() for v in captured]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_on_another_stream(device):
    t = make(400, 256, 128, torch.float16, device, 71, act="silu")
    base = run(t, "silu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = run(t, "silu")
    side.synchronize()
    for name, v in out.items():
        assert torch.equal(v, base[name]), name


def test_nothing_is_written_beside_the_outputs(device):
    """The C entry with outputs inside larger buffers: the values around them stay."""
    lib = _lib.load()
    for m, k, n in ((1, 40, 33), (70, 40, 33), (130, 136, 257)):
        t = make(m, k, n, torch.float16, device, 81, bias=False, residual=False)
        def framed(count):
            return torch.full((count + 128,), 7.0, dtype=torch.float16, device=device)
        y, dx, dw = framed(m * n), framed(m * k), framed(n * k)
        d = _lib.LinearDesc(_lib.FRA_F16, 0, 0, 0, m, k, n, t["x"].data_ptr(), t["w"].data_ptr(), None, None, None, k, k, 0, 0, None)
        stream = _lib.current_stream_ptr(device)
        _lib.check(lib.fra_linear(C.byref(d), None, y.data_ptr() + 128, stream), "fra_linear")
        need = C.c_size_t()
        _lib.check(lib.fra_linear_backward_workspace_bytes(C.byref(d), 1, 1, 0, 0, C.byref(need)), "bytes")
        ws = torch.full((need.value + 256,), 9, dtype=torch.uint8, device=device)
        _lib.check(lib.fra_linear_backward(C.byref(d), None, t["dy"].data_ptr(), n, dx.data_ptr() + 128, dw.data_ptr() + 128, None, None,
                                           ws.data_ptr(), need.value, stream), "fra_linear_backward")
        ref = reference(t, None)
        check({"y": y[64:-64].view(m, n), "dx": dx[64:-64].view(m, k), "dw": dw[64:-64].view(n, k)}, ref)
        for v in (y, dx, dw):
            assert (v[:64] == 7).all() and (v[-64:] == 7).all()
        assert (ws[need.value:] == 9).all()


@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_rows_behind_two_to_the_31_elements(device, act):
    # the last rows, and the group that only they belong to, lie behind 2^31 elements (2^32 bytes) of every operand
    n_last, k, n = 300, 512, 520
    m = 2 ** 31 // k + 5000
    t = make(n_last, k, n, torch.bfloat16, device, 81, lead=(2,), act=act)
    ids = torch.zeros(m, dtype=torch.int32, device=device)
    ids[-n_last:] = 1
    rg = projection.group_rows(ids, 2)
    big = {}
    for name, c in (("x", k), ("r", n), ("dy", n)):
        big[name] = torch.zeros(m, c, dtype=torch.bfloat16, device=device)
        big[name][-n_last:] = t[name]
    out = run(dict(t, **big), act, rg)
    want = reference(t, act, torch.ones(n_last, dtype=torch.int32))
    got = {name: v[-n_last:] if name in ("y", "dx") else v for name, v in out.items()}
    check({name: v if name in ("y", "dx") else v[1] for name, v in got.items()},
          {name: want[name] if name in ("y", "dx") else tuple(p[1] for p in want[name]) for name in want})
    assert not out["dx"][:1000].any() and not out["dw"][0].any()
    # the same without groups: rows beyond the border, and gradients summed over all of them
    one = dict(t, w=t["w"][1], b=t["b"][1])
    plain = run(dict(one, **big), act)
    check({"y": plain["y"][-n_last:], "dx": plain["dx"][-n_last:], "dw": plain["dw"]}, reference(one, act))


@pytest.mark.parametrize("m,k,n", [(40, 24, 33), (300, 64, 72)])
@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_relu_holds_back_any_gradient(device, m, k, n, dt):
    """Where relu's input is below zero its gradient is zero, whatever the output's is: infinities and NaN there change no bit."""
    for groups in (0, 3):
        lead = (groups,) if groups else ()
        t = make(m, k, n, dt, device, 95 + groups, lead=lead, act="relu", residual=False)
        rg = projection.group_rows(torch.arange(m, device=device) % groups, groups) if groups else None
        base = run(t, "relu", rg)
        off = base["y"].detach() == 0
        spoil = torch.tensor([float("inf"), float("-inf"), float("nan")], dtype=dt, device=device)
        dy = torch.where(off, spoil[torch.arange(m * n, device=device).view(m, n) % 3], t["dy"])
        assert off.any() and not dy.isfinite().all()
        for name, v in run(dict(t, dy=dy), "relu", rg).items():
            assert torch.equal(v, base[name]), name
