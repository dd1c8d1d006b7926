"""Operators behind the embeddings: products with a fused epilogue, the same grouped by row, and orthogonalisation.

``run`` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the end) where ``own``
is false, and through ``face_recognition_amd.projection`` where it is true.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def listed():
    """Cases: ``op`` linear / grouped / orthogonalize; ``train`` adds the gradients of every input."""
    return [
        # one face of a camera frame through a 512-wide projection of its embedding: latency
        {"name": "linear_one_face", "op": "linear", "train": False, "dtype": "f16", "m": 1, "k": 512, "n": 512,
         "act": "prelu", "bias": True, "residual": False},
        # the faces of a few frames through a small fp32 head whose width is odd (attribute scores)
        {"name": "linear_attributes", "op": "linear", "train": False, "dtype": "f32", "m": 50, "k": 512, "n": 333,
         "act": "none", "bias": True, "residual": False},
        # a training batch against every identity of a data set, an odd number of them: the logits of a classifier
        {"name": "linear_identities", "op": "linear", "train": False, "dtype": "bf16", "m": 1024, "k": 512, "n": 40961,
         "act": "none", "bias": False, "residual": False},
        # a gallery taken into another network's embedding space in one go, the map added to the rows themselves
        {"name": "linear_gallery", "op": "linear", "train": False, "dtype": "f16", "m": 262144, "k": 512, "n": 512,
         "act": "silu", "bias": True, "residual": True},
        # one training step of a wide hidden layer
        {"name": "train_hidden", "op": "linear", "train": True, "dtype": "bf16", "m": 4096, "k": 1024, "n": 2048,
         "act": "gelu_tanh", "bias": True, "residual": False},
        # one training step of a small fp32 layer with odd sizes on every side and a learnt slope
        {"name": "train_odd", "op": "linear", "train": True, "dtype": "f32", "m": 1000, "k": 500, "n": 301,
         "act": "prelu", "bias": True, "residual": True},
        # the faces of one frame, each through the projection of the camera it came from
        {"name": "grouped_frame", "op": "grouped", "train": False, "dtype": "f16", "m": 9, "k": 512, "n": 512,
         "groups": 12, "act": "none", "bias": True, "residual": True},
        # a large mixed batch, ragged groups (some without a row) and rows of no group
        {"name": "grouped_batch", "op": "grouped", "train": False, "dtype": "bf16", "m": 30001, "k": 512, "n": 768,
         "groups": 37, "act": "gelu_tanh", "bias": True, "residual": False},
        # one training step of sixteen projections on a mixed batch
        {"name": "grouped_train", "op": "grouped", "train": True, "dtype": "bf16", "m": 8192, "k": 512, "n": 1024,
         "groups": 16, "act": "silu", "bias": True, "residual": False},
        # the same in fp32, few groups, odd sizes
        {"name": "grouped_train_odd", "op": "grouped", "train": True, "dtype": "f32", "m": 2999, "k": 250, "n": 513,
         "groups": 5, "act": "relu", "bias": True, "residual": False},
        # the update of one square 512-wide projection
        {"name": "orthogonalize_one", "op": "orthogonalize", "dtype": "f32", "batch": 1, "m": 512, "n": 512},
        # the updates of the wide layers of several groups in one call
        {"name": "orthogonalize_batch", "op": "orthogonalize", "dtype": "bf16", "batch": 8, "m": 2048, "n": 1024},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges: rows from one to the large batches, widths odd or even."""
    kind = rng.choice(["linear", "linear", "linear_train", "grouped", "grouped_train", "orthogonalize"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "orthogonalize":
        m, n = _log_int(rng, 64, 2048), _log_int(rng, 64, 2048)
        lo, hi = min(m, n), max(m, n)
        batch = max(1, min(rng.randint(1, 8), int(2.0e11 / (5.0 * lo * lo * (lo + 3.0 * hi)))))
        return {"op": "orthogonalize", "dtype": dtype, "batch": batch, "m": m, "n": n}
    train = kind.endswith("train")
    k, n = _log_int(rng, 64, 2048), _log_int(rng, 40, 4096)
    # below the largest listed case in products and in bytes
    products = 2.0e10 if dtype == "f32" else 5.0e10
    rows = 6.0e8 / (_SIZE[dtype] * (k + 2 * n) * (2 if train else 1))
    m = _log_int(rng, 1, max(1, min(262144, int(products / (k * n)), int(rows))))
    case = {"op": "grouped" if kind.startswith("grouped") else "linear", "train": train, "dtype": dtype, "m": m, "k": k,
            "n": n, "act": rng.choice(["none", "relu", "prelu", "silu", "gelu_tanh"]),
            "bias": rng.random() < 0.7, "residual": rng.random() < 0.4}
    if case["op"] == "grouped":
        case["groups"] = _log_int(rng, 2, max(2, min(64, (1 << 25) // (k * n))))
    return case


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)

    if case["op"] == "orthogonalize":
        # a gradient: a few strong directions (what a batch has in common) over noise
        b, m, n = case["batch"], case["m"], case["n"]
        g = randn(b, m, n) * 1e-3
        for i in range(4):
            g += randn(b, m, 1) * randn(b, 1, n) * (1e-3 / (1 + i))
        return {"g": (g if b > 1 else g[0]).to(dt)}
    m, k, n = case["m"], case["k"], case["n"]
    lead = (case["groups"],) if case["op"] == "grouped" else ()
    x = randn(m, k)
    x = x / (x * x).sum(1, keepdim=True).sqrt()              # rows of unit length, as embeddings are
    t = {"x": x.to(dt), "w": randn(*lead, n, k).to(dt)}
    if case["bias"]:
        t["b"] = (0.1 * randn(*lead, n)).to(dt)
    if case["act"] == "prelu":
        t["s"] = (0.25 + 0.05 * randn(*lead, n)).to(dt)
    if case["residual"]:
        t["r"] = randn(m, n).to(dt)
    if case["train"]:
        t["dy"] = (randn(m, n) / 8).to(dt)
    if case["op"] == "grouped":
        # uneven shares, one row in 64 of no group
        share = torch.exp(randn(case["groups"]))
        ids = torch.multinomial(share, m, replacement=True, generator=gen)
        t["ids"] = torch.where(torch.rand(m, generator=gen, device=dev) < 1 / 64, torch.full_like(ids, -1), ids)
    return t


def prepare(case, seed):
    state = {"case": case, "t": _inputs(case, seed)}
    if case.get("train"):
        # the parameters and inputs a training program differentiates by
        state["leaves"] = [n for n in ("x", "w", "b", "s", "r") if n in state["t"]]
        for name in state["leaves"]:
            state["t"][name].requires_grad_(True)
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _act(z, act, s):
    if act == "relu":
        return torch.where(z > 0, z, z * 0.0)
    if act == "prelu":
        return torch.where(z > 0, z, z * s)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu_tanh":
        return z / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_grad(z, act, s):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "prelu":
        return torch.where(z > 0, torch.ones_like(z), torch.zeros_like(z) + s)
    if act == "silu":
        q = 1.0 / (1.0 + torch.exp(-z))
        return q * (1.0 + z * (1.0 - q))
    if act == "gelu_tanh":
        c = 2.0 * math.sqrt(2.0 / math.pi)
        q = 1.0 / (1.0 + torch.exp(-c * (z + 0.044715 * z * z * z)))
        return q + z * q * (1.0 - q) * c * (1.0 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_rows(t, rows, g, act, train):
    """One set of rows (all of them: ``rows`` None) through one matrix: (y, gradients), still in 32 bits."""
    pick = (lambda a: a) if rows is None else (lambda a: a[rows])
    par = (lambda a: a) if g is None else (lambda a: a[g])
    x, w = pick(t["x"]).float(), par(t["w"]).float()
    s = par(t["s"]).float() if "s" in t else None
    z = x @ w.t()
    if "b" in t:
        z = z + par(t["b"]).float()
    y = _act(z, act, s)
    if "r" in t:
        y = y + pick(t["r"]).float()
    if not train:
        return y, {}
    dy = pick(t["dy"]).float()
    dz = dy * _act_grad(z, act, s)
    grads = {"x": dz @ w, "w": dz.t() @ x}
    if "b" in t:
        grads["b"] = dz.sum(0)
    if s is not None:
        grads["s"] = torch.where(z > 0, z * 0.0, dy * z).sum(0)
    return y, grads


def _plain_linear(case, t):
    y, grads = _plain_rows(t, None, None, case["act"], case["train"])
    dt = t["x"].dtype
    out = {"y": y.to(dt)}
    for name, v in grads.items():
        out["d" + name] = v.to(dt)
    if case["train"] and "r" in t:
        out["dr"] = t["dy"]
    return out


def _plain_grouped(case, t):
    ids, groups = t["ids"], case["groups"]
    key = torch.where((ids >= 0) & (ids < groups), ids, torch.full_like(ids, groups))
    order = torch.argsort(key, stable=True)
    counts = (key[None, :] == torch.arange(groups, device=ids.device)[:, None]).sum(1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    dt = t["x"].dtype
    y = t["r"].float() if "r" in t else torch.zeros(case["m"], case["n"], device=ids.device)
    names = [n for n in ("x", "w", "b", "s") if n in t] if case["train"] else []
    full = {n: torch.zeros(t[n].shape, device=ids.device) for n in names}
    ends = offsets.tolist()
    for g in range(groups):
        if ends[g + 1] == ends[g]:
            continue
        rows = order[ends[g]:ends[g + 1]]
        yg, grads = _plain_rows(t, rows, g, case["act"], case["train"])
        y[rows] = yg
        for n in names:
            full[n][rows if n == "x" else g] = grads[n]
    out = {"order": order.int(), "offsets": offsets.int(), "y": y.to(dt)}
    for n in names:
        out["d" + n] = full[n].to(dt)
    if case["train"] and "r" in t:
        out["dr"] = t["dy"]
    return out


def _plain_orthogonalize(t):
    g = t["g"].float()
    tall = g.shape[-2] > g.shape[-1]
    x = g.transpose(-1, -2) if tall else g
    x = x / (x * x).sum((-2, -1), keepdim=True).sqrt()
    a, b, c = _COEFFICIENTS
    for _ in range(5):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.transpose(-1, -2) if tall else x).to(t["g"].dtype).contiguous()


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _own_run(case, t, leaves):
    from face_recognition_amd import projection
    if case["op"] == "orthogonalize":
        return projection.orthogonalize(t["g"], steps=5, coefficients=_COEFFICIENTS)
    args = dict(bias=t.get("b"), activation=case["act"], slope=t.get("s"), residual=t.get("r"))
    out = {}
    if case["op"] == "grouped":
        groups = projection.group_rows(t["ids"], case["groups"])
        out["order"], out["offsets"] = groups.order, groups.offsets
        y = projection.grouped_linear(t["x"], t["w"], groups, **args)
    else:
        y = projection.linear(t["x"], t["w"], **args)
    out["y"] = y.detach()
    if case["train"]:
        for name, v in zip(leaves, torch.autograd.grad(y, [t[n] for n in leaves], t["dy"])):
            out["d" + name] = v
    return out


def run(state):
    case, t = state["case"], state["t"]
    if own:
        return _own_run(case, t, state.get("leaves"))
    with torch.no_grad():                                    # the plain forms write their gradients out
        if case["op"] == "orthogonalize":
            return _plain_orthogonalize(t)
        return _plain_grouped(case, t) if case["op"] == "grouped" else _plain_linear(case, t)


# ---- what has to be moved and computed ------------------------------------------------------------------------------

def work(case):
    es = _SIZE[case["dtype"]]
    if case["op"] == "orthogonalize":
        lo, hi = min(case["m"], case["n"]), max(case["m"], case["n"])
        # X X^T and A A are symmetric: half of their products; (b A + c A A) X is not
        flops = 5.0 * (lo * lo * hi + lo ** 3 + 2.0 * lo * lo * hi) * case["batch"]
        return {"bytes": 2.0 * es * lo * hi * case["batch"], "flops": flops}
    m, k, n = case["m"], case["k"], case["n"]
    groups = case.get("groups", 1)
    par = n * k + n * (int(case["bias"]) + int(case["act"] == "prelu"))
    size = m * k + min(groups, m) * par + m * n * (1 + int(case["residual"]))
    flops = 2.0 * m * n * k
    if case["train"]:
        size += m * n + m * k + groups * par                 # dy in; dx and the parameters' gradients out
        flops *= 3
    ints = 4 * (3 * m + groups + 1) if case["op"] == "grouped" else 0       # ids in (8 bytes), order and offsets out
    return {"bytes": float(es * size + ints), "flops": flops}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "orthogonalize":
        x = t["g"].double()
        eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
        if x.shape[-2] > x.shape[-1]:
            eye = torch.eye(x.shape[-1], dtype=torch.float64, device=x.device)
        x = x / torch.linalg.matrix_norm(x, keepdim=True)
        a, b, c = _COEFFICIENTS
        for _ in range(5):
            if x.shape[-2] > x.shape[-1]:
                p = x.mT @ x
                x = x @ (a * eye + p @ (b * eye + c * p))
            else:
                p = x @ x.mT
                x = (a * eye + p @ (b * eye + c * p)) @ x
        return x
    d = {n: v.double().requires_grad_(case["train"]) for n, v in t.items() if n not in ("ids", "dy")}

    def through(x, w, b, s):
        z = torch.nn.functional.linear(x, w, b)
        if case["act"] == "relu":
            return torch.relu(z)
        if case["act"] == "prelu":
            return torch.clamp(z, min=0) + s * torch.clamp(z, max=0)
        if case["act"] == "silu":
            return z * torch.sigmoid(z)
        if case["act"] == "gelu_tanh":
            return torch.nn.functional.gelu(z, approximate="tanh")
        return z

    out = {}
    if case["op"] == "grouped":
        ids, groups = t["ids"], case["groups"]
        rows = [torch.nonzero(ids == g)[:, 0] for g in range(groups)]
        out["offsets"] = torch.tensor([0] + [len(r) for r in rows], device=ids.device).cumsum(0).int()
        rest = torch.nonzero((ids < 0) | (ids >= groups))[:, 0]
        out = {"order": torch.cat(rows + [rest]).int(), "offsets": out["offsets"]}
        y = d["r"] if "r" in d else torch.zeros(case["m"], case["n"], dtype=torch.float64, device=ids.device)
        for g, r in enumerate(rows):
            y = y.index_add(0, r, through(d["x"][r], d["w"][g], d["b"][g] if "b" in d else None,
                                          d["s"][g] if "s" in d else None))
    else:
        y = through(d["x"], d["w"], d.get("b"), d.get("s"))
        if "r" in d:
            y = y + d["r"]
    out["y"] = y.detach()
    if case["train"]:
        names = [n for n in ("x", "w", "b", "s", "r") if n in d]
        for name, v in zip(names, torch.autograd.grad(y, [d[n] for n in names], t["dy"].double())):
            out["d" + name] = v
    return out
