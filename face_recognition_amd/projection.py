"""Matrices behind the embeddings: heads and maps applied to rows, one for all of them or one per group, with gradients.

    linear(x, weight, bias, activation, slope, residual)            y = act(x W^T + b) + r
    group_rows(ids, n_groups) -> RowGroups                          rows sorted by the group they name
    grouped_linear(x, weight[G], groups, ...)                       every row through its group's matrix
    orthogonalize(matrix, steps, coefficients)                      an update made nearly orthogonal, or a fitted map wholly

Uses: a head on top of the 512-wide embeddings, a map that takes one network's embeddings into another's space so that an
existing gallery stays searchable, one such map per camera / tenant / model version, and the training of all of these (a map
that is wholly orthogonal leaves distances, and the thresholds set for them, as they are).  No counterpart in the reference.  All
products run in the HIP library (``fra_linear``, ``fra_group_rows``, ``fra_orthogonalize``); there is no CPU path.

Types: float32, float16, bfloat16; ``x``, ``weight`` and ``residual`` share one, ``bias`` and ``slope`` are of it or float32.
Sums are fp32.  The calls queue on the current stream and neither synchronise nor read anything back, so they can be
captured into a graph.  Capture a backward pass as ``torch.autograd.grad`` on leaves of which no eager graph is alive.
"""
from __future__ import annotations

import ctypes as C
import struct
from functools import lru_cache
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.FRA_F32, torch.bfloat16: _lib.FRA_BF16, torch.float16: _lib.FRA_F16}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "prelu": 2, "silu": 3, "gelu_tanh": 4}
MAX_GROUPS = 4096


def _stream(device: torch.device) -> int:
    """The current stream's handle, without building a ``torch.cuda.Stream`` for it (2 us of a call's 13)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _on_device(device: torch.device, call, *args):
    """``call(*args)`` with `device` as the current one; nothing to do if it is (``torch.cuda.device`` costs 1 us either way)."""
    prev = torch._C._cuda_getDevice()
    if prev == device.index:
        return call(*args)
    torch.cuda.set_device(device.index)
    try:
        return call(*args)
    finally:
        torch.cuda.set_device(prev)


@lru_cache(maxsize=256)
def _group_sizes(rows: int, n_groups: int):
    """(rows of a tile, entries of the tile table, bytes of scratch) of so many rows and groups."""
    lib = _lib.load()
    need = C.c_size_t()
    _lib.check(lib.fra_group_rows_workspace_bytes(rows, n_groups, C.byref(need)), "fra_group_rows_workspace_bytes")
    return lib.fra_group_tile_rows(rows, n_groups), lib.fra_group_tiles(rows, n_groups), need.value


class RowGroups:
    """The rows of a batch sorted by group (``group_rows``).

    ``order`` int32 [rows]: row numbers by group, ascending inside a group, rows of no group last; ``offsets`` int32
    [n_groups + 1]: group g's rows are ``order[offsets[g]:offsets[g + 1]]``.  Serves any number of products of these rows.
    For use on another stream than it was made on it is a tensor like any other: wait for it there, and before it is dropped
    call ``groups.order.record_stream(stream)`` (all its parts are one allocation).
    """

    def __init__(self, rows: int, n_groups: int, ids: torch.Tensor, tile_rows: int, n_tiles: int):
        self.rows, self.n_groups, self.device = rows, n_groups, ids.device
        # one allocation: tiles (16-byte aligned) | order | offsets | tile_offsets
        self._buf = ids.new_empty(4 * n_tiles + rows + 2 * n_groups + 3, dtype=torch.int32)
        base, at = self._buf.data_ptr(), 4 * n_tiles
        self._desc = _lib.RowGroupsDesc(rows, n_groups, tile_rows, n_tiles, base + 4 * at, base + 4 * (at + rows), base,
                                        base + 4 * (at + rows + n_groups + 1))
        self._address = C.addressof(self._desc)

    @property
    def order(self) -> torch.Tensor:
        at = 4 * self._desc.n_tiles
        return self._buf.narrow(0, at, self.rows)

    @property
    def offsets(self) -> torch.Tensor:
        at = 4 * self._desc.n_tiles + self.rows
        return self._buf.narrow(0, at, self.n_groups + 1)


def group_rows(ids: torch.Tensor, n_groups: int) -> RowGroups:
    """Sort rows by group id: ``ids`` int32 / int64 [rows] on the device.  Ids outside [0, n_groups) name no group."""
    if not isinstance(ids, torch.Tensor) or ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("group_rows: ids must be an int32 or int64 vector")
    if not ids.is_cuda:
        raise RuntimeError("group_rows: ids live on the HIP device ('cuda'); there is no CPU path")
    n_groups = int(n_groups)
    if not 1 <= n_groups <= MAX_GROUPS:
        raise RuntimeError(f"group_rows: {n_groups} groups (1 to {MAX_GROUPS})")
    ids = ids.contiguous()
    rows = ids.shape[0]
    tile_rows, n_tiles, need = _group_sizes(rows, n_groups)
    g = RowGroups(rows, n_groups, ids, tile_rows, n_tiles)
    ws = ids.new_empty(need, dtype=torch.uint8) if need else None
    _lib.check(_on_device(g.device, _lib.load().fra_group_rows, ids.data_ptr(), ids.dtype == torch.int64, C.byref(g._desc),
                          ws.data_ptr() if need else None, need, _stream(g.device)), "fra_group_rows")
    return g


# a _lib.LinearDesc as bytes, in C's layout: filling a ctypes structure costs 1 us more
_DESC = struct.Struct("@4iq2i5P4qP")


def _rows(t: torch.Tensor, r: int, c: int):
    """(tensor, pitch) of [r,c]: contiguous rows, copied only if they are not."""
    s0, s1 = t.stride()
    if (s1 != 1 and c > 1) or (r > 1 and s0 < c):
        t = t.contiguous()
        s0 = c
    return t, (s0 if r > 1 else c)


def _weight(weight: torch.Tensor, n: int, k: int):
    """(tensor, row pitch, group pitch) of [N,K] or [G,N,K] with contiguous rows."""
    if weight.dim() == 2:
        return *_rows(weight, n, k), 0
    sg, s0, s1 = weight.stride()
    if (s1 != 1 and k > 1) or (n > 1 and s0 < k):
        weight = weight.contiguous()
        sg, s0 = n * k, k
    return weight, (s0 if n > 1 else k), sg


def _forward(x, weight, bias, slope, residual, act, groups, want_preact):
    """(out, preact, the descriptor's types and sizes, (x, weight, slope) as the kernels read them).  Sizes are taken apart once, and
    `new_empty` gets plain numbers: a shape costs 1 us more."""
    m, k = x.shape
    n = weight.shape[-2]
    dt = _DTYPES[x.dtype]
    x, ldx = _rows(x, m, k)
    weight, ldw, wg = _weight(weight, n, k)
    ldr = 0
    if residual is not None:
        residual, ldr = _rows(residual, m, n)
    if bias is not None:
        bias = bias.contiguous()
    if slope is not None:
        slope = slope.contiguous()
    out = x.new_empty(m, n)
    z = torch.empty_like(out) if want_preact else None
    sizes = (dt, act, _DTYPES[bias.dtype] if bias is not None else 0, _DTYPES[slope.dtype] if slope is not None else 0, m, k, n)
    d = _DESC.pack(*sizes, x.data_ptr(), weight.data_ptr(), bias.data_ptr() if bias is not None else 0,
                   slope.data_ptr() if slope is not None else 0, residual.data_ptr() if residual is not None else 0,
                   ldx, ldw, ldr, wg, groups._address if groups is not None else 0)
    if m:
        device = x.device
        _lib.check(_on_device(device, _lib.load().fra_linear, d, z.data_ptr() if z is not None else None,
                              out.data_ptr(), _stream(device)), "fra_linear")
    return out, z, sizes, (x, weight, slope)


def _backward(ctx, dy):
    need_x, need_w, need_b, need_s, need_r, _, _ = ctx.needs_input_grad
    dx = dw = db = ds = None
    if need_x or need_w or need_b or need_s:
        x, weight, slope, z = ctx.saved_tensors
        sizes, groups = ctx.sizes, ctx.groups
        m, k, n = sizes[4:]
        lead = (groups.n_groups,) if groups is not None else ()
        if need_x:
            dx = x.new_empty(m, k)
        if need_w:
            dw = x.new_empty(*lead, n, k)
        if need_b:
            db = x.new_empty(*lead, n, dtype=ctx.bias_dtype)
        if need_s:
            ds = x.new_empty(*lead, n, dtype=slope.dtype)
        # saved-tensor hooks may bring back other tensors, or the same memory laid out otherwise
        x, ldx = _rows(x, m, k)
        weight, ldw, wg = _weight(weight, n, k)
        if slope is not None:
            slope = slope.contiguous()
        if z is not None:
            z = z.contiguous()
        g, lddy = _rows(dy, m, n)
        d = _DESC.pack(*sizes, x.data_ptr(), weight.data_ptr(), 0, slope.data_ptr() if slope is not None else 0, 0, ldx, ldw, 0, wg,
                       groups._address if groups is not None else 0)
        lib, device, nbytes = _lib.load(), x.device, C.c_size_t()
        _lib.check(lib.fra_linear_backward_workspace_bytes(d, need_x, need_w, need_b, need_s, C.byref(nbytes)),
                   "fra_linear_backward_workspace_bytes")
        ws = x.new_empty(nbytes.value, dtype=torch.uint8)
        _lib.check(_on_device(device, lib.fra_linear_backward, d, z.data_ptr() if z is not None else None,
                              g.data_ptr(), lddy, dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None,
                              db.data_ptr() if need_b else None, ds.data_ptr() if need_s else None,
                              ws.data_ptr(), nbytes.value, _stream(device)), "fra_linear_backward")
    return dx, dw, db, ds, (dy if need_r else None), None, None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, slope, residual, act, groups):
        need = ctx.needs_input_grad
        out, z, sizes, kept = _forward(x, weight, bias, slope, residual, act, groups,
                                       act != 0 and (need[0] or need[1] or need[2] or need[3]))
        ctx.save_for_backward(*kept, z)
        ctx.sizes, ctx.groups = sizes, groups
        ctx.bias_dtype = bias.dtype if bias is not None else None
        return out

    # once differentiable; the wrapper that says so is needed only where a graph of the backward pass is being built
    _once = staticmethod(torch.autograd.function.once_differentiable(_backward))

    @staticmethod
    def backward(ctx, dy):
        return _Linear._once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def _check_parameter(what, name, t, shape, dt, device):
    if t.shape != shape or (t.dtype != dt and t.dtype != torch.float32):
        raise RuntimeError(f"{what}: {name} must be {list(shape)} in {dt} or float32, got {list(t.shape)} {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{what}: {name} is on {t.device}, x on {device}")


def _check(what, x, weight, bias, activation, slope, residual, lead):
    act = ACTIVATIONS.get(activation, -1) if activation is None or isinstance(activation, str) else -1
    if act < 0:
        raise RuntimeError(f"{what}: activation {activation!r} is none of {sorted(k for k in ACTIVATIONS if k)}")
    dt = x.dtype
    if dt not in _DTYPES:
        raise RuntimeError(f"{what}: {dt} is not supported (float32, float16, bfloat16)")
    if not x.is_cuda:
        raise RuntimeError(f"{what}: tensors live on the HIP device ('cuda'); there is no CPU path")
    ws, xs, dev = weight.shape, x.shape, x.device
    if len(ws) != 2 + len(lead) or (lead and ws[:-2] != lead):
        raise RuntimeError(f"{what}: weight must be [{', '.join([str(v) for v in lead] + ['N', 'K'])}], got {tuple(ws)}")
    n, k = ws[-2], ws[-1]
    if n == 0 or k == 0 or not xs or xs[-1] != k:
        raise RuntimeError(f"{what}: x {tuple(xs)} does not go with weight {tuple(ws)}")
    if weight.dtype != dt:
        raise RuntimeError(f"{what}: weight is {weight.dtype}, x is {dt}")
    if weight.device != dev:
        raise RuntimeError(f"{what}: weight is on {weight.device}, x on {dev}")
    if (act == 2) != (slope is not None):
        raise RuntimeError(f"{what}: slope goes with activation 'prelu', and only with it")
    if bias is not None:
        _check_parameter(what, "bias", bias, lead + (n,), dt, dev)
    if slope is not None:
        _check_parameter(what, "slope", slope, lead + (n,), dt, dev)
    if residual is not None:
        if residual.shape != xs[:-1] + (n,):
            raise RuntimeError(f"{what}: residual must be {list(xs[:-1]) + [n]}, got {list(residual.shape)}")
        if residual.dtype != dt:
            raise RuntimeError(f"{what}: residual is {residual.dtype}, x is {dt}")
        if residual.device != dev:
            raise RuntimeError(f"{what}: residual is on {residual.device}, x on {dev}")
    return act


def _apply(x, weight, bias, slope, residual, act, groups):
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (slope is not None and slope.requires_grad) or (residual is not None and residual.requires_grad)) \
            or forward_ad._current_level >= 0:      # torch refuses a tangent there; it would be lost below
        return _Linear.apply(x, weight, bias, slope, residual, act, groups)
    return _forward(x, weight, bias, slope, residual, act, groups, False)[0]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
           slope: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in one kernel: x [..., K], weight [N,K], bias / slope [N], residual [..., N].

    ``activation``: None, 'relu', 'prelu' (with ``slope``, one value per output channel), 'silu' or 'gelu_tanh'.
    Differentiable (once) in every tensor argument.
    """
    act = _check("linear", x, weight, bias, activation, slope, residual, ())
    if x.dim() == 2:
        return _apply(x, weight, bias, slope, residual, act, None)
    k, n = x.shape[-1], weight.shape[0]
    m = x.numel() // k
    y = _apply(x.reshape(m, k), weight, bias, slope, residual.reshape(m, n) if residual is not None else None, act, None)
    return y.reshape(tuple(x.shape[:-1]) + (n,))


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, groups: RowGroups, bias: Optional[torch.Tensor] = None,
                   activation: Optional[str] = None, slope: Optional[torch.Tensor] = None,
                   residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``linear`` with one matrix per group: x [rows,K], weight [G,N,K], bias / slope [G,N], residual [rows,N].

    Row i goes through the matrix of the group its id named (``group_rows``); the result keeps the order of x.  A row of no
    group comes out as its residual, or as zeros, and has a zero gradient.
    """
    if not isinstance(groups, RowGroups):
        raise RuntimeError("grouped_linear: groups must come from group_rows")
    act = _check("grouped_linear", x, weight, bias, activation, slope, residual, (groups.n_groups,))
    if x.dim() != 2 or x.shape[0] != groups.rows:
        raise RuntimeError(f"grouped_linear: x must be [{groups.rows},K], got {tuple(x.shape)}")
    if groups.device != x.device:
        raise RuntimeError(f"grouped_linear: groups are on {groups.device}, x on {x.device}")
    return _apply(x, weight, bias, slope, residual, act, groups)


def _orthogonalize(matrix, steps, coefficients):
    rows, cols = matrix.shape[-2:]
    g = matrix.detach()
    if g.dim() > 3:
        g = g.reshape(-1, rows, cols)
    s0, s1 = g.stride()[-2:]
    if (s1 != 1 and cols > 1) or (rows > 1 and s0 < cols):
        g = g.contiguous()
        s0 = cols
    batch = g.shape[0] if g.dim() == 3 else 1
    lib = _lib.load()
    out = torch.empty(matrix.shape, dtype=matrix.dtype, device=matrix.device)
    need = C.c_size_t()
    _lib.check(lib.fra_orthogonalize_workspace_bytes(batch, rows, cols, C.byref(need)), "fra_orthogonalize_workspace_bytes")
    ws = torch.empty(need.value, dtype=torch.uint8, device=matrix.device)
    _lib.check(_on_device(matrix.device, lib.fra_orthogonalize, _DTYPES[g.dtype], g.data_ptr(), s0 if rows > 1 else cols,
                          g.stride(0) if g.dim() == 3 else 0, batch, rows, cols, steps, *[float(v) for v in coefficients],
                          out.data_ptr(), ws.data_ptr(), need.value, _stream(matrix.device)), "fra_orthogonalize")
    return out


class _ValuesOnly(torch.autograd.Function):
    """``_orthogonalize`` of a matrix whose derivatives are being followed, so that one that goes through it is not lost without a word."""

    @staticmethod
    def forward(ctx, matrix, steps, coefficients):
        return _orthogonalize(matrix, steps, coefficients)

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError("orthogonalize is not differentiable: call it on matrix.detach(), or under torch.no_grad(), for its values")


def orthogonalize(matrix: torch.Tensor, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315)) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of [..., rows, cols] (every leading index a matrix of its own), in its type.

    X = matrix / |matrix|_F, then ``steps`` times X <- a X + (b P + c P P) X with P = X X^T (of the transposed matrix where it
    is taller than wide).  The default coefficients (published by K. Jordan et al. with the Muon optimizer, 2024) take the singular
    values of an update, but the smallest, into about [0.7, 1.2] in five steps and do not converge further: good for an update, not for
    a map that is to leave distances as they are.  Those of the Newton-Schulz iteration, (1.5, -0.5, 0) or (1.875, -1.25, 0.375),
    converge to the nearest orthogonal matrix in more steps (20 to 40, by the smallest singular value).  A matrix of zeros gives zeros.  Between the products values keep 22 bits in a range of +-255 (1 to 100 steps, coefficients within +-16: such that the
    singular values stay near one).  Not differentiable: a derivative asked of it, backward or forward mode, is an error.
    """
    if not isinstance(matrix, torch.Tensor) or matrix.dim() < 2 or matrix.dtype not in _DTYPES:
        raise RuntimeError("orthogonalize: [..., rows, cols] in float32, float16 or bfloat16")
    if not matrix.is_cuda:
        raise RuntimeError("orthogonalize: tensors live on the HIP device ('cuda'); there is no CPU path")
    if len(coefficients) != 3:
        raise RuntimeError("orthogonalize: three coefficients")
    rows, cols = matrix.shape[-2:]
    if rows == 0 or cols == 0:
        raise RuntimeError(f"orthogonalize: empty matrices {tuple(matrix.shape)}")
    if torch.is_grad_enabled() and matrix.requires_grad or forward_ad._current_level >= 0:
        return _ValuesOnly.apply(matrix, int(steps), coefficients)
    return _orthogonalize(matrix, int(steps), coefficients)
