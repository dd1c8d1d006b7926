"""What the products behind the embeddings refuse, before anything reaches the GPU."""
import ctypes as C

import pytest
import torch

from face_recognition_amd import _lib, projection


def test_python_refusals():
    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="HIP device"):
        projection.linear(x, w)
    with pytest.raises(RuntimeError, match="activation"):
        projection.linear(x, w, activation="tanh")
    with pytest.raises(RuntimeError, match="not supported"):
        projection.linear(x.double(), w.double())
    with pytest.raises(RuntimeError, match="HIP device"):
        projection.group_rows(torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        projection.group_rows(torch.zeros(3), 2)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        projection.group_rows(torch.zeros(3, 1, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="group_rows"):
        projection.grouped_linear(x, w[None], None)


def desc(**over):
    """A valid 4 x 8 -> 5 product whose pointers are never followed."""
    d = _lib.LinearDesc(_lib.FRA_F16, 0, _lib.FRA_F16, _lib.FRA_F16, 4, 8, 5, 64, 64, None, None, None, 8, 8, 0, 0, None)
    for name, v in over.items():
        setattr(d, name, v)
    return d


@pytest.mark.parametrize("over,word", [
    (dict(dtype=3), b"dtype"), (dict(M=-1), b"rows"), (dict(M=2 ** 31), b"rows"), (dict(K=0), b"K ="), (dict(N=0), b"N ="),
    (dict(K=2 ** 25), b"K ="), (dict(act=5), b"activation"), (dict(act=2), b"slopes"), (dict(slope=64), b"slopes"),
    (dict(bias=64, bias_dtype=_lib.FRA_BF16), b"bias dtype"), (dict(act=2, slope=64, slope_dtype=_lib.FRA_BF16), b"slope dtype"),
    (dict(x=None), b"null"), (dict(w=None), b"null"), (dict(ldx=7), b"pitches"), (dict(ldw=7), b"pitches"),
    (dict(resid=64, ldr=4), b"residual"),
])
def test_descriptor_refusals(over, word):
    lib = _lib.load()
    d = desc(**over)
    n = C.c_size_t()
    assert lib.fra_linear(C.byref(d), None, 64, None) == 1 and word in lib.fra_last_error()
    assert lib.fra_linear_backward_workspace_bytes(C.byref(d), 1, 1, 0, 0, C.byref(n)) == 1 and word in lib.fra_last_error()
    assert lib.fra_linear_backward(C.byref(d), 64, 64, 5, 64, 64, None, None, None, 0, None) == 1 and word in lib.fra_last_error()


def test_call_refusals():
    lib = _lib.load()
    assert lib.fra_linear(None, None, 64, None) == 1
    assert lib.fra_linear(C.byref(desc()), None, None, None) == 1 and b"output" in lib.fra_last_error()
    back = lib.fra_linear_backward
    assert back(C.byref(desc()), None, None, 5, 64, None, None, None, None, 0, None) == 1 and b"gradient" in lib.fra_last_error()
    assert back(C.byref(desc()), None, 64, 4, 64, None, None, None, None, 0, None) == 1 and b"pitch" in lib.fra_last_error()
    assert back(C.byref(desc(act=1)), None, 64, 5, 64, None, None, None, None, 0, None) == 1 and b"preact" in lib.fra_last_error()
    assert back(C.byref(desc()), None, 64, 5, None, None, None, 64, None, 0, None) == 1 and b"slope" in lib.fra_last_error()
    assert back(C.byref(desc(act=1)), 64, 64, 5, 64, None, None, None, None, 0, None) == 5 and b"workspace" in lib.fra_last_error()
    # no rows: nothing to do, nothing needed
    assert lib.fra_linear(C.byref(desc(M=0, x=None)), None, None, None) == 0


def test_group_refusals():
    lib = _lib.load()
    n = C.c_size_t()
    for rows, groups in ((-1, 4), (2 ** 31, 4), (8, 0), (8, 4097)):
        assert lib.fra_group_rows_workspace_bytes(rows, groups, C.byref(n)) == 1
    assert lib.fra_group_rows_workspace_bytes(8, 4, None) == 1
    tr, nt = lib.fra_group_tile_rows(8, 4), lib.fra_group_tiles(8, 4)

    def groups(**over):
        g = _lib.RowGroupsDesc(8, 4, tr, nt, 64, 64, 64, 64)
        for name, v in over.items():
            setattr(g, name, v)
        return g

    assert lib.fra_group_rows(64, 0, None, None, 0, None) == 1
    assert lib.fra_group_rows(None, 0, C.byref(groups()), None, 0, None) == 1
    for over in (dict(order=None), dict(offsets=None), dict(tiles=None), dict(tile_offsets=None), dict(tile_rows=tr + 1), dict(n_tiles=nt - 1)):
        assert lib.fra_group_rows(64, 0, C.byref(groups(**over)), None, 0, None) == 1, over
    many = groups(rows=100000, tile_rows=lib.fra_group_tile_rows(100000, 4), n_tiles=lib.fra_group_tiles(100000, 4))
    assert lib.fra_group_rows(64, 0, C.byref(many), None, 0, None) == 5 and b"workspace" in lib.fra_last_error()
    for over in (dict(rows=9), dict(n_groups=0), dict(n_tiles=nt + 1), dict(order=None)):
        g = groups(**over)
        d = desc(M=8, groups=C.pointer(g))
        assert lib.fra_linear(C.byref(d), None, 64, None) == 1, over
    # what fra_group_rows fills: every group's tiles and the rest's fit
    for rows in (0, 1, 127, 128, 5000):
        for k in (1, 3, 4096):
            t = lib.fra_group_tile_rows(rows, k)
            assert lib.fra_group_tiles(rows, k) >= rows // t + k + (1 if rows else 0)


def test_orthogonalize_refusals():
    with pytest.raises(RuntimeError, match="HIP device"):
        projection.orthogonalize(torch.zeros(3, 3))
    with pytest.raises(RuntimeError, match="rows, cols"):
        projection.orthogonalize(torch.zeros(3))
    with pytest.raises(RuntimeError, match="rows, cols"):
        projection.orthogonalize(torch.zeros(3, 3, dtype=torch.float64))
    lib = _lib.load()
    n = C.c_size_t()
    usual = (3.4445, -4.775, 2.0315)

    def call(dtype=_lib.FRA_F32, g=64, ldg=8, bs=0, batch=1, rows=4, cols=8, steps=5, abc=usual, out=64, ws=64, nbytes=1 << 40):
        return lib.fra_orthogonalize(dtype, g, ldg, bs, batch, rows, cols, steps, *abc, out, ws, nbytes, None)

    for over in (dict(dtype=5), dict(g=None), dict(ldg=7), dict(bs=-1), dict(batch=-1), dict(batch=65536), dict(rows=0), dict(cols=0),
                 dict(rows=40000), dict(steps=0), dict(steps=101), dict(abc=(17.0, 0.0, 0.0)), dict(abc=(1.0, float("nan"), 0.0)), dict(out=None)):
        assert call(**over) == 1, over
    assert lib.fra_orthogonalize_workspace_bytes(1, 4, 8, C.byref(n)) == 0 and n.value > 0
    assert call(nbytes=n.value - 1) == 5 and call(ws=None) == 5
    assert call(batch=0, g=None, out=None, ws=None, nbytes=0) == 0
    assert lib.fra_orthogonalize_workspace_bytes(1, 0, 8, C.byref(n)) == 1 and lib.fra_orthogonalize_workspace_bytes(1, 4, 8, None) == 1


def test_scratch_and_tables_have_to_be_aligned():
    lib = _lib.load()
    n = C.c_size_t()
    d = desc(act=1)
    assert lib.fra_linear_backward_workspace_bytes(C.byref(d), 1, 1, 0, 0, C.byref(n)) == 0
    assert lib.fra_linear_backward(C.byref(d), 64, 64, 5, 64, 64, None, None, 72, n.value, None) == 1 and b"aligned" in lib.fra_last_error()
    g = _lib.RowGroupsDesc(8, 4, lib.fra_group_tile_rows(8, 4), lib.fra_group_tiles(8, 4), 64, 64, 68, 64)
    assert lib.fra_group_rows(64, 0, C.byref(g), None, 0, None) == 1 and b"aligned" in lib.fra_last_error()
    assert lib.fra_linear(C.byref(desc(M=8, groups=C.pointer(g))), None, 64, None) == 1 and b"aligned" in lib.fra_last_error()
    assert lib.fra_orthogonalize(_lib.FRA_F32, 64, 8, 0, 1, 4, 8, 5, 1.5, -0.5, 0.0, 64, 68, 1 << 40, None) == 1 and b"aligned" in lib.fra_last_error()


def test_more_threads_than_a_launch_takes():
    lib = _lib.load()
    g = _lib.RowGroupsDesc(8, 4096, lib.fra_group_tile_rows(8, 4096), lib.fra_group_tiles(8, 4096), 64, 64, 64, 64)
    d = desc(M=8, N=1 << 16, groups=C.pointer(g))                   # 4097 row tiles x 4096 column tiles of 512 threads
    assert lib.fra_linear(C.byref(d), None, 64, None) == 1 and b"launch" in lib.fra_last_error()


def test_packed_descriptor_is_the_structure():
    values = (1, 2, 3, 4, 5 << 40, 6, 7, 8 << 40, 9 << 40, 10 << 40, 11 << 40, 12 << 40, 13 << 40, 14 << 40, 15 << 40, 16 << 40, 0)
    d = _lib.LinearDesc.from_buffer_copy(projection._DESC.pack(*values))
    assert projection._DESC.size == C.sizeof(_lib.LinearDesc) and not d.groups
    assert tuple(getattr(d, name) for name, _ in d._fields_[:-1]) == values[:-1]
