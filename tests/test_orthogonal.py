"""Orthogonalised updates without a GPU: what the entry points refuse, and what workspace they ask for."""
import ctypes

import numpy as np

from permutohedral_encoding_amd import _native

MUON = (3.4445, -4.7750, 2.0315)


class Orthogonal(ctypes.Structure):  # penc_orthogonal
    _fields_ = [("type", ctypes.c_int), ("halves", ctypes.c_int), ("matrices", ctypes.c_int64), ("rows", ctypes.c_int64), ("columns", ctypes.c_int64), ("steps", ctypes.c_int),
                ("a", ctypes.c_float), ("b", ctypes.c_float), ("c", ctypes.c_float), ("eps", ctypes.c_float)]


def orthogonal(type=0, halves=0, matrices=1, rows=8, columns=9, steps=5, coefficients=MUON, eps=1e-7):
    return Orthogonal(type, halves, matrices, rows, columns, steps, *coefficients, eps)


def workspace(**given):
    return _native.lib().penc_orthogonal_workspace_bytes(ctypes.byref(orthogonal(**given)))


def _memory():
    block = np.zeros(4096, np.uint8)
    return block, block.ctypes.data + (-block.ctypes.data) % 256


def test_matrices_refuse_before_they_launch():
    block, p = _memory()
    z = None

    def call(g=p, to=p + 1024, ws=p, n=1 << 40, **given):
        return _native.lib().penc_orthogonal_matrices(ctypes.byref(orthogonal(**given)), g, to, ws, n, z)

    assert _native.lib().penc_orthogonal_matrices(z, p, p, p, 0, z) == 1 and _native.lib().penc_orthogonal_workspace_bytes(z) == 0
    for halves in (0, 1):
        assert call(type=3, halves=halves) == 10 and call(halves=halves, matrices=-1) == 12 and call(halves=halves, matrices=(1 << 20) + 1) == 12 and call(halves=halves, rows=0) == 12
        assert call(halves=halves, columns=(1 << 16) + 1) == 12 and call(halves=halves, steps=0) == 12 and call(halves=halves, steps=65) == 12
        assert call(halves=halves, eps=0.0) == 11 and call(halves=halves, coefficients=(4.0, 0.0, 0.0)) == 11
        assert call(halves=halves, g=z) == 1 and call(halves=halves, to=z) == 1 and call(halves=halves, g=p + 2) == 5 and call(halves=halves, to=p + 4) == 5 and call(halves=halves, ws=p + 16) == 5
        assert call(halves=halves, matrices=0, g=z, to=z) == 0
        for type in (0, 1, 2):
            need = workspace(type=type, halves=halves, matrices=2, rows=1000, columns=203)
            given = dict(type=type, halves=halves, matrices=2, rows=1000, columns=203)
            assert call(n=need - 1, **given) == 8 and call(ws=z, n=need, **given) == 1


def test_workspace_of_halves():
    large = dict(matrices=16, rows=4096, columns=1024)
    values = 16 * 4096 * 1024
    for type in (0, 1):
        assert workspace(type=type, **large) == workspace(type=type, halves=1, **large) == workspace(type=2, **large) >= 2 * 4 * values
    assert 2 * 2 * values <= workspace(type=2, halves=1, **large) < 2 * 4 * values
    assert _native.lib().penc_orthogonalise_workspace_bytes(2, 16, 4096, 1024) == workspace(type=2, halves=1, **large)


def test_workspace_is_what_the_way_takes():
    """Thin matrices go by sums of their S alone; columns padded to 32 and two copies of X are for steps that they do not survive in 64 bits."""
    gib, lib = 1 << 30, _native.lib()
    for type in (0, 1, 2):
        for (matrices, rows, columns), most in (((16384, 4096, 1), 2.2 * gib), ((1024, 4096, 3), 0.15 * gib), ((4096, 65536, 1), 2.2 * gib)):
            given = dict(type=type, matrices=matrices, rows=rows, columns=columns)
            assert 0 < workspace(**given) <= most
            assert workspace(steps=7, **given) == workspace(steps=1, **given) == workspace(**given)
            assert workspace(steps=8, **given) > 4 * rows * columns * matrices
            assert lib.penc_orthogonalise_workspace_bytes(type, matrices, rows, columns) >= max(workspace(halves=1, **given), workspace(halves=1, steps=8, **given))
    # matrices that stay in the LDS take none, long ones of 48 rows and fewer a little, as long as there are few
    assert workspace(matrices=1000, rows=64, columns=256) == 0 == workspace(matrices=3, rows=64, columns=300, steps=20) == workspace(matrices=65, rows=5, columns=200)
    assert 0 < workspace(matrices=64, rows=5, columns=200) < 1 << 20 and workspace(matrices=64, rows=5, columns=200, steps=8) == 0
    # nothing for what is refused
    for given in (dict(type=3), dict(type=-1), dict(steps=0), dict(steps=65), dict(eps=0.0), dict(coefficients=(4.0, 0.0, 0.0)), dict(matrices=-1), dict(rows=0)):
        assert workspace(**{"rows": 1000, "columns": 203, **given}) == 0


def test_less_workspace_than_the_way_takes_is_refused():
    block, p = _memory()
    given = dict(matrices=3, rows=3000, columns=50)
    need = workspace(**given)
    large = workspace(steps=20, **given)
    assert 0 < need < large

    def call(n, g=p, **more):
        return _native.lib().penc_orthogonal_matrices(ctypes.byref(orthogonal(**given, **more)), g, p + 1024, p, n, None)

    assert call(need - 1) == 8 and call(large - 1, steps=20) == 8 and call(need, steps=20) == 8
    assert _native.lib().penc_orthogonalise(0, 3, 3000, 50, 5, *MUON, 1e-7, p, p + 1024, p, need - 1, None) == 8


def test_the_status_names_what_was_refused():
    block, p = _memory()
    lib = _native.lib()
    lib.penc_status_string.restype = ctypes.c_char_p
    for given in (dict(eps=0.0), dict(coefficients=(4.0, 0.0, 0.0))):
        status = lib.penc_orthogonal_matrices(ctypes.byref(orthogonal(**given)), p, p + 1024, p, 1 << 40, None)
        text = lib.penc_status_string(status).decode()
        assert "coefficients" in text and "eps" in text and "activation" in text
