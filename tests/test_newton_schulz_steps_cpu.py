"""Which way matrices of up to 16 rows go, as the workspaces that calls ask for show it; every check comes before anything
touches the device."""
import ctypes

import pytest

ONE = ctypes.c_void_p(256)   # aligned, never dereferenced
NS = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def lib():
    from _spherical_distortion_ext import _capi
    return _capi.load()


@pytest.mark.parametrize("steps,c", [(8, NS), (20, NS), (100, NS), (30, (1.875, -1.25, 0.375)), (50, (1.5, -0.5, 0.0))])
@pytest.mark.parametrize("rows,columns", [(16, 1000), (2000, 3), (1, 5000)])
def test_many_steps_go_by_the_matrix(lib, rows, columns, steps, c):
    """And need a workspace where it is long; the sizes that are asked for hold whatever the steps are."""
    three = (ctypes.c_double * 3)(*c)
    need = lib.sdk_orthogonalize_workspace_bytes(rows, columns, 1, 0)
    assert need > 0

    def run(ws, bytes_):
        return lib.sdk_orthogonalize(ONE, ONE, rows, columns, 1, steps, three, 1e-7, ws, bytes_, 0, None)
    assert run(None, 0) == -3 and run(ONE, need - 1) == -3
    sizes = [(ctypes.c_int64 * 2)(n, 3) for n in (rows, columns)]
    lists = [(ctypes.c_void_p * 2)(at, at + 256) for at in (1024, 2048, 4096)]
    assert lib.sdk_muon_step_workspace_bytes(*sizes, 2, 0) == need

    def step(ws, bytes_):
        return lib.sdk_muon_step(*lists, *sizes, 2, 0.1, 0.9, 1, 0.0, steps, three, 1e-7, ws, bytes_, 0, None)
    assert step(None, 0) == -3 and step(ONE, need - 1) == -3


def test_workspaces_hold_either_way(lib):
    """65 thin matrices in front of a large one: groups of 64 are dealt otherwise where the thin ones are among them."""
    size = lib.sdk_orthogonalize_workspace_bytes
    thin, large = size(16, 1000, 1, 0), size(100, 100, 1, 0)
    n = 66
    rows, columns = (ctypes.c_int64 * n)(*[16] * 65, 100), (ctypes.c_int64 * n)(*[1000] * 65, 100)
    assert lib.sdk_muon_step_workspace_bytes(rows, columns, n, 0) == max(64 * thin, thin + large, large)
    assert size(16, 300, 9, 0) == 0   # short ones need none either way
