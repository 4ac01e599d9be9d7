"""Which way matrices of up to 16 rows go, as the workspaces that calls ask for show it; every check comes before anything
touches the device."""
import ctypes

import pytest
import torch

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


def _allowed(steps, c):
    from _spherical_distortion_ext import _token_ops
    try:
        _token_ops.check_newton_schulz(steps, c, 1e-7)
    except RuntimeError as e:
        assert "grow too far" in str(e)
        return False
    return True


@pytest.mark.parametrize("c", [1e-20, -1e-20, 1e-300, 5e-324, 1e-12, -1e-9, 0.0])
def test_extremes_beside_a_last_coefficient_of_nearly_nothing(c):
    """15 x - 15 x^3 is 5.77 at sqrt(1/3), 9 x - 9 x^3 3.46; 3 x - x^3 reaches 2 at 1, from where it goes to -2 at 2; 6 x + 3.2 x^3
    only grows; 1.5 x - 0.5 x^3 stays at one."""
    assert not _allowed(1, (15.0, -15.0, c)) and not _allowed(2, (15.0, -15.0, c)) and not _allowed(1, (-15.0, 15.0, c))
    assert _allowed(1, (9.0, -9.0, c)) and _allowed(1, (-9.0, 9.0, c)) and not _allowed(2, (9.0, -9.0, c))
    assert _allowed(3, (3.0, -1.0, c))
    assert not _allowed(1, (6.0, 3.2, c)) and _allowed(100, (1.5, -0.5, c))


def test_extremes_of_small_last_coefficients():
    """Against the polynomial at many points, which miss an extreme by 1e-8 of it."""
    g = torch.Generator().manual_seed(1)
    seen = set()
    for _ in range(300):
        a, b, c = ((torch.rand(3, generator=g, dtype=torch.float64) * 2 - 1) * torch.tensor([15.0, 20.0, 1.0])).tolist()
        c *= 10.0 ** -float(torch.randint(1, 22, (1,), generator=g))
        most, good, near = 1.0, True, False
        for _ in range(2):
            x = torch.linspace(0, most, 20001, dtype=torch.float64)
            q = (a + b * x ** 2 + c * x ** 4).abs()
            good = good and float(q.max()) <= 15 and float((x * q).max()) <= 3.8
            near = near or abs(float(q.max()) - 15) < 1e-5 or abs(float((x * q).max()) - 3.8) < 1e-5
            most = float((x * q).max())
        assert near or _allowed(2, (a, b, c)) == good, (a, b, c)
        seen.add(good)
    assert seen == {True, False}


def test_five_default_steps_as_documented():
    """Singular values of 0.002 of the norm and more end between 0.68 and 1.21, as the documentation of NEWTON_SCHULZ says: the
    polynomial at 2 * 10^6 points, between which five steps of a slope of 3.4445 at most move it by 5e-7 * 3.4445^5 = 2.4e-4."""
    import inspect

    from spherical_distortion.functional import token_ops
    a, b, c = token_ops.NEWTON_SCHULZ
    x = torch.linspace(0.002, 1, 2000001, dtype=torch.float64)
    for _ in range(5):
        x = a * x + b * x ** 3 + c * x ** 5
    assert 0.68 + 2.4e-4 <= float(x.min()) and float(x.max()) <= 1.21 - 2.4e-4
    assert "between 0.68 and 1.21" in inspect.getsource(token_ops) and float(x.max()) > 1.2


def test_coefficients_whose_roundings_grow():
    """3 x - x^3 takes 1 to 2 and 2 to -2, and 2 (1 + e) to -2 (1 + 9 e): what is rounded past 2 leaves.  2.6 x - x^3 stays within
    1.62, its largest value, whatever is rounded (2.6 * 1.62 - 1.62^3 = -0.04)."""
    assert _allowed(3, (3.0, -1.0, 0.0))
    for steps in (6, 8, 30, 100):
        assert not _allowed(steps, (3.0, -1.0, 0.0)) and not _allowed(steps, (-3.0, 1.0, 0.0))
        assert _allowed(steps, (2.6, -1.0, 0.0)) and _allowed(steps, NS) and _allowed(steps, (1.875, -1.25, 0.375))
        assert _allowed(steps, (1.5, -0.5, 0.0)) and _allowed(steps, (2.0, -1.5, 0.5))
