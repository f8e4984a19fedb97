"""Host-only: sizes that the norm's kernels could not count in 32 bits are refused before a launch."""
import ctypes as C

import pytest

import cabi
import cabi_mixer as mixer

OK, E_TOO_LARGE = 0, -16
LAST = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib(cc1d_lib):
    return mixer.declare_mixer(cabi.declare(cc1d_lib))


def block(cls, dim, rows=2):
    p = cls()
    p.rows, p.dim = rows, dim
    for name, _ in cls._fields_:
        if name in ("x", "h", "residual", "y", "y8", "scales", "weight", "dy", "dh", "dx", "dresidual", "dweight"):
            setattr(p, name, 256)
    if cls is mixer.NormParams:
        p.y8 = p.scales = None
    return p


def test_rows_of_nearly_2_31_elements(lib):
    """Lanes step along a row by 8192 elements: the last step of a row longer than 2^31 - 1 - 8192 would leave 32 bits, come back
    negative and read in front of the row, without end."""
    n = C.c_size_t()
    for dim, want in ((LAST - 8192, OK), (LAST - 8191, E_TOO_LARGE), (LAST, E_TOO_LARGE)):
        p = block(mixer.NormParams, dim)
        assert lib.cc1d_validate_norm(p) == want, dim
        if want != OK:
            assert lib.cc1d_norm_fwd(p, None) == want
        assert lib.cc1d_validate_dequantize(block(mixer.DequantizeParams, dim)) == OK          # a vector a thread: no steps
        assert lib.cc1d_validate_norm(block(mixer.NormParams, dim, rows=0)) == OK
    for dim, want in ((2 ** 27 - 32, OK), (2 ** 27 - 31, E_TOO_LARGE), (LAST, E_TOO_LARGE)):   # dweight: 1024 threads for 32 columns, fewer than 2^32 in all
        p = block(mixer.NormBwdParams, dim)
        assert lib.cc1d_validate_norm_bwd(p) == want, dim
        if want != OK:
            assert lib.cc1d_norm_bwd_workspace_bytes(p, C.byref(n)) == want and lib.cc1d_norm_bwd(p, None, 0, None) == want
