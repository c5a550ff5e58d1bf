"""Arguments of the layer norm's and the orthogonalised updates' binding that a C int does not hold, and outputs given twice: refused in front of any launch."""
import pytest
import torch

from encodermap_amd import _lib

P = 1 << 20    # an address that nothing reads


def test_sizes_that_an_int_does_not_hold():
    wide = torch.empty(1, 2 ** 32 + 8, dtype=torch.float16, device="meta")
    with pytest.raises(_lib.EmxError):
        _lib.layernorm_fwd(wide, None, None, 1e-3, wide)
    for n, D in ((4, 2 ** 32 + 8), (4, 0), (-1, 8), (2 ** 63, 8), (4, 2 ** 28 + 1)):
        with pytest.raises(_lib.EmxError, match="layernorm_ws_floats"):
            _lib.layernorm_ws_floats(n, D)
    for value in (2 ** 32 + 5, -2 ** 31 - 1, 2 ** 31):
        with pytest.raises(_lib.EmxError, match="steps"):
            _lib._int32(value, "steps")
    assert _lib._int32(2 ** 31 - 1, "steps") == 2 ** 31 - 1


def test_parts_hold_few_rows():
    """a thread adds a part's rows one after the other: 512 at most, up to 2^25 rows"""
    for n, D in ((1 << 20, 8), (1 << 24, 128), (1 << 25, 1), (10 ** 7, 1 << 17)):
        parts = _lib.layernorm_ws_floats(n, D) // (2 * D)
        assert parts * 512 >= n - 512
    assert _lib.layernorm_ws_floats(1 << 60, 1) == 2 * 65535


def test_outputs_given_twice():
    lib = _lib.load()
    assert lib.emx_layernorm_fwd(P, 0, 4, 8, 8, None, None, 1e-3, 2 * P, 8, 3 * P, 3 * P, None) == -1 and b"the same vector" in lib.emx_last_error()
    ws = _lib.layernorm_ws_floats(4, 8)
    assert lib.emx_layernorm_bwd(P, 8, 2 * P, 8, 0, 4, 8, None, 3 * P, 4 * P, 5 * P, 8, 6 * P, 6 * P, 7 * P, ws, None) == -1
    assert b"the same vector" in lib.emx_last_error()
