"""How large a step with shared prefixes may be: its partial rows, two for every token and
query head and 128 for each of 512 units, are numbered in 32 bits."""
import ctypes

import pytest

from auto_infer_amd import _native

MOST = 2 ** 31 - 1 - 512 * 128


def bytes_of(tokens, hq, hkv, batch=4):
    out = ctypes.c_int64(0)
    code = _native.load().aia_shared_workspace_bytes(batch, tokens, hq, hkv, 128, 16, 64, ctypes.byref(out))
    return code, out.value


@pytest.mark.parametrize("hq,hkv", [(64, 8), (16, 8), (28, 4), (1, 1)])
def test_largest_step(hq, hkv):
    most = MOST // (2 * hq)
    code, size = bytes_of(most, hq, hkv)
    assert code == 0 and size > 2 * most * hq * 128 * 2
    assert bytes_of(most // 3, hq, hkv)[0] == 0
    code, _ = bytes_of(most + 1, hq, hkv)
    assert code == _native.AIA_ERR_UNSUPPORTED and "tokens" in _native.last_error()
