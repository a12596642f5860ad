"""Products of matmul_epilogue launch fewer than 2**32 threads: the library's choice at the largest outputs that a GPU
of 288 GB holds, and a config that would need more is refused."""

import ctypes

import pytest

import kernel_library as kl
from kernel_library import _lib

P = 1 << 44  # an address that nothing is at: these calls only plan

# Outputs of 137 to 280 GB over a short K, narrow and wide.
SHAPES = [(262800139, 531, 2), (218616084, 559, 2), (229501304, 547, 1), (541, 241662035, 8), (1 << 18, 1 << 18, 8),
          (1 << 20, 1 << 17, 64), (2**28 - 2**20, 500, 8)]


def _workspace(M, N, K, transposed, cfg=None):
    args = _lib.EpilogueArgs(P, 2 * P, None, None, 3 * P, None, M, N, K, transposed, 0, 0)
    need = ctypes.c_ulonglong()
    return _lib.lib().mi_matmul_epilogue_workspace(ctypes.byref(args), cfg and ctypes.byref(cfg.to_c()), ctypes.byref(need))


@pytest.mark.parametrize("transposed", [0, 1])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_default(M, N, K, transposed):
    c = _lib.MiTileCfg()
    assert _lib.lib().mi_epilogue_default_config(M, N, K, transposed, ctypes.byref(c)) == _lib.MI_OK
    assert -(-M // c.block_m) * -(-N // c.block_n) * c.split_k * c.waves * 64 < 2**32
    if M != 541 or transposed:  # (rhs[K,N]: loads of a K tile of 64 rows leave 32-bit offsets)
        assert _workspace(M, N, K, transposed) == _lib.MI_OK


def test_a_config_past_it_is_refused():
    small, large = kl.TileConfig(64, 64, 64, 4, 2), kl.TileConfig(256, 256, 64, 8, 2)
    assert _workspace(1 << 20, 1 << 17, 64, 0, large) == _lib.MI_OK
    assert _workspace(1 << 20, 1 << 17, 64, 0, small) == _lib.MI_E_RANGE
    assert _workspace(1 << 18, 1 << 18, 8, 1, small) == _lib.MI_E_RANGE
    assert _workspace(1 << 18, (1 << 18) - 64, 8, 1, small) == _lib.MI_OK


def test_few_rows_as_they_are():
    """Odd rows are read as they are by blocks of 64 x 64, which the widest rhs has too many of for a launch."""
    assert _workspace(256, (1 << 28) - 65, 8, 0) == _lib.MI_OK
    assert _workspace(256, (1 << 28) - 1, 8, 0) == _lib.MI_E_RANGE
