"""Scratch of the dense blocks' launches (K15 - K17): what the size functions ask for, over the sizes that the entries accept."""
import pytest


@pytest.fixture(scope='module')
def lib():
    from ursabench_amd import _native
    return _native.load_library()


@pytest.mark.parametrize('D', [1, 24, 128, 129, 512, 1024, 2048, 4096, 8192, 8193, 16384, 16385, 20000, 1 << 17, 1 << 20, (1 << 22) - 1, 1 << 22, 1 << 25, 1 << 27])
def test_the_norm_backward_stays_within_32_mib(lib, D):
    for M in (1, 2, 4, 5, 17, 64, 1000, 1 << 20, (1 << 31) - 1):
        floats = lib.ursa_layer_norm_ws_floats(M, D)
        assert 0 <= 4 * floats <= 32 << 20, (M, D)
        assert floats % (2 * D) == 0
        assert floats // (2 * D) <= (M + 3) // 4, (M, D)              # a row of partial sums for no less than four rows
    assert lib.ursa_layer_norm_ws_floats(0, D) == 0 and lib.ursa_layer_norm_ws_floats(-1, D) == 0
