"""CPU: limits of the attention's entry points that hold before any HIP call (no pointer here is read)."""
import os

import pytest

from ferret_amd import lib

P = 1 << 20


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(lib.LIB_PATH):
        pytest.skip("libferret_hip.so not built")
    return lib.load()


@pytest.mark.parametrize("B,T,S,H,parts", [(1, 1, 2000, 1, 5), (1, 3, 1200, 1, 3), (1, 5, 2700, 3, 7), (2, 9, 8000, 16, 8)])
def test_partial_outputs_stand_on_16_byte_bounds(L, B, T, S, H, parts):
    """The maxima and sums (8 bytes a row and part) come first in the workspace, then the outputs, read 16 bytes
    at a time."""
    rows = parts * T * H
    assert L.ferret_latent_attention_expanded_workspace(B, T, S, H) == -(-rows * 8 // 16) * 16 + rows * 512
