"""CPU: sizes that the attention refuses before anything is launched (no pointer here is read)."""
import os

import pytest

from ferret_amd import lib

G = 1 << 45  # between tensors that do not overlap


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(lib.LIB_PATH):
        pytest.skip("libferret_hip.so not built")
    return lib.load()


# T * H past 2^26 - 16: the join of the last 16 rows would be the launch's thread 2^32
PAST = [((1 << 26) - 15, 1), (1 << 26, 1), (1 << 20, 64), (1 << 16, 1024), (1 << 24, 128), ((1 << 31) - 1, 1)]


@pytest.mark.parametrize("T,H", PAST)
def test_absorbed_query_rows_past_the_joins_launch(L, T, H):
    """Refused as a whole, so that no kernel has written part of `out` when the join cannot be launched."""
    assert L.ferret_latent_attention_workspace(1, T, H) == 0
    #       ql t        h    qr     t       h   data   scales pages page table lens cu
    args = [G, H * 512, 512, 2 * G, H * 64, 64, 3 * G, 4 * G, 100, 64, 5 * G, 6 * G, 7 * G, 1, 1, T, H, 0.07, 1, 8 * G, None,
            9 * G, 1 << 44, None]  # B max_pages T H scale causal out lse ws bytes stream
    assert L.ferret_latent_attention(*args) == -2


@pytest.mark.parametrize("T,H", PAST)
def test_shared_query_rows_past_the_joins_launch(L, T, H):
    assert L.ferret_latent_attention_shared_workspace(1, 1, T, H) == 0
    args = [G, H * 512, 512, 2 * G, H * 64, 64, 3 * G, 4 * G, 100, 64, 5 * G, 6 * G, 7 * G, 1, 1, 8 * G, 9 * G, 10 * G, 1, 1,
            T, H, 0.07, 1, 11 * G, None, 12 * G, 1 << 44, None]
    assert L.ferret_latent_attention_shared(*args) == -2


def test_the_most_query_rows_have_a_workspace(L):
    for T, H in (((1 << 26) - 16, 1), ((1 << 22) - 1, 16)):
        assert L.ferret_latent_attention_workspace(1, T, H) > 0
        assert L.ferret_latent_attention_shared_workspace(1, 1, T, H) > 0
