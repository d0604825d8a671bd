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


G = 1 << 40  # between tensors that do not overlap


def _refused(f, args, at, value):
    """The call with argument `at` changed; a call that is not refused would reach the device, of which there is none."""
    args = list(args)
    args[at] = value
    return f(*args) == -2


def test_a_read_of_the_cache_into_itself_is_refused(L):
    #       data scales pages page table cu B pages rows latent rotary stream
    args = [G, 2 * G, 100, 64, 3 * G, 4 * G, 3, 8, 50, 5 * G, 6 * G, None]
    end = {0: G + 100 * 64 * 640, 1: 2 * G + 100 * 64 * 4, 4: 3 * G + 3 * 8 * 4, 5: 4 * G + 16}
    for out in (9, 10):
        for read in end:
            assert _refused(L.ferret_latent_cache_read, args, out, args[read]), (out, read)
            assert _refused(L.ferret_latent_cache_read, args, out, (end[read] - 1) & ~15), (out, read)
        assert _refused(L.ferret_latent_cache_read, args, out, args[19 - out] + 16)


def test_a_write_of_what_stands_in_the_cache_is_refused(L):
    #       latent    rotary    table lens cu B pages T  data scales pages page stream
    args = [G, 576, 2 * G, 64, 3 * G, 4 * G, 5 * G, 3, 8, 5, 6 * G, 7 * G, 100, 64, None]
    for at in (0, 2, 4, 5, 6):
        for cache, size in ((10, 640), (11, 4)):
            assert _refused(L.ferret_latent_cache_write, args, at, args[cache] + 100 * 64 * size - 64), (at, cache)
    assert _refused(L.ferret_latent_cache_write, args, 11, 6 * G + 64)
    assert _refused(L.ferret_latent_cache_write, args, 0, 6 * G - 4 * 576 * 2 - 512 * 2 + 16)   # its last row's end


def test_absorbed_outputs_and_workspace_stand_apart(L):
    need = L.ferret_latent_attention_workspace(3, 5, 16)
    #       ql    t     h    qr  t     h   data scales pages page table lens cu B mp T  H  scale causal out lse ws bytes st
    args = [G, 8192, 512, 2 * G, 1024, 64, 3 * G, 4 * G, 100, 64, 5 * G, 6 * G, 7 * G, 3, 8, 5, 16, 0.07, 1, 8 * G, 9 * G,
            10 * G, need, None]
    f = L.ferret_latent_attention
    for written in (19, 20, 21):
        for other in (0, 3, 6, 7, 10, 11, 12, 19, 20, 21):
            if other != written:
                assert _refused(f, args, written, args[other] + (16 if other == 0 else 0)), (written, other)
    # an output exactly on packed queries is in place; on the rows of others it is not
    assert _refused(f, [*args[:1], 8208, *args[2:]], 19, G) and _refused(f, [*args[:2], 1024, *args[3:]], 19, G)


def test_expanded_outputs_and_workspace_stand_apart(L):
    need = L.ferret_latent_attention_expanded_workspace(2, 9, 8000, 16)
    #       qn    t     h    qr   t    h   kn   s     h   kr  s   v   s     h   cu cu B  T  S  H scale causal out lse ws bytes st
    args = [G, 2048, 128, 2 * G, 1024, 64, 3 * G, 4096, 256, 4 * G, 64, 5 * G, 4096, 256, 6 * G, 7 * G, 2, 9, 8000, 16, 0.07, 1,
            8 * G, 9 * G, 10 * G, need, None]
    f = L.ferret_latent_attention_expanded
    for written in (22, 23, 24):
        for other in (0, 3, 6, 9, 11, 14, 15, 22, 23, 24):
            if other != written:
                assert _refused(f, args, written, args[other] + (16 if other == 0 else 0)), (written, other)
    assert _refused(f, [*args[:1], 2056, *args[2:]], 22, G)


def test_keys_that_32_bits_do_not_count_are_refused(L):
    """Steps of 64 keys end past 2^31 where a sequence may have more than 2^31 - 128 keys (a table may name a page
    many times); the expanded form's search for a tile passes 2^31 from about 2.1e9 keys on (keys may have stride 0)."""
    need = L.ferret_latent_attention_workspace(1, 1, 16)
    args = [G, 8192, 512, 2 * G, 1024, 64, 3 * G, 4 * G, 100, 16, 5 * G, 6 * G, 7 * G, 1, 8, 1, 16, 0.07, 1, 8 * G, 9 * G,
            10 * G, need, None]
    for max_pages in ((1 << 27) - 1, (1 << 27) - 7):
        assert _refused(L.ferret_latent_attention, args, 14, max_pages)
    args = [G, 2048, 128, 2 * G, 1024, 64, 3 * G, 0, 0, 4 * G, 0, 5 * G, 0, 0, 6 * G, 7 * G, 1, 9, 8000, 16, 0.07, 1, 8 * G,
            9 * G, 10 * G, 1 << 30, None]
    for keys in ((1 << 30) + 1, (1 << 31) - 1):
        assert _refused(L.ferret_latent_attention_expanded, args, 18, keys)
