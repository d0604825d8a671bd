"""CPU: the workspace of an int8 product that splits K is checked before any HIP call (no pointer here is read)."""
import os

import pytest

from ferret_amd import lib

P = 1 << 24


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(lib.LIB_PATH):
        pytest.skip("libferret_hip.so not built")
    return lib.load()


# shapes whose K is split today: one of each kernel
@pytest.mark.parametrize("M,N,K", [(20, 520, 4096), (33, 2048, 4096)])
def test_workspace_of_a_split_product(L, M, N, K):
    need = L.ferret_int8_gemm_workspace(M, N, K)
    assert need > 0 and need % (4 * M * N) == 0
    a, sa, b, sb, r, y, ws = (i * P for i in (1, 2, 3, 5, 6, 7, 8))
    good = [a, sa, b, sb, r, y, M, N, K, ws, need, None]
    wrong = [(9, None, -3), (10, need - 1, -3), (10, 0, -3), (9, ws + 8, -3), (9, ws + 4, -3),
             # over what is read, and over the output
             (9, a, -2), (9, a + M * K - 16, -2), (9, b, -2), (9, b + N * K - 16, -2), (9, sa, -2), (9, sb, -2),
             (9, r, -2), (9, r + 16, -2), (9, y, -2), (9, y + 2 * M * N - 16, -2), (9, y - need + 16, -2)]
    for at, v, rc in wrong:
        args = list(good)
        args[at] = v
        assert L.ferret_int8_gemm(*args) == rc, (at, v)
    # nor where the output is the residual itself
    args = list(good)
    args[5] = r
    args[9] = r + 16
    assert L.ferret_int8_gemm(*args) == -2
