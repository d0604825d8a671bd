"""GPU: the attention block at the edges of what its entry points take."""
import numpy as np
import pytest
import torch

from ferret_amd import lib
from tests.attention_helpers import bf16_tensor, bf16_values, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip):
    from ferret_amd import ops as O
    return O


@pytest.mark.parametrize("native", [True, False])
def test_expanded_rows_are_refused(ops, native, monkeypatch):
    """Many rows of one row's storage, which a row pitch cannot name; nothing is written."""
    print(f"[case] expanded rows, native={native}", flush=True)
    if not native:
        monkeypatch.setattr(lib, "native", lambda: lib._Absent())
    rng = np.random.default_rng(1)
    x, w, r = (bf16_tensor(bf16_values(rng, *s)) for s in ((64, 512), (512,), (64, 64)))
    one, out = x[:1].expand(64, 512), torch.full((64, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ops.rms_norm(one, w, out=out), lambda: ops.rms_norm_e4m3(one, w)):
        with pytest.raises(ValueError, match="x's rows"):
            call()
    for call in (lambda: ops.rms_norm(x, w, one, out=out), lambda: ops.rms_norm_e4m3(x, w, one)):
        with pytest.raises(ValueError, match="residual's rows"):
            call()
    cache, table = ops.LatentCache.empty(4, 16), i32(range(4)).view(1, 4)
    with pytest.raises(ValueError, match="latent's rows"):
        ops.latent_cache_write(cache, one, r, table, i32([64]), i32([0, 64]))
    with pytest.raises(ValueError, match="rotary's rows"):
        ops.latent_cache_write(cache, x, r[:1].expand(64, 64), table, i32([64]), i32([0, 64]))
    torch.cuda.synchronize()
    assert (out == 7).all() and (cache.data == 0).all()
    # one row has any stride
    assert torch.equal(ops.rms_norm(x[0].expand(1, 512), w)[0], ops.rms_norm(x[:1], w)[0])
