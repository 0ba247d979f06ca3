"""Append, release and plan of the paged 4-bit cache at their documented limits."""
import numpy as np
import pytest

import kv4_ref as R
import zero_b200 as zb
from test_gpu_kv4 import HD, NONE, TYPES, cache, dev, fetch, store, u32

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_refuses_every_magnitude_above_its_limit(ctx, dtype):
    """21760 and the next values above it, of both signs, in K and in V: the
    largest is stored, and a group that holds one above is zeros and recorded."""
    above = {"f32": [np.nextafter(np.float32(21760), np.float32(1e9)), 21770.0, 21823.0, 21824.0],
             "f16": [21776.0, 21792.0, 21824.0], "bf16": [21888.0]}[dtype]
    kv = cache(ctx, 1, 16, 1, 1)
    rng = np.random.default_rng(3)
    for big in above:
        for sign in (1, -1):
            x = rng.standard_normal((3, 1, HD)).astype(np.float32)
            y = rng.standard_normal((3, 1, HD)).astype(np.float32)
            x[0, 0, 5], x[1, 0, 37], y[1, 0, 127] = sign * 21760.0, sign * big, -sign * big
            kt, vt = (torch.from_numpy(a).to(TYPES[dtype][0]).double().numpy() for a in (x, y))
            store(kv, 0, np.arange(3, dtype=np.uint32), x, y, dtype)
            with pytest.raises(zb.ZgpuError) as e:
                kv.check()
            assert e.value.status == 20
            want_k, want_v = R.values(kt), R.values(vt)
            want_k[1, 0, 32:64] = 0
            want_v[1, 0, 96:] = 0
            gk, gv = fetch(kv, 0, np.arange(3), "f32", 1)
            assert np.array_equal(gk, want_k) and np.array_equal(gv, want_v), (big, sign)
    x = np.full((1, 1, HD), 21760.0, np.float32)
    store(kv, 0, np.zeros(1, np.uint32), x, -x, dtype)
    kv.check()
    kv.close()
