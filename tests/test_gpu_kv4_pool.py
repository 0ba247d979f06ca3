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


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv", [1, 7, 96, 1000])
def test_append_and_gather_on_16_byte_boundaries_and_many_heads(ctx, dtype, n_kv):
    """Rows that start 16 bytes behind a wider boundary, at strides that are odd
    multiples of 16 bytes."""
    td, zd = TYPES[dtype]
    unit = 16 // td.itemsize
    n, wide = 21, n_kv * HD + unit
    rng = np.random.default_rng(n_kv)
    kv = cache(ctx, 3, 16, 1, n_kv)
    k, v = (torch.from_numpy(rng.standard_normal(n * wide + unit).astype(np.float32)).to(td).cuda() for _ in range(2))
    gk, gv = (torch.full_like(k, 5.0) for _ in range(2))
    slots = rng.permutation(48)[:n].astype(np.uint32)
    ds = dev(slots)
    at = unit * td.itemsize
    kv.append_device(0, n, k.data_ptr() + at, v.data_ptr() + at, ds.data_ptr(), dtype=zd, k_stride=wide, v_stride=wide, stream=1)
    kv.gather_device(0, n, ds.data_ptr(), gk.data_ptr() + at, gv.data_ptr() + at, dtype=zd, k_stride=wide, v_stride=wide, stream=1)
    torch.cuda.synchronize()
    for x, g in ((k, gk), (v, gv)):
        rows, got = (a[unit:].reshape(n, wide).double().cpu().numpy() for a in (x, g))
        want = torch.from_numpy(R.values(rows[:, :n_kv * HD].reshape(n, n_kv, HD))).to(td).double().numpy()
        assert np.array_equal(got[:, :n_kv * HD].reshape(n, n_kv, HD), want)
        assert (got[:, n_kv * HD:] == 5).all() and (g[:unit] == 5).all()
    kv.check()
    kv.close()


@pytest.mark.parametrize("n,width,block,share", [(1024, 40, 16, 0.5), (1024, 3, 128, 1.0), (37, 5000, 16, 0.3), (1000, 9, 32, 0.0)])
def test_release_of_many_rows(ctx, n, width, block, share):
    rng = np.random.default_rng(n + width)
    lens = rng.integers(0, width * block + 1, n).astype(np.uint32)
    lens[:2] = [0, width * block]
    held = -(-lens.astype(np.int64) // block)
    n_blocks = int(held.sum()) + 7
    order = rng.permutation(n_blocks).astype(np.uint32)
    table = np.full((n, width), NONE, np.uint32)
    at = 0
    for i in range(n):
        table[i, :held[i]] = order[at:at + held[i]]
        at += held[i]
    free = np.full(n_blocks, NONE, np.uint32)
    free[:7] = order[at:]
    done = (rng.random(n) < share).astype(np.uint32) * rng.integers(1, 1 << 32, n).astype(np.uint32)
    kv = cache(ctx, n_blocks, block, 1, 1)

    def go(table, lens):
        b = [dev(a) for a in (done, lens, table, free, np.array([7, 1, 2, 3], np.uint32))]
        kv.release_device(n, width, *[x.data_ptr() for x in b], stream=1)
        torch.cuda.synchronize()
        return [u32(x) for x in b[1:]]

    ln, tab, fl, st = go(table, lens)
    back = np.concatenate([table[i, :held[i]] for i in range(n) if done[i]] + [np.zeros(0, np.uint32)])
    assert np.array_equal(ln, np.where(done != 0, 0, lens)) and list(st) == [7 + len(back), 0, 0, len(back)]
    assert np.array_equal(fl[:7 + len(back)], np.concatenate([free[:7], back])) and (fl[7 + len(back):] == NONE).all()
    assert np.array_equal(tab, np.where(done[:, None] != 0, NONE, table))
    kv.check()
    if done.any():              # one bad block in the last row that ends refuses the whole call
        i = int(np.flatnonzero((done != 0) & (held > 0))[-1])
        broken = table.copy()
        broken[i, held[i] - 1] = n_blocks
        ln, tab, fl, st = go(broken, lens)
        assert np.array_equal(ln, lens) and np.array_equal(tab, broken) and np.array_equal(fl, free) and list(st) == [7, 2, 2, 3]
        with pytest.raises(zb.ZgpuError) as e:
            kv.check()
        assert e.value.status == 13
    kv.close()
