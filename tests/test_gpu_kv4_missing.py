"""Attention of the paged 4-bit cache with blocks that are not in the pool, in
both kernels and at every place that a kernel looks them up, and over sequences
long enough that a warp fetches its addresses several times.

The bounds are those of test_gpu_kv4.check_attn, row by row: a row's result is
what its present keys alone give."""
import numpy as np
import pytest

import kv4_ref as R
import zero_b200 as zb
from test_gpu_kv4 import HD, TYPES, cache, make, run_attn, store

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def check_rows(c, o, q, dtype, i, present, rows=None):
    """Rows of sequence i against the keys that are present and not behind them."""
    half = torch.finfo(TYPES[dtype][0]).eps / 2
    a, b, n = int(c["starts"][i]), int(c["starts"][i + 1]), int(c["lens"][i])
    for t in range(b - a) if rows is None else rows:
        keep = np.flatnonzero(present[:n - (b - a) + t + 1])
        ref, mass, total, ds = R.attention(q[a + t:a + t + 1], c["ks"][i][keep], c["vs"][i][keep], HD ** -0.5)
        rel = 2 * ds[..., None] + 2.0 ** -21 + (n / 16 + 64) * 2.0 ** -23 + (2.0 ** -11 if dtype != "f32" else 0)
        tol = rel * mass + 2.0 ** (-40 if dtype == "f32" else -32) * total + half * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 0)
        err = np.abs(o[a + t:a + t + 1] - ref)
        assert (err <= tol).all(), (i, t, len(keep), float((err / np.maximum(tol, 1e-300)).max()))


def recorded(c):
    with pytest.raises(zb.ZgpuError) as e:
        c["kv"].check()
    assert e.value.status == 10
    c["kv"].check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("nq", [1, 5, 150])
def test_missing_blocks_are_left_out(ctx, dtype, block, nq):
    """Blocks missing in an early key tile, in later ones, at the diagonal of the
    last queries and, for sequence 1, all of them but the last."""
    lens = [900, 400]
    c = make(ctx, block + nq, lens, [nq, nq], 4, 2, block)
    n_blocks = [-(-n // block) for n in lens]
    gone = [{1, 300 // block, 500 // block + 1, n_blocks[0] - 1}, set(range(n_blocks[1] - 1))]
    present = []
    for i, n in enumerate(lens):
        for j in gone[i]:
            c["table"][i, j] = (0x7FFFFFFF, 0xFFFFFFFF, len(c["table"]) * 1000)[j % 3]
        present.append(~np.isin(np.arange(n) // block, list(gone[i])))
    o, q = run_attn(c, dtype)
    recorded(c)
    rows = sorted({0, nq // 3, nq // 2, nq - 1} | set(range(max(0, nq - 12), nq)))
    for i in range(2):
        check_rows(c, o, q, dtype, i, present[i], rows)
    first = (n_blocks[1] - 1) * block - (lens[1] - nq)       # queries of sequence 1 before its only block
    if first > 0:
        a = int(c["starts"][1])
        assert not o[a:a + first].any() and o[a + first:a + nq].any(-1).all()
    c["kv"].close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("block,nq,n_q", [(16, 1, 2), (64, 1, 2), (16, 2, 8), (32, 1, 2), (16, 130, 2)])
def test_long_sequences_with_and_without_missing_blocks(ctx, dtype, block, nq, n_q):
    """128 sequences (8 of prompt chunks) of up to 12000 keys on the same blocks in
    orders of their own: a CTA's range is over 8192 keys of a piece, so each warp
    fetches its addresses more than once.  Some sequences lack a twentieth of
    their blocks, at places of their own."""
    n, n_kv, n_seq = 12000, 2, 128 if nq < 100 else 8
    rng = np.random.default_rng(block + nq)
    n_blocks = n // block + 1
    kv = cache(ctx, n_blocks, block, 1, n_kv)
    k, v = (rng.standard_normal((n_blocks * block, n_kv, HD)).astype(np.float32) for _ in range(2))
    store(kv, 0, np.arange(n_blocks * block, dtype=np.uint32), k, v)
    k, v = R.values(k), R.values(v)
    lens = [n - int(x) for x in rng.integers(0, 2000, n_seq)]
    table = np.stack([rng.permutation(n_blocks) for _ in range(n_seq)]).astype(np.uint32)
    checked = list(range(0, n_seq, n_seq // 4)) + [n_seq - 1]
    present = {}
    c = dict(kv=kv, lens=np.asarray(lens, np.uint32), starts=(np.arange(n_seq + 1) * nq).astype(np.uint32), layer=0,
             n_q=n_q, n_kv=n_kv, width=n_blocks, ks={}, vs={},
             q=rng.standard_normal((n_seq * nq, n_q, HD)).astype(np.float32))
    for i in range(n_seq):
        gone = rng.choice(n_blocks, n_blocks // 20, replace=False) if i % 2 else np.zeros(0, int)
        pos = np.arange(lens[i])
        if i in checked:
            slots = table[i][pos // block].astype(np.int64) * block + pos % block
            c["ks"][i], c["vs"][i] = k[slots], v[slots]
            present[i] = ~np.isin(pos // block, gone)
        table[i, gone] = n_blocks + 5
    c["table"] = table
    o, q = run_attn(c, dtype)
    recorded(c)
    for i in checked:
        check_rows(c, o, q, dtype, i, present[i], None if nq < 100 else [0, nq // 2, nq - 1])
    kv.close()
