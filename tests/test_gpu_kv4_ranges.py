"""Attention of the paged 4-bit cache at the ends of its number ranges: rows of
zeros and tiny rows under tiny scales, rows as large and as small as their type
holds, and scores whose products are far larger than their sums.

Bounds are those of test_gpu_kv4.check_attn unless a test derives its own."""
import numpy as np
import pytest

import kv4_ref as R
import zero_b200 as zb
from test_gpu_kv4 import HD, NONE, TYPES, cache, check_attn, make, run_attn, store

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 3, 140])
@pytest.mark.parametrize("scale", [1e-10, 9e-16, 1e-30, 1e-38])
def test_zero_and_tiny_rows_under_a_tiny_scale(ctx, dtype, nq, scale):
    """Scores of nearly 0: a row's result is the mean of the values that it sees."""
    c = make(ctx, 40 + nq, [300, nq + 2], [nq, nq], 4, 2, 16)
    c["q"][0] = 0
    c["q"][nq:, 1] = 0
    c["q"][nq // 2, 2] *= 1e-5 if dtype == "f16" else 2.0 ** -100
    o, q = run_attn(c, dtype, scale)
    check_attn(c, o, q, dtype, float(np.float32(scale)))
    c["kv"].check()
    c["kv"].close()


def cancelling(rng, n, n_kv, amp):
    """A query of all magnitudes up to 2 amp and keys [n, n_kv, HD] of whole numbers
    -8..7 (scale 1, exact in the cache), whose products reach 16 amp while
    their sum is at most about 1."""
    q = rng.choice([-1.0, 1.0], HD) * amp * np.exp2(-rng.integers(0, 12, HD)) * (1 + rng.random(HD))
    q = q.astype(np.float16).astype(np.float64)
    keys = np.zeros((n, n_kv, HD))
    for t in range(n):
        for h in range(n_kv):
            k = rng.integers(-7, 8, HD).astype(np.float64)
            k[::32] = -8                     # the group's largest: its scale is 1
            free = np.arange(HD) % 32 != 0
            for _ in range(400):             # the step that leaves least
                s = q @ k
                if abs(s) < 1:
                    break
                up, down = np.where(free & (k < 7), abs(s + q), np.inf), np.where(free & (k > -7), abs(s - q), np.inf)
                i, j = up.argmin(), down.argmin()
                if min(up[i], down[j]) < abs(s):
                    k[i if up[i] < down[j] else j] += 1 if up[i] < down[j] else -1
                else:
                    k[rng.choice(np.flatnonzero(free))] = rng.integers(-7, 8)
            keys[t, h] = k
    return q, keys


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 40])
def test_scores_of_16_bit_rows_are_summed_as_exactly_as_those_of_f32_rows(ctx, dtype, nq):
    """The same rows in f32 and in 16 bits.  Beside what the f32 call is off by, a
    16-bit result is off by its own rounding and by a probability of 11 bits;
    a sum of scores in fewer than f32's bits would show: the largest product is 2048,
    and a probability's last place is worth 2^-11 of a score."""
    rng = np.random.default_rng(6)
    n, n_kv, block = 16 + nq - 1, 2, 16
    q1, keys = cancelling(rng, n, n_kv, 128.0)
    q1 = torch.from_numpy(q1).to(TYPES[dtype][0]).double().numpy()
    kv = cache(ctx, -(-n // block), block, 1, n_kv)
    vals = rng.standard_normal((n, n_kv, HD)).astype(np.float32)
    store(kv, 0, np.arange(n, dtype=np.uint32), keys, vals)
    c = dict(kv=kv, table=np.arange(-(-n // block), dtype=np.uint32)[None], lens=np.array([n], np.uint32),
             starts=np.array([0, nq], np.uint32), layer=0, n_q=n_kv, n_kv=n_kv, width=-(-n // block),
             q=np.broadcast_to(q1, (nq, n_kv, HD)).astype(np.float32).copy(), ks=[keys], vs=[R.values(vals)])
    assert np.array_equal(R.values(keys), keys)
    wide, q = run_attn(c, "f32", 1.0)
    o, _ = run_attn(c, dtype, 1.0)
    ref, mass, _, _ = R.attention(q, keys, c["vs"][0], 1.0)
    half = torch.finfo(TYPES[dtype][0]).eps / 2
    tol = 2 * np.abs(wide - ref).max() + 2.0 ** -11 * mass + half * np.abs(ref) + 2.0 ** -21
    err = np.abs(o - ref)
    assert (err <= tol).all(), float((err / tol).max())
    kv.check()
    kv.close()


@pytest.mark.parametrize("dtype,gain,scale", [
    ("f32", 4e37, 2.2e-39), ("f32", 3e36, 2.9e-38), ("f32", 1e-33, 8.8e31), ("f32", 1e-37, 8.8e35), ("f32", 1e-40, 3.3e38),
    ("bf16", 4e37, 2.2e-39), ("bf16", 3e36, 2.9e-38), ("bf16", 1e-33, 8.8e31), ("bf16", 1e-37, 8.8e35), ("bf16", 1e-40, 3.3e38),
    ("f16", 1e4, 8.8e-6), ("f16", 3e-7, 3e5), ("f16", 30.0, 0.09), ("bf16", 30.0, 0.09), ("bf16", 1e4, 1e-3)])
@pytest.mark.parametrize("lens,nq", [([300, 41], [1, 3]), ([300, 141], [160, 141])])
def test_rows_at_the_ends_of_their_types(ctx, dtype, gain, scale, lens, nq):
    """Rows of the largest and of subnormal values in both kernels, and sharp
    scores of 16-bit rows."""
    c = make(ctx, 50, lens, nq, 4, 2, 16, qgain=gain)
    o, q = run_attn(c, dtype, scale)
    assert np.isfinite(q).all() and q.any()
    check_attn(c, o, q, dtype, float(np.float32(scale)))
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 3, 140])
@pytest.mark.parametrize("size", [1e5, 3e6, 4e7, 1e8])
def test_scores_far_apart(ctx, dtype, nq, size):
    """Scores up to 10^8: a row is the value of its largest score, to that value's
    rounding, where the next score is clearly smaller, and finite anyway.  With
    16-bit rows the probability, 1 up to a power of two that need not be whole, is
    one binary16 value over an f32 sum: 2^-11 on top."""
    c = make(ctx, 60, [700, nq + 90], [nq, nq], 4, 2, 16, qgain=30.0)
    scale = float(np.float32(size / (30 * 40)))         # the largest q k of some hundred keys is about 30 x 40
    o, q = run_attn(c, dtype, scale)
    half = torch.finfo(TYPES[dtype][0]).eps / 2
    clear = 0
    for i, n in enumerate(c["lens"]):
        a = int(c["starts"][i])
        _, _, _, ds = R.attention(q[a:a + nq], c["ks"][i], c["vs"][i], scale)
        for t in range(nq):
            see = int(n) - nq + t + 1
            for h in range(4):
                s = c["ks"][i][:see, h // 2] @ q[a + t, h] * scale
                first, second = np.argsort(-s)[:2]
                row, v = o[a + t, h], c["vs"][i][:see, h // 2]
                assert np.isfinite(row).all() and (np.abs(row) <= np.abs(v).max(0) * (1 + 2 * half + 2.0 ** -11) + 2.0 ** -20).all()
                if s[first] - s[second] > 2 * ds[t, h] + 40:      # the others weigh less than e^-40
                    clear += 1
                    assert (np.abs(row - v[first]) <= (half + 2.0 ** -20 + (2.0 ** -11 if dtype != "f32" else 0)) * np.abs(v[first]) + 2.0 ** -30).all()
    assert clear > nq or size > 1e7
    c["kv"].check()
    c["kv"].close()
