"""The paged 4-bit KV cache on the GPU, through the C ABI, against plain
64-bit restatements (kv4_ref).

Whole numbers (plan, quantised values) are equal.  The attention is held to a
bound that its arithmetic gives: a score is off by at most ds (queries kept to
22 bits, products exact, f32 sums), which moves a probability by 2 ds
relatively; exp2 and the split of P in two halves add 2^-21, the f32 sums over
the keys 2^-23 for each of the about len / 16 steps; all of it times
sum p |v|.  The halves of a probability are held times 2^15 in binary16, whose
last place is 2^-24 at least: a probability is off by up to 2^-25 / 2^15 = 2^-40
of the row's largest on top, hence 2^-40 sum |v| (where the row's largest key
has a value of 0, nothing else is left); with 16-bit rows and many queries
times 2^7, hence 2^-32.  A 16-bit result is off by another half step, and a kernel that
takes 16-bit rows may hold a probability in binary16 (2^-11 of it)."""
import numpy as np
import pytest

import kv4_ref as R
import zero_b200 as zb
from zero_b200._lib import LIB

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HD, NONE = 128, R.NONE
TYPES = {"f32": (torch.float32, zb.F32), "f16": (torch.float16, zb.F16), "bf16": (torch.bfloat16, zb.BF16)}


def dev(a):
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint32:
        a = a.view(np.int32)
    return torch.from_numpy(a).to("cuda")


def u32(t):
    return t.cpu().numpy().view(np.uint32)


def cache(ctx, n_blocks=8, block=16, layers=1, n_kv=2):
    return zb.KvCache4(ctx, n_blocks, block, layers, n_kv, HD)


def store(kv, layer, slots, k, v, dtype="f32"):
    td, zd = TYPES[dtype]
    dk, dv, ds = dev(np.asarray(k, np.float32)).to(td), dev(np.asarray(v, np.float32)).to(td), dev(slots)
    kv.append_device(layer, len(slots), dk.data_ptr(), dv.data_ptr(), ds.data_ptr(), dtype=zd, stream=1)
    torch.cuda.synchronize()


def fetch(kv, layer, slots, dtype="f32", n_kv=2):
    td, zd = TYPES[dtype]
    k = torch.full((len(slots), n_kv, HD), 7.0, dtype=td, device="cuda")
    v = torch.full_like(k, 7.0)
    ds = dev(np.asarray(slots, np.uint32))
    kv.gather_device(layer, len(slots), ds.data_ptr(), k.data_ptr(), v.data_ptr(), dtype=zd, stream=1)
    torch.cuda.synchronize()
    return k.double().cpu().numpy(), v.double().cpu().numpy()


# ---------------------------------------------------------- append / gather
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block,n,n_kv", [(16, 1, 1), (16, 37, 2), (32, 64, 3), (64, 200, 8), (128, 131, 2)])
def test_append_then_gather_gives_the_formats_values(ctx, dtype, block, n, n_kv):
    rng = np.random.default_rng(n * 7 + n_kv)
    n_blocks = -(-n // block) + 3
    kv = cache(ctx, n_blocks, block, 2, n_kv)
    k = torch.from_numpy(rng.standard_normal((n, n_kv, HD)).astype(np.float32)).to(TYPES[dtype][0]).double().numpy()
    v = torch.from_numpy((0.3 * rng.standard_normal((n, n_kv, HD))).astype(np.float32)).to(TYPES[dtype][0]).double().numpy()
    slots = rng.permutation(n_blocks * block)[:n].astype(np.uint32)
    store(kv, 1, slots, k, v, dtype)
    gk, gv = fetch(kv, 1, slots, "f32", n_kv)
    assert np.array_equal(gk, R.values(k)) and np.array_equal(gv, R.values(v))
    hk, _ = fetch(kv, 1, slots, "f16", n_kv)
    assert np.array_equal(hk, gk)
    bk, _ = fetch(kv, 1, slots, "bf16", n_kv)
    assert np.array_equal(bk, torch.from_numpy(gk).to(torch.bfloat16).double().numpy())
    rest = np.setdiff1d(np.arange(n_blocks * block), slots).astype(np.uint32)
    ok, ov = fetch(kv, 1, rest, "f32", n_kv)
    assert not ok.any() and not ov.any(), "other slots untouched"
    ok, ov = fetch(kv, 0, slots, "f32", n_kv)
    assert not ok.any() and not ov.any(), "other layer untouched"
    kv.check()
    kv.close()


def test_append_borders_ties_and_scales(ctx):
    """Values on the borders between integers, equal magnitudes of both signs,
    zero groups, the smallest and largest scales: equal to the definition."""
    rng = np.random.default_rng(3)
    rows = [np.zeros(HD)]
    for d in (1.0, 2.0 ** -14, 2.0 ** -24, 3 * 2.0 ** -24, 255 * 2.0 ** -20, 2720.0, 171 / 256):
        x = (rng.integers(-17, 16, HD) / 2.0) * d           # halves: every second one is a tie
        x[::32] = -8 * d
        rows += [x, -x, np.nextafter(x.astype(np.float32), np.float32(0)), np.nextafter(x.astype(np.float32), np.float32(1e9))]
    x = rng.standard_normal(HD)
    x[5], x[9] = 4.0, -4.0
    y = x.copy()
    y[5], y[9] = -4.0, 4.0
    rows += [x, y, np.full(HD, 2.0 ** -26), np.full(HD, 2.0 ** -22), np.full(HD, 1e-30), np.full(HD, 21760.0),
             np.where(np.arange(HD) % 32 == 31, 1e4, 1e-3)]
    for s in np.exp2(rng.uniform(-26, 13, 300)):
        rows.append(s * rng.standard_normal(HD))
    x = np.clip(np.array(rows), -21760, 21760).astype(np.float32)[:, None, :]
    n = len(x)
    kv = cache(ctx, -(-n // 16), 16, 1, 1)
    store(kv, 0, np.arange(n, dtype=np.uint32), x, -x[::-1].copy())
    gk, gv = fetch(kv, 0, np.arange(n), "f32", 1)
    assert np.array_equal(gk, R.values(x)) and np.array_equal(gv, R.values(-x[::-1]))
    kv.check()
    kv.close()


def test_append_refuses_what_it_cannot_hold(ctx):
    x = np.ones((4, 1, HD), np.float32)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 70], x[3, 0, 127] = np.nan, np.inf, -21900.0, -np.inf
    kv = cache(ctx, 1, 16, 1, 1)
    store(kv, 0, np.arange(4, dtype=np.uint32), x, np.ones_like(x))
    with pytest.raises(zb.ZgpuError) as e:
        kv.check()
    assert e.value.status == 20
    kv.check()      # reported once
    gk, _ = fetch(kv, 0, np.arange(4), "f32", 1)
    want = np.ones((4, 1, 4, 32))
    for i, g in enumerate((0, 1, 2, 3)):
        want[i, 0, g] = 0       # the whole group
    assert np.array_equal(gk, want.reshape(4, 1, HD))
    kv.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_reads_fused_rows_and_skips_padding(ctx, dtype):
    """k and v as columns of wider rows; NONE skips, a slot behind the pool is
    recorded and skipped."""
    rng = np.random.default_rng(11)
    td, zd = TYPES[dtype]
    n, n_kv, n_q = 33, 2, 4
    qkv = torch.from_numpy(rng.standard_normal((n, (n_q + 2 * n_kv) * HD)).astype(np.float32)).to(td).cuda()
    slots = rng.permutation(64)[:n].astype(np.uint32)
    slots[[4, 20]] = NONE
    slots[7] = 64
    kv = cache(ctx, 4, 16, 1, n_kv)
    ds = dev(slots)
    es = qkv.element_size()
    kv.append_device(0, n, qkv.data_ptr() + n_q * HD * es, qkv.data_ptr() + (n_q + n_kv) * HD * es, ds.data_ptr(),
                     dtype=zd, k_stride=qkv.stride(0), v_stride=qkv.stride(0), stream=1)
    torch.cuda.synchronize()
    with pytest.raises(zb.ZgpuError) as e:
        kv.check()
    assert e.value.status == 10
    host = qkv.double().cpu().numpy()
    keep = [i for i in range(n) if i not in (4, 7, 20)]
    gk, gv = fetch(kv, 0, slots[keep])
    assert np.array_equal(gk, R.values(host[keep, n_q * HD:(n_q + n_kv) * HD].reshape(-1, n_kv, HD)))
    assert np.array_equal(gv, R.values(host[keep, (n_q + n_kv) * HD:].reshape(-1, n_kv, HD)))
    rest = np.setdiff1d(np.arange(64), slots[keep])
    assert not fetch(kv, 0, rest)[0].any()
    gk, gv = fetch(kv, 0, [NONE, int(slots[0])])
    assert not gk[0].any() and not gv[0].any() and gk[1].any()
    # wide rows out, one side only: the gap stays
    out = torch.full((len(keep), 3 * n_kv * HD), 5.0, device="cuda")
    ks = dev(slots[keep])
    kv.gather_device(0, len(keep), ks.data_ptr(), 0, out.data_ptr() + n_kv * HD * 4, v_stride=3 * n_kv * HD, stream=1)
    torch.cuda.synchronize()
    o = out.cpu().numpy()
    assert (o[:, :n_kv * HD] == 5).all() and (o[:, 2 * n_kv * HD:] == 5).all()
    assert np.array_equal(o[:, n_kv * HD:2 * n_kv * HD].reshape(-1, n_kv, HD), fetch(kv, 0, slots[keep])[1])
    kv.check()
    kv.close()


# --------------------------------------------------------------------- plan
def run_plan(kv, old, new, table, free, count, n_slots, in_place=False):
    n, w = table.shape
    t_in = dev(table)
    t_out = t_in if in_place else torch.full_like(t_in, 77)
    bufs = dict(old=dev(np.asarray(old, np.uint32)), new=dev(np.asarray(new, np.uint32)), free=dev(free),
                st=dev(np.array([count, 9, 9, 9], np.uint32)), so=dev(np.zeros(4, np.uint32)),
                slots=dev(np.full(n_slots + 3, 77, np.uint32)), starts=dev(np.zeros(n + 2, np.uint32) + 77),
                kv=dev(np.zeros(n + 1, np.uint32) + 77))
    kv.plan_device(n, w, bufs["old"].data_ptr(), bufs["new"].data_ptr(), t_in.data_ptr(), t_out.data_ptr(),
                   bufs["free"].data_ptr(), bufs["st"].data_ptr(), bufs["so"].data_ptr(), n_slots,
                   bufs["slots"].data_ptr(), bufs["starts"].data_ptr(), bufs["kv"].data_ptr(), stream=1)
    torch.cuda.synchronize()
    assert (u32(bufs["slots"])[n_slots:] == 77).all() and u32(bufs["starts"])[-1] == 77 and u32(bufs["kv"])[-1] == 77
    return (u32(t_out), u32(bufs["slots"])[:n_slots], u32(bufs["starts"])[:-1], u32(bufs["kv"])[:-1], u32(bufs["so"]))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,block,width,old_hi,new_hi,pad", [
    (1, 16, 1, 0, 16, 0), (1, 16, 9, 100, 1, 3), (5, 32, 7, 130, 60, 0), (16, 16, 160, 2047, 1, 0),
    (33, 64, 40, 2000, 300, 17), (300, 16, 70, 1000, 3, 1), (1024, 128, 3, 300, 2, 5), (2, 16, 5000, 60000, 9000, 0)])
def test_plan_matches_restatement(ctx, n, block, width, old_hi, new_hi, pad, in_place):
    rng = np.random.default_rng(n + width)
    old = rng.integers(0, old_hi + 1, n)
    new = rng.integers(0, new_hi + 1, n)
    old[0] = old_hi
    new[0] = min(new_hi, width * block - old_hi)
    held = -(-old // block)
    want = -(-(old + new) // block)
    n_blocks = int(want.sum()) + 4
    order = rng.permutation(n_blocks).astype(np.uint32)
    table = np.full((n, width), NONE, np.uint32)
    at = 0
    for i in range(n):
        table[i, :held[i]] = order[at:at + held[i]]
        at += held[i]
    free = np.full(n_blocks, NONE, np.uint32)
    free[:n_blocks - at] = order[at:]
    kv = cache(ctx, n_blocks, block, 1, 1)
    n_slots = int(new.sum()) + pad
    got = run_plan(kv, old, new, table, free, n_blocks - at, n_slots, in_place)
    ref = R.plan(old, new, table, free, n_blocks - at, block, n_slots, n_blocks)
    for g, w in zip(got, ref):
        assert np.array_equal(g, w)
    kv.check()
    kv.close()


def test_plan_refuses_whole_steps(ctx):
    kv = cache(ctx, 8, 16, 1, 1)
    table = np.array([[3, NONE, NONE], [5, 1, NONE]], np.uint32)
    free = np.array([0, 2, 4, 6, 7, NONE, NONE, NONE], np.uint32)
    cases = [([10, 20], [1, 13], 2, 14, 0), ([10, 20], [1, 13], 1, 14, 0), ([10, 20], [7, 13], 1, 20, 1),
             ([10, 20], [7, 30], 5, 37, 2), ([10, 20], [1, 13], 2, 13, 2), ([10, 20], [1, 1], 9, 2, 2),
             ([10, 20], [0xFFFFFFFF, 1], 5, 40, 2), ([60, 20], [0, 1], 5, 4, 2)]
    for old, new, count, n_slots, code in cases:
        got = run_plan(kv, old, new, table, free, count, n_slots)
        ref = R.plan(old, new, table, free, count, 16, n_slots, 8)
        assert ref[4][1] == code
        for g, w in zip(got, ref):
            assert np.array_equal(g, w), (old, new, count)
        if code:
            with pytest.raises(zb.ZgpuError) as e:
                kv.check()
            assert e.value.status == 13
        else:
            kv.check()
    # a row's last block is not in the pool: its tokens get no slot
    bad = table.copy()
    bad[0, 0] = 8
    got = run_plan(kv, [10, 20], [2, 1], bad, free, 5, 3)
    assert list(got[1]) == [NONE, NONE, 1 * 16 + 4]
    with pytest.raises(zb.ZgpuError) as e:
        kv.check()
    assert e.value.status == 10
    kv.close()


def test_release_returns_blocks_and_refuses_bad_tables(ctx):
    kv = cache(ctx, 12, 16, 1, 1)
    table = np.array([[3, 9, NONE], [5, NONE, NONE], [1, 2, 8]], np.uint32)
    free = np.full(12, NONE, np.uint32)
    free[:3] = [0, 4, 6]

    def go(done, lens, table, count):
        b = [dev(np.asarray(a, np.uint32)) for a in (done, lens, table, free, [count, 1, 2, 3])]
        kv.release_device(3, 3, *[x.data_ptr() for x in b], stream=1)
        torch.cuda.synchronize()
        return [u32(x) for x in b[1:]]

    lens, tab, fl, st = go([1, 0, 7], [17, 16, 48], table, 3)
    assert list(lens) == [0, 16, 0] and list(st) == [8, 0, 0, 5]
    assert list(fl[:8]) == [0, 4, 6, 3, 9, 1, 2, 8] and (fl[8:] == NONE).all()
    assert (tab[[0, 2]] == NONE).all() and np.array_equal(tab[1], table[1])
    kv.check()
    lens, tab, fl, st = go([0, 0, 0], [17, 16, 48], table, 3)
    assert list(lens) == [17, 16, 48] and list(st) == [3, 0, 0, 0] and np.array_equal(tab, table)
    kv.check()
    broken = table.copy()
    broken[2, 1] = 12
    for t, ln, count in ((broken, [17, 16, 48], 3), (table, [17, 16, 49], 3), (table, [17, 16, 48], 8), (table, [17, 16, 48], 13)):
        lens, tab, fl, st = go([1, 0, 1], ln, t, count)
        assert list(lens) == ln and list(st) == [count, 2, 2, 3]
        assert np.array_equal(tab, t) and np.array_equal(fl, free)
        with pytest.raises(zb.ZgpuError) as e:
            kv.check()
        assert e.value.status == 13
    kv.close()


# ---------------------------------------------------------------- attention
def make(ctx, seed, lens, nq, n_q, n_kv, block, layers=1, qgain=1.0):
    """A cache holding random rows for sequences of `lens` keys, and queries."""
    rng = np.random.default_rng(seed)
    held = [-(-n // block) for n in lens]
    n_blocks = sum(held) + 2
    order = rng.permutation(n_blocks).astype(np.uint32)
    width = max(held + [1]) + 1
    table = np.full((len(lens), width), NONE, np.uint32)
    at = 0
    kv = cache(ctx, n_blocks, block, layers, n_kv)
    ks, vs = [], []
    # every slot of the pool holds something: what lies behind a row is not zeros
    allk = rng.standard_normal((n_blocks * block, n_kv, HD)).astype(np.float32)
    allv = rng.standard_normal((n_blocks * block, n_kv, HD)).astype(np.float32)
    store(kv, layers - 1, np.arange(n_blocks * block, dtype=np.uint32), allk, allv)
    vk, vv = R.values(allk), R.values(allv)
    for i, n in enumerate(lens):
        table[i, :held[i]] = order[at:at + held[i]]
        at += held[i]
        pos = np.arange(n)
        sl = table[i][pos // block].astype(np.int64) * block + pos % block
        ks.append(vk[sl])
        vs.append(vv[sl])
    starts = np.concatenate([[0], np.cumsum(nq)]).astype(np.uint32)
    q = (qgain * rng.standard_normal((int(starts[-1]), n_q, HD))).astype(np.float32)
    return dict(kv=kv, table=table, lens=np.asarray(lens, np.uint32), starts=starts, q=q, ks=ks, vs=vs, layer=layers - 1,
                n_q=n_q, n_kv=n_kv, width=width)


def run_attn(c, dtype="f32", scale=None, pad=2, max_q=None, stream=None, fused=False, work=None):
    td, zd = TYPES[dtype]
    T = c["q"].shape[0]
    scale = HD ** -0.5 if scale is None else scale
    q = dev(c["q"]).to(td)
    if fused:       # q as columns of wider rows, out likewise
        wide = torch.zeros(T, (c["n_q"] + 2) * HD, dtype=td, device="cuda")
        wide[:, HD:-HD] = q.flatten(1)
        out = torch.full((T + pad, (c["n_q"] + 1) * HD), 3.0, dtype=td, device="cuda")
        args = dict(q_stride=wide.stride(0), out_stride=out.stride(0))
        qp, op = wide.data_ptr() + HD * wide.element_size(), out.data_ptr()
    else:
        out = torch.full((T + pad, c["n_q"], HD), 3.0, dtype=td, device="cuda")
        args, qp, op = {}, q.data_ptr(), out.data_ptr()
    st, ln, tb = dev(c["starts"]), dev(c["lens"]), dev(c["table"])
    nq = np.diff(c["starts"].astype(np.int64))
    torch.cuda.synchronize()
    c["kv"].attention_device(c["layer"], len(c["lens"]), T, int(nq.max()) if max_q is None else max_q, c["n_q"], qp, op,
                             st.data_ptr(), ln.data_ptr(), tb.data_ptr(), c["width"], dtype=zd, scale=scale,
                             stream=1 if stream is None else stream.cuda_stream, work=work, **args)
    torch.cuda.synchronize()
    o = out.double().cpu().numpy()
    assert (o[T:] == 3.0).all(), "rows behind the last sequence are left alone"
    if fused:
        assert (o[:, c["n_q"] * HD:] == 3.0).all()
        o = o[:, :c["n_q"] * HD].reshape(-1, c["n_q"], HD)
    return o[:T], q.double().cpu().numpy()


def check_attn(c, o, q, dtype, scale=None, rows=None):
    scale = HD ** -0.5 if scale is None else scale
    half = torch.finfo(TYPES[dtype][0]).eps / 2
    for i, n in enumerate(c["lens"]):
        a, b = int(c["starts"][i]), int(c["starts"][i + 1])
        if a == b or (rows is not None and i not in rows):
            continue
        ref, mass, total, ds = R.attention(q[a:b], c["ks"][i], c["vs"][i], scale)
        rel = 2 * ds[..., None] + 2.0 ** -21 + (int(n) / 16 + 64) * 2.0 ** -23 + (2.0 ** -11 if dtype != "f32" else 0)
        tol = rel * mass + 2.0 ** (-40 if dtype == "f32" else -32) * total + half * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 0)
        err = np.abs(o[a:b] - ref)
        assert (err <= tol).all(), (i, int(n), float((err / np.maximum(tol, 1e-300)).max()))


DECODE = [
    # lens, queries per sequence, q heads, kv heads, block
    ([1], [1], 1, 1, 16), ([2], [1], 2, 1, 16), ([15, 16, 17], [1, 1, 1], 4, 2, 16), ([500], [1], 16, 8, 16),
    ([129, 0, 1, 700, 64], [1, 0, 1, 1, 1], 8, 2, 32), ([333, 90], [1, 1], 8, 1, 64), ([2500, 3, 40], [1, 1, 1], 32, 8, 128),
    ([5000], [1], 5, 1, 16), ([200, 31], [1, 1], 32, 2, 16), ([70, 71], [1, 1], 6, 2, 64), ([1000] * 40, [1] * 40, 4, 2, 16),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,nq,n_q,n_kv,block", DECODE)
def test_attention_single_tokens(ctx, lens, nq, n_q, n_kv, block, dtype):
    c = make(ctx, sum(lens) + n_q, lens, nq, n_q, n_kv, block)
    o, q = run_attn(c, dtype)
    check_attn(c, o, q, dtype)
    c["kv"].check()
    c["kv"].close()


CHUNKS = [
    ([5], [5], 2, 1, 16), ([16], [16], 1, 1, 16), ([33, 40], [2, 7], 4, 2, 16), ([300], [300], 4, 2, 16),
    ([257, 64, 900], [129, 64, 33], 4, 1, 64), ([700, 90, 513, 20], [1, 90, 130, 0], 8, 2, 32),
    ([65, 64, 63, 128], [65, 64, 63, 128], 3, 1, 128), ([1500], [37], 16, 2, 16), ([400], [200], 16, 1, 64),
    ([2100], [260], 2, 1, 32), ([140, 150], [140, 1], 14, 2, 16),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,nq,n_q,n_kv,block", CHUNKS)
def test_attention_chunks(ctx, lens, nq, n_q, n_kv, block, dtype):
    c = make(ctx, sum(lens) * 3 + n_q, lens, nq, n_q, n_kv, block, layers=2)
    o, q = run_attn(c, dtype)
    check_attn(c, o, q, dtype)
    # a bound above the largest chunk, q and out as columns of wider rows
    o2, _ = run_attn(c, dtype, max_q=max(nq) + 1000, fused=True)
    check_attn(c, o2, q, dtype)
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("gain,scale", [(1e-3, None), (30.0, None), (1.0, 1e-4), (1e4, 1e-3), (1e-30, 1e28), (1e30, 1e-32)])
@pytest.mark.parametrize("lens,nq", [([300, 41], [1, 1]), ([300, 141], [160, 141])])
def test_attention_query_ranges(ctx, gain, scale, lens, nq):
    """Flat and sharp softmax, queries far below and above binary16's range."""
    c = make(ctx, 5, lens, nq, 4, 2, 16, qgain=gain)
    o, q = run_attn(c, "f32", scale)
    check_attn(c, o, q, "f32", scale)
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("nq", [4, 140])
def test_attention_rows_before_position_zero_are_zero(ctx, nq):
    c = make(ctx, 6, [nq, 3, 0, nq - 1], [nq, nq, nq, 1], 4, 2, 16)
    o, q = run_attn(c)
    check_attn(c, o, q, "f32")
    a = int(c["starts"][1])
    assert not o[a:a + nq - 3].any() and o[a + nq - 3:a + nq].any(-1).all()
    assert not o[2 * nq:3 * nq].any()
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("nq", [1, 150])
def test_attention_bad_blocks_lengths_and_starts_are_recorded(ctx, nq):
    def status(c):
        with pytest.raises(zb.ZgpuError) as e:
            c["kv"].check()
        assert e.value.status == 10
        c["kv"].check()

    lens = [300, 200, 90 + nq]
    c = make(ctx, 8, lens, [nq, 1, 1], 4, 2, 16)
    good = c["table"].copy()
    c["table"] = good.copy()
    c["table"][0, 3] = 0x7FFFFFFF          # keys 48..63 of sequence 0 are left out
    o, q = run_attn(c)
    status(c)
    check_attn(c, o, q, "f32", rows=[1, 2])
    keep = np.r_[0:48, 64:300]
    if nq == 1:
        d = dict(c, ks=[c["ks"][0][keep]], vs=[c["vs"][0][keep]], lens=np.array([len(keep)]), starts=c["starts"][:2])
        check_attn(d, o, q, "f32")
    c["table"] = good
    c["lens"] = np.array([300, c["width"] * 16 + 1, lens[2]], np.uint32)      # longer than its table row
    o, q = run_attn(c)
    status(c)
    c["lens"] = np.asarray(lens, np.uint32)
    check_attn(c, o, q, "f32", rows=[0, 2])
    keep_starts = c["starts"]
    T = nq + 2
    for starts, rows in (([0, nq, nq - 1, nq - 1], [0]), ([0, nq, nq + 1, T + 1], [0, 1]), ([0, nq, nq + 1, 0xFFFFFFFF], [0, 1])):
        c["starts"] = np.asarray(starts, np.uint32)
        o, q = run_attn(c, max_q=max(nq, 4))
        status(c)
        c["starts"] = keep_starts
        check_attn(c, o, q, "f32", rows=rows)
    if nq > 1:                     # more queries than max_q: that sequence alone gets no output
        o, q = run_attn(c, max_q=nq - 1)
        status(c)
        check_attn(c, o, q, "f32", rows=[1, 2])
        assert (o[:nq] == 3.0).all()
    o, q = run_attn(c)
    check_attn(c, o, q, "f32")
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("nq", [1, 70])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_attention_non_finite_queries_stay_in_their_rows(ctx, nq, value):
    c = make(ctx, 9, [100, 90], [nq, 1], 4, 2, 16)
    c["q"][nq // 2, 1, 77] = value
    o, q = run_attn(c)
    with pytest.raises(zb.ZgpuError) as e:
        c["kv"].check()
    assert e.value.status == 20
    assert np.isnan(o[nq // 2, 1]).all()
    o[nq // 2, 1] = 0
    q[nq // 2, 1] = 0
    c["q"][nq // 2, 1] = 0
    o0, _ = run_attn(c)
    o0[nq // 2, 1] = 0
    assert np.array_equal(o, o0), "every other row is what it is without the bad one"
    c["kv"].close()


def test_attention_repeats_bit_for_bit_and_on_any_stream(ctx):
    c = make(ctx, 10, [3000, 17, 260], [1, 1, 130], 8, 2, 64)
    o, _ = run_attn(c, "f16")
    s = torch.cuda.Stream()
    for _ in range(3):
        o2, _ = run_attn(c, "f16", stream=s)
        assert np.array_equal(o, o2)
    c["kv"].check()
    c["kv"].close()


def test_two_attentions_at_once_with_a_workspace_each(ctx):
    c = make(ctx, 12, [9000, 4000], [1, 1], 8, 2, 64)
    alone, _ = run_attn(c, "f32")
    st, ln, tb, q = dev(c["starts"]), dev(c["lens"]), dev(c["table"]), dev(c["q"])
    streams = [torch.cuda.Stream() for _ in range(3)]
    works = [c["kv"].new_work() for _ in streams]
    outs = [torch.zeros_like(q) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, w, o in zip(streams, works, outs):
            c["kv"].attention_device(0, 2, 2, 1, 8, q.data_ptr(), o.data_ptr(), st.data_ptr(), ln.data_ptr(),
                                     tb.data_ptr(), c["width"], stream=s.cuda_stream, work=w)
    torch.cuda.synchronize()
    for o in outs:
        assert np.array_equal(o.double().cpu().numpy(), alone)
    for w in works:
        w.close()
    c["kv"].close()


# ---------------------------------------------------- a run of them together
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_serving_steps(ctx, captured, dtype):
    """Prompts and decode steps of several sequences through plan, append and
    attention, with sequences that end and begin; in the captured form the
    decode step is one graph whose lengths live on the device."""
    td, zd = TYPES[dtype]
    n_seq, n_q, n_kv, block, width, n_blocks, cap = 4, 4, 2, 16, 8, 30, 96
    rng = np.random.default_rng(1)
    kv = cache(ctx, n_blocks, block, 1, n_kv)
    lens = [dev(np.zeros(n_seq, np.uint32)) for _ in range(2)]
    state = [dev(np.array([n_blocks, 0, 0, 0], np.uint32)) for _ in range(2)]
    table = dev(np.full((n_seq, width), NONE, np.uint32))
    free = dev(np.arange(n_blocks, dtype=np.uint32))
    new = dev(np.zeros(n_seq, np.uint32))
    slots, starts = dev(np.zeros(cap, np.uint32)), dev(np.zeros(n_seq + 1, np.uint32))
    qkv = torch.zeros(cap, (n_q + 2 * n_kv) * HD, dtype=td, device="cuda")
    out = torch.zeros(cap, n_q * HD, dtype=td, device="cuda")
    es = qkv.element_size()
    hist = [(np.zeros((0, n_kv, HD)), np.zeros((0, n_kv, HD))) for _ in range(n_seq)]

    def step(stream, src, max_q):
        kv.plan_device(n_seq, width, lens[src].data_ptr(), new.data_ptr(), table.data_ptr(), table.data_ptr(),
                       free.data_ptr(), state[src].data_ptr(), state[1 - src].data_ptr(), cap, slots.data_ptr(),
                       starts.data_ptr(), lens[1 - src].data_ptr(), stream=stream)
        kv.append_device(0, cap, qkv.data_ptr() + n_q * HD * es, qkv.data_ptr() + (n_q + n_kv) * HD * es,
                         slots.data_ptr(), dtype=zd, k_stride=qkv.stride(0), v_stride=qkv.stride(0), stream=stream)
        kv.attention_device(0, n_seq, cap, max_q, n_q, qkv.data_ptr(), out.data_ptr(), starts.data_ptr(),
                            lens[1 - src].data_ptr(), table.data_ptr(), width, dtype=zd, q_stride=qkv.stride(0),
                            stream=stream)

    graphs = []
    if captured:
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        for src in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step(s.cuda_stream, src, cap)
            graphs.append(g)
    counts = [[40, 0, 7, 1], [1, 33, 1, 0], [1, 1, 1, 1], [0, 1, 50, 1], [1, 1, 1, 1], [16, 1, 1, 1], [1, 1, 1, 1]]
    src = 0
    for i, n in enumerate(counts):
        if i == 4:      # sequences 0 and 2 end
            done = dev(np.array([1, 0, 1, 0], np.uint32))
            kv.release_device(n_seq, width, done.data_ptr(), lens[src].data_ptr(), table.data_ptr(), free.data_ptr(),
                              state[src].data_ptr(), stream=1)
            for k in (0, 2):
                hist[k] = (hist[k][0][:0], hist[k][1][:0])
        x = rng.standard_normal((cap, (n_q + 2 * n_kv) * HD)).astype(np.float32)
        qkv.copy_(dev(x).to(td))
        new.copy_(dev(np.array(n, np.uint32)))
        out.fill_(9.0)
        torch.cuda.synchronize()
        if captured:
            graphs[src].replay()
        else:
            step(1, src, max(n))
        torch.cuda.synchronize()
        kv.check()
        src = 1 - src
        host = qkv.double().cpu().numpy()
        o = out.double().cpu().numpy()
        assert (o[sum(n):] == 9.0).all()
        at = 0
        for k in range(n_seq):
            rows = host[at:at + n[k]]
            hist[k] = (np.concatenate([hist[k][0], R.values(rows[:, n_q * HD:(n_q + n_kv) * HD].reshape(-1, n_kv, HD))]),
                       np.concatenate([hist[k][1], R.values(rows[:, (n_q + n_kv) * HD:].reshape(-1, n_kv, HD))]))
            if n[k]:
                c = dict(lens=[len(hist[k][0])], starts=[0, n[k]], ks=[hist[k][0]], vs=[hist[k][1]])
                check_attn(c, o[at:at + n[k]].reshape(-1, n_q, HD), rows[:, :n_q * HD].reshape(-1, n_q, HD), dtype)
            at += n[k]
        assert list(u32(lens[src])) == [len(h[0]) for h in hist]
        assert u32(state[src])[0] == n_blocks - sum(-(-len(h[0]) // block) for h in hist)
    kv.close()


# ------------------------------------------------------------------ refusals
def test_calls_leave_the_current_device_and_null_rows_alone(ctx):
    c = make(ctx, 14, [20], [1], 4, 2, 16)
    kv = c["kv"]
    assert LIB.zgpu_kv4_append_device(kv.h, 0, 0, None, 0, None, 0, 0, None, None) == 0
    assert LIB.zgpu_kv4_gather_device(kv.h, 0, 0, None, None, 0, None, 0, 0, None) == 0
    before = torch.cuda.current_device()
    run_attn(c)
    assert torch.cuda.current_device() == before
    kv.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,nq", [
    (2, 2, [31, 32, 33]), (6, 2, [10, 11, 12]), (4, 1, [8, 9, 1]), (16, 2, [4, 5, 3]), (16, 1, [2, 3, 0]), (11, 1, [3, 2, 3]),
    (2, 2, [24, 25, 23]), (4, 1, [6, 7, 5]), (12, 1, [2, 3, 1])])
def test_attention_around_the_border_of_the_two_kernels(ctx, dtype, n_q, n_kv, nq):
    """Up to 32 query rows per kv head (24 in f32) and more, in one call."""
    c = make(ctx, n_q + n_kv, [nq[0] + 200, nq[1], nq[2] + 999], nq, n_q, n_kv, 32)
    o, q = run_attn(c, dtype)
    check_attn(c, o, q, dtype)
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n_seq,n", [(40, 100), (300, 20), (3, 1000)])
def test_attention_many_short_pieces_per_cta(ctx, dtype, n_seq, n):
    """Prompts of one key tile each, several to a CTA, one after the other."""
    c = make(ctx, n_seq, [n + i % 3 for i in range(n_seq)], [n] * n_seq, 8, 4, 16)
    o, q = run_attn(c, dtype)
    check_attn(c, o, q, dtype, rows=range(0, n_seq, max(1, n_seq // 6)))
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("seed", range(6))
def test_attention_short_and_long_sequences_in_any_order(ctx, dtype, seed):
    """Pieces that are cut between CTAs beside ones that are not (512 keys and fewer)."""
    rng = np.random.default_rng(900 + seed)
    n = int(rng.integers(5, 90))
    lens = [int(x) for x in np.where(rng.random(n) < 0.5, rng.integers(1, 514, n), rng.integers(500, 2600, n))]
    nq = [min(x, int(y)) for x, y in zip(lens, rng.integers(0, 4, n))]
    c = make(ctx, seed, lens, nq, 4, 2, 16 << (seed % 4))
    o, q = run_attn(c, dtype)
    check_attn(c, o, q, dtype)
    o2, _ = run_attn(c, dtype)
    assert np.array_equal(o, o2)
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("nq", [1, 9, 20])
def test_attention_of_the_most_sequences(ctx, nq):
    """1024 sequences, the largest table of sums; every 64th is checked."""
    lens = [nq + (i * 37) % 90 for i in range(1024)]
    c = make(ctx, 21, lens, [nq] * 1024, 4, 2, 16)
    o, q = run_attn(c, "f32")
    check_attn(c, o, q, "f32", rows=range(0, 1024, 64))
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_at_the_end_of_a_pool_of_many_gigabytes(ctx, dtype):
    """Blocks whose bytes lie far beyond 2^32, single tokens and a chunk."""
    n_kv, block, n_blocks = 8, 16, 300_000                  # 5.5 GB
    kv = cache(ctx, n_blocks, block, 1, n_kv)
    lens, nq, n_q = [70, 130], [1, 65], 16
    rng = np.random.default_rng(4)
    table = np.full((2, 10), NONE, np.uint32)
    ids = n_blocks - 1 - rng.permutation(40)[:14]
    table[0, :5], table[1, :9] = ids[:5], ids[5:14]
    c = dict(kv=kv, table=table, lens=np.asarray(lens, np.uint32), starts=np.array([0, 1, 66], np.uint32), layer=0,
             n_q=n_q, n_kv=n_kv, width=10, ks=[], vs=[], q=rng.standard_normal((66, n_q, HD)).astype(np.float32))
    for i, n in enumerate(lens):
        pos = np.arange(n)
        slots = (table[i][pos // block].astype(np.int64) * block + pos % block).astype(np.uint32)
        k, v = (rng.standard_normal((n, n_kv, HD)).astype(np.float32) for _ in range(2))
        store(kv, 0, slots, k, v)
        c["ks"].append(R.values(k))
        c["vs"].append(R.values(v))
        gk, gv = fetch(kv, 0, slots, "f32", n_kv)
        assert np.array_equal(gk, c["ks"][i]) and np.array_equal(gv, c["vs"][i])
    o, q = run_attn(c, dtype)
    check_attn(c, o, q, dtype)
    kv.check()
    kv.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_sequences_that_share_blocks_and_rows_in_odd_order(ctx, dtype):
    """Two sequences on one prefix's blocks, and a gap in the query rows."""
    c = make(ctx, 31, [96, 200], [40, 1], 6, 2, 32)
    c["table"][1, :3] = c["table"][0, :3]                  # 96 keys of the other sequence
    c["ks"][1] = np.concatenate([c["ks"][0], c["ks"][1][96:]])
    c["vs"][1] = np.concatenate([c["vs"][0], c["vs"][1][96:]])
    o, q = run_attn(c, dtype)
    check_attn(c, o, q, dtype)
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_attention_non_finite_16_bit_queries(ctx, dtype, value):
    c = make(ctx, 9, [200, 90], [150, 1], 4, 2, 16)
    c["q"][70, 1, 77] = value
    o, q = run_attn(c, dtype)
    with pytest.raises(zb.ZgpuError) as e:
        c["kv"].check()
    assert e.value.status == 20
    assert np.isnan(o[70, 1]).all()
    c["q"][70, 1] = 0
    o0, _ = run_attn(c, dtype)
    o[70, 1] = o0[70, 1] = 0
    assert np.array_equal(o, o0)
    c["kv"].close()


def test_a_graph_of_each_of_two_chunks_replayed_side_by_side(ctx):
    """Two captured calls with a workspace each, on two streams at once."""
    c = make(ctx, 17, [700, 300], [200, 1], 8, 2, 16)
    alone, _ = run_attn(c, "f16")
    td = torch.float16
    st, ln, tb, q = dev(c["starts"]), dev(c["lens"]), dev(c["table"]), dev(c["q"]).to(td)
    outs, graphs, works = [torch.zeros_like(q) for _ in range(2)], [], []
    torch.cuda.synchronize()
    for o in outs:
        works.append(c["kv"].new_work())
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=s):
            c["kv"].attention_device(0, 2, 201, 200, 8, q.data_ptr(), o.data_ptr(), st.data_ptr(), ln.data_ptr(),
                                     tb.data_ptr(), c["width"], dtype=zb.F16, stream=s.cuda_stream, work=works[-1])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert np.array_equal(o.double().cpu().numpy(), alone)
    del graphs
    c["kv"].check()
    for w in works:
        w.close()
    c["kv"].close()
