"""Which of its two kernels the 4-bit cache's attention takes, and that both are
right on either side of the border: it falls from 96 query rows per kv head
for small calls to 24 (f32) and 32 for calls that may read many keys, which a wide
table stands for here."""
import numpy as np
import pytest

from test_gpu_kv4 import NONE, TYPES, check_attn, dev, make, run_attn

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
runtime = pytest.importorskip("cuda.bindings.runtime")

WIDE = 1 << 19      # keys of a table row that put the border at its lowest


def widen(c, block):
    t = np.full((len(c["lens"]), WIDE // block), NONE, np.uint32)
    t[:, :c["width"]] = c["table"]
    return dict(c, table=t, width=WIDE // block)


def kernels(c, dtype):
    """Kernels that the call captured into a graph consists of."""
    td, zd = TYPES[dtype]
    T = c["q"].shape[0]
    q, st, ln, tb = dev(c["q"]).to(td), dev(c["starts"]), dev(c["lens"]), dev(c["table"])
    g, s = torch.cuda.CUDAGraph(keep_graph=True), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        c["kv"].attention_device(0, len(c["lens"]), T, int(np.diff(c["starts"].astype(np.int64)).max()), c["n_q"],
                                 q.data_ptr(), torch.empty_like(q).data_ptr(), st.data_ptr(), ln.data_ptr(),
                                 tb.data_ptr(), c["width"], dtype=zd, stream=s.cuda_stream)
    err, _, n = runtime.cudaGraphGetNodes(runtime.cudaGraph_t(g.raw_cuda_graph()))
    assert int(err) == 0
    return n


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,nq", [
    (4, 1, [6, 7, 1]), (4, 1, [8, 9, 5]), (16, 2, [5, 12, 3]), (3, 1, [32, 33, 13]), (2, 2, [96, 97, 40]), (16, 1, [6, 7, 0]),
    (8, 8, [95, 1, 33])])
def test_both_kernels_on_both_sides_of_the_border(ctx, dtype, n_q, n_kv, nq):
    c = make(ctx, n_q * n_kv + nq[0], [nq[0] + 300, nq[1], nq[2] + 777], nq, n_q, n_kv, 32)
    rows, least = max(nq) * (n_q // n_kv), 24 if dtype == "f32" else 32
    assert kernels(c, dtype) == (2 if rows > 96 else 1)
    o, q = run_attn(c, dtype)
    check_attn(c, o, q, dtype)
    wide = widen(c, 32)
    assert kernels(wide, dtype) == (2 if rows > least else 1)
    o, q = run_attn(wide, dtype, fused=True)
    check_attn(c, o, q, dtype)
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_small_chunks_by_the_prompt_kernel(ctx, dtype):
    """Row tiles that are a tenth full, several to a CTA and cut between CTAs."""
    lens = [33 + 7 * i for i in range(30)] + [3000, 2500]
    nq = [33 + i for i in range(30)] + [40, 63]
    c = make(ctx, 77, lens, nq, 4, 4, 16)
    wide = widen(c, 16)
    assert kernels(wide, dtype) == 2
    o, q = run_attn(wide, dtype)
    check_attn(c, o, q, dtype)
    o2, _ = run_attn(wide, dtype)
    assert np.array_equal(o, o2)
    c["kv"].check()
    c["kv"].close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_q,n_kv,nq", [(6, 2, [40, 1]), (192, 96, [17, 2]), (96, 96, [33, 1])])
def test_rows_on_16_byte_boundaries(ctx, dtype, n_q, n_kv, nq):
    """q and out 16 bytes behind a wider boundary, at strides that are odd multiples of
    16 bytes, through both kernels; the gaps stay as they are."""
    td, zd = TYPES[dtype]
    unit = 16 // td.itemsize
    c = make(ctx, n_q, [nq[0] + 300, nq[1] + 40], nq, n_q, n_kv, 16)
    T, width = sum(nq), n_q * 128 + unit
    q = torch.zeros(T * width + unit, dtype=td, device="cuda")
    q[unit:].view(T, width)[:, :n_q * 128] = dev(c["q"]).to(td).flatten(1)
    host = q[unit:].view(T, width)[:, :n_q * 128].reshape(T, n_q, 128).double().cpu().numpy()
    for x in (c, widen(c, 16)):
        out = torch.full_like(q, 3.0)
        st, ln, tb = dev(x["starts"]), dev(x["lens"]), dev(x["table"])
        torch.cuda.synchronize()
        c["kv"].attention_device(0, 2, T, max(nq), n_q, q.data_ptr() + 16, out.data_ptr() + 16, st.data_ptr(),
                                 ln.data_ptr(), tb.data_ptr(), x["width"], dtype=zd, q_stride=width, out_stride=width,
                                 stream=1)
        torch.cuda.synchronize()
        o = out.double().cpu().numpy()
        assert (o[:unit] == 3).all() and (o[unit:].reshape(T, width)[:, n_q * 128:] == 3).all()
        check_attn(c, o[unit:].reshape(T, width)[:, :n_q * 128].reshape(T, n_q, 128), host, dtype)
    c["kv"].check()
    c["kv"].close()
