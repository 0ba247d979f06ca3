"""Plain 64-bit restatements of the paged 4-bit cache, for its tests."""
import numpy as np

NONE = 0xFFFFFFFF
HD = 128


def quantise(x):
    """(q int [..., 4, 32], d float64 [..., 4]) of rows x [..., 128], from the
    format's definition; x holds finite values below the format's limit."""
    g = np.asarray(x, np.float64).reshape(*np.shape(x)[:-1], 4, 32)
    first = np.abs(g).argmax(-1)                      # the first of equals
    m = np.take_along_axis(g, first[..., None], -1)[..., 0]
    mant, ex = np.frexp(-m / 8)
    d = np.ldexp(np.rint(mant * 256), ex - 8)         # 8 significant bits
    d = d.astype(np.float16).astype(np.float64)       # exact above 2^-17, the binary16 grid below
    q = np.rint(np.divide(g, d[..., None], out=np.zeros_like(g), where=d[..., None] != 0))
    return np.clip(q, -8, 7).astype(np.int64), d


def values(x):
    q, d = quantise(x)
    return (q * d[..., None]).reshape(np.shape(x))


def plan(old, new, table, free, count, block, n_slots, n_blocks):
    """table, slots, starts, kv lengths, state of one step."""
    n, width = table.shape
    old, new = [int(o) for o in old], [int(x) for x in new]
    need = [-(-(o + x) // block) - -(-o // block) for o, x in zip(old, new)]
    code = 0
    if any(o + x > width * block for o, x in zip(old, new)) or sum(new) > n_slots or count > n_blocks:
        code = 2
    elif sum(need) > count:
        code = 1
    out = np.full((n, width), NONE, np.uint32)
    slots = np.full(n_slots, NONE, np.uint32)
    starts = np.zeros(n + 1, np.uint32)
    top, at = count, 0
    for i in range(n):
        held = min(-(-old[i] // block), width)
        out[i, :held] = table[i, :held]
        if code:
            continue
        for j in range(need[i]):
            top -= 1
            out[i, held + j] = free[top]
        for t in range(new[i]):
            pos = old[i] + t
            b = int(out[i, pos // block])
            slots[at] = b * block + pos % block if b < n_blocks else NONE
            at += 1
        starts[i + 1] = at
    kv = np.array(old if code else [o + x for o, x in zip(old, new)], np.uint32)
    return out, slots, starts, kv, np.array([top, code, at, count - top], np.uint32)


def attention(q, k, v, scale):
    """(o, bound inputs) of queries q [n, heads, 128] that are the last n of
    the keys k, v [len, kv heads, 128], all float64.  Returns o and, per
    output, sum p |v| and sum |v|, and per row the largest error of a score for queries
    and products that are right to 2^-22 and summed in f32."""
    n, nq, _ = q.shape
    length, nkv, _ = k.shape
    g = nq // nkv
    o = np.zeros_like(q)
    mass, total = np.zeros_like(q), np.zeros_like(q)
    ds = np.zeros((n, nq))
    for h in range(nq):
        kh, vh = k[:, h // g], v[:, h // g]
        s = q[:, h] @ kh.T * scale
        err = (2.0 ** -22 * np.abs(q[:, h]).max(-1, keepdims=True) * np.abs(kh).sum(-1)
               + 2.0 ** -23 * 24 * (np.abs(q[:, h]) @ np.abs(kh).T)) * scale + 2.0 ** -22 * np.abs(s)
        seen = np.arange(length)[None, :] <= (length - n + np.arange(n))[:, None]
        for t in range(n):
            m = seen[t]
            if not m.any():
                continue
            p = np.exp(s[t, m] - s[t, m].max())
            p /= p.sum()
            o[t, h], mass[t, h], total[t, h] = p @ vh[m], p @ np.abs(vh[m]), np.abs(vh[m]).sum(0)
            ds[t, h] = err[t, m].max()
    return o, mass, total, ds
