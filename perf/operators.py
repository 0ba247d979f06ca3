"""Timed cases of the paged 4-bit KV cache: step plan, append, attention.

``run`` computes a case in its plain form (elementary torch operations in 32
bits) while ``own`` is false, and through ``zero_b200.KvCache4`` while it is
true.  The cache format both share: a token's K (or V) row of one kv head is
four groups of 32 values; a group is one signed scale d and 32 integers q in
-8..7, and stands for q * d.  With m the group's value of largest magnitude
(the first of equals), d is -m / 8 rounded to 8 significant bits and then to
binary16, and q the integer nearest to x / d (ties to even), clamped to -8..7.
"""
import random

import torch

own = False

HEAD = 128          # values per head
GROUP = 32          # values per scale
TOKEN_BYTES = 2 * (HEAD // 2 + HEAD // GROUP * 2)   # K and V of one token and kv head
NONE = -1           # a slot or a block that is not there
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of the benchmark's 16 sequences: one new token each,
        # launch latency counts
        dict(name="plan_decode_16", op="plan", n_seq=16, block=16, table=160, ctx_lo=128, ctx_hi=2047, q_lo=1, q_hi=1,
             chunks=0, chunk=0, pad=0, lens=1),
        # a busy server's mixed step: decoding sequences, some idle, and prompt
        # chunks, with the slot map padded to a fixed size
        dict(name="plan_mixed_512", op="plan", n_seq=512, block=16, table=1056, ctx_lo=0, ctx_hi=16384, q_lo=0, q_hi=2,
             chunks=40, chunk=401, pad=129, lens=2),
        # one sequence's next token: the smallest call
        dict(name="append_token_f32", op="append", tokens=1, n_q=16, n_kv=8, block=16, dtype="f32", fused=True, skip=0),
        # a decode step of many sequences at a padded batch size
        dict(name="append_decode_250_f16", op="append", tokens=250, n_q=32, n_kv=8, block=32, dtype="f16", fused=False,
             skip=13),
        # eight prompts of 2048 tokens, k and v taken from the fused projection
        dict(name="append_prompts_16384_f32", op="append", tokens=16384, n_q=16, n_kv=8, block=64, dtype="f32",
             fused=True, skip=0),
        # the model's batch-1 decode at a short context: latency
        dict(name="attn_decode_1_500_f32", op="attention", n_seq=1, n_q=16, n_kv=8, block=16, dtype="f32", ctx_lo=500,
             ctx_hi=500, q_lo=1, q_hi=1, chunks=0, chunk=0, lens=3),
        # batched decode of 16 sequences of the larger model
        dict(name="attn_decode_16_f32", op="attention", n_seq=16, n_q=32, n_kv=8, block=16, dtype="f32", ctx_lo=128,
             ctx_hi=2047, q_lo=1, q_hi=1, chunks=0, chunk=0, lens=1),
        # 32 long conversations of odd lengths: the cache read counts
        dict(name="attn_decode_32_long_bf16", op="attention", n_seq=32, n_q=32, n_kv=8, block=64, dtype="bf16",
             ctx_lo=8191, ctx_hi=32767, q_lo=1, q_hi=1, chunks=0, chunk=0, lens=4),
        # one very long document, one token: work split over the long axis
        dict(name="attn_decode_1_131071_f16", op="attention", n_seq=1, n_q=16, n_kv=8, block=32, dtype="f16",
             ctx_lo=131071, ctx_hi=131071, q_lo=1, q_hi=1, chunks=0, chunk=0, lens=5),
        # the prefill benchmark's prompt of 2048 tokens in the model's type
        dict(name="attn_prompt_2048_f32", op="attention", n_seq=1, n_q=16, n_kv=8, block=16, dtype="f32", ctx_lo=0,
             ctx_hi=0, q_lo=2048, q_hi=2048, chunks=0, chunk=0, lens=6),
        # eight ragged prompts of the larger model
        dict(name="attn_prompts_8_f16", op="attention", n_seq=8, n_q=32, n_kv=8, block=64, dtype="f16", ctx_lo=0,
             ctx_hi=0, q_lo=1021, q_hi=2048, chunks=0, chunk=0, lens=7),
        # a serving step: decoding sequences beside prompt chunks that continue
        # long contexts
        dict(name="attn_chunks_24_bf16", op="attention", n_seq=24, n_q=32, n_kv=8, block=64, dtype="bf16", ctx_lo=4000,
             ctx_hi=16384, q_lo=1, q_hi=1, chunks=4, chunk=509, lens=8),
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    while True:
        case = _drawn(rng)
        w = work(case)
        if w["bytes"] <= 650e6 and w["flops"] <= 280e9:     # the largest listed
            return case


def _drawn(rng):
    op = rng.choice(["plan", "append", "append", "attention", "attention", "attention"])
    lens = rng.randrange(1 << 30)
    block = rng.choice([16, 32, 64, 128])
    if op == "plan":
        n_seq, hi, chunks = _log(rng, 1, 512), _log(rng, 64, 16384), 0
        if rng.random() < 0.5:
            chunks = rng.randint(1, 1 + n_seq // 13)
        chunk = _log(rng, 2, 401) if chunks else 0
        return dict(op=op, n_seq=n_seq, block=block, table=(hi + 402 + block) // block + rng.randint(0, 7), ctx_lo=0,
                    ctx_hi=hi, q_lo=rng.randint(0, 1), q_hi=rng.randint(1, 3), chunks=chunks, chunk=chunk,
                    pad=rng.choice([0, 1, 77]), lens=lens)
    n_kv, g = rng.choice([1, 2, 8]), rng.choice([1, 2, 3, 4, 8])
    head = dict(n_q=n_kv * g, n_kv=n_kv, block=block, dtype=rng.choice(["f32", "f16", "bf16"]))
    if op == "append":
        tokens = _log(rng, 1, 16384)
        return dict(op=op, tokens=tokens, fused=rng.random() < 0.5, skip=rng.randint(0, tokens // 5), **head)
    if rng.random() < 0.6:                                                   # single tokens
        n_seq = _log(rng, 1, 48)
        hi = _log(rng, 16, min(131071, 480000 // n_seq))
        spec = dict(n_seq=n_seq, ctx_lo=rng.randint(0, hi), ctx_hi=hi, q_lo=rng.randint(0, 1), q_hi=rng.choice([1, 1, 4]),
                    chunks=0, chunk=0)
    elif rng.random() < 0.5:                                                 # prompts
        n_seq = rng.randint(1, 8)
        hi = _log(rng, 24, 2048)
        spec = dict(n_seq=n_seq, ctx_lo=0, ctx_hi=0, q_lo=rng.randint(1, hi), q_hi=hi, chunks=0, chunk=0)
    else:                                                                    # chunks beside single tokens
        n_seq, hi = rng.randint(2, 24), _log(rng, 64, 16384)
        spec = dict(n_seq=n_seq, ctx_lo=rng.randint(0, hi), ctx_hi=hi, q_lo=1, q_hi=1, chunks=rng.randint(1, min(3, n_seq)),
                    chunk=_log(rng, 2, 509))
    return dict(op=op, lens=lens, **spec, **head)


def _lengths(case):
    """Per sequence the tokens cached before the step and the step's new ones."""
    rng = random.Random(case["lens"])
    old = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["n_seq"])]
    new = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n_seq"])]
    if case["n_seq"] == 1:
        old, new = [case["ctx_hi"]], [max(1, case["q_hi"])]
    for i in rng.sample(range(case["n_seq"]), case["chunks"]):
        new[i] = case["chunk"]
    if not any(new):
        new[0] = 1
    return old, new


def work(case):
    if case["op"] == "plan":
        old, new = _lengths(case)
        b = case["block"]
        rows = case["n_seq"] * case["table"]
        read = sum(-(-o // b) for o in old) + sum(-(-(o + n) // b) - -(-o // b) for o, n in zip(old, new))
        return {"bytes": 4 * (2 * case["n_seq"] + read + rows + sum(new) + case["pad"] + 2 * case["n_seq"] + 1 + 8),
                "flops": 0}
    if case["op"] == "append":
        t, kept = case["tokens"], case["tokens"] - case["skip"]
        # rows in, cache written, cache read again, rows out, the slots twice
        return {"bytes": 2 * kept * case["n_kv"] * HEAD * SIZE[case["dtype"]] + 2 * kept * case["n_kv"] * TOKEN_BYTES
                + 2 * t * case["n_kv"] * HEAD * SIZE[case["dtype"]] + 8 * t,
                "flops": 6 * kept * case["n_kv"] * HEAD}
    old, new = _lengths(case)
    seen = sum(o + n for o, n in zip(old, new) if n)
    pairs = sum(n * o + n * (n + 1) // 2 for o, n in zip(old, new))
    return {"bytes": seen * case["n_kv"] * TOKEN_BYTES + 2 * sum(new) * case["n_q"] * HEAD * SIZE[case["dtype"]]
            + 4 * (sum(-(-(o + n) // case["block"]) for o, n in zip(old, new)) + 2 * case["n_seq"] + 1),
            "flops": 4 * pairs * case["n_q"] * HEAD}


# --------------------------------------------------------------- the inputs
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _plan_inputs(case, seed):
    """A pool half in use: the rows' blocks and the free list are a shuffle."""
    old, new = _lengths(case)
    b, n_seq = case["block"], case["n_seq"]
    held = [-(-o // b) for o in old]
    need = sum(-(-(o + n) // b) for o, n in zip(old, new)) - sum(held)
    n_blocks = sum(held) + need + 64
    order = torch.randperm(n_blocks, generator=_gen(seed, 1), device=DEV).to(torch.int32)
    table = torch.full((n_seq, case["table"]), NONE, dtype=torch.int32, device=DEV)
    cols = torch.arange(case["table"], device=DEV)
    table[cols[None, :] < torch.tensor(held, device=DEV)[:, None]] = order[:sum(held)]
    free = torch.full((n_blocks,), NONE, dtype=torch.int32, device=DEV)
    free[:n_blocks - sum(held)] = order[sum(held):]
    return dict(n_blocks=n_blocks, old=_ints(old), new=_ints(new), table=table, free=free,
                count=_ints([n_blocks - sum(held), 0, 0, 0]), tokens=sum(new) + case["pad"])


def _rows(n, n_kv, gain, gen, dtype):
    return (torch.randn(n, n_kv, HEAD, generator=gen, device=DEV) * gain).to(dtype)


def _gains(case, seed):
    """Channel gains of keys and values: a few channels stand out, as in trained keys."""
    g = _gen(seed, 2)
    k = torch.exp(0.4 * torch.randn(case["n_kv"], HEAD, generator=g, device=DEV))
    return k, 0.5 * torch.exp(0.3 * torch.randn(case["n_kv"], HEAD, generator=g, device=DEV))


def _append_inputs(case, seed):
    t, n_kv, dt = case["tokens"], case["n_kv"], DTYPES[case["dtype"]]
    kg, vg = _gains(case, seed)
    gen = _gen(seed, 3)
    if case["fused"]:       # k and v are columns of the projection's q | k | v rows
        qkv = torch.zeros(t, (case["n_q"] + 2 * n_kv) * HEAD, dtype=dt, device=DEV)
        k = qkv[:, case["n_q"] * HEAD:(case["n_q"] + n_kv) * HEAD].unflatten(1, (n_kv, HEAD))
        v = qkv[:, (case["n_q"] + n_kv) * HEAD:].unflatten(1, (n_kv, HEAD))
    else:
        k = torch.empty(t, n_kv, HEAD, dtype=dt, device=DEV)
        v = torch.empty(t, n_kv, HEAD, dtype=dt, device=DEV)
    k.copy_(_rows(t, n_kv, kg, gen, dt))
    v.copy_(_rows(t, n_kv, vg, gen, dt))
    n_blocks = -(-t // case["block"]) + 5
    blocks = torch.randperm(n_blocks, generator=gen, device=DEV)
    at = torch.arange(t, device=DEV)
    slots = (blocks[at // case["block"]] * case["block"] + at % case["block"]).to(torch.int32)
    slots[torch.randperm(t, generator=gen, device=DEV)[:case["skip"]]] = NONE
    return dict(n_blocks=n_blocks, k=k, v=v, slots=slots)


STRIP = 32768       # tokens whose keys and values are made at a time


def _attention_inputs(case, seed):
    """Block table, queries, and a maker of the cache's rows in strips of slots."""
    old, new = _lengths(case)
    b, dt = case["block"], DTYPES[case["dtype"]]
    kv = [o + n for o, n in zip(old, new)]
    held = [-(-n // b) for n in kv]
    n_blocks = sum(held) + 3
    order = torch.randperm(n_blocks, generator=_gen(seed, 1), device=DEV).to(torch.int32)
    width = max(held) + 1
    table = torch.full((case["n_seq"], width), NONE, dtype=torch.int32, device=DEV)
    table[torch.arange(width, device=DEV)[None, :] < torch.tensor(held, device=DEV)[:, None]] = order[:sum(held)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], case["n_q"], HEAD, generator=_gen(seed, 4), device=DEV)
    q = (q * torch.exp(0.3 * torch.randn(case["n_q"], HEAD, generator=_gen(seed, 5), device=DEV))).to(dt)
    kg, vg = _gains(case, seed)

    def strips():
        for s in range(0, n_blocks * b, STRIP):
            n = min(STRIP, n_blocks * b - s)
            gen = _gen(seed, 1000 + s // STRIP)
            yield s, _rows(n, case["n_kv"], kg, gen, torch.float32), _rows(n, case["n_kv"], vg, gen, torch.float32)

    return dict(n_blocks=n_blocks, starts_host=starts, kv_host=kv, starts=_ints(starts), kv=_ints(kv), table=table, q=q,
                strips=strips, scale=HEAD ** -0.5)


# ------------------------------------------------------------ the framework
_context = []


def _ctx():
    """The program's device context, one for all its caches."""
    import zero_b200 as zb

    if not _context:
        _context.append(zb.Context(device=torch.cuda.current_device()))
    return _context[0]


def _stream():
    """The current stream's handle; 1 names the legacy default stream."""
    return torch.cuda.current_stream().cuda_stream or 1


def _cache(case, n_blocks):
    import zero_b200 as zb

    return zb.KvCache4(_ctx(), n_blocks, case["block"], 1, case.get("n_kv", 1), HEAD)


def _type(case):
    import zero_b200 as zb

    return {"f32": zb.F32, "f16": zb.F16, "bf16": zb.BF16}[case["dtype"]]


# ------------------------------------------------------- prepare, run, exact
def prepare(case, seed):
    if case["op"] == "plan":
        st = _plan_inputs(case, seed)
        if own:
            st["cache"] = _cache(case, st["n_blocks"])
            n, c = case["n_seq"], st["tokens"]
            st["out"] = dict(table=torch.empty_like(st["table"]), slots=torch.empty(c, dtype=torch.int32, device=DEV),
                             starts=torch.empty(n + 1, dtype=torch.int32, device=DEV),
                             kv=torch.empty(n, dtype=torch.int32, device=DEV), count=torch.empty_like(st["count"]))
    elif case["op"] == "append":
        st = _append_inputs(case, seed)
        shape = (case["tokens"], case["n_kv"], HEAD)
        if own:
            st["cache"] = _cache(case, st["n_blocks"])
            st["k_out"] = torch.empty(shape, dtype=DTYPES[case["dtype"]], device=DEV)
            st["v_out"] = torch.empty(shape, dtype=DTYPES[case["dtype"]], device=DEV)
        else:
            n = st["n_blocks"] * case["block"]
            st["pool"] = [torch.zeros(n, case["n_kv"], HEAD, dtype=torch.int8, device=DEV) for _ in range(2)]
            st["scales"] = [torch.zeros(n, case["n_kv"], HEAD // GROUP, dtype=torch.float16, device=DEV) for _ in range(2)]
    else:
        st = _attention_inputs(case, seed)
        n = st["n_blocks"] * case["block"]
        if own:
            st["cache"] = _cache(case, st["n_blocks"])
            st["out"] = torch.empty_like(st["q"])
            for s, k, v in st["strips"]():
                slots = torch.arange(s, s + k.shape[0], dtype=torch.int32, device=DEV)
                st["cache"].append_device(0, k.shape[0], k.data_ptr(), v.data_ptr(), slots.data_ptr(), stream=_stream())
            torch.cuda.synchronize()
        else:
            st["pool"] = [torch.empty(n, case["n_kv"], HEAD // 2, dtype=torch.uint8, device=DEV) for _ in range(2)]
            st["scales"] = [torch.empty(n, case["n_kv"], HEAD // GROUP, dtype=torch.float16, device=DEV) for _ in range(2)]
            for s, k, v in st["strips"]():
                for x, pool, scales in zip((k, v), st["pool"], st["scales"]):
                    q, d = _quantise(x)
                    n8 = (q + 8).to(torch.uint8)
                    pool[s:s + k.shape[0]] = n8[..., 0::2] | (n8[..., 1::2] << 4)
                    scales[s:s + k.shape[0]] = d
    st["case"] = dict(case)
    return st


def run(st):
    case = st["case"]
    return {"plan": _run_plan, "append": _run_append, "attention": _run_attention}[case["op"]](case, st)


def _run_plan(case, st):
    if own:
        o = st["out"]
        st["cache"].plan_device(case["n_seq"], case["table"], st["old"].data_ptr(), st["new"].data_ptr(),
                                st["table"].data_ptr(), o["table"].data_ptr(), st["free"].data_ptr(),
                                st["count"].data_ptr(), o["count"].data_ptr(), st["tokens"], o["slots"].data_ptr(),
                                o["starts"].data_ptr(), o["kv"].data_ptr(), stream=_stream())
        return o
    b, width = case["block"], case["table"]
    old, new = st["old"].long(), st["new"].long()
    kv = old + new
    held, want = (old + b - 1) // b, (kv + b - 1) // b
    first = torch.cumsum(want - held, 0) - (want - held)          # blocks taken by the rows before
    taken = (want - held).sum()
    cols = torch.arange(width, device=DEV)[None, :]
    pick = st["count"][0].long() - 1 - (first[:, None] + cols - held[:, None])
    fresh = st["free"][pick.clamp(0, st["n_blocks"] - 1)]
    table = torch.where(cols < held[:, None], st["table"], torch.where(cols < want[:, None], fresh, NONE))
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), torch.cumsum(new, 0)])
    t = torch.arange(st["tokens"], device=DEV)
    row = torch.searchsorted(starts, t, right=True) - 1
    real = t < starts[-1]
    row = row.clamp(max=case["n_seq"] - 1)
    pos = torch.where(real, old[row] + t - starts[row], 0)
    slots = torch.where(real, table[row, pos // b].long() * b + pos % b, NONE)
    count = torch.stack([st["count"][0].long() - taken, torch.zeros_like(taken), starts[-1], taken])
    return dict(table=table.to(torch.int32), slots=slots.to(torch.int32), starts=starts.to(torch.int32),
                kv=kv.to(torch.int32), count=count.to(torch.int32))


def _quantise(x):
    """Integers -8..7 [..., 128] and binary16 scales [..., 4] of rows x."""
    g = x.float().unflatten(-1, (HEAD // GROUP, GROUP))
    a = g.abs()
    place = torch.arange(GROUP, device=x.device)
    first = torch.where(a == a.amax(-1, keepdim=True), place, GROUP).amin(-1, keepdim=True)
    d = (g.gather(-1, first) * -0.125).to(torch.bfloat16).to(torch.float16)
    # the quotient in 64 bits: in 32 it can round onto a border between integers
    q = torch.round(g.double() / d.double()).clamp(-8, 7)
    q = torch.where(d == 0, 0, q)
    return q.flatten(-2).to(torch.int8), d.squeeze(-1)


def _values(q, d):
    return (q.unflatten(-1, (HEAD // GROUP, GROUP)).float() * d.float()[..., None]).flatten(-2)


def _run_append(case, st):
    t = case["tokens"]
    if own:
        c, dt = st["cache"], _type(case)
        c.append_device(0, t, st["k"].data_ptr(), st["v"].data_ptr(), st["slots"].data_ptr(), dtype=dt,
                        k_stride=st["k"].stride(0), v_stride=st["v"].stride(0), stream=_stream())
        c.gather_device(0, t, st["slots"].data_ptr(), st["k_out"].data_ptr(), st["v_out"].data_ptr(), dtype=dt,
                        stream=_stream())
        return [st["k_out"], st["v_out"]]
    kept = st["slots"] >= 0
    at = st["slots"].long().clamp(min=0)
    out = []
    for x, pool, scales in zip((st["k"], st["v"]), st["pool"], st["scales"]):
        q, d = _quantise(x)
        keep = kept[:, None, None]
        # a padded token goes to a row behind the pool, which is dropped
        for to, what in ((pool, q), (scales, d)):
            wide = torch.cat([to, to[:1]])
            wide[torch.where(kept, at, to.shape[0])] = what
            to.copy_(wide[:-1])
        out.append(torch.where(keep, _values(pool[at], scales[at]), 0).to(x.dtype))
    return out


def _slots(st, case, i, n):
    pos = torch.arange(n, device=DEV)
    return st["table"][i].long()[pos // case["block"]] * case["block"] + pos % case["block"]


SCORES = 1 << 27    # scores held at a time


def _run_attention(case, st):
    if own:
        st["cache"].attention_device(0, case["n_seq"], st["q"].shape[0], max(1, max(b - a for a, b in zip(
            st["starts_host"], st["starts_host"][1:]))), case["n_q"], st["q"].data_ptr(), st["out"].data_ptr(),
            st["starts"].data_ptr(), st["kv"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1],
            dtype=_type(case), scale=st["scale"], stream=_stream())
        return st["out"]
    out = torch.empty_like(st["q"])
    group = case["n_q"] // case["n_kv"]
    for i, n in enumerate(st["kv_host"]):
        a, b = st["starts_host"][i], st["starts_host"][i + 1]
        if a == b:
            continue
        at = _slots(st, case, i, n)
        k, v = (_values(_unpack(pool[at]), scales[at]).transpose(0, 1) for pool, scales in zip(st["pool"], st["scales"]))
        step = max(1, SCORES // (n * case["n_q"]))
        for c in range(a, b, step):
            e = min(b, c + step)
            q = st["q"][c:e].float().unflatten(1, (case["n_kv"], group)).permute(1, 2, 0, 3)     # kv head, head, token
            s = torch.matmul(q.flatten(1, 2), k.transpose(1, 2)) * st["scale"]
            s = s.unflatten(1, (group, e - c))
            if b - a > 1:
                last = n - b + torch.arange(c, e, device=DEV)
                s = s.masked_fill(torch.arange(n, device=DEV) > last[:, None], float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(p.flatten(1, 2), v).unflatten(1, (group, e - c)) / p.sum(-1, keepdim=True)
            out[c:e] = o.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
    return out


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2).to(torch.int8) - 8


# ------------------------------------------------------ 64-bit definitions
def _exact_values(x):
    """What the cache stands for after storing rows x, from the definition."""
    g = x.double().reshape(*x.shape[:-1], HEAD // GROUP, GROUP)
    hi, lo = g.amax(-1), g.amin(-1)
    # the first of equals only matters where +m and -m are both there
    back = torch.arange(GROUP, 0, -1, device=x.device)
    at_hi, at_lo = ((back * (g == e[..., None])).amax(-1) for e in (hi, lo))      # larger: earlier
    m = torch.where((hi > -lo) | ((hi == -lo) & (at_hi > at_lo)), hi, lo)
    mant, ex = torch.frexp(-m / 8)
    d = torch.ldexp(torch.round(mant * 256), ex - 8)              # 8 significant bits
    grid = torch.clamp(torch.frexp(d)[1] - 11, min=-24)           # binary16's last place
    d = torch.ldexp(torch.round(torch.ldexp(d, -grid)), grid)[..., None]
    q = torch.where(d == 0, torch.zeros_like(g), torch.round(g / torch.where(d == 0, torch.ones_like(d), d)))
    return (q.clamp(-8, 7) * d).reshape(x.shape)


def exact(case, seed):
    if case["op"] == "plan":
        return None                 # whole numbers: the plain form is exact
    if case["op"] == "append":
        st = _append_inputs(case, seed)
        keep = (st["slots"] >= 0)[:, None, None]
        return [torch.where(keep, _exact_values(x), torch.zeros((), dtype=torch.float64, device=DEV))
                for x in (st["k"], st["v"])]
    st = _attention_inputs(case, seed)
    n = st["n_blocks"] * case["block"]
    k, v = (torch.empty(n, case["n_kv"], HEAD, dtype=torch.float32, device=DEV) for _ in range(2))
    for s, ks, vs in st["strips"]():
        k[s:s + ks.shape[0]] = _exact_values(ks)                  # 11 significant bits at most: held exactly
        v[s:s + ks.shape[0]] = _exact_values(vs)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    group = case["n_q"] // case["n_kv"]
    for i, total in enumerate(st["kv_host"]):
        a, b = st["starts_host"][i], st["starts_host"][i + 1]
        at = _slots(st, case, i, total)
        for h in range(case["n_kv"] if b > a else 0):
            kh, vh = k[at, h].double(), v[at, h].double()
            step = max(1, (1 << 26) // (total * group))
            for c in range(a, b, step):
                e = min(b, c + step)
                s = torch.einsum("tgd,nd->tgn", st["q"][c:e, h * group:(h + 1) * group].double(), kh) * st["scale"]
                seen = torch.arange(total, device=DEV)[None, :] <= (total - b + torch.arange(c, e, device=DEV))[:, None]
                w = torch.softmax(s.masked_fill(~seen[:, None], float("-inf")), -1)
                out[c:e, h * group:(h + 1) * group] = torch.einsum("tgn,nd->tgd", w, vh)
    return out
