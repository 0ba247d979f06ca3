"""CPU tests of the paged 4-bit KV cache: the tile layout is a bijection whose
bytes belong to one token each, the format's values are exact in binary16, and
every refusal comes before the library touches a device."""
import subprocess
from pathlib import Path

import numpy as np

import kv4_ref as R
from zero_b200 import _lib

ROOT = Path(__file__).resolve().parent.parent


def k_bits(t, dim):
    g, c, i = dim // 32, dim % 32 // 8, dim % 8
    return [8 * (64 * t + 16 * c + 4 * g) + 16 * (i % 2) + 4 * (i // 2) + b for b in range(4)]


def v_bits(t, dim):
    g, s, r = dim // 32, dim % 32 // 8, dim % 8
    at = 8 * (1152 + 512 * (t // 8) + 16 * (4 * r + t % 8 // 2) + 4 * g + 2 * (t % 2))
    return [at + (([6, 2, 10, 14][s] + b) % 16) for b in range(4)]


def test_tile_layout_is_a_bijection_with_whole_bytes_per_token():
    seen, owner = set(), {}
    for t in range(16):
        for dim in range(128):
            for b in k_bits(t, dim) + v_bits(t, dim):
                assert b not in seen
                seen.add(b)
                assert owner.setdefault(b // 8, t) == t
    assert seen == set(range(8 * 1024)) | set(range(8 * 1152, 8 * 2176))
    scale = {2 * (2 * (16 * (t // 8) + 4 * (t % 8 // 2) + g) + t % 2) for t in range(16) for g in range(4)}
    assert scale == set(range(0, 128, 2))


def test_values_and_the_dequantising_constant_are_exact_in_binary16():
    """q d and 24 d for every scale the format can hold."""
    bits = np.arange(0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)
    mant, _ = np.frexp(bits)
    d = bits[(mant * 256 == np.rint(mant * 256)) & (bits <= 2720)]
    assert len(d) > 3000 and d.max() == 2720
    for q in list(range(-8, 8)) + [24]:
        assert np.array_equal((q * d).astype(np.float16).astype(np.float64), q * d)
    # what the quantiser gives is among them
    x = np.random.default_rng(0).standard_normal((2000, 128)) * np.exp2(np.random.default_rng(1).uniform(-30, 12, (2000, 1)))
    _, got = R.quantise(x.astype(np.float32))
    assert np.isin(np.abs(got), d).all()


def test_work_ranges_cover_every_unit_once_and_name_their_sharers():
    """The attention cuts W units into G ranges [W b / G, W (b + 1) / G); the
    range that holds unit x is ((x + 1) G - 1) / W."""
    rng = np.random.default_rng(2)
    for _ in range(300):
        G = int(rng.integers(1, 400))
        W = int(rng.integers(G, 5000 if rng.random() < 0.9 else 1 << 40))
        for b in [0, G - 1] + [int(v) for v in rng.integers(0, G, 20)]:
            lo, hi = W * b // G, W * (b + 1) // G
            assert lo < hi
            for x in (lo, hi - 1, (lo + hi) // 2):
                assert ((x + 1) * G - 1) // W == b


REFUSALS = r"""
#include <stdio.h>
#include "kv4.h"
static int fails = 0, n = 0;
#define WANT(code, call) do { ++n; int got = (int)(call); if (got != (int)(code)) { printf("%d: %s gave %d\n", __LINE__, #call, got); ++fails; } } while (0)
int main() {
  // never a device call: the handles are made by hand, the addresses mean nothing
  zgpu_ctx ctx, other;
  zgpu_kv4 kv, *out = 0;
  zgpu_kv4_work w, w2;
  kv.ctx = &ctx; kv.n_blocks = 10; kv.block_tokens = 16; kv.bt_log2 = 4; kv.n_layers = 2; kv.n_kv = 2;
  w.ctx = &ctx; w2.ctx = &other;
  char *m = (char *)0x10000;
  uint32_t *a = (uint32_t *)m, *o = (uint32_t *)(m + 0x100000);
  const int ARG = ZGPU_ERR_INVALID_ARG;
  WANT(ARG, zgpu_kv4_create(0, 4, 16, 1, 1, 128, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 4, 16, 1, 1, 128, 0));
  WANT(ARG, zgpu_kv4_create(&ctx, 0, 16, 1, 1, 128, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 4, 16, 0, 1, 128, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 4, 16, 1, 0, 128, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 4, 16, 1, 1, 64, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 4, 8, 1, 1, 128, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 4, 24, 1, 1, 128, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 4, 256, 1, 1, 128, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 4, 16, 1, 1025, 128, &out));
  WANT(ARG, zgpu_kv4_create(&ctx, 1u << 27, 16, 1, 1, 128, &out));
  WANT(ARG, zgpu_kv4_work_create(0, 0));
  WANT(ARG, zgpu_kv4_check(0));
  zgpu_kv4_destroy(0);
  zgpu_kv4_work_destroy(0);
  // plan: n_seq, width, old, new, tin, tout, free, sin, sout, n_slots, slots, starts, kv
#define PLAN(ns, wd, old, nw, ti, to, fr, si, so, nl, sl, st, kl) zgpu_kv4_plan_device(&kv, ns, wd, old, nw, ti, to, fr, si, so, nl, sl, st, kl, 0)
  uint32_t *i1 = a, *i2 = a + 4096, *i3 = a + 8192, *i4 = a + 100000, *i5 = a + 110000;
  uint32_t *o1 = o, *o2 = o + 100000, *o3 = o + 110000, *o4 = o + 120000, *o5 = o + 130000;
  WANT(ARG, zgpu_kv4_plan_device(0, 4, 8, i1, i2, i3, o1, i4, i5, o2, 9, o3, o4, o5, 0));
  WANT(ARG, PLAN(0, 8, i1, i2, i3, o1, i4, i5, o2, 9, o3, o4, o5));
  WANT(ARG, PLAN(1025, 8, i1, i2, i3, o1, i4, i5, o2, 9, o3, o4, o5));
  WANT(ARG, PLAN(4, 0, i1, i2, i3, o1, i4, i5, o2, 9, o3, o4, o5));
  WANT(ARG, PLAN(4, 1u << 28, i1, i2, i3, o1, i4, i5, o2, 9, o3, o4, o5));
  WANT(ARG, PLAN(4, 8, 0, i2, i3, o1, i4, i5, o2, 9, o3, o4, o5));
  WANT(ARG, PLAN(4, 8, i1, i2, i3, o1, i4, i5, o2, 9, 0, o4, o5));
  WANT(ARG, PLAN(4, 8, i1, i2, i3, o1, i4, i5, o2, 0x80000000u, o3, o4, o5));
  WANT(ARG, PLAN(4, 8, (uint32_t *)(m + 2), i2, i3, o1, i4, i5, o2, 9, o3, o4, o5));
  WANT(ARG, PLAN(4, 8, i1, i2, i3, i3 + 1, i4, i5, o2, 9, o3, o4, o5));   // shifted in place
  WANT(ARG, PLAN(4, 8, i1, i2, i3, o1, i4, i5, i5, 9, o3, o4, o5));       // state in place
  WANT(ARG, PLAN(4, 8, i1, i2, i3, o1, i4, i5, o2, 9, o3, o4, i1));       // lengths in place
  WANT(ARG, PLAN(4, 8, i1, i2, i3, o1, i4, i5, o2, 9, o3, o3 + 8, o5));   // outputs overlap
  WANT(ARG, PLAN(4, 8, i1, i2, i3, o1, i4, i5, o2, 9, i4 + 9, o4, o5));   // slots over the free list
#define REL(ns, wd, dn, ln, tb, fr, st) zgpu_kv4_release_device(&kv, ns, wd, dn, ln, tb, fr, st, 0)
  WANT(ARG, REL(0, 8, i1, o1, o2, o3, o4));
  WANT(ARG, REL(1025, 8, i1, o1, o2, o3, o4));
  WANT(ARG, REL(4, 0, i1, o1, o2, o3, o4));
  WANT(ARG, REL(4, 8, i1, o1, o2, o3, 0));
  WANT(ARG, REL(4, 8, i1, i1, o2, o3, o4));
  WANT(ARG, REL(4, 8, i1, o1, o2, o2 + 31, o4));
  // rows
  void *k = m + 0x400000, *v = m + 0x800000;
#define APP(l, n, k, ks, v, vs, t, s) zgpu_kv4_append_device(&kv, l, n, k, ks, v, vs, t, s, 0)
  WANT(ARG, zgpu_kv4_append_device(0, 0, 1, k, 0, v, 0, ZGPU_F32, a, 0));
  WANT(ARG, APP(0, 1, 0, 0, v, 0, ZGPU_F32, a));
  WANT(ARG, APP(0, 1, k, 0, v, 0, ZGPU_F32, 0));
  WANT(ZGPU_ERR_KV_LAYER_OUT_OF_RANGE, APP(2, 1, k, 0, v, 0, ZGPU_F32, a));
  WANT(ZGPU_ERR_UNSUPPORTED_QUANT, APP(0, 1, k, 0, v, 0, ZGPU_Q4_0, a));
  WANT(ARG, APP(0, 0x80000000u, k, 0, v, 0, ZGPU_F32, a));
  WANT(ARG, APP(0, 1, k, 255, v, 0, ZGPU_F32, a));
  WANT(ARG, APP(0, 1, k, 0, v, 258, ZGPU_F32, a));
  WANT(ARG, APP(0, 1, k, 260, v, 0, ZGPU_F16, a));
  WANT(ARG, APP(0, 1, (char *)k + 8, 0, v, 0, ZGPU_F32, a));
  WANT(ARG, APP(0, 1, k, 0, v, 0, ZGPU_BF16, (uint32_t *)(m + 1)));
  WANT(ZGPU_OK, APP(0, 0, 0, 0, 0, 0, ZGPU_F32, 0));
  WANT(ARG, zgpu_kv4_gather_device(&kv, 0, 1, a, 0, 0, 0, 0, ZGPU_F32, 0));
  WANT(ARG, zgpu_kv4_gather_device(&kv, 0, 1, a, (char *)k + 4, 0, 0, 0, ZGPU_F32, 0));
  WANT(ZGPU_ERR_KV_LAYER_OUT_OF_RANGE, zgpu_kv4_gather_device(&kv, 9, 1, a, k, 0, v, 0, ZGPU_F32, 0));
  // attention: work, layer, n_seq, rows, max_q, heads, q, qs, out, os, type, starts, lens, table, width, scale
#define ATT(wk, l, ns, nr, mq, h, q, qs, u, us, t, st, ln, tb, wd, sc) zgpu_kv4_attention_device(&kv, wk, l, ns, nr, mq, h, q, qs, u, us, t, st, ln, tb, wd, sc, 0)
  WANT(ARG, ATT(0, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w2, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ZGPU_ERR_KV_LAYER_OUT_OF_RANGE, ATT(&w, 2, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ZGPU_ERR_UNSUPPORTED_QUANT, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_Q8_0, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 0, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1025, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 0, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 3, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 34, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 508, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 514, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, (char *)v + 8, 0, ZGPU_F16, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, (uint32_t *)(m + 2), a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 0, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 1u << 28, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 0.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, -1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1e39));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, __builtin_nanf("")));
  WANT(ARG, ATT(&w, 0, 1, 0x80000000u, 1, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 0x80000000u, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ARG, ATT(&w, 0, 1, 1, 1, 4, 0, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ZGPU_OK, ATT(&w, 0, 1, 0, 1, 4, 0, 0, 0, 0, ZGPU_F32, a, a, a, 4, 1.f));
  WANT(ZGPU_OK, ATT(&w, 0, 1, 1, 0, 4, k, 0, v, 0, ZGPU_F32, a, a, a, 4, 1.f));
  printf("%d calls, %d wrong\n", n, fails);
  return fails != 0;
}
"""


def test_refusals_come_before_any_device_call(tmp_path):
    src = tmp_path / "refuse.cpp"
    src.write_text(REFUSALS)
    exe = tmp_path / "refuse"
    lib = Path(_lib.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-O0", "-w", f"-I{ROOT / 'zero_b200' / 'csrc'}", "-I/usr/local/cuda/include",
                    str(src), str(lib), f"-Wl,-rpath,{lib.parent}", "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
