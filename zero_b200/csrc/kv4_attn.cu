// kv4_attn.cu — attention of a ragged batch over the paged 4-bit KV cache.
//
// o = softmax(scale * q K^T) V per query row, over the keys up to the row's
// own position: row i's queries are its last ones, query t of n at position
// kv_len - n + t.
//
// kv4_rows_kernel: few query rows per kv head (decode, short continuations).
// Bound by the cache read, 144 bytes per key and kv head, and close behind it
// by instruction issue: unpacking 256 values per key and head.
//
//   Rows.  The query rows of a kv head (its group of heads, times the new
//   tokens) are taken eight at a time.  The tensor cores multiply 16-bit
//   values (m16n8k16, f32 sums); a row is put in as hi + lo, two binary16
//   values whose sum holds 22 bits, in rows r and r + 8 of the fragment.  The
//   cache's values are exact in binary16, so q K^T and P V keep f32 accuracy
//   at the price of eight rows instead of sixteen, which a memory-bound
//   kernel has to spare; both halves of a sum land in one thread.  A query
//   row is scaled by a power of two first (its largest value in [1, 2)), so
//   neither half leaves binary16's range; P is held times 2^15, which keeps
//   probabilities down to 2^-39 of the row's largest.
//
//   Loads.  Each warp streams its own tiles (16 keys, 2304 contiguous bytes)
//   through a private ring of bulk copies, one mbarrier a stage, and no
//   barrier joins the warps until a piece of work ends.  The tile's layout is
//   the fragment's (kv4.h): 16-byte shared loads without bank conflicts, and
//   per two values a shift, a logical operation and one half2 fma:
//   (16 + n) d - 24 d = (n - 8) d, exact because 24 d is.
//
//   Split.  All pieces of work (sequence, kv head, eight rows) are laid end to
//   end in units of one tile and cut into equal ranges, one per CTA, so a
//   ragged batch or one long sequence keeps every SM equally busy.  A piece
//   cut by a range boundary leaves unnormalised partials (max, sum, o) in the
//   workspace; the CTA that arrives last merges them in range order, so the
//   result does not depend on which one that is.
#include <cuda_bf16.h>

#include "common.cuh"
#include "kv4.h"

namespace zgpu {

namespace {

constexpr uint32_t kWarps = 8;
constexpr uint32_t kCtasPerSm = 2;
constexpr uint32_t kStages = 4;                  // tiles in flight per warp
constexpr uint32_t kRows = 8;                    // query rows of a piece
constexpr uint32_t kPartFloats = kRows * (kKv4Head + 2);   // o, max, sum
constexpr float kPShift = 15.f;                  // P is held times 2^15
constexpr uint32_t kMinTiles = kWarps;           // a range is worth a tile per warp

// Dynamic shared memory: the warps' rings, the warps' partials, the sums of
// work over the sequences.
constexpr uint32_t kRingBytes = kWarps * kStages * kKv4TileBytes;
constexpr uint32_t kMergeBytes = kWarps * kPartFloats * 4;
constexpr uint32_t kOffMerge = kRingBytes;
constexpr uint32_t kOffSums = kOffMerge + kMergeBytes;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 bits2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Nibble s of both halves of w as (n - 8) d: the nibble becomes bits 6..9 of
// a binary16 with 16's exponent, 16 + n.
template <int S>
__device__ __forceinline__ uint32_t dequant2(uint32_t w, __half2 d, __half2 m24d) {
  const uint32_t sh = S == 0 ? w << 6 : S == 1 ? w << 2 : S == 2 ? w >> 2 : w >> 6;
  const uint32_t x = (sh & 0x03C003C0u) | 0x4C004C00u;
  return h2bits(__hfma2(bits2h(x), d, m24d));
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}

template <class T>
__device__ __forceinline__ float4 q4(const T *p);
template <>
__device__ __forceinline__ float4 q4<float>(const float *p) {
  return __ldg(reinterpret_cast<const float4 *>(p));
}
template <>
__device__ __forceinline__ float4 q4<__half>(const __half *p) {
  const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
  const float2 a = __half22float2(bits2h(u.x)), b = __half22float2(bits2h(u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 q4<__nv_bfloat16>(const __nv_bfloat16 *p) {
  const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xFFFF0000u));
}
__device__ __forceinline__ void put4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void put4(__half *p, float4 v) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(h2bits(__floats2half2_rn(v.x, v.y)), h2bits(__floats2half2_rn(v.z, v.w)));
}
__device__ __forceinline__ void put4(__nv_bfloat16 *p, float4 v) {
  __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
}

// One sequence as the call gives it, with lengths that cannot lead outside
// the buffers; *bad says that they would have.
struct Seq {
  uint32_t q0, nq, len;
};
__device__ __forceinline__ Seq load_seq(const Kv4AttnParams &p, uint32_t i, bool *bad) {
  Seq s;
  s.q0 = p.starts[i];
  const uint32_t q1 = p.starts[i + 1];
  s.len = p.kv_lens[i];
  s.nq = q1 - s.q0;
  if (q1 < s.q0 || q1 > p.n_rows || s.nq > p.max_q) {
    s.nq = 0;
    *bad = true;
  }
  const uint64_t most = static_cast<uint64_t>(p.table_width) << p.bt_log2;
  if (s.len > most) {
    s.len = static_cast<uint32_t>(most);
    *bad = true;
  }
  return s;
}

struct WarpState {
  float o[16][4];
  float m, l;
};

template <class T>
__global__ void __launch_bounds__(32 * kWarps, kCtasPerSm) kv4_rows_kernel(const Kv4AttnParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps * kStages];
  __shared__ uint64_t s_scan[kWarps];
  __shared__ uint32_t s_last;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  uint64_t *sums = reinterpret_cast<uint64_t *>(smem + kOffSums);   // work before sequence i, n_seq + 1
  float *merge = reinterpret_cast<float *>(smem + kOffMerge);
  const uint32_t ring = smem_addr(smem) + warp * kStages * kKv4TileBytes;
  const uint32_t bar0 = smem_addr(&bars[warp * kStages]);

  if (lane == 0) {
    for (uint32_t s = 0; s < kStages; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_barrier_init();
  }
  // work of sequence i: kv heads x pieces of eight rows x tiles
  {
    uint64_t base = 0;
    bool bad = false, blind = false;
    for (uint32_t i0 = 0; i0 < p.n_seq; i0 += 32 * kWarps) {
      const uint32_t i = i0 + tid;
      uint64_t w = 0;
      if (i < p.n_seq) {
        const Seq s = load_seq(p, i, &bad);
        blind |= s.len < s.nq;
        w = static_cast<uint64_t>((s.nq * p.group + kRows - 1) / kRows) * p.n_kv * ((s.len + kKv4Tile - 1) / kKv4Tile);
      }
      uint64_t inc = w;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= static_cast<uint32_t>(off)) inc += u;
      }
      if (lane == 31) s_scan[warp] = inc;
      __syncthreads();
      uint64_t before = base, all = 0;
      for (uint32_t k = 0; k < kWarps; ++k) {
        if (k < warp) before += s_scan[k];
        all += s_scan[k];
      }
      if (i < p.n_seq) sums[i] = before + inc - w;
      base += all;
      __syncthreads();
    }
    if (tid == 0) sums[p.n_seq] = base;
    if (bad && blockIdx.x == 0) atomicOr(p.status, ZDEV_ERR_BOUNDS);
    // queries before position 0 see no key and are in no range: zeros
    if (__syncthreads_or(blind) && blockIdx.x == 0)
      for (uint32_t i = 0; i < p.n_seq; ++i) {
        const Seq s = load_seq(p, i, &bad);
        const uint32_t cols = p.n_kv * p.group * (kKv4Head / 4);
        const uint64_t n = s.len < s.nq ? static_cast<uint64_t>(s.nq - s.len) * cols : 0;
        for (uint64_t k = tid; k < n; k += 32 * kWarps)
          put4(static_cast<T *>(p.out) + (s.q0 + k / cols) * p.out_stride + 4 * (k % cols),
               make_float4(0.f, 0.f, 0.f, 0.f));
      }
  }

  const uint64_t W = sums[p.n_seq];
  uint64_t G = (W + kMinTiles - 1) / kMinTiles;
  if (G > gridDim.x) G = gridDim.x;
  if (blockIdx.x >= G) return;
  uint64_t at = W * blockIdx.x / G;
  const uint64_t end = W * (blockIdx.x + 1) / G;
  uint32_t seq = 0;
  {
    uint32_t lo = 0, hi = p.n_seq;   // sums[lo] <= at < sums[hi]
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (sums[mid] <= at) lo = mid;
      else hi = mid;
    }
    seq = lo;
  }
  uint32_t it0 = 0;         // tiles that this warp took before the piece: stage and phase of the ring
  bool dead = false;        // a wait of this warp ran out

  while (at < end) {
    while (sums[seq + 1] <= at) ++seq;
    bool bad = false;
    const Seq s = load_seq(p, seq, &bad);
    const uint32_t n_tiles = (s.len + kKv4Tile - 1) / kKv4Tile;
    const uint32_t pieces = (s.nq * p.group + kRows - 1) / kRows;
    const uint64_t piece = (at - sums[seq]) / n_tiles;
    const uint64_t piece_at = sums[seq] + piece * n_tiles;   // the piece in units of work
    const uint32_t head = static_cast<uint32_t>(piece / pieces), rt = static_cast<uint32_t>(piece % pieces);
    const uint32_t t0 = static_cast<uint32_t>(at - piece_at);
    const uint32_t t1 = static_cast<uint32_t>(end - piece_at < n_tiles ? end - piece_at : n_tiles);
    const uint32_t *table = p.table + static_cast<size_t>(seq) * p.table_width;
    const uint32_t tpb_log2 = p.bt_log2 - 4;
    // this warp's tiles: t0 + warp + 8 k, k < nk
    const uint32_t nk = t1 - t0 > warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;

    // blocks of the next 32 tiles to be copied, one per lane, and of the 32 after
    auto entry = [&](uint32_t k) -> uint32_t {
      return k < nk ? __ldg(table + ((t0 + warp + kWarps * k) >> tpb_log2)) : 0u;
    };
    uint32_t ent = entry(lane), ent_next = entry(32 + lane), issued = 0;
    uint32_t bad_block = 0;      // bit k % 32 of the tiles in flight
    auto issue = [&]() {
      const uint32_t k = issued, tile = t0 + warp + kWarps * k;
      const uint32_t block = __shfl_sync(0xffffffffu, ent, k & 31u);
      const uint32_t stage = (it0 + k) % kStages, bar = bar0 + 8 * stage, dst = ring + stage * kKv4TileBytes;
      const bool ok = block < p.n_blocks;
      if (lane == 0) {
        if (ok) {
          const uint8_t *src =
              p.pool + (((static_cast<size_t>(block) * p.n_kv + head) << tpb_log2) + (tile & ((1u << tpb_log2) - 1u))) *
                           kKv4TileBytes;
          mbar_arrive_expect_tx(bar, kKv4TileBytes);
          bulk_copy_g2s(dst, src, kKv4TileBytes, bar);
        } else {
          mbar_arrive(bar);
          atomicOr(p.status, ZDEV_ERR_BOUNDS);
        }
      }
      bad_block = (bad_block & ~(1u << (k & 31u))) | (ok ? 0u : 1u << (k & 31u));
      ++issued;
      if ((issued & 31u) == 0) {
        ent = ent_next;
        ent_next = entry(issued + 32 + lane);
      }
    };
    const uint32_t ahead = nk < kStages ? nk : kStages;
    if (!dead)
      while (issued < ahead) issue();

    // the queries: row r of the piece, dims 32 c .. 32 c + 31, hi and lo
    const uint32_t row = rt * kRows + r, n_rows = s.nq * p.group;
    const uint32_t tok = row < n_rows ? row / p.group : 0, hd = row < n_rows ? row % p.group : 0;
    uint32_t qh[8][2], ql[8][2];
    float scl;
    {
      const T *qp = static_cast<const T *>(p.q) + (s.q0 + tok) * p.q_stride +
                    (static_cast<size_t>(head) * p.group + hd) * kKv4Head + 32 * c;
      float4 x[8];
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] = q4(qp + 4 * k);
        amax = fmaxf(fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w))), amax);
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
      e = e < -100 ? -100 : e > 126 ? 126 : e;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      scl = p.scale * 1.44269504088896341f * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float y[4] = {x[k].x * down, x[k].y * down, x[k].z * down, x[k].w * down};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const __half2 hi = __floats2half2_rn(y[2 * h], y[2 * h + 1]);
          const float2 f = __half22float2(hi);
          qh[k][h] = h2bits(hi);
          ql[k][h] = h2bits(__floats2half2_rn(y[2 * h] - f.x, y[2 * h + 1] - f.y));
        }
      }
    }
    // keys that row r sees: 0 .. limit - 1 (none when its position is negative)
    const int64_t pos1 = static_cast<int64_t>(s.len) - s.nq + tok + 1;
    const uint32_t limit = row < n_rows && pos1 > 0 ? static_cast<uint32_t>(pos1) : 0u;

    WarpState st;
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int n = 0; n < 16; ++n) st.o[n][0] = st.o[n][1] = st.o[n][2] = st.o[n][3] = 0.f;

    for (uint32_t k = 0; k < nk && !dead; ++k) {
      const uint32_t stage = (it0 + k) % kStages, base = ring + stage * kKv4TileBytes;
      dead = __any_sync(0xffffffffu, !mbar_wait(bar0 + 8 * stage, ((it0 + k) / kStages) & 1u, p.status));
      if (dead) {       // the copies in flight land before the CTA may end
        for (++k; k < issued; ++k) mbar_wait(bar0 + 8 * ((it0 + k) % kStages), ((it0 + k) / kStages) & 1u, p.status);
        break;
      }
      const uint32_t key0 = (t0 + warp + kWarps * k) * kKv4Tile;
      if (!((bad_block >> (k & 31u)) & 1u)) {
        float sc[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 w = lds128(base + 512 * u + 16 * lane);
          const uint32_t dw = lds16(base + kKv4Ks + 64 * u + 2 * lane);
          const __half2 d = bits2h(dw | dw << 16), m24 = __hmul2(d, __float2half2_rn(-24.f));
          sc[u][0] = sc[u][1] = sc[u][2] = sc[u][3] = 0.f;
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma16816(sc[u], qh[2 * j][0], ql[2 * j][0], qh[2 * j][1], ql[2 * j][1], dequant2<0>(ww[j], d, m24),
                     dequant2<1>(ww[j], d, m24));
            mma16816(sc[u], qh[2 * j + 1][0], ql[2 * j + 1][0], qh[2 * j + 1][1], ql[2 * j + 1][1],
                     dequant2<2>(ww[j], d, m24), dequant2<3>(ww[j], d, m24));
          }
        }
        float v[4];
        float mx = st.m;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t key = key0 + 8 * u + 2 * c + e;
            v[2 * u + e] = key < limit ? (sc[u][e] + sc[u][2 + e]) * scl : -INFINITY;
            mx = fmaxf(mx, v[2 * u + e]);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float ms = mx == -INFINITY ? 0.f : mx;
        if (__any_sync(0xffffffffu, mx > st.m)) {
          const float a = ex2(st.m - ms);
          st.l *= a;
#pragma unroll
          for (int n = 0; n < 16; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[n][e] *= a;
          st.m = mx;
        }
        uint32_t ph[2], pl[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float p0 = ex2(v[2 * u] - (ms - kPShift)), p1 = ex2(v[2 * u + 1] - (ms - kPShift));
          st.l += p0 + p1;
          const __half2 hi = __floats2half2_rn(p0, p1);
          const float2 f = __half22float2(hi);
          ph[u] = h2bits(hi);
          pl[u] = h2bits(__floats2half2_rn(p0 - f.x, p1 - f.y));
        }
        const uint4 w0 = lds128(base + kKv4V + 16 * lane), w1 = lds128(base + kKv4V + 512 + 16 * lane);
        const uint4 d0 = lds128(base + kKv4Vs + 16 * c), d1 = lds128(base + kKv4Vs + 64 + 16 * c);
        const uint32_t a0[4] = {w0.x, w0.y, w0.z, w0.w}, a1[4] = {w1.x, w1.y, w1.z, w1.w};
        const uint32_t e0[4] = {d0.x, d0.y, d0.z, d0.w}, e1[4] = {d1.x, d1.y, d1.z, d1.w};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const __half2 x0 = bits2h(e0[g]), x1 = bits2h(e1[g]);
          const __half2 y0 = __hmul2(x0, __float2half2_rn(-24.f)), y1 = __hmul2(x1, __float2half2_rn(-24.f));
          mma16816(st.o[4 * g], ph[0], pl[0], ph[1], pl[1], dequant2<0>(a0[g], x0, y0), dequant2<0>(a1[g], x1, y1));
          mma16816(st.o[4 * g + 1], ph[0], pl[0], ph[1], pl[1], dequant2<1>(a0[g], x0, y0), dequant2<1>(a1[g], x1, y1));
          mma16816(st.o[4 * g + 2], ph[0], pl[0], ph[1], pl[1], dequant2<2>(a0[g], x0, y0), dequant2<2>(a1[g], x1, y1));
          mma16816(st.o[4 * g + 3], ph[0], pl[0], ph[1], pl[1], dequant2<3>(a0[g], x0, y0), dequant2<3>(a1[g], x1, y1));
        }
      }
      __syncwarp();       // every lane has read the stage before it is filled again
      if (issued < nk) issue();
    }
    it0 += nk;

    // the warps' states, then the piece
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
    float *mine = merge + warp * kPartFloats;
#pragma unroll
    for (int n = 0; n < 16; ++n)
      *reinterpret_cast<float2 *>(mine + r * kKv4Head + 8 * n + 2 * c) =
          make_float2(st.o[n][0] + st.o[n][2], st.o[n][1] + st.o[n][3]);
    if (c == 0) {
      mine[kRows * kKv4Head + 2 * r] = st.m;
      mine[kRows * kKv4Head + 2 * r + 1] = st.l;
    }
    __syncthreads();
    // thread: row mr, dims 4 mc ..
    const uint32_t mr = tid >> 5, mc = tid & 31;
    float M = -INFINITY, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    auto fold = [&](float m, float l, float4 o) {
      if (m == -INFINITY && l == 0.f) return;      // saw no key
      const float nm = fmaxf(M, m), a = ex2(M - nm), b = ex2(m - nm);
      L = L * a + l * b;
      O.x = O.x * a + o.x * b;
      O.y = O.y * a + o.y * b;
      O.z = O.z * a + o.z * b;
      O.w = O.w * a + o.w * b;
      M = nm;
    };
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      const float *src = merge + w * kPartFloats;
      fold(src[kRows * kKv4Head + 2 * mr], src[kRows * kKv4Head + 2 * mr + 1],
           *reinterpret_cast<const float4 *>(src + mr * kKv4Head + 4 * mc));
    }
    bool whole = t0 == 0 && t1 == n_tiles;
    if (!whole) {
      float *dst = p.part + (2ull * blockIdx.x + (t0 == 0 ? 1 : 0)) * kPartFloats;
      *reinterpret_cast<float4 *>(dst + mr * kKv4Head + 4 * mc) = O;
      if (mc == 0) {
        dst[kRows * kKv4Head + 2 * mr] = M;
        dst[kRows * kKv4Head + 2 * mr + 1] = L;
      }
      __threadfence();
      __syncthreads();
      // the ranges that share the piece
      const uint32_t c0 = static_cast<uint32_t>(((piece_at + 1) * G - 1) / W);
      const uint32_t c1 = static_cast<uint32_t>(((piece_at + n_tiles) * G - 1) / W);
      if (tid == 0) {
        const uint32_t n = atomicAdd(&p.counters[c0], 1u);
        s_last = n == c1 - c0;
        if (s_last) p.counters[c0] = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        M = -INFINITY;
        L = 0.f;
        O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (uint32_t k = c0; k <= c1; ++k) {
          const float *src = p.part + (2ull * k + (k == c0 ? 1 : 0)) * kPartFloats;
          fold(__ldcg(src + kRows * kKv4Head + 2 * mr), __ldcg(src + kRows * kKv4Head + 2 * mr + 1),
               __ldcg(reinterpret_cast<const float4 *>(src + mr * kKv4Head + 4 * mc)));
        }
        whole = true;
      }
    }
    if (whole) {
      const uint32_t orow = rt * kRows + mr;
      if (orow < n_rows) {
        const uint32_t otok = orow / p.group, ohd = orow % p.group;
        if (static_cast<int64_t>(s.len) - s.nq + otok >= 0) {      // a row before position 0 was written above
          // sees at least one key: the sum is positive unless the state is broken or its blocks are not there
          const bool none = M == -INFINITY && L == 0.f;
          const float inv = none ? 0.f : 1.f / L;
          if (!none && !(L > 0.f && L < INFINITY && fabsf(M) < INFINITY)) atomicOr(p.status, ZDEV_ERR_NUMERICAL);
          put4(static_cast<T *>(p.out) + (s.q0 + otok) * p.out_stride +
                   (static_cast<size_t>(head) * p.group + ohd) * kKv4Head + 4 * mc,
               make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv));
        }
      }
    }
    __syncthreads();       // the merge area and s_last are free again
    at = piece_at + t1;
  }
}

template <class T>
cudaError_t launch_rows(const Kv4AttnParams &p, int sm_count, cudaStream_t s) {
  const uint32_t smem = kOffSums + (p.n_seq + 1) * 8;
  kv4_rows_kernel<T><<<sm_count * kCtasPerSm, 32 * kWarps, smem, s>>>(p);
  return cudaGetLastError();
}

template <class T>
cudaError_t rows_setup() {
  return cudaFuncSetAttribute(kv4_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              kOffSums + (kKv4MaxSeqs + 1) * 8);
}

}  // namespace

size_t kv4_attn_part_bytes(int sm_count) {
  return static_cast<size_t>(sm_count) * kCtasPerSm * 2 * kPartFloats * sizeof(float);
}
uint32_t kv4_attn_counters(int sm_count) { return static_cast<uint32_t>(sm_count) * kCtasPerSm; }

cudaError_t kv4_attn_setup() {
  cudaError_t e = rows_setup<float>();
  if (e == cudaSuccess) e = rows_setup<__half>();
  if (e == cudaSuccess) e = rows_setup<__nv_bfloat16>();
  return e;
}

cudaError_t launch_kv4_attention(const Kv4AttnParams &p, Kv4Type t, int sm_count, uint32_t *launches, cudaStream_t s) {
  cudaError_t e;
  if (t == KV4_F32) e = launch_rows<float>(p, sm_count, s);
  else if (t == KV4_F16) e = launch_rows<__half>(p, sm_count, s);
  else e = launch_rows<__nv_bfloat16>(p, sm_count, s);
  if (e == cudaSuccess && launches) ++*launches;
  return e;
}

}  // namespace zgpu
