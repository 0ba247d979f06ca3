// kv4.cu — the paged 4-bit KV cache (layout in kv4.h): creation, the step
// plan (block tables, slot map and row starts built on the GPU from request
// lengths), release of finished rows, append and gather.
#include <cuda_bf16.h>

#include <new>
#include <string>
#include <vector>

#include "common.cuh"
#include "kv4.h"

namespace zgpu {

namespace {

// ------------------------------------------------------------------- plan
// Row i holds old_i tokens in ceil(old_i / B) blocks and gets new_i more.
// With first_i the exclusive sum of the blocks that the rows before need, its
// j-th new block is free_list[count - 1 - first_i - j]; token t of row i goes
// to slot table[i][pos / B] * B + pos % B, pos = old_i + t.  The sums over at
// most 1024 rows are cheap, so every CTA makes them for itself and no CTA
// waits for another; the table rows and the slots are then spread over the
// grid.  Bound by latency: one launch, two dependent reads (3.0 us in a graph for
// 16 rows, 4.5 us for 512 rows of 1056 table entries and 16 thousand slots).
constexpr uint32_t kPlanThreads = 256;
constexpr uint32_t kPlanPer = kKv4MaxSeqs / kPlanThreads;   // rows per thread

// Exclusive sums over the block's threads of two values; *ta, *tb the totals.
__device__ __forceinline__ void block_scan2(uint64_t &a, uint64_t &b, uint64_t *ta, uint64_t *tb, uint64_t *sh) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  uint64_t ia = a, ib = b;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t ua = __shfl_up_sync(0xffffffffu, ia, off), ub = __shfl_up_sync(0xffffffffu, ib, off);
    if (lane >= static_cast<uint32_t>(off)) {
      ia += ua;
      ib += ub;
    }
  }
  if (lane == 31) {
    sh[2 * warp] = ia;
    sh[2 * warp + 1] = ib;
  }
  __syncthreads();
  uint64_t pa = 0, pb = 0, sa = 0, sb = 0;
  for (uint32_t w = 0; w < nw; ++w) {
    if (w == warp) {
      pa = sa;
      pb = sb;
    }
    sa += sh[2 * w];
    sb += sh[2 * w + 1];
  }
  a = pa + ia - a;
  b = pb + ib - b;
  *ta = sa;
  *tb = sb;
}

__global__ void __launch_bounds__(kPlanThreads) kv4_plan_kernel(const Kv4PlanParams p) {
  __shared__ uint32_t s_old[kKv4MaxSeqs], s_first[kKv4MaxSeqs], s_start[kKv4MaxSeqs + 1];
  __shared__ uint64_t sh[2 * kPlanThreads / 32];
  const uint32_t tid = threadIdx.x, B = 1u << p.bt_log2;
  const uint32_t count = p.state_in[0];

  uint64_t need[kPlanPer], fresh[kPlanPer], sum_need = 0, sum_new = 0;
  bool too_long = false;
#pragma unroll
  for (uint32_t e = 0; e < kPlanPer; ++e) {
    const uint32_t i = tid * kPlanPer + e;
    need[e] = fresh[e] = 0;
    if (i < p.n_seq) {
      const uint64_t o = p.old_lens[i], n = p.new_lens[i];
      too_long |= o + n > static_cast<uint64_t>(p.table_width) * B;
      fresh[e] = n;
      need[e] = ((o + n + B - 1) >> p.bt_log2) - ((o + B - 1) >> p.bt_log2);
      s_old[i] = static_cast<uint32_t>(o);
    }
    sum_need += need[e];
    sum_new += fresh[e];
  }
  uint64_t first = sum_need, start = sum_new, total_need, total_new;
  block_scan2(first, start, &total_need, &total_new, sh);
  // 2: a row beyond its table or more tokens than slots; 1: the pool is used up
  const bool bad = __syncthreads_or(too_long) || total_new > p.n_slots || count > p.n_blocks;
  const uint32_t code = bad ? 2u : total_need > count ? 1u : 0u;
#pragma unroll
  for (uint32_t e = 0; e < kPlanPer; ++e) {
    const uint32_t i = tid * kPlanPer + e;
    if (i < p.n_seq) {
      s_first[i] = static_cast<uint32_t>(first);
      s_start[i] = code ? 0u : static_cast<uint32_t>(start);
    }
    first += need[e];
    start += fresh[e];
  }
  if (tid == 0) s_start[p.n_seq] = code ? 0u : static_cast<uint32_t>(total_new);
  __syncthreads();

  const uint32_t cta = blockIdx.y * gridDim.x + blockIdx.x, ctas = gridDim.x * gridDim.y;
  if (cta == 0) {
    for (uint32_t i = tid; i <= p.n_seq; i += kPlanThreads) {
      p.starts[i] = s_start[i];
      if (i < p.n_seq) p.kv_lens[i] = s_old[i] + (code ? 0u : s_start[i + 1] - s_start[i]);
    }
    if (tid == 0) {
      p.state_out[0] = code ? count : count - static_cast<uint32_t>(total_need);
      p.state_out[1] = code;
      p.state_out[2] = code ? 0u : static_cast<uint32_t>(total_new);
      p.state_out[3] = code ? 0u : static_cast<uint32_t>(total_need);
      if (code) atomicOr(p.status, ZDEV_ERR_POOL);
    }
  }
  // blocks of a row: what it held, then what it takes, then none
  auto block_at = [&](uint32_t i, uint32_t j, uint32_t held, uint32_t want) -> uint32_t {
    if (j < held) return p.table_in[static_cast<size_t>(i) * p.table_width + j];
    if (j < want) return p.free_list[count - 1 - (s_first[i] + (j - held))];
    return kKv4NoSlot;
  };
  for (uint32_t i = blockIdx.x; i < p.n_seq; i += gridDim.x) {
    const uint32_t o = s_old[i], n = s_start[i + 1] - s_start[i];
    // a refused plan keeps what the table can hold of each row
    const uint32_t held = min(static_cast<uint32_t>((static_cast<uint64_t>(o) + B - 1) >> p.bt_log2), p.table_width);
    const uint32_t want = code ? held : (o + n + B - 1) >> p.bt_log2;
    for (uint32_t j = blockIdx.y * kPlanThreads + tid; j < p.table_width; j += gridDim.y * kPlanThreads)
      p.table_out[static_cast<size_t>(i) * p.table_width + j] = block_at(i, j, held, want);
  }
  for (uint32_t t = cta * kPlanThreads + tid; t < p.n_slots; t += ctas * kPlanThreads) {
    uint32_t slot = kKv4NoSlot;
    if (t < s_start[p.n_seq]) {
      uint32_t lo = 0, hi = p.n_seq;   // last row with start <= t that has tokens: s_start[lo] <= t < s_start[hi]
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s_start[mid] <= t) lo = mid;
        else hi = mid;
      }
      const uint32_t o = s_old[lo], n = s_start[lo + 1] - s_start[lo], pos = o + (t - s_start[lo]);
      const uint32_t block = block_at(lo, pos >> p.bt_log2, (o + B - 1) >> p.bt_log2, (o + n + B - 1) >> p.bt_log2);
      if (block < p.n_blocks) slot = (block << p.bt_log2) + (pos & (B - 1));
      else atomicOr(p.status, ZDEV_ERR_BOUNDS);
    }
    p.slots[t] = slot;
  }
}

// ---------------------------------------------------------------- release
// One CTA: pushes the blocks of the rows marked done onto the free list in
// row order.  A row whose table or the list cannot be right (a block outside
// the pool, more blocks than the pool has) changes nothing at all.  16 rows of
// up to 128 blocks take 4.2 us in a graph, bound by latency; beyond some
// thousand blocks the one CTA's accesses bound it: 1024 rows of 64 blocks 40 us,
// of 1056 blocks 284 us.
constexpr uint32_t kReleaseThreads = kKv4MaxSeqs;

__global__ void __launch_bounds__(kReleaseThreads) kv4_release_kernel(const Kv4ReleaseParams p) {
  __shared__ uint64_t sh[2 * kReleaseThreads / 32];
  __shared__ uint32_t s_first[kReleaseThreads], s_held[kReleaseThreads];
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, B = 1u << p.bt_log2;
  const uint32_t count = p.state[0];
  bool bad = count > p.n_blocks;
  uint64_t held = 0;
  if (tid < p.n_seq && p.done[tid]) {
    held = (static_cast<uint64_t>(p.lens[tid]) + B - 1) >> p.bt_log2;
    if (held > p.table_width) bad = true;
  }
  uint64_t first = held, unused = 0, total, t2;
  block_scan2(first, unused, &total, &t2, sh);
  bad = bad || count + total > p.n_blocks;
  s_first[tid] = static_cast<uint32_t>(first);
  s_held[tid] = static_cast<uint32_t>(held);
  if (!__syncthreads_or(bad)) {
    bad = false;
    for (uint32_t i = warp; i < p.n_seq; i += kReleaseThreads / 32)
      for (uint32_t j = lane; j < s_held[i]; j += 32)
        bad |= p.table[static_cast<size_t>(i) * p.table_width + j] >= p.n_blocks;
    if (!__syncthreads_or(bad)) {
      for (uint32_t i = warp; i < p.n_seq; i += kReleaseThreads / 32)
        for (uint32_t j = lane; j < s_held[i]; j += 32) {
          uint32_t *e = p.table + static_cast<size_t>(i) * p.table_width + j;
          p.free_list[count + s_first[i] + j] = *e;
          *e = kKv4NoSlot;
        }
      if (tid < p.n_seq && p.done[tid]) p.lens[tid] = 0;
      if (tid == 0) {
        p.state[0] = count + static_cast<uint32_t>(total);
        p.state[1] = 0;
        p.state[2] = 0;
        p.state[3] = static_cast<uint32_t>(total);
      }
      return;
    }
  }
  if (tid == 0) {
    p.state[1] = 2;
    atomicOr(p.status, ZDEV_ERR_POOL);
  }
}

// -------------------------------------------------------- append / gather
template <class T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__half>(const __half *p, float (&x)[8]) {
  const uint4 u = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
    x[2 * e] = f.x, x[2 * e + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&x)[8]) {
  const uint4 u = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
}
__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(__half *p, float4 v) {
  __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 v) {
  __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
}

// n = q + 8 of one value where the quick rounding of x / d cannot be trusted:
// r is within one of the quotient, and the remainder x - r d, which the fma
// gives exactly (a multiple of both last places and at most about |d|, so at
// most 24 bits), says on which side of a border x lies.
__device__ __forceinline__ uint32_t nibble_exact(float x, float d, float inv) {
  float r = rintf(x * inv);
  const float e = fmaf(-r, d, x), h = 0.5f * fabsf(d);
  if (fabsf(e) >= h) {
    const float r1 = r + ((e > 0.f) == (d > 0.f) ? 1.f : -1.f);
    if (fabsf(e) > h || (static_cast<int>(r) & 1)) r = r1;
  }
  r = fminf(fmaxf(r, -8.f), 7.f);
  return static_cast<uint32_t>(static_cast<int>(r) + 8);
}

// Eight values of a row a lane, four lanes a group: the lane's n, the even
// dims' at bits 4 s of the low half and the odd dims' of the high half, and the
// group's scale.  A group that cannot be held (a non-finite value, a magnitude
// above 8 * 2720) is stored as zeros and recorded as a numerical error.  The
// work is bound by instruction issue, so the common case is kept short: the
// sign of the group's largest magnitude comes from its maximum and minimum,
// and only a warp in which the two are of one magnitude looks for the first;
// x / d is rounded by adding 1.5 * 2^23, and only a warp in which some
// remainder reaches d / 2 (a tie, or a quotient rounded onto a border), or some
// scale is subnormal (a quotient may then be far outside -8..8), takes the
// exact form.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t lane, __half *scale, uint32_t *status) {
  float mx, mn = fminf(fminf(fminf(x[0], x[1]), x[2]), fminf(fminf(x[3], x[4]), x[5]));
  mn = fminf(fminf(mn, x[6]), x[7]);
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(mx) : "f"(x[0]), "f"(x[1]), "f"(x[2]));
  asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(mx) : "f"(x[3]), "f"(x[4]));
  asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(mx) : "f"(x[5]), "f"(x[6]));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(mx) : "f"(x[7]));
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    const float a = __shfl_xor_sync(0xffffffffu, mx, off);
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(mx) : "f"(a));
  }
  float amax;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(amax) : "f"(mx), "f"(-mn));
  bool neg = -mn > mx;
  if (__any_sync(0xffffffffu, mx == -mn && mx > 0.f)) {
    float mine = 0.f;      // the lane's first value of that magnitude
#pragma unroll
    for (int e = 7; e >= 0; --e) mine = fabsf(x[e]) == amax ? x[e] : mine;
    const uint32_t any = __ballot_sync(0xffffffffu, mine != 0.f) & (0xFu << (lane & 28u));
    const uint32_t below = __ballot_sync(0xffffffffu, mine < 0.f);
    neg = any & (0u - any) & below;                                // the group's lowest lane that has it
  }
  float d = (neg ? 0.125f : -0.125f) * amax;
  __half dh = __float2half_rn(__bfloat162float(__float2bfloat16_rn(d)));
  d = __half2float(dh);
  if (!(amax <= 8.f * kKv4MaxScale)) {      // the scale alone would round 21823 down to the limit
    if ((lane & 3u) == 0) atomicOr(status, ZDEV_ERR_NUMERICAL);
    d = 0.f;
    dh = __float2half_rn(0.f);
  }
  *scale = dh;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d));
  constexpr float kAdd = 12582912.f + 8.f;     // its last four bits are n
  float worst = 0.f;
  uint32_t n[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 v = make_float2(x[e], x[e + 1]);
    const float2 t = fma2_rn(v, make_float2(inv, inv), make_float2(kAdd, kAdd));
    const float2 r = add2_rn(make_float2(kAdd, kAdd), make_float2(-t.x, -t.y));
    const float2 left = fma2_rn(r, make_float2(d, d), v);
    worst = fmaxf(fmaxf(worst, fabsf(left.x)), fabsf(left.y));
    n[e] = __float_as_uint(fminf(t.x, kAdd + 7.f));
    n[e + 1] = __float_as_uint(fminf(t.y, kAdd + 7.f));
  }
  if (__any_sync(0xffffffffu, !(worst < (fabsf(d) < 0x1p-14f ? 0.f : 0.5f * fabsf(d))))) {
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = d != 0.f ? nibble_exact(x[e], d, inv) : 8u;
  }
  uint32_t w = __byte_perm(n[0], n[1], 0x5410u);
#pragma unroll
  for (int e = 2; e < 8; e += 2) w += __byte_perm(n[e], n[e + 1], 0x5410u) << (2 * e);
  return w;
}

// A 4 x 4 transpose of nibbles over the four lanes of this lane's parity in
// its group (its own inverse): lane s's nibble e becomes lane e's nibble s.
__device__ __forceinline__ uint32_t transpose_nibbles(uint32_t n, uint32_t lane) {
  const uint32_t q = __shfl_xor_sync(0xffffffffu, n, 4);
  n = __byte_perm(n, q, lane & 4u ? 0x7715u : 0x7740u) & 0xFFFFu;
  const uint32_t p = __shfl_xor_sync(0xffffffffu, n, 2);
  return lane & 2u ? (n & 0xF0F0u) | ((p >> 4) & 0x0F0Fu) : (n & 0x0F0Fu) | ((p << 4) & 0xF0F0u);
}

// Nibble pairs (bits 0..3 and 16..19) as (n - 8) d, exact in binary16.
__device__ __forceinline__ float2 pair_values(uint32_t n, __half2 d) {
  const uint32_t x = (n & 0x000F000Fu) | 0x64006400u;      // 1024 + n
  return __half22float2(__hmul2(__hadd2(*reinterpret_cast<const __half2 *>(&x), __half2half2(__ushort_as_half(0xE408))), d));
}

// Byte offsets in a tile: lane's K word (shared by two lanes) and 16 V bits of
// token t, and the scale of its group g.
__device__ __forceinline__ uint32_t v_off(uint32_t t, uint32_t lane) {
  const uint32_t r = 4u * (lane & 1u) + ((lane >> 1) & 3u);
  return kKv4V + (t >> 3) * 512u + 16u * (4u * r + ((t & 7u) >> 1)) + 4u * (lane >> 3) + 2u * (t & 1u);
}
__device__ __forceinline__ uint32_t k_off(uint32_t t, uint32_t lane) {
  return 64u * t + 16u * ((lane & 7u) >> 1) + 4u * (lane >> 3);
}
__device__ __forceinline__ uint32_t scale_off(uint32_t t, uint32_t g) {
  return 2u * (2u * (16u * (t >> 3) + 4u * ((t & 7u) >> 1) + g) + (t & 1u));
}

constexpr uint32_t kRowWarps = 8;

// A warp per (token, kv head): lanes 0..15 take the K row, 16..31 the V row,
// lane 4 g + c of a half its dims 32 g + 8 c + 0..7.
// Bound by instruction issue, close above the reads of the rows: 16384 tokens
// of 8 kv heads in f32 take 37.6 us (134 MB in, 19 MB out, 4.1 TB/s), 203
// instructions a warp and row pair at 72 % issue (33.3 us in a graph).  16-bit
// rows are coarser: of normal values a tie sends 34 % of the warps in f16 and 49 %
// in bf16 into the exact rounding, 47.0 and 50.3 us in a graph (67 MB in).  Four values of both rows a
// lane took 47 us: the group's maximum, scale and sign cost as much for four
// values as for eight.  Four CTAs fit an SM at 57 registers; bounds for five and
// six, at the price of the values on their way, measured 40 and 49 us.
template <class T>
__global__ void __launch_bounds__(32 * kRowWarps) kv4_append_kernel(const Kv4RowsParams p) {
  // the number of warps is a multiple of n_kv: a warp keeps its head
  const uint32_t lane = threadIdx.x & 31, w0 = blockIdx.x * kRowWarps + (threadIdx.x >> 5), head = w0 % p.n_kv;
  const uint32_t step = gridDim.x * kRowWarps / p.n_kv, c = lane & 3u, g = (lane >> 2) & 3u;
  const bool is_v = lane >= 16;
  uint32_t token = w0 / p.n_kv;
  if (token >= p.n_tokens) return;
  const T *rows = static_cast<const T *>(is_v ? p.v : p.k) + head * kKv4Head + 8 * (lane & 15u);
  const uint64_t stride = is_v ? p.v_stride : p.k_stride;
  // V: the lane's pieces of a token are dims r and r + 2 of each eight
  const uint32_t r = 4 * (c & 1u) + (c >> 1);
  const uint32_t lane_off = is_v ? kKv4V + 64 * r + 4 * g : 16 * c + 4 * g;
  const uint32_t scale_off0 = (is_v ? kKv4Vs : kKv4Ks) + 4 * g;
  uint32_t next_slot = p.slots[token];
  float next[8];
  load8(rows + token * stride, next);
  while (true) {
    const uint32_t slot = next_slot;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = next[e];
    // the next token's rows are on their way while this one's are worked on
    const bool more = p.n_tokens - token > step;
    token += step;
    if (more) {
      next_slot = p.slots[token];
      load8(rows + token * stride, next);
    }
    if (slot >= p.n_slots) {
      if (slot != kKv4NoSlot && lane == 0) atomicOr(p.status, ZDEV_ERR_BOUNDS);
      if (!more) return;
      continue;
    }
    uint8_t *tile = p.pool + kv4_tile_off(slot, head, p.n_kv, p.bt_log2);
    const uint32_t t = slot % kKv4Tile, half = t >> 3, at = 16 * ((t >> 1) & 3u) + 2 * (t & 1u);
    __half scale;
    const uint32_t w = quantise8(x, lane, &scale, p.status);
    // V: a 4 x 4 transpose of bytes over the group's lanes, after which byte s
    // holds dims 8 s + r and 8 s + r + 2 in its low and high four bits
    uint32_t q = __shfl_xor_sync(0xffffffffu, w, 2);
    uint32_t v = __byte_perm(w, q, c & 2u ? 0x3276u : 0x5410u);
    q = __shfl_xor_sync(0xffffffffu, v, 1);
    v = __byte_perm(v, q, c & 1u ? 0x3715u : 0x6240u);
    if (is_v) {
      const uint32_t lo = v & 0x0F0F0F0Fu, hi = (v >> 4) & 0x0F0F0F0Fu;
      const uint32_t s3 = __byte_perm(lo, hi, 0x0703u) & 0x000F000Fu;
      const uint32_t both = (__byte_perm(lo, hi, 0x0400u) & 0x000F000Fu) << 6 | (__byte_perm(lo, hi, 0x0501u) & 0x000F000Fu) << 2 |
                            (__byte_perm(lo, hi, 0x0602u) & 0x000F000Fu) << 10 | (s3 & 0x00030003u) << 14 |
                            ((s3 >> 2) & 0x00030003u);
      uint8_t *to = tile + lane_off + 512 * half + at;
      *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(both);
      *reinterpret_cast<uint16_t *>(to + 128) = static_cast<uint16_t>(both >> 16);
    } else {
      *reinterpret_cast<uint32_t *>(tile + lane_off + 64 * t) = w;
    }
    if (c == 0) *reinterpret_cast<__half *>(tile + scale_off0 + 64 * half + at) = scale;
    if (!more) return;
  }
}

// A warp per (token, kv head), four values of both rows a lane, so that a store
// is 512 contiguous bytes.  Bound by the writes: 16384 tokens of 8 kv heads to f32
// take 29.5 us (134 MB out, 19 MB in, 5.2 TB/s), to f16 or bf16 25.5 us.
template <class T>
__global__ void __launch_bounds__(32 * kRowWarps) kv4_gather_kernel(const Kv4RowsParams p) {
  // the number of warps is a multiple of n_kv: a warp keeps its head
  const uint32_t lane = threadIdx.x & 31, w0 = blockIdx.x * kRowWarps + (threadIdx.x >> 5), head = w0 % p.n_kv;
  const uint32_t step = gridDim.x * kRowWarps / p.n_kv;
  for (uint32_t token = w0 / p.n_kv; token < p.n_tokens; token += step) {
    const uint32_t slot = p.slots[token];
    float4 kx = make_float4(0.f, 0.f, 0.f, 0.f), vx = kx;
    if (slot < p.n_slots) {
      const uint8_t *tile = p.pool + kv4_tile_off(slot, head, p.n_kv, p.bt_log2);
      const uint32_t t = slot % kKv4Tile;
      if (p.k_out) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(tile + k_off(t, lane));
        const __half2 d = __half2half2(*reinterpret_cast<const __half *>(tile + kKv4Ks + scale_off(t, lane / 8)));
        const uint32_t mine = lane & 1u ? w >> 8 : w;
        const float2 a = pair_values(mine, d), b = pair_values(mine >> 4, d);
        kx = make_float4(a.x, a.y, b.x, b.y);
      }
      if (p.v_out) {
        const uint32_t u = *reinterpret_cast<const uint16_t *>(tile + v_off(t, lane));
        const __half2 d = __half2half2(*reinterpret_cast<const __half *>(tile + kKv4Vs + scale_off(t, lane / 8)));
        const uint32_t n = transpose_nibbles(kv4_v_nibbles(u), lane);
        const float2 a = pair_values(n | n << 12, d), b = pair_values(n >> 8 | (n >> 8) << 12, d);
        vx = make_float4(a.x, a.y, b.x, b.y);
      }
    } else if (slot != kKv4NoSlot && lane == 0) {
      atomicOr(p.status, ZDEV_ERR_BOUNDS);
    }
    if (p.k_out) store4(static_cast<T *>(p.k_out) + token * p.k_stride + head * kKv4Head + 4 * lane, kx);
    if (p.v_out) store4(static_cast<T *>(p.v_out) + token * p.v_stride + head * kKv4Head + 4 * lane, vx);
  }
}

// CTAs: eight per SM at most, and a number whose warps are a multiple of n_kv.
uint32_t row_grid(const Kv4RowsParams &p, int sm_count) {
  uint32_t unit = p.n_kv;
  for (uint32_t k = 0; k < 3 && unit % 2 == 0; ++k) unit /= 2;      // n_kv / gcd(n_kv, 8)
  const uint64_t want = (static_cast<uint64_t>(p.n_tokens) * p.n_kv + kRowWarps - 1) / kRowWarps;
  const uint64_t most = static_cast<uint64_t>(sm_count) * 8, n = want < most ? want : most;
  return static_cast<uint32_t>((n + unit - 1) / unit * unit);
}
static_assert(kRowWarps == 8, "row_grid");

}  // namespace

cudaError_t launch_kv4_plan(const Kv4PlanParams &p, int sm_count, cudaStream_t s) {
  // a CTA per table row, more for a row above 2048 entries; enough CTAs for
  // 1024 slots each
  const uint32_t ny = (p.table_width + 2047) / 2048;
  uint32_t nx = p.n_seq;
  const uint32_t slot_ctas = (p.n_slots + 1023) / 1024;
  if (nx * ny < slot_ctas) nx = (slot_ctas + ny - 1) / ny;
  const uint32_t most = static_cast<uint32_t>(sm_count) * 4;
  if (nx > most) nx = most;
  kv4_plan_kernel<<<dim3(nx, ny > 64 ? 64 : ny), kPlanThreads, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv4_release(const Kv4ReleaseParams &p, cudaStream_t s) {
  kv4_release_kernel<<<1, kReleaseThreads, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv4_append(const Kv4RowsParams &p, Kv4Type t, int sm_count, cudaStream_t s) {
  const uint32_t g = row_grid(p, sm_count);
  if (t == KV4_F32) kv4_append_kernel<float><<<g, 32 * kRowWarps, 0, s>>>(p);
  else if (t == KV4_F16) kv4_append_kernel<__half><<<g, 32 * kRowWarps, 0, s>>>(p);
  else kv4_append_kernel<__nv_bfloat16><<<g, 32 * kRowWarps, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv4_gather(const Kv4RowsParams &p, Kv4Type t, int sm_count, cudaStream_t s) {
  const uint32_t g = row_grid(p, sm_count);
  if (t == KV4_F32) kv4_gather_kernel<float><<<g, 32 * kRowWarps, 0, s>>>(p);
  else if (t == KV4_F16) kv4_gather_kernel<__half><<<g, 32 * kRowWarps, 0, s>>>(p);
  else kv4_gather_kernel<__nv_bfloat16><<<g, 32 * kRowWarps, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace zgpu

// ------------------------------------------------------------ entry points
namespace {

// Makes the context's device current for a call and puts the caller's back.
struct DeviceGuard {
  int old = -1;
  bool ok = false;
  explicit DeviceGuard(int device) {
    if (cudaGetDevice(&old) != cudaSuccess) {
      cudaGetLastError();
      old = -1;
    }
    ok = old == device || cudaSetDevice(device) == cudaSuccess;
    if (old == device) old = -1;
  }
  ~DeviceGuard() {
    if (old >= 0) cudaSetDevice(old);
  }
};

bool kv4_type(uint32_t dtype, zgpu::Kv4Type *t, uint32_t *size) {
  if (dtype == ZGPU_F32) *t = zgpu::KV4_F32, *size = 4;
  else if (dtype == ZGPU_F16) *t = zgpu::KV4_F16, *size = 2;
  else if (dtype == ZGPU_BF16) *t = zgpu::KV4_BF16, *size = 2;
  else return false;
  return true;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na && nb && x < y + nb && y < x + na;
}

// A row stride in elements: 0 stands for dense rows; rows are read and
// written in 16-byte pieces.
bool row_stride(uint64_t *stride, uint64_t width, uint32_t size) {
  if (*stride == 0) *stride = width;
  return *stride >= width && (*stride * size) % 16 == 0 && *stride <= (1ull << 40);
}

zgpu_status bad(zgpu_ctx *ctx, const char *what) { return zgpu_fail(ctx, ZGPU_ERR_INVALID_ARG, what); }

}  // namespace

#define KV4_CUDA(call, what)                                     \
  do {                                                           \
    const cudaError_t e_ = (call);                               \
    if (e_ != cudaSuccess) return zgpu_cuda_fail(ctx, e_, what); \
  } while (0)

extern "C" {

zgpu_status zgpu_kv4_create(zgpu_ctx *ctx, uint32_t n_blocks, uint32_t block_tokens, uint32_t n_layers,
                            uint32_t n_kv_heads, uint32_t head_dim, zgpu_kv4 **out) {
  if (out) *out = nullptr;
  if (!ctx || !out || !n_blocks || !n_layers || !n_kv_heads) return ZGPU_ERR_INVALID_ARG;
  if (head_dim != zgpu::kKv4Head) return bad(ctx, "kv4: head_dim must be 128");
  uint32_t lg = 0;
  while (lg < 8 && (1u << lg) != block_tokens) ++lg;
  if (lg < 4 || lg > 7) return bad(ctx, "kv4: block_tokens must be 16, 32, 64 or 128");
  if (n_kv_heads > 1024) return bad(ctx, "kv4: at most 1024 kv heads");
  const uint64_t slots = static_cast<uint64_t>(n_blocks) * block_tokens;
  if (slots > 0x7FFFFFFFull) return bad(ctx, "kv4: more than 2^31 - 1 token slots");
  DeviceGuard g(ctx->device);
  if (!g.ok) return zgpu_cuda_fail(ctx, cudaGetLastError(), "kv4: cudaSetDevice");
  const unsigned __int128 want = static_cast<unsigned __int128>(slots) / zgpu::kKv4Tile * zgpu::kKv4TileBytes *
                                 n_kv_heads * n_layers;
  if (want > (static_cast<unsigned __int128>(1) << 46)) return zgpu_fail(ctx, ZGPU_ERR_OUT_OF_MEMORY, "kv4: pool size");
  zgpu_kv4 *kv = new (std::nothrow) zgpu_kv4();
  if (!kv) return zgpu_fail(ctx, ZGPU_ERR_OUT_OF_MEMORY, "kv4: host allocation");
  kv->ctx = ctx;
  kv->device = ctx->device;
  kv->sm_count = ctx->sm_count;
  kv->n_blocks = n_blocks;
  kv->block_tokens = block_tokens;
  kv->bt_log2 = lg;
  kv->n_layers = n_layers;
  kv->n_kv = n_kv_heads;
  kv->layer_bytes = slots / zgpu::kKv4Tile * zgpu::kKv4TileBytes * n_kv_heads;
  // zeroed: every scale in the pool is finite from the start, and append
  // stores only finite ones, so a slot outside a row's mask can hold no
  // infinity or NaN
  cudaError_t e = cudaMalloc(&kv->d, kv->layer_bytes * n_layers);
  if (e == cudaSuccess) e = cudaMemset(kv->d, 0, kv->layer_bytes * n_layers);
  if (e == cudaSuccess) e = cudaMalloc(&kv->d_status, zgpu::kStatusWords * sizeof(uint32_t));
  if (e == cudaSuccess) e = cudaMemset(kv->d_status, 0, zgpu::kStatusWords * sizeof(uint32_t));
  // the clearing runs on the default stream: done before any stream uses it
  if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
  if (e != cudaSuccess) {
    cudaGetLastError();
    cudaFree(kv->d);
    cudaFree(kv->d_status);
    delete kv;
    return zgpu_cuda_fail(ctx, e, "kv4: pool allocation");
  }
  *out = kv;
  return ZGPU_OK;
}

void zgpu_kv4_destroy(zgpu_kv4 *kv) {
  if (!kv) return;
  DeviceGuard g(kv->device);
  cudaFree(kv->d);
  cudaFree(kv->d_status);
  delete kv;
}

zgpu_status zgpu_kv4_work_create(zgpu_ctx *ctx, zgpu_kv4_work **out) {
  if (out) *out = nullptr;
  if (!ctx || !out) return ZGPU_ERR_INVALID_ARG;
  DeviceGuard g(ctx->device);
  if (!g.ok) return zgpu_cuda_fail(ctx, cudaGetLastError(), "kv4 work: cudaSetDevice");
  zgpu_kv4_work *w = new (std::nothrow) zgpu_kv4_work();
  if (!w) return zgpu_fail(ctx, ZGPU_ERR_OUT_OF_MEMORY, "kv4 work: host allocation");
  w->ctx = ctx;
  w->device = ctx->device;
  const size_t nc = zgpu::kv4_attn_counters(ctx->sm_count) * sizeof(uint32_t);
  cudaError_t e = cudaMalloc(&w->part, zgpu::kv4_attn_part_bytes(ctx->sm_count));
  if (e == cudaSuccess) e = cudaMalloc(&w->counters, nc);
  if (e == cudaSuccess) e = cudaMemset(w->counters, 0, nc);
  if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
  if (e != cudaSuccess) {
    cudaGetLastError();
    cudaFree(w->part);
    cudaFree(w->counters);
    delete w;
    return zgpu_cuda_fail(ctx, e, "kv4 work: allocation");
  }
  *out = w;
  return ZGPU_OK;
}

void zgpu_kv4_work_destroy(zgpu_kv4_work *w) {
  if (!w) return;
  DeviceGuard g(w->device);
  cudaFree(w->part);
  cudaFree(w->counters);
  delete w;
}

zgpu_status zgpu_kv4_check(zgpu_kv4 *kv) {
  if (!kv) return ZGPU_ERR_INVALID_ARG;
  zgpu_ctx *ctx = kv->ctx;
  DeviceGuard g(kv->device);
  if (!g.ok) return zgpu_cuda_fail(ctx, cudaGetLastError(), "kv4 check: cudaSetDevice");
  uint32_t st[zgpu::kStatusWords] = {0};
  KV4_CUDA(cudaMemcpyAsync(st, kv->d_status, sizeof(st), cudaMemcpyDeviceToHost, ctx->stream), "kv4 check: status");
  KV4_CUDA(cudaStreamSynchronize(ctx->stream), "kv4 check: sync");
  if (!st[0]) return ZGPU_OK;
  KV4_CUDA(cudaMemsetAsync(kv->d_status, 0, sizeof(st), ctx->stream), "kv4 check: clear");
  KV4_CUDA(cudaStreamSynchronize(ctx->stream), "kv4 check: sync");
  if (st[0] & zgpu::ZDEV_ERR_TIMEOUT) return zgpu_fail(ctx, ZGPU_ERR_DEVICE_TIMEOUT, "kv4: device wait timed out");
  if (st[0] & zgpu::ZDEV_ERR_BOUNDS)
    return zgpu_fail(ctx, ZGPU_ERR_KV_TOKEN_OUT_OF_RANGE, "kv4: a slot, block or length outside the cache");
  if (st[0] & zgpu::ZDEV_ERR_POOL)
    return zgpu_fail(ctx, ZGPU_ERR_KV_TOKEN_COUNT_EXCEEDS_MAX,
                     "kv4: plan or release refused (blocks used up, or lengths beyond the table or the slots)");
  return zgpu_fail(ctx, ZGPU_ERR_NUMERICAL_INSTABILITY,
                   "kv4: a value that the cache cannot hold, or a non-finite softmax state");
}

zgpu_status zgpu_kv4_plan_device(zgpu_kv4 *kv, uint32_t n_seq, uint32_t table_width, const uint32_t *d_old_lens,
                                 const uint32_t *d_new_lens, const uint32_t *d_table_in, uint32_t *d_table_out,
                                 const uint32_t *d_free_list, const uint32_t *d_state_in, uint32_t *d_state_out,
                                 uint32_t n_slots, uint32_t *d_slots, uint32_t *d_starts, uint32_t *d_kv_lens,
                                 void *stream) {
  if (!kv || !d_old_lens || !d_new_lens || !d_table_in || !d_table_out || !d_free_list || !d_state_in ||
      !d_state_out || !d_starts || !d_kv_lens || (n_slots && !d_slots))
    return ZGPU_ERR_INVALID_ARG;
  zgpu_ctx *ctx = kv->ctx;
  if (n_seq == 0 || n_seq > zgpu::kKv4MaxSeqs) return bad(ctx, "kv4 plan: 1 to 1024 rows");
  if (table_width == 0 || static_cast<uint64_t>(table_width) * kv->block_tokens > 0x7FFFFFFFull)
    return bad(ctx, "kv4 plan: table width");
  if (n_slots > 0x7FFFFFFFu) return bad(ctx, "kv4 plan: slot count");
  const void *ptrs[] = {d_old_lens, d_new_lens, d_table_in, d_table_out, d_free_list, d_state_in, d_state_out,
                        d_slots,    d_starts,   d_kv_lens};
  for (const void *p : ptrs)
    if (!aligned4(p)) return bad(ctx, "kv4 plan: arrays of 4-byte words");
  // the table may be updated in place; nothing else may overlap: the CTAs
  // read the inputs without waiting for one another
  const size_t lens = n_seq * 4ull, tab = 4ull * n_seq * table_width, st = 16;
  const struct { const void *p; size_t n; } in[] = {{d_old_lens, lens}, {d_new_lens, lens}, {d_table_in, tab},
                                                    {d_free_list, 4ull * kv->n_blocks}, {d_state_in, st}},
      outs[] = {{d_table_out, tab}, {d_state_out, st}, {d_slots, 4ull * n_slots}, {d_starts, lens + 4}, {d_kv_lens, lens}};
  for (const auto &o : outs) {
    for (const auto &i : in)
      if (overlap(o.p, o.n, i.p, i.n) && !(o.p == d_table_out && i.p == d_table_in && d_table_out == d_table_in))
        return bad(ctx, "kv4 plan: an output overlaps an input (only the table may be updated in place)");
    for (const auto &o2 : outs)
      if (&o != &o2 && overlap(o.p, o.n, o2.p, o2.n)) return bad(ctx, "kv4 plan: outputs overlap");
  }
  DeviceGuard g(kv->device);
  if (!g.ok) return zgpu_cuda_fail(ctx, cudaGetLastError(), "kv4 plan: cudaSetDevice");
  zgpu::Kv4PlanParams p = {};
  p.old_lens = d_old_lens;
  p.new_lens = d_new_lens;
  p.table_in = d_table_in;
  p.table_out = d_table_out;
  p.free_list = d_free_list;
  p.state_in = d_state_in;
  p.state_out = d_state_out;
  p.slots = d_slots;
  p.starts = d_starts;
  p.kv_lens = d_kv_lens;
  p.n_seq = n_seq;
  p.table_width = table_width;
  p.n_slots = n_slots;
  p.n_blocks = kv->n_blocks;
  p.bt_log2 = kv->bt_log2;
  p.status = kv->d_status;
  KV4_CUDA(zgpu::launch_kv4_plan(p, kv->sm_count, stream ? static_cast<cudaStream_t>(stream) : ctx->stream),
           "kv4 plan");
  ++ctx->launches;
  return ZGPU_OK;
}

zgpu_status zgpu_kv4_release_device(zgpu_kv4 *kv, uint32_t n_seq, uint32_t table_width, const uint32_t *d_done,
                                    uint32_t *d_lens, uint32_t *d_table, uint32_t *d_free_list, uint32_t *d_state,
                                    void *stream) {
  if (!kv || !d_done || !d_lens || !d_table || !d_free_list || !d_state) return ZGPU_ERR_INVALID_ARG;
  zgpu_ctx *ctx = kv->ctx;
  if (n_seq == 0 || n_seq > zgpu::kKv4MaxSeqs) return bad(ctx, "kv4 release: 1 to 1024 rows");
  if (table_width == 0 || static_cast<uint64_t>(table_width) * kv->block_tokens > 0x7FFFFFFFull)
    return bad(ctx, "kv4 release: table width");
  const size_t lens = n_seq * 4ull, tab = 4ull * n_seq * table_width;
  const struct { const void *p; size_t n; } a[] = {
      {d_done, lens}, {d_lens, lens}, {d_table, tab}, {d_free_list, 4ull * kv->n_blocks}, {d_state, 16}};
  for (const auto &x : a) {
    if (!aligned4(x.p)) return bad(ctx, "kv4 release: arrays of 4-byte words");
    for (const auto &y : a)
      if (&x != &y && overlap(x.p, x.n, y.p, y.n)) return bad(ctx, "kv4 release: arrays overlap");
  }
  DeviceGuard g(kv->device);
  if (!g.ok) return zgpu_cuda_fail(ctx, cudaGetLastError(), "kv4 release: cudaSetDevice");
  zgpu::Kv4ReleaseParams p = {};
  p.done = d_done;
  p.lens = d_lens;
  p.table = d_table;
  p.free_list = d_free_list;
  p.state = d_state;
  p.n_seq = n_seq;
  p.table_width = table_width;
  p.n_blocks = kv->n_blocks;
  p.bt_log2 = kv->bt_log2;
  p.status = kv->d_status;
  KV4_CUDA(zgpu::launch_kv4_release(p, stream ? static_cast<cudaStream_t>(stream) : ctx->stream), "kv4 release");
  ++ctx->launches;
  return ZGPU_OK;
}

static zgpu_status rows_params(zgpu_kv4 *kv, uint32_t layer, uint32_t n_tokens, const void *k, const void *v,
                               uint64_t k_stride, uint64_t v_stride, uint32_t dtype, const uint32_t *d_slots,
                               zgpu::Kv4RowsParams *p, zgpu::Kv4Type *t) {
  zgpu_ctx *ctx = kv->ctx;
  uint32_t size = 0;
  if (layer >= kv->n_layers) return zgpu_fail(ctx, ZGPU_ERR_KV_LAYER_OUT_OF_RANGE, "kv4 rows: layer out of range");
  if (!kv4_type(dtype, t, &size))
    return zgpu_fail(ctx, ZGPU_ERR_UNSUPPORTED_QUANT, "kv4 rows: element type must be f32, f16 or bf16");
  if (n_tokens > 0x7FFFFFFFu) return bad(ctx, "kv4 rows: token count");
  const uint64_t width = static_cast<uint64_t>(kv->n_kv) * zgpu::kKv4Head;
  if (!row_stride(&k_stride, width, size) || !row_stride(&v_stride, width, size))
    return bad(ctx, "kv4 rows: a row stride must hold a token's heads and be a multiple of 16 bytes");
  if (!aligned16(k) || !aligned16(v) || !aligned4(d_slots))
    return bad(ctx, "kv4 rows: rows must start on 16-byte boundaries");
  p->pool = kv->d + layer * kv->layer_bytes;
  p->slots = d_slots;
  p->k_stride = k_stride;
  p->v_stride = v_stride;
  p->n_tokens = n_tokens;
  p->n_kv = kv->n_kv;
  p->n_slots = kv->n_blocks * kv->block_tokens;
  p->bt_log2 = kv->bt_log2;
  p->status = kv->d_status;
  return ZGPU_OK;
}

zgpu_status zgpu_kv4_append_device(zgpu_kv4 *kv, uint32_t layer, uint32_t n_tokens, const void *d_k, uint64_t k_stride,
                                   const void *d_v, uint64_t v_stride, uint32_t dtype, const uint32_t *d_slots,
                                   void *stream) {
  if (!kv || (n_tokens && (!d_k || !d_v || !d_slots))) return ZGPU_ERR_INVALID_ARG;
  zgpu_ctx *ctx = kv->ctx;
  zgpu::Kv4RowsParams p = {};
  zgpu::Kv4Type t = zgpu::KV4_F32;
  const zgpu_status s = rows_params(kv, layer, n_tokens, d_k, d_v, k_stride, v_stride, dtype, d_slots, &p, &t);
  if (s || !n_tokens) return s;
  p.k = d_k;
  p.v = d_v;
  DeviceGuard g(kv->device);
  if (!g.ok) return zgpu_cuda_fail(ctx, cudaGetLastError(), "kv4 append: cudaSetDevice");
  KV4_CUDA(zgpu::launch_kv4_append(p, t, kv->sm_count, stream ? static_cast<cudaStream_t>(stream) : ctx->stream),
           "kv4 append");
  ++ctx->launches;
  return ZGPU_OK;
}

zgpu_status zgpu_kv4_gather_device(zgpu_kv4 *kv, uint32_t layer, uint32_t n_tokens, const uint32_t *d_slots, void *d_k,
                                   uint64_t k_stride, void *d_v, uint64_t v_stride, uint32_t dtype, void *stream) {
  if (!kv || (n_tokens && ((!d_k && !d_v) || !d_slots))) return ZGPU_ERR_INVALID_ARG;
  zgpu_ctx *ctx = kv->ctx;
  zgpu::Kv4RowsParams p = {};
  zgpu::Kv4Type t = zgpu::KV4_F32;
  const zgpu_status s = rows_params(kv, layer, n_tokens, d_k, d_v, k_stride, v_stride, dtype, d_slots, &p, &t);
  if (s || !n_tokens) return s;
  p.k_out = d_k;
  p.v_out = d_v;
  DeviceGuard g(kv->device);
  if (!g.ok) return zgpu_cuda_fail(ctx, cudaGetLastError(), "kv4 gather: cudaSetDevice");
  KV4_CUDA(zgpu::launch_kv4_gather(p, t, kv->sm_count, stream ? static_cast<cudaStream_t>(stream) : ctx->stream),
           "kv4 gather");
  ++ctx->launches;
  return ZGPU_OK;
}

zgpu_status zgpu_kv4_attention_device(zgpu_kv4 *kv, zgpu_kv4_work *work, uint32_t layer, uint32_t n_seq,
                                      uint32_t n_rows, uint32_t max_q, uint32_t n_q_heads, const void *d_q,
                                      uint64_t q_stride, void *d_out, uint64_t out_stride, uint32_t dtype,
                                      const uint32_t *d_starts, const uint32_t *d_kv_lens, const uint32_t *d_table,
                                      uint32_t table_width, float scale, void *stream) {
  if (!kv || !work || !d_starts || !d_kv_lens || !d_table || (n_rows && (!d_q || !d_out))) return ZGPU_ERR_INVALID_ARG;
  zgpu_ctx *ctx = kv->ctx;
  zgpu::Kv4Type t = zgpu::KV4_F32;
  uint32_t size = 0;
  if (work->ctx != ctx) return bad(ctx, "kv4 attention: workspace belongs to another context");
  if (layer >= kv->n_layers) return zgpu_fail(ctx, ZGPU_ERR_KV_LAYER_OUT_OF_RANGE, "kv4 attention: layer out of range");
  if (!kv4_type(dtype, &t, &size))
    return zgpu_fail(ctx, ZGPU_ERR_UNSUPPORTED_QUANT, "kv4 attention: element type must be f32, f16 or bf16");
  if (n_seq == 0 || n_seq > zgpu::kKv4MaxSeqs) return bad(ctx, "kv4 attention: 1 to 1024 sequences");
  if (n_rows > 0x7FFFFFFFu || max_q > 0x7FFFFFFFu / 16u) return bad(ctx, "kv4 attention: row count");
  if (n_q_heads == 0 || n_q_heads % kv->n_kv != 0 || n_q_heads / kv->n_kv > 16)
    return bad(ctx, "kv4 attention: n_q_heads must be 1..16 x n_kv_heads");
  if (table_width == 0 || static_cast<uint64_t>(table_width) * kv->block_tokens > 0x7FFFFFFFull)
    return bad(ctx, "kv4 attention: table width");
  const uint64_t width = static_cast<uint64_t>(n_q_heads) * zgpu::kKv4Head;
  if (!row_stride(&q_stride, width, size) || !row_stride(&out_stride, width, size))
    return bad(ctx, "kv4 attention: a row stride must hold a token's heads and be a multiple of 16 bytes");
  if (!aligned16(d_q) || !aligned16(d_out) || !aligned4(d_starts) || !aligned4(d_kv_lens) || !aligned4(d_table))
    return bad(ctx, "kv4 attention: rows must start on 16-byte boundaries");
  if (!(scale > 0.f) || !(scale <= 3.4e38f)) return bad(ctx, "kv4 attention: scale must be positive and finite");
  if (n_rows == 0 || max_q == 0) return ZGPU_OK;
  DeviceGuard g(kv->device);
  if (!g.ok) return zgpu_cuda_fail(ctx, cudaGetLastError(), "kv4 attention: cudaSetDevice");
  zgpu::Kv4AttnParams p = {};
  p.pool = kv->d + layer * kv->layer_bytes;
  p.q = d_q;
  p.out = d_out;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.starts = d_starts;
  p.kv_lens = d_kv_lens;
  p.table = d_table;
  p.table_width = table_width;
  p.n_seq = n_seq;
  p.n_rows = n_rows;
  p.max_q = max_q;
  p.n_kv = kv->n_kv;
  p.group = n_q_heads / kv->n_kv;
  p.n_blocks = kv->n_blocks;
  p.bt_log2 = kv->bt_log2;
  p.scale = scale;
  p.part = work->part;
  p.counters = work->counters;
  p.status = kv->d_status;
  KV4_CUDA(zgpu::launch_kv4_attention(p, t, kv->sm_count, &ctx->launches,
                                      stream ? static_cast<cudaStream_t>(stream) : ctx->stream),
           "kv4 attention");
  return ZGPU_OK;
}

}  // extern "C"
