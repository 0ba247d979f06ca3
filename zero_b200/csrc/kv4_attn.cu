// kv4_attn.cu — attention of a ragged batch over the paged 4-bit KV cache.
//
// o = softmax(scale * q K^T) V per query row, over the keys up to the row's
// own position: row i's queries are its last ones, query t of n at position
// kv_len - n + t.
//
// kv4_rows_kernel: few query rows per kv head (decode, short continuations;
// kv4_few_rows below); kv4_prompt.cu takes the sequences with more.
// Bound by the cache read, 144 bytes per key and kv head, and close behind it
// by instruction issue: unpacking 256 values per key and head.
//
//   Rows.  The query rows of a kv head (its group of heads, times the new
//   tokens) are taken eight at a time.  The tensor cores multiply 16-bit
//   values (m16n8k16, f32 sums); a row is put in as hi + lo, two binary16
//   values whose sum holds 22 bits, in rows r and r + 8 of the fragment.  The
//   cache's values are exact in binary16, so q K^T and P V keep f32 accuracy
//   at the price of eight rows instead of sixteen, which a memory-bound
//   kernel has to spare; both halves of a score land in one thread.  P V is
//   taken transposed, V^T P^T: the scores' fragment is P^T's as it stands, the
//   values are the sixteen rows, and the result takes half the registers.  For
//   16-bit rows P is one binary16 value, 11 bits, as many as an f16 result has: the
//   second half would double P V's products (an f16 result is 2.5e-4 off with one
//   half, 2.0e-4 by its own rounding; a bf16 result 1.7e-3 either way).  A query
//   row is scaled by a power of two first (its largest value in [256, 512); a row
//   below 2^-119 by 2^127), so neither half leaves binary16's range; P is held times 2^15, which
//   keeps probabilities down to 2^-39 of the row's largest.
//
//   Keys enter as the whole numbers n - 8, exact: a nibble under the exponent of
//   1024 (bits 0..3) or of 64 (bits 4..7), less 1032 or 72.  Each group of 32
//   dims has its own sum, scaled by d_g in f32.  The masked nibble itself would be a
//   subnormal, n 2^-24, for one operation less a pair, but the matrix unit
//   aligns a subnormal's products by its exponent, not by its leading bit, so
//   that their sum keeps some 17 bits: an f16 result whose products reach 2048
//   was 4e-3 off, and is 3e-4 off with these.
//   Values are made binary16 by the bits' place: under a fixed exponent a
//   nibble is a constant plus n, and (16 + n) d - 24 d is one exact fma since
//   24 d is exact; for 256 + n an add takes the constant off first.
//
//   Loads.  Each warp streams its own units (32 keys, two tiles of 2304 bytes)
//   through a private ring of bulk copies, one mbarrier a stage, and no
//   barrier joins the warps until a piece of work ends.
//
//   Split.  All pieces of work (sequence, kv head, eight rows) are laid end to
//   end in units of 32 keys, each behind kPieceCost units for what a piece
//   costs by itself (queries, merging), and cut into equal ranges, one per
//   CTA, so a ragged batch or one long sequence keeps every SM equally busy.  A piece
//   of at most 512 keys is not cut: the border moves to its nearer end.  One
//   cut by a range boundary leaves unnormalised partials (max, sum, o) in the
//   workspace; the CTA that arrives last merges them in range order, so the
//   result does not depend on which one that is.
//
//   Measured: 32 sequences of 8191..32767 keys, 32 heads on 8, bf16: 164 us with
//   inputs that change (4.0 TB/s; 148 in a graph, f32 164); one of 131071 keys, 16
//   heads on 8, f16: 48.7 us (46.8 in a graph); one of 500: 7.8 us in a graph, of
//   which the lengths, the table, the words, the split's bookkeeping and the join
//   are each about a microsecond.  128 registers; the 16-bit forms spill 84 bytes
//   a thread, f32 16.
#include "kv4_rows.cuh"

namespace zgpu {

namespace {

constexpr uint32_t kWarps = 8;
constexpr uint32_t kCtasPerSm = 2;
constexpr uint32_t kUnit = 2 * kKv4Tile;         // keys a warp takes at a time
constexpr uint32_t kUnitBytes = 2 * kKv4TileBytes;
constexpr uint32_t kStages = 2;                  // units in flight per warp
constexpr uint32_t kRows = 8;                    // query rows of a piece
constexpr uint32_t kPartFloats = kRows * (kKv4Head + 2);   // o, max, sum
constexpr uint32_t kMergeRow = kKv4Head + 4;     // floats between a warp's rows: its stores hit 32 banks
constexpr uint32_t kMergeFloats = kRows * (kMergeRow + 2);
constexpr float kPShift = 15.f;                  // P is held times 2^15
// A range is worth a unit for every second warp.  4, 8, 16, 32 units measured in a
// graph, 16 heads on 8, f32: one sequence of 1000 keys 7.8, 8.0, 9.2, 10.9 us; four
// of 500 7.9, 9.2, 8.0, 8.0; 16 of 300 11.5, 11.5, 10.7, 13.1; 16 of 1000 14.8,
// 14.8, 14.8, 15.8.
constexpr uint32_t kMinUnits = kWarps / 2;
// What a piece costs beside its units, in units.  4, 8, 16, 32 measured: 16
// sequences of 128..2047 keys, 32 heads on 8, 19.4, 19.3, 17.9, 20.1 us; in a graph
// and 16 heads on 8, four of 500 8.6, 8.4, 7.8, 9.6, 64 of 300 20.8, 20.4, 20.1, 17.0;
// 131071 keys 45.6 to 45.9 with all four.
constexpr uint32_t kPieceCost = 16;
// A piece of no more units than this is not cut: joining costs as much as it
// computes.  None, 12, 16 and 32 units, in a graph, 16 heads on 8, f32: 64 sequences
// of 300 keys 20.1, 16.4, 16.4, 16.4 us, 64 of 500 22.6, 22.8, 18.5, 18.5, 32 of 400
// 14.8, 14.8, 10.5, 10.5, four of 1000 10.4, 10.5, 10.5, 15.8; one of 131071 46.2,
// 46.7, 46.9 (the borders' search).
constexpr uint32_t kWholeUnits = 2 * kWarps;

// Dynamic shared memory: the warps' rings (and, when a piece is done, the
// warps' states in their places: two CTAs then fit an SM whatever the number of
// sequences), the queries, the sums of work over the sequences.
constexpr uint32_t kRingBytes = kWarps * kStages * kUnitBytes;
static_assert(kMergeFloats * 4 <= kStages * kUnitBytes, "a warp's state fits its ring");
constexpr uint32_t kQBytes = 8 * 512;            // hi and lo of eight rows, as fragments
constexpr uint32_t kOffQ = kRingBytes;
constexpr uint32_t kOffSums = kOffQ + kQBytes;

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}

__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Units of a piece over len keys, its own cost included.
__device__ __forceinline__ uint32_t units_of(uint32_t len) { return len ? (len + kUnit - 1) / kUnit + kPieceCost : 0u; }

// a / b; the 64-bit division is long, and hardly ever needed.
__device__ __noinline__ uint64_t long_div(uint64_t a, uint64_t b) { return a / b; }
__device__ __forceinline__ uint64_t div64(uint64_t a, uint64_t b) {
  return (a | b) >> 32 ? long_div(a, b) : static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}

__device__ __forceinline__ uint32_t count_arrival(uint32_t *counter) {
  uint32_t n;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(counter) : "memory");
  return n;
}

template <class T>
__global__ void __launch_bounds__(32 * kWarps, kCtasPerSm) kv4_rows_kernel(const Kv4AttnParams p) {
  // a 16-bit row is exact as hi alone, and so near enough is a probability
  // that a 16-bit result is made of
  constexpr bool kLo = sizeof(T) == 4;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps * kStages];
  __shared__ uint64_t s_scan[kWarps];
  __shared__ uint32_t s_last, s_limit[kRows];
  __shared__ float s_scl[kRows];
  __shared__ __align__(8) uint32_t s_magic[4];
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  uint64_t *sums = reinterpret_cast<uint64_t *>(smem + kOffSums);   // work before sequence i, n_seq + 1
  auto state_of = [&](uint32_t w) { return reinterpret_cast<float *>(smem + w * kStages * kUnitBytes); };
  const uint32_t ring = smem_addr(smem) + warp * kStages * kUnitBytes;
  const uint32_t bar0 = smem_addr(&bars[warp * kStages]);

  if (lane == 0) {
    for (uint32_t s = 0; s < kStages; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_barrier_init();
  }
  // work of sequence i: kv heads x pieces of eight rows x units
  {
    uint64_t base = 0;
    bool bad = false, blind = false;
    for (uint32_t i0 = 0; i0 < p.n_seq; i0 += 32 * kWarps) {
      const uint32_t i = i0 + tid;
      uint64_t w = 0;
      if (i < p.n_seq) {
        const Kv4Seq s = kv4_seq(p, i, &bad);
        blind |= s.len < s.nq;
        if (s.nq * p.group <= p.few_rows)
          w = static_cast<uint64_t>((s.nq * p.group + kRows - 1) / kRows) * p.n_kv * units_of(s.len);
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
    // queries before position 0 see no key and are in no range: zeros, written
    // by every CTA, `share` of them to a sequence (one CTA for all: 1024 sequences of
    // 100 keys, half of them idle, 457 us in place of 126)
    if (__syncthreads_or(blind)) {
      const uint32_t share = gridDim.x > p.n_seq ? gridDim.x / p.n_seq : 1u, cols = p.n_kv * p.group * (kKv4Head / 4);
      for (uint32_t i = blockIdx.x / share; i < p.n_seq; i += gridDim.x / share) {
        const Kv4Seq s = kv4_seq(p, i, &bad);
        for (uint32_t t = blockIdx.x % share; t < s.nq && t + s.len < s.nq; t += share)
          for (uint32_t k = tid; k < cols; k += 32 * kWarps)
            put4(static_cast<T *>(p.out) + (s.q0 + t) * p.out_stride + 4 * k, make_float4(0.f, 0.f, 0.f, 0.f));
      }
    }
  }

  const uint64_t W = sums[p.n_seq];
  uint64_t G = (W + kMinUnits - 1) / kMinUnits;
  if (G > gridDim.x) G = gridDim.x;
  if (blockIdx.x >= G) {
    pdl_wait();
    return;
  }
  // the range's borders, one to a lane; a border inside a short piece moves to
  // the nearer end of it (which moves no border into, or out of, a longer one)
  uint64_t at, end;
  uint32_t seq;
  {
    uint64_t border = div64(W * (blockIdx.x + (lane & 1u)), G);
    uint32_t lo = 0, hi = p.n_seq;   // sums[lo] <= border < sums[hi]
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (sums[mid] <= border) lo = mid;
      else hi = mid;
    }
    bool bad = false;
    const uint32_t all = units_of(kv4_seq(p, lo, &bad).len);
    if (border < W && all <= kWholeUnits + kPieceCost) {
      const uint64_t in = border - sums[lo];
      const uint32_t off = static_cast<uint32_t>(in - div64(in, all) * all);
      border = 2 * off < all ? border - off : border + (all - off);
    }
    at = __shfl_sync(0xffffffffu, border, 0);
    end = __shfl_sync(0xffffffffu, border, 1);
    seq = __shfl_sync(0xffffffffu, lo, 0);
  }
  uint32_t it0 = 0;         // units that this warp took before the piece: stage and phase of the ring
  bool dead = false;        // a wait of this warp ran out
  const Magic mg = magic(smem_addr(s_magic));
  const KMagic kg = k_magic(smem_addr(s_magic + 2));

  while (at < end) {
    while (sums[seq + 1] <= at) ++seq;
    bool bad = false;
    const Kv4Seq s = kv4_seq(p, seq, &bad);
    const uint32_t n_units = (s.len + kUnit - 1) / kUnit, all_units = n_units + kPieceCost;
    const uint32_t pieces = (s.nq * p.group + kRows - 1) / kRows;
    const uint64_t piece = div64(at - sums[seq], all_units);
    const uint64_t piece_at = sums[seq] + piece * all_units + kPieceCost;   // its first unit of keys
    const uint32_t head = static_cast<uint32_t>(div64(piece, pieces)), rt = static_cast<uint32_t>(piece - static_cast<uint64_t>(head) * pieces);
    const uint64_t piece_end = piece_at + n_units, stop = end < piece_end ? end : piece_end;
    if (stop <= piece_at) break;        // the range ends in what the piece costs
    const uint32_t t0 = at > piece_at ? static_cast<uint32_t>(at - piece_at) : 0u;
    const uint32_t t1 = static_cast<uint32_t>(stop - piece_at);
    // the queries' loads go first: warp w takes row w of the piece, four dims
    // per lane (a row behind the last is the first one again, for no use)
    const uint32_t n_rows = s.nq * p.group, qrow = rt * kRows + warp;
    const uint32_t qtok = qrow < n_rows ? qrow / p.group : 0, qhd = qrow < n_rows ? qrow - qtok * p.group : 0;
    const float4 qx = q4(static_cast<const T *>(p.q) + (s.q0 + qtok) * p.q_stride +
                         (static_cast<size_t>(head) * p.group + qhd) * kKv4Head + 4 * lane);
    const uint32_t *table = p.table + static_cast<size_t>(seq) * p.table_width;
    const uint32_t tpb_log2 = p.bt_log2 - 4;
    // this warp's units: t0 + warp + 8 k, k < nk
    const uint32_t nk = t1 - t0 > warp ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;

    // Where the next units lie: lane i holds the address of unit k0 + i, or
    // with blocks of 16 tokens lanes 2 i and 2 i + 1 those of unit k0 + i's
    // tiles, and the lane that holds an address issues its copy.  Table
    // entries are fetched a batch ahead of the addresses.
    const bool split = tpb_log2 == 0;
    const uint32_t batch = split ? 16 : 32;
    auto tile_of = [&](uint32_t k0) { return 2 * (t0 + warp + kWarps * (k0 + (split ? lane >> 1 : lane))) + (split ? lane & 1u : 0u); };
    auto entry = [&](uint32_t k0) -> uint32_t {
      const uint32_t tile = tile_of(k0);
      return k0 + (split ? lane >> 1 : lane) < nk && tile * kKv4Tile < s.len ? __ldg(table + (tile >> tpb_log2)) : kKv4NoSlot;
    };
    const uint8_t *src = nullptr;
    uint32_t ent = entry(0), issued = 0;
    // units of this batch and the one before with a block outside the pool
    uint32_t bad_now = 0, bad_before = 0;
    auto addresses = [&](uint32_t k0) {
      const uint32_t tile = tile_of(k0);
      const bool is = k0 + (split ? lane >> 1 : lane) < nk && tile * kKv4Tile < s.len, ok = ent < p.n_blocks;
      // a tile that is not there is copied from block 0, for the mask to drop
      src = p.pool + (((static_cast<size_t>(ok ? ent : 0u) * p.n_kv + head) << tpb_log2) + (tile & ((1u << tpb_log2) - 1u))) *
                         kKv4TileBytes;
      bad_before = bad_now;
      bad_now = __ballot_sync(0xffffffffu, is && !ok);
      if (is && !ok) atomicOr(p.status, ZDEV_ERR_BOUNDS);
      ent = entry(k0 + batch);
    };
    auto issue = [&]() {
      const uint32_t i = issued & (batch - 1);
      if (i == 0) addresses(issued);
      const uint32_t stage = (it0 + issued) % kStages, bar = bar0 + 8 * stage, dst = ring + stage * kUnitBytes;
      if (split) {
        if (lane == 2 * i) mbar_arrive_expect_tx(bar, kUnitBytes);
        __syncwarp();
        if ((lane >> 1) == i) bulk_copy_g2s(dst + (lane & 1u) * kKv4TileBytes, src, kKv4TileBytes, bar);
      } else if (lane == i) {
        mbar_arrive_expect_tx(bar, kUnitBytes);
        bulk_copy_g2s(dst, src, kUnitBytes, bar);
      }
      ++issued;
    };
    const uint32_t ahead = nk < kStages ? nk : kStages;
    if (!dead)
      while (issued < ahead) issue();

    // the queries, scaled by a power of two and split in hi and lo; fragment kk
    // of lane (r, c) is the 16 bytes at 512 kk + 16 lane: dims 32 (kk / 2) + 8 c +
    // 4 (kk % 2) + 0..3
    {
      const float4 x = qx;
      float amax = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      // 256 times: the low halves stay far from binary16's subnormals
      int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
      e = e < -119 ? -119 : e > 127 ? 127 : e;
      const float down = __uint_as_float(static_cast<uint32_t>(127 + 8 - e) << 23);
      const float4 y = make_float4(x.x * down, x.y * down, x.z * down, x.w * down);
      const __half2 h0 = __floats2half2_rn(y.x, y.y), h1 = __floats2half2_rn(y.z, y.w);
      const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
      *reinterpret_cast<uint4 *>(smem + kOffQ + 512 * (2 * (lane >> 3) + (lane & 1u)) + 16 * (4 * warp + ((lane & 7u) >> 1))) =
          make_uint4(h2bits(h0), h2bits(__floats2half2_rn(y.x - f0.x, y.y - f0.y)), h2bits(h1),
                     h2bits(__floats2half2_rn(y.z - f1.x, y.w - f1.y)));
      if (lane == 0) {
        // keys that the row sees: 0 .. limit - 1 (none when its position is negative)
        const int64_t pos1 = static_cast<int64_t>(s.len) - s.nq + qtok + 1;
        s_limit[warp] = pos1 > 0 ? static_cast<uint32_t>(pos1) : 0u;
        s_scl[warp] = score_factor(p.scale, e - 8);
      }
    }
    __syncthreads();
    const uint32_t limit = s_limit[r], qs = smem_addr(smem) + kOffQ + 16 * lane;
    const float scl = s_scl[r];
    uint32_t all_see = limit;       // keys that every row sees need no mask
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, off));

    // o[n]: dims 16 n + r (and + 8) of rows 2 c and 2 c + 1; m (the exponent that P is
    // held relative to), l: row r
    float o[8][4], m = -INFINITY;
    float2 l = make_float2(0.f, 0.f);
#pragma unroll
    for (int n = 0; n < 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

    for (uint32_t k = 0; k < nk && !dead; ++k) {
      const uint32_t stage = (it0 + k) % kStages;
      dead = __any_sync(0xffffffffu, !mbar_wait(bar0 + 8 * stage, ((it0 + k) / kStages) & 1u, p.status));
      if (dead) {       // the copies in flight land before the CTA may end
        for (uint32_t x = k + 1; x < issued; ++x)
          mbar_wait(bar0 + 8 * ((it0 + x) % kStages), ((it0 + x) / kStages) & 1u, p.status);
        break;
      }
      const uint32_t base0 = ring + stage * kUnitBytes, key0 = (t0 + warp + kWarps * k) * kUnit;
      // scores of keys 8 u + 2 c and + 1 of row r
      float2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = make_float2(0.f, 0.f);
      uint4 kw[4], kd[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        kw[u] = lds128(base0 + kKv4TileBytes * (u >> 1) + 512 * (u & 1) + 16 * lane);
        kd[u] = lds128(base0 + kKv4TileBytes * (u >> 1) + kKv4Ks + 64 * (u & 1) + 16 * c);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint4 qa = lds128(qs + 1024 * g), qb = lds128(qs + 1024 * g + 512);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t w = g == 0 ? kw[u].x : g == 1 ? kw[u].y : g == 2 ? kw[u].z : kw[u].w, w8 = w >> 8;
          const uint32_t dw = g == 0 ? kd[u].x : g == 1 ? kd[u].y : g == 2 ? kd[u].z : kd[u].w;
          float sc[4];
          // 1024 + n, less 1032; 64 + n, less 72
          uint32_t n[4] = {(w & 0x000F000Fu) | kg.x1024, (w & 0x00F000F0u) | kg.x64, (w8 & 0x000F000Fu) | kg.x1024,
                           (w8 & 0x00F000F0u) | kg.x64};
#pragma unroll
          for (int x = 0; x < 4; ++x) n[x] = h2bits(__hsub2(bits2h(n[x]), bits2h(x & 1 ? 0x54805480u : 0x64086408u)));
          mma16816_zero(sc, qa.x, qa.y, qa.z, qa.w, n[0], n[1]);
          mma16816(sc, qb.x, qb.y, qb.z, qb.w, n[2], n[3]);
          float2 t = make_float2(sc[0], sc[1]);
          if (kLo) t = add2_rn(t, make_float2(sc[2], sc[3]));
          v[u] = fma2_rn(t, __half22float2(bits2h(dw)), v[u]);
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = mul2_rn(v[u], make_float2(scl, scl));
      if (key0 + kUnit > all_see || (bad_now | bad_before)) {
        // which of the unit's tiles lie in the pool: its batch is the last
        // one addressed or, with units in flight, the one before
        const uint32_t bm = (issued - 1) / batch == k / batch ? bad_now : bad_before, i = k & (batch - 1);
        const bool gone0 = (bm >> (split ? 2 * i : i)) & 1u, gone1 = (bm >> (split ? 2 * i + 1 : i)) & 1u;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t key = key0 + 8 * u + 2 * c;
          if (key >= limit || (u < 2 ? gone0 : gone1)) v[u].x = -INFINITY;
          if (key + 1 >= limit || (u < 2 ? gone0 : gone1)) v[u].y = -INFINITY;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) mx = fmaxf(mx, fmaxf(v[u].x, v[u].y));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // P is 2^(v - m) with m the largest score less kPShift, rounded up: rounded
      // otherwise, P could pass binary16's range for scores from 2^24
      mx = fmaxf(m, __fadd_ru(mx, -kPShift));
      const float ms = mx == -INFINITY ? 0.f : mx;
      if (__any_sync(0xffffffffu, mx > m)) {
        const float a = ex2(m - ms);
        const float2 aa = make_float2(__shfl_sync(0xffffffffu, a, 8 * c), __shfl_sync(0xffffffffu, a, 8 * c + 4));
        l = mul2_rn(l, make_float2(a, a));
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 x = mul2_rn(make_float2(o[n][0], o[n][1]), aa), y = mul2_rn(make_float2(o[n][2], o[n][3]), aa);
          o[n][0] = x.x, o[n][1] = x.y, o[n][2] = y.x, o[n][3] = y.y;
        }
        m = mx;
      }
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float2 e = add2_rn(v[u], make_float2(-ms, -ms)), pr = make_float2(ex2(e.x), ex2(e.y));
        l = add2_rn(l, pr);
        const __half2 hi = __floats2half2_rn(pr.x, pr.y);
        ph[u] = h2bits(hi);
        if (kLo) {
          const float2 lo = sub2_rn(pr, __half22float2(hi));
          pl[u] = h2bits(__floats2half2_rn(lo.x, lo.y));
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t b = base0 + kKv4TileBytes * t + kKv4V;
        const uint4 w0 = lds128(b + 16 * lane), w1 = lds128(b + 512 + 16 * lane);
        const uint4 d0 = lds128(b + kKv4Vs - kKv4V + 16 * c), d1 = lds128(b + kKv4Vs - kKv4V + 64 + 16 * c);
        const uint32_t a0[4] = {w0.x, w0.y, w0.z, w0.w}, a1[4] = {w1.x, w1.y, w1.z, w1.w};
        const uint32_t e0[4] = {d0.x, d0.y, d0.z, d0.w}, e1[4] = {d1.x, d1.y, d1.z, d1.w};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const __half2 x0 = bits2h(e0[g]), x1 = bits2h(e1[g]);
          uint32_t v0[4], v1[4];
          v_values(a0[g], x0, __hmul2(x0, __float2half2_rn(-24.f)), mg, v0);
          v_values(a1[g], x1, __hmul2(x1, __float2half2_rn(-24.f)), mg, v1);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            mma16816(o[2 * g + n], v0[2 * n], v0[2 * n + 1], v1[2 * n], v1[2 * n + 1], ph[2 * t], ph[2 * t + 1]);
            if (kLo) mma16816(o[2 * g + n], v0[2 * n], v0[2 * n + 1], v1[2 * n], v1[2 * n + 1], pl[2 * t], pl[2 * t + 1]);
          }
        }
      }
      __syncwarp();       // every lane has read the stage before it is filled again
      if (issued < nk) issue();
    }
    it0 += nk;

    // the warps' states, then the piece
    float lsum = l.x + l.y;
    lsum += __shfl_xor_sync(0xffffffffu, lsum, 1);
    lsum += __shfl_xor_sync(0xffffffffu, lsum, 2);
    float *mine = state_of(warp);
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(2 * c + (e & 1)) * kMergeRow + 16 * n + 8 * (e >> 1) + r] = o[n][e];
    if (c == 0) {
      mine[kRows * kMergeRow + 2 * r] = m;
      mine[kRows * kMergeRow + 2 * r + 1] = lsum;
    }
    __syncthreads();
    // thread: row mr, dims 4 mc ..
    const uint32_t mr = tid >> 5, mc = tid & 31;
    // weights of states by their maxima: a state that saw no key has nothing
    // to add, and a broken one (a NaN sum) breaks the whole
    auto weight = [](float m, float top) { return m == top ? 1.f : ex2(m - top); };
    float M = -INFINITY, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    {
      float2 ml[kWarps];
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) {
        ml[w] = *reinterpret_cast<const float2 *>(state_of(w) + kRows * kMergeRow + 2 * mr);
        M = fmaxf(M, ml[w].x);
      }
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4 *>(state_of(w) + mr * kMergeRow + 4 * mc);
        const float a = weight(ml[w].x, M);
        L += ml[w].y * a;
        O.x += x.x * a, O.y += x.y * a, O.z += x.z * a, O.w += x.w * a;
      }
    }
    bool whole = t0 == 0 && t1 == n_units;
    if (!whole) {
      float *dst = p.part + (2ull * blockIdx.x + (t0 == 0 ? 1 : 0)) * kPartFloats;
      *reinterpret_cast<float4 *>(dst + mr * kKv4Head + 4 * mc) = O;
      if (mc == 0) *reinterpret_cast<float2 *>(dst + kRows * kKv4Head + 2 * mr) = make_float2(M, L);
      // the ranges that share the piece
      const uint32_t c0 = static_cast<uint32_t>(div64((piece_at + 1) * G - 1, W));
      const uint32_t c1 = static_cast<uint32_t>(div64(piece_end * G - 1, W));
      __syncthreads();
      if (tid == 0) {
        s_last = count_arrival(&p.counters[c0]) == c1 - c0;
        if (s_last) p.counters[c0] = 0;
      }
      __syncthreads();
      if (s_last) {
        // the row's largest maximum and the ranges' weights, a lane each, then
        // the sums: the loads of a batch do not wait for one another
        M = -INFINITY;
        L = 0.f;
        O = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t k0 = c0; k0 <= c1; k0 += 32) {
          const uint32_t k = k0 + mc, n = min(32u, c1 - k0 + 1);
          auto sums_of = [&](uint32_t j) {
            return __ldcg(reinterpret_cast<const float4 *>(p.part + (2ull * (k0 + j) + (k0 + j == c0 ? 1 : 0)) * kPartFloats +
                                                           mr * kKv4Head + 4 * mc));
          };
          // the first sums come with the states: most pieces are cut in few
          constexpr uint32_t kFirst = 4;
          float4 first[kFirst];
#pragma unroll
          for (uint32_t j = 0; j < kFirst; ++j) first[j] = j < n ? sums_of(j) : make_float4(0.f, 0.f, 0.f, 0.f);
          float2 st = make_float2(-INFINITY, 0.f);
          if (k <= c1)
            st = __ldcg(reinterpret_cast<const float2 *>(p.part + (2ull * k + (k == c0 ? 1 : 0)) * kPartFloats +
                                                         kRows * kKv4Head + 2 * mr));
          float nm = fmaxf(M, st.x);
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, off));
          const float keep = weight(M, nm), w = weight(st.x, nm);
          L *= keep;
          O.x *= keep, O.y *= keep, O.z *= keep, O.w *= keep;
          auto add = [&](uint32_t j, const float4 x) {
            const float wj = __shfl_sync(0xffffffffu, w, j);
            L += __shfl_sync(0xffffffffu, st.y, j) * wj;
            O.x += x.x * wj, O.y += x.y * wj, O.z += x.z * wj, O.w += x.w * wj;
          };
#pragma unroll
          for (uint32_t j = 0; j < kFirst; ++j)
            if (j < n) add(j, first[j]);
#pragma unroll 8
          for (uint32_t j = kFirst; j < n; ++j) add(j, sums_of(j));
          M = nm;
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
    // the rings are free again, for bulk copies behind these plain accesses
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    at = stop;
  }
  pdl_wait();              // the launch ends no earlier than the one before it
}

template <class T>
cudaError_t launch_rows(const Kv4AttnParams &p, bool behind, int sm_count, cudaStream_t s) {
  const uint32_t smem = kOffSums + (p.n_seq + 1) * 8;
  if (!behind) {
    kv4_rows_kernel<T><<<sm_count * kCtasPerSm, 32 * kWarps, smem, s>>>(p);
    return cudaGetLastError();
  }
  // behind the prompt kernel, which it does not depend on: it may start as
  // that one's CTAs end, and ends after it
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sm_count * kCtasPerSm);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_rows_kernel<T>, p);
}

template <class T>
cudaError_t rows_setup() {
  return cudaFuncSetAttribute(kv4_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              kOffSums + (kKv4MaxSeqs + 1) * 8);
}

// Query rows per kv head above which a sequence goes to the prompt kernel
// (kv4_prompt.cu).  That one's time hardly depends on the rows of a tile, but it
// starts slowly and joins long sequences in one CTA per kv head; this one's
// grows by a pass over the cache with every eighth row.  So the border falls with
// what a pass costs: the keys that the call can read, sequences x kv heads x
// (table row + 512, a piece's own cost).  us, few rows / prompt kernel, in a graph:
//                               rows  16          32          48          64          96
//   f32  1 x   700, 8 kv heads     8.8/20.7    9.8/21.2   10.5/21.9   11.0/22.2   12.0/23.4
//        1 x  8000, 8             15.0/41.4   19.3/40.6   23.2/41.6   27.8/42.1   35.7/44.1
//       64 x   700, 1             13.9/26.3   17.9/26.6   23.4/27.3   27.1/27.7   36.4/28.7
//       16 x   700, 8             17.8/31.8   27.2/32.1   36.3/32.3   44.1/33.0   62.3/33.9
//        1 x 65536, 8             46.1/85.2   79.3/86.2  113.2/87.5  147.2/88.6  214.8/89.8
//       16 x  4096, 8             47.4/71.7   84.0/72.6  120.9/74.2  158.6/74.8  231.2/76.3
//       64 x   700, 8             44.4/69.4   79.5/70.0  114.5/71.9  149.7/73.2  220.9/79.9
//   f16  1 x   700, 8              9.0/23.3    9.8/23.7   10.8/24.0   10.8/24.6   12.0/25.4
//        1 x  8000, 8             14.6/57.6   18.2/59.3   21.7/59.9   25.9/60.0   33.5/61.1
//       64 x   700, 1             13.2/30.1   17.6/30.4   22.5/30.9   26.4/31.2   35.3/32.0
//       16 x   700, 8             17.6/34.2   26.6/34.5   35.3/34.9   42.7/35.3   60.3/36.1
//        1 x 65536, 8             43.2/109     73.4/109    104/110     135/110     196/112
//       16 x  4096, 8             44.7/85.6   78.7/85.9    112/85.7    147/86.5    214/87.1
//       64 x   700, 8             42.6/76.3   76.7/77.1    110/77.9    144/78.5    210/79.6
// Groups of 1, 4 and 8 measured alike.  The lengths themselves are on the
// device: a table wider than its sequences, or idle rows, count as keys and
// lower the border, to no less than 24 and 32, which is right for large calls.
uint32_t kv4_few_rows(const Kv4AttnParams &p, bool f32) {
  const uint64_t keys = static_cast<uint64_t>(p.n_seq) * p.n_kv * ((static_cast<uint64_t>(p.table_width) << p.bt_log2) + 512);
  const uint64_t rows = (f32 ? 6400000u : 7500000u) / keys, least = f32 ? 24 : 32;
  return static_cast<uint32_t>(rows < least ? least : rows > 96 ? 96 : rows);
}

size_t rows_part_floats(int sm_count) { return static_cast<size_t>(sm_count) * kCtasPerSm * 2 * kPartFloats; }

}  // namespace

size_t kv4_attn_part_bytes(int sm_count) {
  return rows_part_floats(sm_count) * sizeof(float) + kv4_prompt_part_bytes(sm_count);
}
uint32_t kv4_attn_counters(int sm_count) {
  return static_cast<uint32_t>(sm_count) * kCtasPerSm + kv4_prompt_counters(sm_count);
}

cudaError_t kv4_attn_setup() {
  cudaError_t e = rows_setup<float>();
  if (e == cudaSuccess) e = rows_setup<__half>();
  if (e == cudaSuccess) e = rows_setup<__nv_bfloat16>();
  if (e == cudaSuccess) e = kv4_prompt_setup();
  return e;
}

cudaError_t launch_kv4_attention(const Kv4AttnParams &p, Kv4Type t, int sm_count, uint32_t *launches, cudaStream_t s) {
  Kv4AttnParams few = p;
  few.few_rows = kv4_few_rows(p, t == KV4_F32);
  const bool both = static_cast<uint64_t>(p.max_q) * p.group > few.few_rows;
  cudaError_t e = cudaSuccess;
  if (both) {
    Kv4AttnParams many = few;
    many.part = p.part + rows_part_floats(sm_count);
    many.counters = p.counters + static_cast<uint32_t>(sm_count) * kCtasPerSm;
    e = launch_kv4_prompt(many, t, sm_count, s);
    if (e != cudaSuccess) return e;
    if (launches) ++*launches;
  }
  if (t == KV4_F32) e = launch_rows<float>(few, both, sm_count, s);
  else if (t == KV4_F16) e = launch_rows<__half>(few, both, sm_count, s);
  else e = launch_rows<__nv_bfloat16>(few, both, sm_count, s);
  if (e == cudaSuccess && launches) ++*launches;
  return e;
}

}  // namespace zgpu
