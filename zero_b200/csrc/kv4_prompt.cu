// kv4_prompt.cu — attention of prompts and prompt chunks over the paged 4-bit
// KV cache, on tcgen05.
//
// The same formula as kv4_attn.cu for sequences with many query rows per kv head
// (kv4_few_rows there).  Bound by the tensor cores (4 * 128 flops per query head and
// key, twice that for f32 rows) and, as closely, by the exponentials: 128 x
// 128 scores are 1024 cycles of either.
//
// A persistent CTA per SM works through pieces (sequence, kv head, row tile);
// a row tile is 256 query rows of the kv head's group for 16-bit types, 128
// for f32.  Keys come 128 at a time.  Two streams of softmax run side by
// side, each 128 rows with its own score columns and accumulator in TMEM, so
// that one stream's exponentials overlap the other's products:
//   16-bit rows  stream i is rows 128 i.. of the tile, both see every key tile;
//   f32 rows     q = hi + lo (binary16 each), S = hi K^T + lo K^T in one
//                accumulator, P = hi + lo likewise; the streams take the key
//                tiles in turn and are joined at the end of the piece.
// The cache's values are exact in binary16 (kv4.h), so f32 rows keep 22 bits.
//
// Warps:
//   0-7    softmax, a row per thread: the scores' maximum, then exponentials
//          written back over the scores as the A operand of P V.  For 16-bit
//          rows the accumulator is rescaled only when a row's maximum has
//          grown by more than 2^8, with P held times 2^7; for f32 rows at
//          once, with P times 2^15, which keeps it to 2^-40 of the largest;
//   8-11   keys and values, tile after tile, from 4-bit words to binary16
//          operands in a ring of three, a key word being one 16-byte chunk of
//          the canonical layout;
//   12     one thread issues the MMAs: PV(t), then S(t + 2), in order;
//   13     bulk copies of the tiles' words, two key tiles ahead;
//   14-15  the next piece's query rows, together with 8-11.
// TMEM (512 columns): S of stream 0 and 1 at 0 and 128, O at 256 and 384.  P
// lies on its own scores: 32 score columns become 16 of hi and 16 of lo.
//
// The work is cut into equal ranges of key tiles as in kv4_attn.cu; pieces cut
// by a range boundary leave partials that the last CTA to arrive joins.
// Measured: eight prompts of 1021..2048 tokens, 32 heads on 8, f16: 225 us with
// inputs that change (207 in a graph, 36 % of the tensor cores' time); a prompt of 2048 in
// f32, 16 heads on 8: 59 us.  The MMA warp, the conversion and the streams'
// chains take about as long as each other (3000 to 4400 cycles a key tile).
// Every wait is bounded; on an expired one each role stops, the MMA thread
// waits for its own MMAs, and TMEM is freed.
#include "kv4_rows.cuh"
#include "tcgen05.cuh"

namespace zgpu {

namespace {

constexpr uint32_t kSoftWarps = 8, kConvWarps = 4, kQWarps = 2, kThreads = 512;
constexpr uint32_t kConv0 = kSoftWarps, kMmaWarp = kConv0 + kConvWarps, kLoadWarp = kMmaWarp + 1, kQ0 = kLoadWarp + 1;
static_assert(32 * (kQ0 + kQWarps) == kThreads, "every warp has a role");
constexpr uint32_t kKeys = 128;                       // keys of a tile
constexpr uint32_t kOpBytes = 128 * kKv4Head * 2;     // one operand tile: 128 rows x 128 binary16
constexpr uint32_t kSlots = 3;                        // operand tiles of keys and values, in turn
constexpr uint32_t kHalfBytes = kKv4TileBytes / 2;    // K's or V's words and scales of 16 keys
constexpr uint32_t kRawBytes = kKeys / kKv4Tile * kHalfBytes, kRawStages = 2;   // of each kind
constexpr uint32_t kOffQ = 0, kOffOp = 2 * kOpBytes, kOffRaw = kOffOp + kSlots * kOpBytes;
constexpr uint32_t kOffTab = kOffRaw + 2 * kRawStages * kRawBytes;
constexpr uint32_t kMaxRows = 256;
constexpr uint32_t kPartFloats = kMaxRows * (kKv4Head + 2);
constexpr uint32_t kMinTiles = 2;                     // units of work that a range is worth
constexpr uint32_t kTmemS = 0, kTmemO = 256, kTmemCols = 512;
// kind::f16: D f32, A and B binary16, both K-major, N = 128, M = 128
constexpr uint32_t kIdesc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
// Operand tiles: [row / 8][16-byte chunk][row % 8][16 bytes]
constexpr uint32_t kLbo = 128, kSbo = 2048;
constexpr uint32_t kPieces = 4;                       // pieces made known ahead

struct Bars {
  uint64_t nfull[kPieces], nempty[kPieces];
  uint64_t qfull, qempty, rfull[2][kRawStages], rempty[2][kRawStages], full[kSlots], empty[kSlots];
  uint64_t sfull[2], pfull[2], ofull[2], oempty[2], join, drain;
};

// K's four nibble pairs of a word (bits 0, 4, 8, 12 of each half) as (n - 8) d.
__device__ __forceinline__ void k_values(uint32_t w, __half2 d, const KMagic &g, uint32_t (&v)[4]) {
  const uint32_t w8 = w >> 8;
  const __half2 m1032 = __half2half2(__ushort_as_half(0xE408)), m72 = __half2half2(__ushort_as_half(0xD480));
  v[0] = h2bits(__hmul2(__hadd2(bits2h((w & 0x000F000Fu) | g.x1024), m1032), d));
  v[1] = h2bits(__hmul2(__hadd2(bits2h((w & 0x00F000F0u) | g.x64), m72), d));
  v[2] = h2bits(__hmul2(__hadd2(bits2h((w8 & 0x000F000Fu) | g.x1024), m1032), d));
  v[3] = h2bits(__hmul2(__hadd2(bits2h((w8 & 0x00F000F0u) | g.x64), m72), d));
}

// 32 bytes to a 32-byte boundary: a whole sector a lane.
__device__ __forceinline__ void st_sector(void *p, const uint32_t *v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// 32 values of a row.  A lane writes its own row, so a store is worth as many
// bytes as it can carry: whole sectors where the rows allow it (eight f16 prompts
// 209 us, with 16-byte stores alone 218; a prompt of 2048 in f32 60.7 and 61.6).
template <class T>
__device__ __forceinline__ void put32(T *p, const float (&o)[32], bool sectors) {
  constexpr int kWords = 8 * sizeof(T);
  uint32_t w[kWords];
#pragma unroll
  for (int x = 0; x < kWords; ++x) {
    if (sizeof(T) == 4) {
      w[x] = __float_as_uint(o[x]);
    } else if (__is_same(T, __half)) {
      w[x] = h2bits(__floats2half2_rn(o[(2 * x) & 31], o[(2 * x + 1) & 31]));
    } else {
      const __nv_bfloat162 b = __floats2bfloat162_rn(o[(2 * x) & 31], o[(2 * x + 1) & 31]);
      w[x] = *reinterpret_cast<const uint32_t *>(&b);
    }
  }
  uint32_t *d = reinterpret_cast<uint32_t *>(p);
  if (sectors) {
#pragma unroll
    for (int x = 0; x < kWords; x += 8) st_sector(d + x, w + x);
  } else {
#pragma unroll
    for (int x = 0; x < kWords; x += 4) *reinterpret_cast<uint4 *>(d + x) = make_uint4(w[x], w[x + 1], w[x + 2], w[x + 3]);
  }
}

// Waits with the polling loop out of line: six roles share the instruction
// cache, and their loops have to stay small (with everything unrolled and
// inlined the kernel spent more time fetching instructions than issuing them).
__device__ __noinline__ bool slow_wait(uint32_t bar, uint32_t parity, uint32_t *status) {
  return mbar_wait(bar, parity, status);
}
__device__ __forceinline__ bool wait(uint64_t &bar, uint32_t parity, uint32_t *status) {
  return mbar_try_wait(smem_addr(&bar), parity) || slow_wait(smem_addr(&bar), parity, status);
}
// A bounded wait of a whole warp with one answer for all lanes.
__device__ __forceinline__ bool warp_wait(uint64_t &bar, uint32_t parity, uint32_t *status) {
  return __all_sync(0xffffffffu, wait(bar, parity, status));
}

// A piece of work, as the loading warp makes it known to the others: code that
// runs once a piece comes from behind the instruction cache (some 16 cycles an
// instruction), so one warp walks, ahead of the rest, and they read.
struct Piece {
  uint32_t seq, head, rt;        // what
  uint32_t t0, t1, n;            // key tiles t0 .. t1 - 1 of n; t1 = 0 ends the range
  Kv4Seq s;
  uint32_t c0, c1;               // the ranges that share the piece
  uint32_t tok0, rem0;           // the row tile's first row as token and head of the group
  // token and head of the tile's row r: r + rem0 < 272, so 2^16 / group, rounded
  // up, divides exactly
  __device__ __forceinline__ void place(uint32_t r, uint32_t group, uint32_t inv, uint32_t *tok, uint32_t *hd) const {
    const uint32_t x = r + rem0, y = x * inv >> 16;
    *tok = tok0 + y;
    *hd = x - y * group;
  }
};

// Walks the pieces of a range.  A piece of n key tiles is n + kPieceCost units
// of work, the tiles being the last n.

template <uint32_t MR>
struct Walk {
  // What a piece costs beside its key tiles, in key tiles (1, 2, 3, 4 measured:
  // a prompt of 2048 in f32 67.3, 62.7, 60.5, 62.4 us; eight prompts in f16 220,
  // 212, 218, 224).
  static constexpr uint32_t kPieceCost = MR == 128 ? 3 : 2;
  const uint64_t *sums;
  const uint32_t *lens, *nqs, *q0s;
  uint32_t n_kv, group;
  uint64_t at, end;
  Piece p = {};
  uint64_t first = 0;            // the piece's first tile in units of work
  uint32_t n_rt, off;            // units of the piece before `at`
  bool fresh;

  __device__ __forceinline__ static uint32_t row_tiles(uint32_t nq, uint32_t group) { return (nq * group + MR - 1) / MR; }
  // key tiles that row tile rt sees
  __device__ __forceinline__ static uint32_t tiles(uint32_t len, uint32_t nq, uint32_t group, uint32_t rt) {
    const uint32_t toks = min(nq, ((rt + 1) * MR - 1) / group + 1);    // tokens up to the tile's last row's
    const int64_t see = static_cast<int64_t>(len) - nq + toks;
    return see > 0 ? static_cast<uint32_t>((see + kKeys - 1) / kKeys) : 0u;
  }
  __device__ __forceinline__ static uint32_t units(uint32_t len, uint32_t nq, uint32_t group, uint32_t rt) {
    const uint32_t n = tiles(len, nq, group, rt);
    return n ? n + kPieceCost : 0u;
  }
  __device__ __forceinline__ void load() {
    p.s.len = lens[p.seq];
    p.s.nq = nqs[p.seq];
    p.s.q0 = q0s[p.seq];
    n_rt = row_tiles(p.s.nq, group);
  }
  // The first piece: all lanes of the warp take part.
  __device__ __forceinline__ void start(uint32_t n_seq) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, hi = n_seq;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (sums[mid] <= at) lo = mid;
      else hi = mid;
    }
    while (sums[lo + 1] <= at) ++lo;
    p.seq = lo;
    load();
    const uint64_t per_head = (sums[lo + 1] - sums[lo]) / n_kv, rem0 = at - sums[lo];
    p.head = static_cast<uint32_t>(rem0 / per_head);
    uint64_t rem = rem0 % per_head;
    for (uint32_t r0 = 0; r0 < n_rt; r0 += 32) {
      const uint32_t mine = r0 + lane < n_rt ? units(p.s.len, p.s.nq, group, r0 + lane) : 0u;
      uint32_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= static_cast<uint32_t>(o)) inc += u;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, rem < inc);
      if (hit) {
        const uint32_t l = __ffs(hit) - 1;
        p.rt = r0 + l;
        p.n = __shfl_sync(0xffffffffu, mine, l) - kPieceCost;
        off = static_cast<uint32_t>(rem) - (__shfl_sync(0xffffffffu, inc, l) - p.n - kPieceCost);
        break;
      }
      rem -= __shfl_sync(0xffffffffu, inc, 31);
    }
    fresh = true;
  }
  // The next piece of the range with a key tile in it, or false.
  __device__ __forceinline__ bool next() {
    while (at < end) {
      if (!fresh) {
        off = 0;
        while (true) {
          if (++p.rt == n_rt) {
            p.rt = 0;
            if (++p.head == n_kv) {
              p.head = 0;
              do ++p.seq;
              while (sums[p.seq + 1] <= at);
              load();
            }
          }
          p.n = tiles(p.s.len, p.s.nq, group, p.rt);
          if (p.n) break;
        }
      }
      fresh = false;
      first = at - off + kPieceCost;
      const uint64_t left = end - at;
      const uint32_t last = left < p.n + kPieceCost - off ? off + static_cast<uint32_t>(left) : p.n + kPieceCost;
      p.t0 = off > kPieceCost ? off - kPieceCost : 0u;
      p.t1 = last > kPieceCost ? last - kPieceCost : 0u;
      at += last - off;
      if (p.t1 > p.t0) return true;
    }
    return false;
  }
};

// One of kConvWarps + kQWarps warps' share of a piece's query rows: binary16
// (hi and lo for f32) in the operand layout, and each row's factor of the
// scores.  Eight rows at a time, lane (kr, kq) taking chunks kq, kq + 4, kq + 8,
// kq + 12 of row kr: the eight lanes of a 16-byte store phase write 128
// contiguous bytes.  All of a warp's rows are on their way at once, copied to
// where they end up (an f32 chunk's two halves to its hi and its lo place);
// then f32 and bf16 rows are scaled by a power of two (the largest value in
// [2, 4); subnormal rows by 2^127) to fit binary16's range, in place, each lane
// its own chunks.
template <class T>
__device__ __forceinline__ void load_queries(const Kv4AttnParams &p, const Piece &pc, uint8_t *q_op, float *s_scl,
                                             uint32_t inv, uint32_t share) {
  constexpr bool kLo = sizeof(T) == 4, kCopy = __is_same(T, __half);
  constexpr uint32_t MR = kLo ? 128 : 256, kShares = kConvWarps + kQWarps;
  const uint32_t lane = threadIdx.x & 31, kr = lane & 7, kq = lane >> 3, n_rows = pc.s.nq * p.group;
  const uint32_t row0 = pc.rt * MR, at = smem_addr(q_op) + 16 * kr + kLbo * kq;
  const T *q = static_cast<const T *>(p.q) + pc.s.q0 * p.q_stride + static_cast<size_t>(pc.head) * p.group * kKv4Head + 8 * kq;
#pragma unroll 1
  for (uint32_t g = share; g < MR / 8; g += kShares) {
    uint32_t tok, hd;
    pc.place(8 * g + kr, p.group, inv, &tok, &hd);
    const bool is = row0 + 8 * g + kr < n_rows;       // zeros behind the last row
    const T *src = is ? q + tok * p.q_stride + hd * kKv4Head : static_cast<const T *>(p.q);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      cp_async16(at + kSbo * g + 4 * kLbo * k, src + (is ? 32 * k : 0), is ? 16u : 0u);
      if (kLo) cp_async16(at + kOpBytes + kSbo * g + 4 * kLbo * k, src + (is ? 32 * k + 4 : 0), is ? 16u : 0u);
    }
    if (kCopy && kq == 0) s_scl[8 * g + kr] = score_factor(p.scale, 0);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!kCopy) {
#pragma unroll 1
    for (uint32_t g = share; g < MR / 8; g += kShares) {
      uint8_t *dst = q_op + kSbo * g + 16 * kr + kLbo * kq;
      uint4 a[4], b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] = *reinterpret_cast<const uint4 *>(dst + 4 * kLbo * k);
        if (kLo) b[k] = *reinterpret_cast<const uint4 *>(dst + kOpBytes + 4 * kLbo * k);
      }
      float amax = 0.f;
      if (kLo) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          amax = fmaxf(fmaxf(fmaxf(fabsf(__uint_as_float(a[k].x)), fabsf(__uint_as_float(a[k].y))),
                             fmaxf(fabsf(__uint_as_float(a[k].z)), fabsf(__uint_as_float(a[k].w)))), amax);
          amax = fmaxf(fmaxf(fmaxf(fabsf(__uint_as_float(b[k].x)), fabsf(__uint_as_float(b[k].y))),
                             fmaxf(fabsf(__uint_as_float(b[k].z)), fabsf(__uint_as_float(b[k].w)))), amax);
        }
      } else {
        __nv_bfloat162 mx = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t u[4] = {a[k].x, a[k].y, a[k].z, a[k].w};
#pragma unroll
          for (int x = 0; x < 4; ++x) mx = __hmax2(mx, __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&u[x])));
        }
        amax = fmaxf(__low2float(mx), __high2float(mx));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
      int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
      e = e < -126 ? -126 : e > 127 ? 127 : e;
      const float down = __uint_as_float(static_cast<uint32_t>(127 + 1 - e) << 23);
      if (kq == 0)
        s_scl[8 * g + kr] = score_factor(p.scale, e - 1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float2 f;
          if (kLo) {
            const uint4 u = x < 2 ? a[k] : b[k];
            f = x & 1 ? make_float2(__uint_as_float(u.z), __uint_as_float(u.w))
                      : make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
          } else {
            const uint32_t w = x == 0 ? a[k].x : x == 1 ? a[k].y : x == 2 ? a[k].z : a[k].w;
            f = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
          }
          f = mul2_rn(f, make_float2(down, down));
          const __half2 h = __floats2half2_rn(f.x, f.y);
          hi[x] = h2bits(h);
          if (kLo) {
            const float2 r = __half22float2(h);
            lo[x] = h2bits(__floats2half2_rn(f.x - r.x, f.y - r.y));
          }
        }
        *reinterpret_cast<uint4 *>(dst + 4 * kLbo * k) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (kLo) *reinterpret_cast<uint4 *>(dst + kOpBytes + 4 * kLbo * k) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

template <class T>
__global__ void __launch_bounds__(kThreads, 1) kv4_prompt_kernel(const Kv4AttnParams p) {
  constexpr bool kLo = sizeof(T) == 4;
  constexpr uint32_t MR = kLo ? 128 : 256;
  // P is held times 2^kPShift, and the accumulator is left alone until a
  // maximum has grown by kLazy: their sum keeps P below 2^15
  constexpr float kPShift = kLo ? 15.f : 7.f, kLazy = kLo ? 0.f : 8.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) Bars bars;
  __shared__ Piece s_piece[kPieces];
  __shared__ uint32_t tmem_base, s_last;
  __shared__ float s_scl[kMaxRows];
  __shared__ float s_ml[2][2][128][2];
  __shared__ __align__(8) uint8_t s_bad[8][8];                 // 16-key tiles of a key tile that are not in the pool
  __shared__ __align__(8) uint32_t s_magic[4];
  // the shuffle makes the roles' branches uniform: the MMA warp's operands
  // stay in uniform registers
  const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  uint64_t *sums = reinterpret_cast<uint64_t *>(smem + kOffTab);
  uint32_t *lens = reinterpret_cast<uint32_t *>(sums + p.n_seq + 1), *nqs = lens + p.n_seq, *q0s = nqs + p.n_seq;

  // the few-rows kernel behind this one reads nothing that this one writes
  pdl_launch_dependents();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 32) {
    for (uint32_t i = 0; i < kPieces; ++i) {
      mbar_init(smem_addr(&bars.nfull[i]), 1);
      mbar_init(smem_addr(&bars.nempty[i]), kThreads / 32 - 1);
    }
    mbar_init(smem_addr(&bars.qfull), kQWarps + kConvWarps);
    mbar_init(smem_addr(&bars.qempty), 1 + kSoftWarps);     // the last S, and every reader of s_scl
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&bars.sfull[i]), 1);
      mbar_init(smem_addr(&bars.pfull[i]), kSoftWarps / 2);
      mbar_init(smem_addr(&bars.ofull[i]), 1);
      mbar_init(smem_addr(&bars.oempty[i]), kLo ? kSoftWarps : kSoftWarps / 2);
    }
    for (uint32_t i = 0; i < kRawStages; ++i) {
      for (uint32_t v = 0; v < 2; ++v) {
        mbar_init(smem_addr(&bars.rfull[v][i]), 1);
        mbar_init(smem_addr(&bars.rempty[v][i]), kConvWarps);
      }
    }
    for (uint32_t i = 0; i < kSlots; ++i) {
      mbar_init(smem_addr(&bars.full[i]), kConvWarps);
      mbar_init(smem_addr(&bars.empty[i]), 1);
    }
    mbar_init(smem_addr(&bars.join), kSoftWarps);
    mbar_init(smem_addr(&bars.drain), 1);
    fence_barrier_init();
  }
  // lengths, then the work of each sequence (a warp each), then its sums
  for (uint32_t i = tid; i < p.n_seq; i += kThreads) {
    bool bad = false;                     // recorded by the few-rows kernel
    const Kv4Seq s = kv4_seq(p, i, &bad);
    lens[i] = s.len;
    nqs[i] = s.nq * p.group > p.few_rows ? s.nq : 0u;
    q0s[i] = s.q0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  for (uint32_t i = warp; i < p.n_seq; i += kThreads / 32) {
    const uint32_t nq = nqs[i], n_rt = Walk<MR>::row_tiles(nq, p.group);
    uint64_t w = 0;
    for (uint32_t r = lane; r < n_rt; r += 32) w += Walk<MR>::units(lens[i], nq, p.group, r);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (lane == 0) sums[i + 1] = w * p.n_kv;
  }
  if (tid == 0) sums[0] = 0;
  __syncthreads();
  if (warp == 0) {
    uint64_t carry = 0;
    for (uint32_t i0 = 0; i0 < p.n_seq; i0 += 32) {
      uint64_t inc = i0 + lane < p.n_seq ? sums[i0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= static_cast<uint32_t>(o)) inc += u;
      }
      if (i0 + lane < p.n_seq) sums[i0 + lane + 1] = carry + inc;
      carry += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  __syncthreads();
  const uint32_t tmem = tmem_base;
  const uint64_t W = sums[p.n_seq];
  uint64_t G = (W + kMinTiles - 1) / kMinTiles;
  if (G > gridDim.x) G = gridDim.x;

  if (blockIdx.x < G) {
    // steps of a piece with key tiles 0 .. n - 1: stream t & 1, key tile kv_of(t)
    auto steps = [](uint32_t n) { return kLo ? n : 2 * n; };
    // The place of key tile j and of its values in the ring's order.  f32 rows
    // ask for K(t + 2) right behind PV(t): their keys come two tiles before
    // their values (K0 K1 V0 K2 V1 ..), or they would wait for PV(t)'s slot;
    // 16-bit rows' come in turn (K0 V0 K1 V1 ..).
    auto key_tile = [](uint32_t j) { return kLo ? (j < 2 ? j : 2 * j - 1) : 2 * j; };
    auto value_tile = [](uint32_t j) { return kLo ? 2 * j + 2 : 2 * j + 1; };
    bool ok = true;
    const uint32_t inv = 65536u / p.group + 1;
    // The range's next piece, for every warp but the loading one.
    uint32_t pieces = 0;
    Piece pc;
    auto next_piece = [&]() -> bool {
      const uint32_t slot = pieces % kPieces;
      ok = warp_wait(bars.nfull[slot], (pieces / kPieces) & 1, p.status);
      if (!ok) return false;
      ++pieces;
      pc = s_piece[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&bars.nempty[slot]));
      return pc.t1 != 0;
    };

    if (warp == kMmaWarp) {
      // ------------------------------------------------------- MMA issuer
      // The whole warp waits and counts; one elected lane issues.  The streams
      // wait on each other here, so the loop is kept short: places in the ring
      // are counted on, what a step needs is looked for at once, and PV and S go
      // out together.
      uint32_t item = 0, oc[2] = {0, 0}, p_parity[2] = {0, 0};
      // the next tile of keys and of values in the ring: place and phase
      uint32_t k_slot = 0, k_phase = 0, v_slot = kLo ? 2 : 1, v_phase = 0;
      bool first_key = kLo;
      auto two_on = [](uint32_t &slot, uint32_t &phase) {
        phase ^= slot != 0;
        slot = slot ? slot - 1 : 2;
      };
      static_assert(kSlots == 3, "two_on");
      // operand descriptors: 16 more per K step of 16 (two 128-byte chunks)
      const uint64_t q_desc = umma_desc(smem_addr(smem) + kOffQ, kLbo, kSbo);
      const uint64_t op_desc = umma_desc(smem_addr(smem) + kOffOp, kLbo, kSbo);
      while (ok && next_piece()) {
        const uint32_t n = pc.t1 - pc.t0, n_steps = steps(n);
        ok = warp_wait(bars.qfull, item & 1, p.status);
        // S(0), S(1), then PV(t - 2) and S(t)
        for (uint32_t t = 0; ok && t < n_steps + 2; ++t) {
          const uint32_t i = t & 1, d = tmem + kTmemO + 128 * i, sc = tmem + kTmemS + 128 * i;
          const bool pv = t >= 2, more = t < n_steps;     // PV(t - 2), S(t)
          if (pv && t < 4 && oc[i] > 0) ok = warp_wait(bars.oempty[i], (oc[i] - 1) & 1, p.status);
          // the next S's keys are looked for before P, so that S follows PV at once
          const uint32_t v_bar = smem_addr(&bars.full[v_slot]), k_bar = smem_addr(&bars.full[k_slot]);
          const uint32_t p_bar = smem_addr(&bars.pfull[i]), p_par = i ? p_parity[1] : p_parity[0];
          const bool v_there = !pv || mbar_try_wait(v_bar, v_phase), k_there = !more || mbar_try_wait(k_bar, k_phase);
          const bool p_there = !pv || mbar_try_wait(p_bar, p_par);
          if (!__all_sync(0xffffffffu, v_there && k_there && p_there))
            ok = ok && __all_sync(0xffffffffu, (!pv || slow_wait(v_bar, v_phase, p.status)) && (!more || slow_wait(k_bar, k_phase, p.status)) &&
                                                   (!pv || slow_wait(p_bar, p_par, p.status)));
          if (!ok) break;
          tc_fence_after();
          const uint64_t bv = op_desc + v_slot * (kOpBytes >> 4), bk = op_desc + k_slot * (kOpBytes >> 4);
          const uint64_t a0 = q_desc + (kLo ? 0 : i) * (kOpBytes >> 4);
          const bool last = kLo || i == 1;                // the last stream to read the tiles
          if (elect_one()) {
            if (pv) {
#pragma unroll
              for (uint32_t part = 0; part < (kLo ? 2u : 1u); ++part)
#pragma unroll
                for (uint32_t kk = 0; kk < 8; ++kk)
                  umma_f16_ts(d, sc + 32 * (kk / 2) + 8 * (kk & 1) + 16 * (kLo ? 1 - part : 0), bv + 16 * kk, kIdesc, t >= 4 || kk || part);
              if (!more) umma_commit(smem_addr(&bars.ofull[i]));
              if (last) umma_commit(v_bar - smem_addr(&bars.full[0]) + smem_addr(&bars.empty[0]));
            }
            if (more) {
#pragma unroll
              for (uint32_t part = 0; part < (kLo ? 2u : 1u); ++part)
#pragma unroll
                for (uint32_t kk = 0; kk < 8; ++kk)
                  umma_f16_ss(sc, a0 + (kLo ? 1 - part : 0) * (kOpBytes >> 4) + 16 * kk, bk + 16 * kk, kIdesc, part || kk);
              umma_commit(smem_addr(&bars.sfull[i]));
              if (last) umma_commit(k_bar - smem_addr(&bars.full[0]) + smem_addr(&bars.empty[0]));
              if (t + 1 == n_steps) umma_commit(smem_addr(&bars.qempty));
            }
          }
          __syncwarp();
          if (pv) {
            if (i) p_parity[1] ^= 1;
            else p_parity[0] ^= 1;
            if (last) two_on(v_slot, v_phase);
          }
          if (more && last) {
            if (first_key) k_slot = 1, first_key = false;   // K0 K1 V0 K2 ..
            else two_on(k_slot, k_phase);
          }
        }
        ++oc[0];
        if (n_steps > 1) ++oc[1];
        ++item;
      }
      // every MMA has completed before TMEM is freed
      if (elect_one()) umma_commit(smem_addr(&bars.drain));
      __syncwarp();
      wait(bars.drain, 0, p.status);
    } else if (warp == kLoadWarp) {
      // ------------------------------------------ the key tiles' 4-bit words
      // lane h < 8: keys 16 h .. of the tile, table entries a tile ahead
      const uint32_t tpb_log2 = p.bt_log2 - 4;
      uint32_t kc = 0, issued[2] = {0, 0};
      Walk<MR> walk;
      walk.sums = sums, walk.lens = lens, walk.nqs = nqs, walk.q0s = q0s;
      walk.n_kv = p.n_kv, walk.group = p.group;
      walk.at = W * blockIdx.x / G;
      walk.end = W * (blockIdx.x + 1) / G;
      walk.start(p.n_seq);
      for (bool more = true; ok && more; ++pieces) {
        const uint32_t piece_slot = pieces % kPieces;
        if (pieces >= kPieces) ok = warp_wait(bars.nempty[piece_slot], (pieces / kPieces - 1) & 1, p.status);
        if (!ok) break;
        more = walk.next();
        pc = walk.p;
        if (!more) pc.t0 = pc.t1 = 0;
        const uint64_t last = walk.first + pc.n;
        pc.c0 = static_cast<uint32_t>(((walk.first + 1) * G - 1) / W);
        pc.c1 = static_cast<uint32_t>((last * G - 1) / W);
        pc.tok0 = pc.rt * MR / p.group;
        pc.rem0 = pc.rt * MR - pc.tok0 * p.group;
        if (lane == 0) {
          s_piece[piece_slot] = pc;
          mbar_arrive(smem_addr(&bars.nfull[piece_slot]));
        }
        const uint32_t *table = p.table + static_cast<size_t>(pc.seq) * p.table_width;
        auto entry = [&](uint32_t t) -> uint32_t {
          const uint32_t tile = 8 * t + lane;
          return lane < 8 && t < pc.t1 && tile * kKv4Tile < pc.s.len ? __ldg(table + (tile >> tpb_log2)) : kKv4NoSlot;
        };
        uint32_t ent = entry(pc.t0);
        for (uint32_t t = pc.t0; t < pc.t1; ++t, ++kc) {
          const uint32_t stage = kc % kRawStages, tile = 8 * t + lane;
          const bool there = ent < p.n_blocks, bad = lane < 8 && !there && tile * kKv4Tile < pc.s.len;
          // keys that are not there are read from block 0, for the mask to drop
          const uint8_t *src = p.pool + (((static_cast<size_t>(there ? ent : 0u) * p.n_kv + pc.head) << tpb_log2) +
                                         (tile & ((1u << tpb_log2) - 1u))) * kKv4TileBytes;
          ent = entry(t + 1);
          if (lane < 8) s_bad[kc & 7][lane] = bad;
          if (bad) atomicOr(p.status, ZDEV_ERR_BOUNDS);
          __syncwarp();          // lane 0's arrival on rfull publishes what eight lanes stored
#pragma unroll 1
          for (uint32_t v = 0; ok && v < 2; ++v) {
            if (kc >= kRawStages) ok = warp_wait(bars.rempty[v][stage], (kc / kRawStages - 1) & 1, p.status);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(smem_addr(&bars.rfull[v][stage]), kRawBytes);
            __syncwarp();
            if (lane < 8)
              bulk_copy_g2s(smem_addr(smem) + kOffRaw + (v * kRawStages + stage) * kRawBytes + lane * kHalfBytes,
                            src + v * kHalfBytes, kHalfBytes, smem_addr(&bars.rfull[v][stage]));
            issued[v] = kc + 1;
          }
          if (!ok) break;
        }
      }
      // never leave a copy in flight when the CTA may exit
      for (uint32_t v = 0; v < 2; ++v)
        for (uint32_t x = issued[v] > kRawStages ? issued[v] - kRawStages : 0; x < issued[v]; ++x)
          wait(bars.rfull[v][x % kRawStages], (x / kRawStages) & 1, p.status);
    } else if (warp >= kQ0) {
      // -------------------------------------------------------- query rows
      uint32_t item = 0;
      while (ok && next_piece()) {
        // the rows on their way to L2 while the last piece's are in their place:
        // a lane a row and 128 bytes
        for (uint32_t x = 32 * (warp - kQ0) + lane; x < MR * (kLo ? 4u : 2u); x += 32 * kQWarps) {
          const uint32_t r = x / (kLo ? 4u : 2u), part = x % (kLo ? 4u : 2u);
          uint32_t tok, hd;
          pc.place(r, p.group, inv, &tok, &hd);
          if (pc.rt * MR + r < pc.s.nq * p.group)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(
                reinterpret_cast<const uint8_t *>(static_cast<const T *>(p.q) + (pc.s.q0 + static_cast<uint64_t>(tok)) * p.q_stride +
                                                  (static_cast<size_t>(pc.head) * p.group + hd) * kKv4Head) + 128 * part));
        }
        ok = item == 0 || warp_wait(bars.qempty, (item - 1) & 1, p.status);
        if (ok) load_queries<T>(p, pc, smem + kOffQ, s_scl, inv, warp - kQ0);
        if (ok && lane == 0) mbar_arrive(smem_addr(&bars.qfull));
        ++item;
      }
    } else if (warp >= kConv0) {
      // --------------------------------------- keys and values to binary16
      const uint32_t cw = warp - kConv0, r = lane >> 2, c = lane & 3, kr = lane & 7, kq = lane >> 3;
      const Magic mg = magic(smem_addr(s_magic));
      const KMagic kg = k_magic(smem_addr(s_magic + 2));
      // operand tile x may be written once the MMAs that read tile x - 3 are done
      auto slot_free = [&](uint32_t x) { return x < kSlots || warp_wait(bars.empty[x % kSlots], (x / kSlots - 1) & 1, p.status); };
      auto hand_over = [&](uint32_t x) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&bars.full[x % kSlots]));
      };
      // this warp's sixteen keys of each half of tile j: 16 (4 h + cw) ..
      auto raw_ready = [&](uint32_t v, uint32_t j) { return warp_wait(bars.rfull[v][j % kRawStages], (j / kRawStages) & 1, p.status); };
      auto raw_of = [&](uint32_t v, uint32_t j) {
        return smem + kOffRaw + (v * kRawStages + j % kRawStages) * kRawBytes + cw * kHalfBytes;
      };
      auto raw_done = [&](uint32_t v, uint32_t j) {
        if (lane == 0) mbar_arrive(smem_addr(&bars.rempty[v][j % kRawStages]));
      };
      auto keys = [&](uint32_t j) -> bool {
        const uint32_t x = key_tile(j);
        if (!raw_ready(0, j) || !slot_free(x)) return false;
        // row = key 64 h + 16 cw + 8 u + kr, chunk 4 g + kq
        uint8_t *kd = smem + kOffOp + (x % kSlots) * kOpBytes + kSbo * (2 * cw) + 16 * kr + kLbo * kq;
#pragma unroll 2
        for (int hu = 0; hu < 4; ++hu) {
          const int h = hu >> 1, u = hu & 1;
          const uint8_t *src = raw_of(0, j) + 4 * h * kHalfBytes;
          const uint4 kw = *reinterpret_cast<const uint4 *>(src + 512 * u + 64 * kr + 16 * kq);
          const uint4 ks = *reinterpret_cast<const uint4 *>(src + kKv4Ks + 64 * u + 16 * (kr >> 1));
          const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w}, s4[4] = {ks.x, ks.y, ks.z, ks.w};
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const __half2 dd = bits2h(s4[g]);
            const __half2 d = kr & 1 ? __high2half2(dd) : __low2half2(dd);
            uint32_t v[4];
            k_values(w[g], d, kg, v);
            *reinterpret_cast<uint4 *>(kd + kSbo * (8 * h + u) + kLbo * 4 * g) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        hand_over(x);
        raw_done(0, j);
        return true;
      };
      // transposed: row = dim 32 g + 8 s + r, keys 64 h + 16 cw + 8 u + 2 c and + 1
      auto values = [&](uint32_t j) -> bool {
        const uint32_t x = value_tile(j);
        if (!raw_ready(1, j) || !slot_free(x)) return false;
        uint8_t *vd = smem + kOffOp + (x % kSlots) * kOpBytes + kLbo * (2 * cw) + 16 * r + 4 * c;
#pragma unroll 2
        for (int hu = 0; hu < 4; ++hu) {
          const int h = hu >> 1, u = hu & 1;
          const uint8_t *src = raw_of(1, j) + 4 * h * kHalfBytes;
          const uint4 vw = *reinterpret_cast<const uint4 *>(src + 512 * u + 16 * lane);
          const uint4 vs = *reinterpret_cast<const uint4 *>(src + (kKv4Vs - kKv4V) + 64 * u + 16 * c);
          const uint32_t w[4] = {vw.x, vw.y, vw.z, vw.w}, s4[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const __half2 d = bits2h(s4[g]);
            uint32_t v[4];
            v_values(w[g], d, __hmul2(d, __float2half2_rn(-24.f)), mg, v);
#pragma unroll
            for (int s2 = 0; s2 < 4; ++s2)
              *reinterpret_cast<uint32_t *>(vd + kLbo * (8 * h + u) + kSbo * (4 * g + s2)) = v[s2];
          }
        }
        hand_over(x);
        raw_done(1, j);
        return true;
      };
      uint32_t kc = 0, item = 0;
      while (ok && next_piece()) {
        const uint32_t n = pc.t1 - pc.t0;
        for (uint32_t t = 0; ok && t < n; ++t, ++kc) {
          ok = keys(kc);
          if (ok && (!kLo || kc > 0) && !(!kLo && t == 0)) ok = values(kLo ? kc - 1 : kc);
          // the piece's first keys are on their way while the queries' place
          // is still taken; then this warp's share of the rows
          if (ok && t == 0) {
            ok = item == 0 || warp_wait(bars.qempty, (item - 1) & 1, p.status);
            if (!ok) break;
            load_queries<T>(p, pc, smem + kOffQ, s_scl, inv, kQWarps + cw);
            if (lane == 0) mbar_arrive(smem_addr(&bars.qfull));
            ++item;
            if (!kLo) ok = values(kc);
          }
        }
      }
      if (ok && kLo && kc > 0) values(kc - 1);
    } else {
      // ------------------------------------------------------------ softmax
      const uint32_t i = warp >> 2, row = 32 * (warp & 3) + lane;     // stream, row of the stream
      const uint32_t lane_base = tmem + ((32u * (warp & 3)) << 16);
      const uint32_t s_col = lane_base + kTmemS + 128 * i, o_col = lane_base + kTmemO;
      uint32_t item = 0, kc0 = 0, ns = 0, oc[2] = {0, 0}, joins = 0;
      const bool sectors = ((reinterpret_cast<uintptr_t>(p.out) | p.out_stride * sizeof(T)) & 31u) == 0;
      // all softmax warps, with a bounded wait
      auto join = [&]() -> bool {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&bars.join));
        return warp_wait(bars.join, joins++ & 1, p.status);
      };
      while (ok && next_piece()) {
        const uint32_t n = pc.t1 - pc.t0, n_steps = steps(n), trow = kLo ? row : 128 * i + row;
        const uint32_t grow = pc.rt * MR + trow, n_rows = pc.s.nq * p.group;
        uint32_t tok, hd;
        pc.place(trow, p.group, inv, &tok, &hd);
        // keys that the row sees; a row behind the last is for no use
        const int64_t pos1 = static_cast<int64_t>(pc.s.len) - pc.s.nq + tok + 1;
        const uint32_t limit = grow >= n_rows ? pc.s.len : pos1 > 0 ? static_cast<uint32_t>(pos1) : 0u;
        uint32_t all_see = limit;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, o));
        ok = warp_wait(bars.qfull, item & 1, p.status);
        if (!ok) break;
        const float scl = s_scl[trow];
        // the next piece's queries wait for this: a piece of one key tile
        // would otherwise let them run two phases of qfull ahead
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&bars.qempty));
        float m = -INFINITY;
        float2 l[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        for (uint32_t t = i; ok && t < n_steps; t += 2) {
          const uint32_t kv = kLo ? t : t >> 1, key0 = (pc.t0 + kv) * kKeys;
          ok = warp_wait(bars.sfull[i], ns & 1, p.status);
          ++ns;
          if (!ok) break;
          tc_fence_after();
          const uint2 bad8 = *reinterpret_cast<const uint2 *>(s_bad[(kc0 + kv) & 7]);
          // a key that the row does not see is -inf; written back, so that the
          // second pass need not ask
          if (key0 + kKeys > all_see || (bad8.x | bad8.y)) {
            const uint64_t bad = bad8.x | static_cast<uint64_t>(bad8.y) << 32;
#pragma unroll 1
            for (uint32_t q = 0; q < 4; ++q) {
              const uint32_t k0 = key0 + 32 * q, see = limit > k0 ? limit - k0 : 0u;
              const bool bad0 = (bad >> (16 * q)) & 1u, bad1 = (bad >> (16 * q + 8)) & 1u;
              uint32_t v[32];
              tmem_ld32(s_col + 32 * q, v);
              tmem_ld_wait32(v);
#pragma unroll
              for (uint32_t x = 0; x < 32; ++x)
                if (x >= see || (x < 16 ? bad0 : bad1)) v[x] = 0xFF800000u;
              tmem_st32(s_col + 32 * q, v);
            }
            tmem_st_wait();
          }
          // the largest score, in four chains of maxima
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          uint32_t va[32];
#pragma unroll 1
          for (uint32_t q = 0; q < 4; ++q) {
            tmem_ld32(s_col + 32 * q, va);
            tmem_ld_wait32(va);
#pragma unroll
            for (int x = 0; x < 32; x += 2)
              mx4[(x >> 1) & 3] = fmaxf(fmaxf(mx4[(x >> 1) & 3], __uint_as_float(va[x])), __uint_as_float(va[x + 1]));
          }
          // P is 2^(score - m) with m the largest score less kPShift, rounded up:
          // rounded otherwise, P could pass binary16's range for scores from 2^24
          const float mx = __fmaf_ru(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), scl, -kPShift);
          if (t < 2) {
            m = mx;
          } else if (__any_sync(0xffffffffu, mx > m + kLazy)) {
            // S(t) was issued after PV(t - 2): the accumulator is at rest
            const float nm = mx > m + kLazy ? mx : m, f = nm == m ? 1.f : ex2(m - nm);
            const float2 ff = make_float2(f, f);
            l[0] = mul2_rn(l[0], ff), l[1] = mul2_rn(l[1], ff);
            m = nm;
#pragma unroll 1
            for (uint32_t q = 0; q < 4; ++q) {
              tmem_ld32(o_col + 128 * i + 32 * q, va);
              tmem_ld_wait32(va);
#pragma unroll
              for (int x = 0; x < 32; ++x) va[x] = __float_as_uint(__uint_as_float(va[x]) * f);
              tmem_st32(o_col + 128 * i + 32 * q, va);
            }
          }
          const float sub = m == -INFINITY ? 0.f : -m;
          const float2 scl2 = make_float2(scl, scl), sub2 = make_float2(sub, sub);
          // 32 scores to P in their own columns: 16 of hi, 16 of lo
          auto probs = [&](uint32_t q, const uint32_t (&va)[32]) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const float2 y = fma2_rn(make_float2(__uint_as_float(va[2 * x]), __uint_as_float(va[2 * x + 1])), scl2, sub2);
              const float2 e = make_float2(ex2(y.x), ex2(y.y));
              l[x & 1] = add2_rn(l[x & 1], e);
              const __half2 h = __floats2half2_rn(e.x, e.y);
              hi[x] = h2bits(h);
              if (kLo) {
                const float2 d = sub2_rn(e, __half22float2(h));
                lo[x] = h2bits(__floats2half2_rn(d.x, d.y));
              }
            }
            tmem_st16(s_col + 32 * q, hi);
            if (kLo) tmem_st16(s_col + 32 * q + 16, lo);
          };
          tmem_ld32(s_col, va);
          if (kLo) {
#pragma unroll 1
            for (uint32_t q = 0; q < 4; ++q) {
              tmem_ld_wait32(va);
              probs(q, va);
              if (q < 3) tmem_ld32(s_col + 32 * q + 32, va);
            }
          } else {      // the next scores on their way
            uint32_t vb[32];
#pragma unroll 1
            for (uint32_t q = 0; q < 4; q += 2) {
              tmem_ld_wait32(va);
              tmem_ld32(s_col + 32 * q + 32, vb);
              probs(q, va);
              tmem_ld_wait32(vb);
              if (q == 0) tmem_ld32(s_col + 64, va);
              probs(q + 1, vb);
            }
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&bars.pfull[i]));
        }
        // ------------------------------------------ the piece's accumulator
        const bool use1 = n_steps > 1;
        if (ok && (kLo || i == 0)) ok = warp_wait(bars.ofull[0], oc[0] & 1, p.status);
        if (ok && (kLo ? use1 : i == 1)) ok = warp_wait(bars.ofull[1], oc[1] & 1, p.status);
        ++oc[0];
        if (use1) ++oc[1];
        if (!ok) break;
        tc_fence_after();
        float M = m, L = (l[0].x + l[0].y) + (l[1].x + l[1].y), w0 = 1.f, w1 = 0.f;
        if (kLo) {
          // the streams' states of a row: both halves of the warps need both
          float(*ml)[128][2] = s_ml[item & 1];
          ml[i][row][0] = M;
          ml[i][row][1] = L;
          if (!(ok = join())) break;
          const float m0 = ml[0][row][0], m1 = ml[1][row][0];
          M = fmaxf(m0, m1);
          w0 = m0 == M ? 1.f : ex2(m0 - M);
          w1 = m1 == M ? 1.f : ex2(m1 - M);
          L = ml[0][row][1] * w0 + ml[1][row][1] * w1;
        }
        const bool whole = pc.t0 == 0 && pc.t1 == pc.n;
        const bool blind = limit == 0 || grow >= n_rows;
        const float share = whole ? 1.f / L : 1.f;
        if (whole && !blind && !(M == -INFINITY && L == 0.f) && !(L > 0.f && L < INFINITY && fabsf(M) < INFINITY))
          atomicOr(p.status, ZDEV_ERR_NUMERICAL);
        T *orow = static_cast<T *>(p.out) + (pc.s.q0 + static_cast<uint64_t>(tok)) * p.out_stride +
                  (static_cast<size_t>(pc.head) * p.group + hd) * kKv4Head;
        const bool none = M == -INFINITY && L == 0.f;
        float *part = p.part + (2ull * blockIdx.x + (pc.t0 == 0 ? 1 : 0)) * kPartFloats;
        // 32 dims at a time: f32 rows share the row's dims between the streams' warps
        const uint32_t q0 = kLo ? 2 * i : 0, q1 = kLo ? 2 * i + 2 : 4;
        uint32_t v[32];
        tmem_ld32(o_col + (kLo ? 0 : 128 * i) + 32 * q0, v);
#pragma unroll 1
        for (uint32_t q = q0; q < q1; ++q) {
          tmem_ld_wait32(v);
          float o[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = __uint_as_float(v[x]) * w0;
          if (kLo && use1) {
            tmem_ld32(o_col + 128 + 32 * q, v);
            tmem_ld_wait32(v);
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = fmaf(__uint_as_float(v[x]), w1, o[x]);
          }
          if (q + 1 < q1) tmem_ld32(o_col + (kLo ? 0 : 128 * i) + 32 * (q + 1), v);
          if (whole) {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = none ? 0.f : o[x] * share;
            if (!blind) put32(orow + 32 * q, o, sectors);
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x)
              *reinterpret_cast<float4 *>(part + 4 * ((8 * q + x) * MR + trow)) =
                  make_float4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (kLo) {
            mbar_arrive(smem_addr(&bars.oempty[0]));
            if (use1) mbar_arrive(smem_addr(&bars.oempty[1]));
          } else {
            mbar_arrive(smem_addr(&bars.oempty[i]));
          }
        }
        if (!whole) {
          if (!kLo || i == 0) *reinterpret_cast<float2 *>(part + MR * kKv4Head + 2 * trow) = make_float2(M, L);
          __threadfence();
          if (!(ok = join())) break;
          // the ranges that share the piece
          const uint32_t c0 = pc.c0, c1 = pc.c1;
          if (tid == 0) {
            s_last = atomicAdd(&p.counters[c0], 1u) == c1 - c0;
            if (s_last) p.counters[c0] = 0;
          }
          if (!(ok = join())) break;
          if (s_last) {
            __threadfence();
            auto from = [&](uint32_t k) { return p.part + (2ull * k + (k == c0 ? 1 : 0)) * kPartFloats; };
            M = -INFINITY;
            L = 0.f;
            for (uint32_t k = c0; k <= c1; ++k) {
              const float2 x = __ldcg(reinterpret_cast<const float2 *>(from(k) + MR * kKv4Head + 2 * trow));
              if (x.x == -INFINITY && x.y == 0.f) continue;
              const float nm = fmaxf(M, x.x);
              L = (M == nm ? L : L * ex2(M - nm)) + (x.x == nm ? x.y : x.y * ex2(x.x - nm));
              M = nm;
            }
            const bool empty = M == -INFINITY && L == 0.f;
            if (!blind && !empty && !(L > 0.f && L < INFINITY && fabsf(M) < INFINITY)) atomicOr(p.status, ZDEV_ERR_NUMERICAL);
            const float li = empty ? 0.f : 1.f / L;
#pragma unroll 1
            for (uint32_t d0 = kLo ? 16 * i : 0; d0 < (kLo ? 16 * i + 16 : 32u); d0 += 8) {
              float4 a[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) a[x] = make_float4(0.f, 0.f, 0.f, 0.f);
              for (uint32_t k = c0; k <= c1; ++k) {
                const float *src = from(k);
                const float2 st = __ldcg(reinterpret_cast<const float2 *>(src + MR * kKv4Head + 2 * trow));
                const float w = st.x == -INFINITY && st.y == 0.f ? 0.f : st.x == M ? 1.f : ex2(st.x - M);
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                  const float4 y = __ldcg(reinterpret_cast<const float4 *>(src + 4 * ((d0 + x) * MR + trow)));
                  a[x].x += y.x * w, a[x].y += y.y * w, a[x].z += y.z * w, a[x].w += y.w * w;
                }
              }
              if (!blind)
#pragma unroll
                for (int x = 0; x < 8; ++x)
                  put4(orow + 4 * (d0 + x), make_float4(a[x].x * li, a[x].y * li, a[x].z * li, a[x].w * li));
            }
          }
          if (!(ok = join())) break;      // s_last is free again
        }
        kc0 += n;
        ++item;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

template <class T>
cudaError_t launch(const Kv4AttnParams &p, int sm_count, cudaStream_t s) {
  const uint32_t smem = kOffTab + (p.n_seq + 1) * 8 + p.n_seq * 12;
  kv4_prompt_kernel<T><<<sm_count, kThreads, smem, s>>>(p);
  return cudaGetLastError();
}
template <class T>
cudaError_t setup() {
  return cudaFuncSetAttribute(kv4_prompt_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              kOffTab + (kKv4MaxSeqs + 1) * 8 + kKv4MaxSeqs * 12);
}

}  // namespace

size_t kv4_prompt_part_bytes(int sm_count) { return static_cast<size_t>(sm_count) * 2 * kPartFloats * sizeof(float); }
uint32_t kv4_prompt_counters(int sm_count) { return static_cast<uint32_t>(sm_count); }

cudaError_t kv4_prompt_setup() {
  cudaError_t e = setup<float>();
  if (e == cudaSuccess) e = setup<__half>();
  if (e == cudaSuccess) e = setup<__nv_bfloat16>();
  return e;
}

cudaError_t launch_kv4_prompt(const Kv4AttnParams &p, Kv4Type t, int sm_count, cudaStream_t s) {
  if (t == KV4_F32) return launch<float>(p, sm_count, s);
  if (t == KV4_F16) return launch<__half>(p, sm_count, s);
  return launch<__nv_bfloat16>(p, sm_count, s);
}

}  // namespace zgpu
