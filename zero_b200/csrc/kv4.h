// kv4.h — the paged 4-bit KV cache: layout, parameter blocks and launchers.
//
// A cache is a pool of n_blocks blocks of block_tokens (16, 32, 64 or 128)
// token slots per layer.  A token's K or V row of one kv head is four groups
// of 32 values; a group is a signed scale d and integers q in -8..7 and
// stands for q * d.  With m the group's value of largest magnitude (the first
// of equals), d = binary16(bfloat16(-m / 8)) and q is the integer nearest to
// x / d, ties to even, clamped.  d has at most 8 significant bits and q at
// most 3, so q * d has at most 11 and is exact in binary16: the attention
// kernels feed the tensor cores the cache's values without a rounding.
//
// Why 8 bits of scale: binary16's own 11 would make q * d a 14-bit product
// that the 16-bit operands round, and the rounding of d costs next to nothing,
// since q is chosen against the d that is stored: normal rows are 8.596 % off
// (root mean square) with 8 bits of d, with 11 and with 24, and 8.602 % with 6.
//
// Storage is by tiles of 16 tokens of one kv head, 2304 contiguous bytes (one
// bulk copy, or one for each half): K nibbles (1024), K scales (128), V nibbles
// (1024), V scales (128), with n = q + 8 as the nibble.
//   K: token t's row is bytes 64 t..; word g of column c (bytes 64 t + 16 c +
//      4 g) holds dims 32 g + 8 c + 0..7, even dims in its low half and odd
//      dims in its high half, bits 4 s of a half being dim pair 2 s.
//   V: half p = t / 8, column c = (t % 8) / 2, odd = t % 2; the 16 bits at
//      512 p + 16 (4 r + c) + 4 g + 2 odd of its half hold dims 32 g + 8 s + r, s = 0..3:
//      s = 0 at bits 6..9, 1 at 2..5, 2 at 10..13, 3 at 14, 15, 0, 1 (after a
//      swap of the two bytes, 2 is at 2..5 and 3 at 6..9).
//   Scales of K and of V: half index 2 (16 p + 4 c + g) + odd.
// These are the m16n8k16 B fragments: lane (r, c) = (lane / 4, lane % 4) of a
// warp reads its K words of 8 tokens, or its V words of 16, with one 16-byte
// shared-memory load per 512 bytes.  Every byte belongs to one token, so
// tokens are stored without touching their neighbours.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "internal.h"

namespace zgpu {

constexpr uint32_t kKv4Head = 128;          // head_dim
constexpr uint32_t kKv4Tile = 16;           // tokens per tile
constexpr uint32_t kKv4TileBytes = 2304;
constexpr uint32_t kKv4Ks = 1024, kKv4V = 1152, kKv4Vs = 2176;   // offsets in a tile
constexpr uint32_t kKv4MaxSeqs = 1024;
constexpr uint32_t kKv4NoSlot = 0xFFFFFFFFu;
// The largest scale: 24 d has to be finite in binary16 (the dequantising fma
// subtracts it), so the cache holds magnitudes up to 8 * 2720.
constexpr float kKv4MaxScale = 2720.f;

// Byte offset of the tile that holds slot `slot` of kv head `head`, from the
// layer's first byte.  bt_log2 = log2(block_tokens).
__host__ __device__ inline size_t kv4_tile_off(uint32_t slot, uint32_t head, uint32_t n_kv, uint32_t bt_log2) {
  const uint32_t block = slot >> bt_log2, tile = (slot & ((1u << bt_log2) - 1u)) / kKv4Tile;
  return (((static_cast<size_t>(block) * n_kv + head) << (bt_log2 - 4)) + tile) * kKv4TileBytes;
}

// The nibbles s of a token's 16 bits of V, at bits 4 s.
__host__ __device__ inline uint32_t kv4_v_nibbles(uint32_t v) {
  return ((v >> 6) & 15u) | ((v >> 2) & 15u) << 4 | ((v >> 10) & 15u) << 8 | ((v >> 14) | (v & 3u) << 2) << 12;
}

// A bit of the cache's status word beside those of common.cuh: a plan or
// release that was refused.
enum : uint32_t { ZDEV_ERR_POOL = 1u << 5 };

// Element types of rows given to append / gather / attention.
enum Kv4Type { KV4_F32 = 0, KV4_F16 = 1, KV4_BF16 = 2 };

struct Kv4PlanParams {
  const uint32_t *old_lens, *new_lens, *table_in, *free_list, *state_in;
  uint32_t *table_out, *state_out, *slots, *starts, *kv_lens;
  uint32_t n_seq, table_width, n_slots, n_blocks, bt_log2;
  uint32_t *status;
};
cudaError_t launch_kv4_plan(const Kv4PlanParams &p, int sm_count, cudaStream_t s);

struct Kv4ReleaseParams {
  const uint32_t *done;
  uint32_t *lens, *table, *free_list, *state;
  uint32_t n_seq, table_width, n_blocks, bt_log2;
  uint32_t *status;
};
cudaError_t launch_kv4_release(const Kv4ReleaseParams &p, cudaStream_t s);

struct Kv4RowsParams {
  uint8_t *pool;              // the layer's first byte
  const uint32_t *slots;
  const void *k, *v;          // append: rows in
  void *k_out, *v_out;        // gather: rows out (either may be null)
  uint64_t k_stride, v_stride;   // elements between tokens
  uint32_t n_tokens, n_kv, n_slots, bt_log2;
  uint32_t *status;
};
cudaError_t launch_kv4_append(const Kv4RowsParams &p, Kv4Type t, int sm_count, cudaStream_t s);
cudaError_t launch_kv4_gather(const Kv4RowsParams &p, Kv4Type t, int sm_count, cudaStream_t s);

struct Kv4AttnParams {
  const uint8_t *pool;        // the layer's first byte
  const void *q;
  void *out;
  uint64_t q_stride, out_stride;
  const uint32_t *starts, *kv_lens, *table;
  uint32_t table_width, n_seq, n_rows, max_q, n_kv, group, n_blocks, bt_log2;
  float scale;
  float *part;                // partial slots of the launch's CTAs
  uint32_t *counters;         // zero between calls
  uint32_t few_rows;          // sequences of more rows per kv head go to kv4_prompt.cu
  uint32_t *status;
};
// Bytes of the partials and the number of counters a workspace needs.
size_t kv4_attn_part_bytes(int sm_count);
uint32_t kv4_attn_counters(int sm_count);
cudaError_t kv4_attn_setup();
cudaError_t launch_kv4_attention(const Kv4AttnParams &p, Kv4Type t, int sm_count, uint32_t *launches, cudaStream_t s);
// The part of it for sequences with many query rows (kv4_prompt.cu).
size_t kv4_prompt_part_bytes(int sm_count);
uint32_t kv4_prompt_counters(int sm_count);
cudaError_t kv4_prompt_setup();
cudaError_t launch_kv4_prompt(const Kv4AttnParams &p, Kv4Type t, int sm_count, cudaStream_t s);

}  // namespace zgpu

struct zgpu_kv4 {
  zgpu_ctx *ctx = nullptr;
  int device = 0, sm_count = 0;
  uint8_t *d = nullptr;
  uint32_t *d_status = nullptr;   // kStatusWords words of this cache
  uint32_t n_blocks = 0, block_tokens = 0, bt_log2 = 0, n_layers = 0, n_kv = 0;
  size_t layer_bytes = 0;
};

struct zgpu_kv4_work {
  zgpu_ctx *ctx = nullptr;
  int device = 0;
  float *part = nullptr;
  uint32_t *counters = nullptr;
};
