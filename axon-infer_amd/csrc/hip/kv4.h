// The 4-bit KV cache: its layout, and the launchers of the kernels that write it (kv4.hip), read it back
// and attend over it (attention_kv4.hip).
//
// A block is 32 consecutive values of one head of one position. It holds one fp16 scale d and 32 codes
// c in 0..15, code c standing for d * (c - 8). A layer of one sequence is n_kv head regions, a region
// ceil(max_ctx / 32) tiles of 32 positions, and a tile of NB = head_dim / 32 blocks a position is
//   key codes     16 * head_dim bytes
//   value codes   16 * head_dim bytes
//   key scales     2 * head_dim bytes
//   value scales   2 * head_dim bytes
// ordered inside as the lanes of a wave take them into v_mfma_f32_16x16x32_f16 operands (lane
// 16 g + i), so that a lane's share of a tile is one run of bytes and the wave's loads are whole lines:
//   keys    position 16 s + i, values 32 b + 8 g + t (t 0..7) of every block: dword [g][i][s][b], value t
//           in nibble t / 2 + 4 (t mod 2) (nibbles 0 and 4 of a dword mask out as the two halves of a
//           register at once, and so on);
//   values  positions 16 s + 4 g + r as byte e = 4 s + r, values 32 b + i (low nibble) and 32 b + 16 + i:
//           byte [g][i][b][e]. A lane of the scores' product holds positions 16 s + 4 g + r of its
//           column, so the probabilities enter the second product without crossing lanes;
//   scales  position 16 s + 4 g + r: half [g][s][b][r], for keys and values alike.
// No byte is shared by two positions: rows are written without reading what is there.
#pragma once

#include "elementwise.h"

#include <cstddef>
#include <cstdint>

namespace axon_hip {

constexpr uint32_t kKv4Tile = 32;  // positions per tile
constexpr size_t kKv4MaxCtx = size_t{1} << 24;  // positions, which floats count exactly

// Bytes of one tile: 32 positions of one head, keys and values.
constexpr uint32_t kv4_tile_bytes(uint32_t head_dim) { return 36 * head_dim; }
constexpr uint32_t kv4_tiles(uint32_t positions) { return (positions + kKv4Tile - 1) / kKv4Tile; }
// The head sizes of the kernels.
constexpr bool kv4_head_dim_ok(size_t head_dim) {
  return head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 192 || head_dim == 256;
}

// Byte offsets inside a tile. p: the position within the tile, b: the block of the head, g8: which
// eighth-row of eight values (value index within the block / 8).
constexpr uint32_t kv4_key_dword(uint32_t nb, uint32_t p, uint32_t b, uint32_t g8) {
  return 4 * (((g8 * 16 + p % 16) * 2 + p / 16) * nb + b);
}
constexpr uint32_t kv4_value_byte(uint32_t nb, uint32_t p, uint32_t b, uint32_t i) {
  return 16 * 32 * nb + ((p % 16 / 4 * 16 + i) * nb + b) * 8 + p / 16 * 4 + p % 4;
}
constexpr uint32_t kv4_scale_half(uint32_t nb, uint32_t p, uint32_t b) {
  return ((p % 16 / 4 * 2 + p / 16) * nb + b) * 4 + p % 4;
}

// What a launch can take: fewer than 2^32 threads along x, 65535 workgroups along y.
inline int launch_fits(const char* what, size_t x, size_t threads, size_t y) {
  if (x > 0xffffffffu / threads || y > 65535) return fail(kInvalidArgument, "%s: %zu by %zu workgroups of %zu threads", what, x, y, threads);
  return kOk;
}

// Rotates (rope_rows' arithmetic) and quantizes new rows into a 4-bit cache: a.cache_off and
// a.k_layer_off in bytes.
int rope_rows_kv4_launch(const RopeRowsArgs& a, uint32_t max_ctx, uint32_t n_rows);
int rope_rows_kv4_check_size(const RopeRowsArgs& a, size_t n_rows);

struct Kv4ReadArgs {
  const void* cache;
  const int64_t* cache_off;  // per-row byte offset of the row's sequence, or null
  int64_t layer_off;         // bytes
  const int32_t* pos;        // per row, or null for pos0 + row
  int32_t pos0;
  uint32_t n_kv, head_dim, max_ctx;
  float* k;                  // [rows][stride], or null
  float* v;
  uint32_t stride;
};
int kv4_read_launch(const Kv4ReadArgs& a, uint32_t n_rows);
int kv4_read_check_size(const Kv4ReadArgs& a, size_t n_rows);

struct AttnKv4Args {
  const float* q;
  float* out;
  uint32_t q_stride, out_stride;
  const void* cache;
  const int64_t* cache_off;  // per-row byte offsets, or null
  const int32_t* n_vis;      // per row, or null for n_past + row + 1
  int64_t layer_off;
  int32_t n_past;
  uint32_t n_head, n_kv, head_dim;
  uint32_t max_ctx, max_vis;
  float scale;
  uint32_t chunk_rows;       // the first rows belong to one sequence
  float* scratch;
  void* outq;                // Q8_0 blocks [rows][n_head * head_dim / 32], or null
};
int attention_kv4_launch(const AttnKv4Args& a, uint32_t n_rows);
int attention_kv4_check_size(const AttnKv4Args& a, uint32_t n_rows);
size_t attention_kv4_scratch_floats(const AttnKv4Args& a, uint32_t n_rows);

}  // namespace axon_hip
