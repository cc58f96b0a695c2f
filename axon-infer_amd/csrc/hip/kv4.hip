// Rows into and out of the 4-bit KV cache (layout: kv4.h).
//
// A block x[0..31] is held as d = fp16(m / -8), m its value of largest magnitude (the first of equal
// ones; the quotient within fp16's finite range), and the codes c = floor(x / d + 8.5) within 0..15 in
// exact arithmetic: the nearest level, the higher code between two. d = 0 (every value below half of
// fp16's smallest) holds zeros. A block with an infinity or a NaN is held as a NaN scale, so that what
// reads it reads NaN, as it would from a float cache.
//
// The code is found in 32 bits and then set right: x / d can round across a border, but the border
// (c - 8.5) * d is a product of a 5-bit and an 11-bit number, which 32 bits hold exactly, and so is its
// comparison with x.
//
// One half-wave per block, one value per lane; each lane turns its own value of a rotary pair, reading
// its partner too (from cache lines the wave holds anyway), which spares the barrier between rotation
// and quantization. One row (8 KV heads of 64) takes 2.8 us, the launch; 33 rows (2 heads) 3.4; 512 rows (8 heads)
// 5.0 to 5.3, where their 2.4 MB ask for 0.5: a position's codes are single bytes and dwords over its tile, so a line is
// written by the workgroups of 8 or more positions. Reading 512 positions back takes 3.0 to 3.3 us.
#include "common.h"
#include "kv4.h"

namespace axon_hip {

namespace {

// The row's cos and sin of pair i.
__device__ __forceinline__ float2 kv4_angle(const RopeRowsArgs& a, int32_t pos, uint32_t i) {
  const uint32_t half = a.rotary_dim / 2;
  if (a.table != nullptr) return reinterpret_cast<const float2*>(a.table)[static_cast<size_t>(pos) * half + i];
  double inv_freq = pow(static_cast<double>(a.theta), -static_cast<double>(2 * i) / static_cast<double>(a.rotary_dim));
  if (a.freq_factors != nullptr) inv_freq /= static_cast<double>(a.freq_factors[i]);
  const double angle = static_cast<double>(pos) * inv_freq;
  return make_float2(static_cast<float>(cos(angle)), static_cast<float>(sin(angle)));
}

// Pair i of a head: the indexes of its two values.
__device__ __forceinline__ void kv4_pair(const RopeRowsArgs& a, uint32_t i, uint32_t& ia, uint32_t& ib) {
  ia = a.neox ? i : 2 * i;
  ib = a.neox ? i + a.rotary_dim / 2 : 2 * i + 1;
}

// floor(x / d + 8.5) within 0..15, exactly. d finite and not 0, x finite.
__device__ __forceinline__ uint32_t kv4_code(float x, float d) {
  int c = static_cast<int>(fminf(fmaxf(floorf(x / d + 8.5f), 0.0f), 15.0f));
  // Code c begins at (c - 8.5) * d; both products are exact. With d below zero the order turns around.
  const float lo = (static_cast<float>(c) - 8.5f) * d;
  const float hi = (static_cast<float>(c) - 7.5f) * d;
  if (d > 0.0f ? x < lo : x > lo) --c;
  else if (d > 0.0f ? x >= hi : x <= hi) ++c;
  return static_cast<uint32_t>(min(max(c, 0), 15));
}

// grid (rows, groups of 8 blocks): blocks 0 .. n_kv * NB - 1 of a row are its keys, as many of values
// follow, and then, 256 pairs a workgroup, the query's pairs are turned in place.
__global__ __launch_bounds__(256) void rope_rows_kv4_kernel(RopeRowsArgs a, uint32_t max_ctx, uint32_t store_groups) {
  const uint32_t r = blockIdx.x;
  const int32_t pos = a.pos != nullptr ? a.pos[r] : a.pos0 + static_cast<int32_t>(r);
  if (pos < 0 || static_cast<uint32_t>(pos) >= max_ctx) return;  // a padded row
  const uint32_t half = a.rotary_dim / 2;
  if (blockIdx.y >= store_groups) {
    const uint32_t t = (blockIdx.y - store_groups) * 256 + threadIdx.x;
    // Without rotation a "pair" is two neighbours, for the bias alone.
    const uint32_t per_head = a.head_dim / 2;
    if (t >= a.n_head * per_head) return;
    const uint32_t h = t / per_head, i = t - h * per_head;
    uint32_t ia, ib;
    if (i < half) {
      kv4_pair(a, i, ia, ib);
    } else {
      ia = a.rotary_dim + 2 * (i - half);
      ib = ia + 1;
    }
    float* head = a.q + static_cast<size_t>(r) * a.q_stride + h * a.head_dim;
    float x0 = head[ia], x1 = head[ib];
    if (a.bq != nullptr) {
      x0 = x0 + a.bq[h * a.head_dim + ia];
      x1 = x1 + a.bq[h * a.head_dim + ib];
    }
    if (i < half) {
      const float2 cs = kv4_angle(a, pos, i);
      head[ia] = x0 * cs.x - x1 * cs.y;
      head[ib] = x0 * cs.y + x1 * cs.x;
    } else if (a.bq != nullptr) {
      head[ia] = x0;
      head[ib] = x1;
    }
    return;
  }
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t nb = a.head_dim / kQK;
  const uint32_t blocks = a.n_kv * nb;
  const uint32_t at = blockIdx.y * 8 + threadIdx.x / 32;
  // A half-wave past the last block repeats it up to the stores: the lane operations below take whole waves.
  const bool active = at < 2 * blocks;
  const uint32_t which = min(at, 2 * blocks - 1);
  const bool is_v = which >= blocks;
  const uint32_t hb = is_v ? which - blocks : which;
  const uint32_t h = hb / nb, b = hb - h * nb;
  const uint32_t j = b * kQK + lane;  // the value's index in its head
  float x;
  if (is_v) {
    const uint32_t e = h * a.head_dim + j;
    x = a.v[static_cast<size_t>(r) * a.k_stride + e];
    if (a.bv != nullptr) x = x + a.bv[e];
  } else {
    const float* row = a.k + static_cast<size_t>(r) * a.k_stride + h * a.head_dim;
    const float* bias = a.bk != nullptr ? a.bk + h * a.head_dim : nullptr;
    if (j < a.rotary_dim) {
      const uint32_t i = a.neox ? (j < half ? j : j - half) : j / 2;
      uint32_t ia, ib;
      kv4_pair(a, i, ia, ib);
      float x0 = row[ia], x1 = row[ib];
      if (bias != nullptr) {
        x0 = x0 + bias[ia];
        x1 = x1 + bias[ib];
      }
      const float2 cs = kv4_angle(a, pos, i);
      x = j == ia ? x0 * cs.x - x1 * cs.y : x0 * cs.y + x1 * cs.x;
    } else {
      x = row[j];
      if (bias != nullptr) x = x + bias[j];
    }
  }
  // The block's value of largest magnitude: magnitudes compare as their bits do, infinities and NaN above.
  const uint32_t mag = __float_as_uint(x) & 0x7fffffffu;
  uint32_t top = mag;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 32)));
  const uint32_t holders = static_cast<uint32_t>(__ballot(mag == top) >> (threadIdx.x & 32u));
  const float m = __shfl(x, __ffs(static_cast<int>(holders)) - 1, 32);
  uint32_t dbits, code = 8;
  if (top >= 0x7f800000u) {
    dbits = 0x7e00u;
  } else {
    dbits = float_to_half_bits(fminf(fmaxf(m / -8.0f, -65504.0f), 65504.0f));
    const float d = half_value(dbits);
    if (d != 0.0f) code = kv4_code(x, d);
  }
  uint8_t* tile = static_cast<uint8_t*>(a.cache) + (a.cache_off != nullptr ? a.cache_off[r] : 0) + a.k_layer_off +
                  (static_cast<size_t>(h) * kv4_tiles(max_ctx) + static_cast<uint32_t>(pos) / kKv4Tile) *
                      kv4_tile_bytes(a.head_dim);
  const uint32_t p = static_cast<uint32_t>(pos) % kKv4Tile;
  if (is_v) {
    const uint32_t high = static_cast<uint32_t>(__shfl_down(static_cast<int>(code), 16, 32));
    if (active && lane < 16) tile[kv4_value_byte(nb, p, b, lane)] = static_cast<uint8_t>(code | (high << 4));
  } else {
    const uint32_t t = lane & 7u;
    uint32_t w = code << (4 * (t / 2 + 4 * (t & 1u)));
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) w |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(w), off, 32));
    if (active && t == 0) *reinterpret_cast<uint32_t*>(tile + kv4_key_dword(nb, p, b, lane / 8)) = w;
  }
  if (active && lane == 0)
    reinterpret_cast<uint16_t*>(tile + (is_v ? 34 : 32) * a.head_dim)[kv4_scale_half(nb, p, b)] = static_cast<uint16_t>(dbits);
}

// One thread per value: grid (rows, 256 values of the row's keys and values).
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4ReadArgs a) {
  const uint32_t r = blockIdx.x;
  const uint32_t width = a.n_kv * a.head_dim;
  uint32_t e = blockIdx.y * 256 + threadIdx.x;
  if (e >= 2 * width) return;
  const bool is_v = e >= width;
  if (is_v) e -= width;
  float* out = is_v ? a.v : a.k;
  if (out == nullptr) return;
  const int32_t pos = a.pos != nullptr ? a.pos[r] : a.pos0 + static_cast<int32_t>(r);
  if (pos < 0 || static_cast<uint32_t>(pos) >= a.max_ctx) return;
  const uint32_t h = e / a.head_dim, j = e - h * a.head_dim;
  const uint32_t nb = a.head_dim / kQK, b = j / kQK, p = static_cast<uint32_t>(pos) % kKv4Tile;
  const uint8_t* tile = static_cast<const uint8_t*>(a.cache) + (a.cache_off != nullptr ? a.cache_off[r] : 0) +
                        a.layer_off +
                        (static_cast<size_t>(h) * kv4_tiles(a.max_ctx) + static_cast<uint32_t>(pos) / kKv4Tile) *
                            kv4_tile_bytes(a.head_dim);
  uint32_t code;
  if (is_v) {
    code = tile[kv4_value_byte(nb, p, b, j % 16)] >> (j % kQK < 16 ? 0 : 4);
  } else {
    const uint32_t t = j % 8;
    code = *reinterpret_cast<const uint32_t*>(tile + kv4_key_dword(nb, p, b, j % kQK / 8)) >> (4 * (t / 2 + 4 * (t & 1u)));
  }
  const float d =
      half_value(reinterpret_cast<const uint16_t*>(tile + (is_v ? 34 : 32) * a.head_dim)[kv4_scale_half(nb, p, b)]);
  out[static_cast<size_t>(r) * a.stride + e] = d * (static_cast<float>(code & 15u) - 8.0f);
}

// Workgroups of a row that store, and that turn its query.
uint32_t store_groups_of(const RopeRowsArgs& a) { return static_cast<uint32_t>(ceil_div(2 * a.n_kv * (a.head_dim / kQK), 8)); }
uint32_t query_groups_of(const RopeRowsArgs& a) {
  const bool turn = a.q != nullptr && (a.rotary_dim != 0 || a.bq != nullptr);
  return turn ? static_cast<uint32_t>(ceil_div(static_cast<size_t>(a.n_head) * (a.head_dim / 2), 256)) : 0;
}
uint32_t read_groups_of(const Kv4ReadArgs& a) { return static_cast<uint32_t>(ceil_div(2 * static_cast<size_t>(a.n_kv) * a.head_dim, 256)); }

}  // namespace

int rope_rows_kv4_check_size(const RopeRowsArgs& a, size_t n_rows) {
  return launch_fits("rope_rows_kv4", n_rows, 256, store_groups_of(a) + query_groups_of(a));
}
int kv4_read_check_size(const Kv4ReadArgs& a, size_t n_rows) { return launch_fits("kv4_read_rows", n_rows, 256, read_groups_of(a)); }

int rope_rows_kv4_launch(const RopeRowsArgs& a, uint32_t max_ctx, uint32_t n_rows) {
  if (n_rows == 0) return kOk;
  const uint32_t store_groups = store_groups_of(a);
  hipLaunchKernelGGL(rope_rows_kv4_kernel, dim3(n_rows, store_groups + query_groups_of(a)), dim3(256), 0, stream(), a, max_ctx,
                     store_groups);
  return check_launch("rope_rows_kv4");
}

int kv4_read_launch(const Kv4ReadArgs& a, uint32_t n_rows) {
  if (n_rows == 0) return kOk;
  hipLaunchKernelGGL(kv4_read_kernel, dim3(n_rows, read_groups_of(a)), dim3(256), 0, stream(), a);
  return check_launch("kv4_read_rows");
}

}  // namespace axon_hip
