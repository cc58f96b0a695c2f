// Grouped-query attention over the 4-bit KV cache (layout: kv4.h).
//
//   out_h = sum_p softmax_p(scale q_h . K_p) V_p,  p < n_vis(row)
//
// With K_p = d_k (c - 8) per block of 32 values, q . K_p = sum_b d_k(p, b) (q_b . (c - 8)): the codes go
// into the matrix cores as the small integers they are, exactly, and the scale is applied to each block's
// sum in 32 bits. For values the scale goes on the probability: out_b = sum_p (P_p d_v(p, b)) (c - 8).
// The other operand of each product is split into two fp16 terms, hi = fp16(x) and lo = fp16(x - hi),
// which together hold 22 bits of x; products and sums are in 32 bits, so the outputs keep the accuracy
// of a 32-bit computation (one fp16 term alone would cost 2^-12 relative). Queries are first multiplied by
// the mantissa of scale log2(e) and brought to a power of two near 2^9 per row, so that what is left of the
// factor from a product's sum to the exponent is a power of two, and a score and its reference are compared
// exactly however large they are. Probabilities carry a factor of 2^11, so that with scales below 2
// nothing overflows, and the products of probabilities and scales are held to 2^-34 at the least. A tile with a
// value scale of 2 or more has each block's products brought to the same place first, by the power of two
// of the largest among them, and what they add up to brought back in 32 bits (where every tile is such a one,
// 2000 rows behind none, 32 heads of size 64 over 8, take 88 us, else 57; 32 rows of 64 to 2048 11.0 and 9.6).
//
// A workgroup takes sets of 16 CT columns, a column being one (row, head) pair of one KV head: the
// heads of a group for one row, or of several rows of a prompt chunk. The waves that share a set take its
// tiles of 32 positions in turn and keep the running maximum, sum and output of their own tiles (the online
// softmax); they meet in LDS at the end. Scores are computed transposed (positions are the rows of the product),
// so a lane's scores belong to one column, and with the tile's position order they are already where the
// second product wants its probabilities: nothing crosses lanes between the products.
//
// Single rows with groups of up to 8 heads would leave most of 16 columns empty and spend their vector
// instructions on them; they take v_mfma_f32_4x4x4_16b_f16 instead, 16 products of 4 x 4 x 4 at once:
// 64 positions are the 16 products' rows, 4 heads their columns. The four lanes of a product hold 4
// positions of 4 heads each, which is what the second product, with probabilities as its rows, takes;
// there each product's probabilities are broadcast to the 16 lanes that hold a block's values.
//
// Few rows over long contexts are split further, one workgroup per run of positions, and a second
// kernel joins the parts by their maxima.
//
// Bounds, as measured (heads over KV heads, head size; a large copy runs at 4.9 TB/s here, reads alone at 6.3, a
// large fp16 product at 1.1 PFLOP/s):
//   16 rows of 32768 positions (32/8, 128): 597 MB in 114 us, 5.2 TB/s: the codes' bytes, and vector instructions,
//   issued two thirds of the time;
//   32 rows of 64 to 2048 (32/8, 64): 19 MB in 9.6 us: the longest row's steps, one workgroup a CU;
//   1 row of 512 (9/3, 64): 4.8 us, the launch and one step after another;
//   2000 rows behind none (32/8, 64): 16.4 GFLOP, twice that for the two terms, in 57 us: vector
//   instructions are issued 61 % of the time (a wave's step of 32 positions by 32 columns is 230 of them:
//   codes 72, scores' scales 32, maxima and exponentials 64, probabilities' terms 96) and the matrix cores busy
//   20 %; 8192 rows 680 us, 404 TFLOP/s.
#include "common.h"
#include "kv4.h"

#include <algorithm>
#include <type_traits>

namespace axon_hip {

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2E = 1.4426950408889634f;
// The probabilities' power of two, and how far above the reference a score may rise (in powers of two)
// before the reference follows it: most maxima after the first tile's stay within that, and following costs
// a multiplication of every output. 2^(11 + 3) times a scale below 2 fits fp16.
constexpr float kShift = 11.0f, kRoom = 3.0f;

// What a column's largest score so far sets: `ref`, which is subtracted in the exponent, and `limit`, the score above
// which both are set anew. `factor` is a power of two, so t, the score in powers of two, is exact, and the reference
// is t less kShift: the largest probability is 2^kShift. Where 32 bits do not hold that number (t from 2^24 on; the
// nearest they hold would leave fp16's range from 2^25 on) it is t less 8, or t: all scores are whole multiples of a
// power of two there, probabilities whole powers of two, and what they lose of their room below is not used.
struct Reference {
  float ref, limit;
  __device__ __forceinline__ Reference(float top, float factor) {
    const float t = top * factor;
    ref = t - kShift;
    limit = __builtin_fmaf(kRoom, __uint_as_float((254u << 23) - __float_as_uint(factor)), top);
    if (__builtin_expect(fabsf((t - ref) - kShift) > 0.5f, 0)) {
      ref = t - 8.0f;
      if (t - ref > 8.5f) ref = t;
      limit = top;
    }
  }
};

// What brings the queries of a head to 2^9 and more, their largest magnitude being `top`: first a power of two, then
// a mantissa; and the power of two that the scores are left to be multiplied by.
struct QueryScale {
  float power, mantissa, factor;
  // A query as it is split: rounded to 32 bits (split2).
  __device__ __forceinline__ float operator()(float q) const {
    float x = q * power * mantissa;
    asm("" : "+v"(x));
    return x;
  }
};
__device__ __forceinline__ QueryScale query_scale(float top, float scale) {
  const uint32_t up = min(263u - min(__float_as_uint(top) >> 23, 255u), 253u);
  const float by = scale * kLog2E;
  const int32_t left = __builtin_amdgcn_frexp_expf(by) + 127 - static_cast<int32_t>(up);
  return QueryScale{__uint_as_float(up << 23), __builtin_amdgcn_frexp_mantf(by),
                    __uint_as_float(static_cast<uint32_t>(min(max(left, -126), 127) + 127) << 23)};
}

// The power of two that brings a largest magnitude to [2^14, 2^15), within what has an inverse, and the inverse.
__device__ __forceinline__ float to_fp16_range(float largest, float& inverse) {
  const uint32_t up = min(268u - min(__float_as_uint(largest) >> 23, 255u), 253u);
  inverse = __uint_as_float((254u - up) << 23);
  return __uint_as_float(up << 23);
}

// 2^x, and 0 for -inf (the instruction; 1 ulp).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The larger / the sum over the four lanes that share a column (lane ^ 16, lane ^ 32).
__device__ __forceinline__ float column_max(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float column_sum(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Four values' sums over the four rows of 16 lanes: row g gets v[g]'s.
__device__ __forceinline__ float row_sums(f32x4 v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[0]), __float_as_uint(v[1]), false, false);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[2]), __float_as_uint(v[3]), false, false);
  const float x = __uint_as_float(a[0]) + __uint_as_float(a[1]), y = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}

// Masks and the fp16 exponent of 1024, kept in registers: "and" and "or" with them are one instruction
// (v_and_or_b32 takes no literals).
struct CodeBits {
  uint32_t low = 0x000f000fu, high = 0x00f000f0u, magic = 0x64006400u;
  __device__ __forceinline__ CodeBits() {
    asm("" : "+s"(low));
    asm("" : "+s"(high));
    asm("" : "+v"(magic));
  }
};
// Nibbles 0 and 4 of w as code - 8: 0x6400 | n is 1024 + n in fp16.
__device__ __forceinline__ half2_t codes_low(const CodeBits& k, uint32_t w) {
  const uint32_t x = (w & k.low) | k.magic;
  return __builtin_bit_cast(half2_t, x) + half2_t{static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
}
// Nibbles 1 and 5: 1024 + 16 n, brought to n - 8 by one multiply-add (exact).
__device__ __forceinline__ half2_t codes_high(const CodeBits& k, uint32_t w) {
  const uint32_t x = (w & k.high) | k.magic;
  const half2_t m = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
  const half2_t c = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
  return __builtin_elementwise_fma(__builtin_bit_cast(half2_t, x), m, c);
}
// x and y as two fp16 terms each: hi the nearest, lo the nearest to the rest (the difference is one
// mixed instruction, which the compiler makes two of). x and y are no products that round: the conversion would be
// joined with the product, whose own rounding can part from that of the number it is in 32 bits.
__device__ __forceinline__ void split2(float x, float y, half2_t& hi, half2_t& lo) {
  hi = half2_t{static_cast<_Float16>(x), static_cast<_Float16>(y)};
  float a, b;
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(hi), "v"(x));
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(hi), "v"(y));
  lo = half2_t{static_cast<_Float16>(a), static_cast<_Float16>(b)};
}
__device__ __forceinline__ half8_t join8(half2_t a, half2_t b, half2_t c, half2_t d) {
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float half_of(u32x2 d, int r) {
  const uint32_t word = d[r / 2];  // (a bit cast of the vector's element itself takes its first one)
  return static_cast<float>(__builtin_bit_cast(half2_t, word)[r & 1]);
}

// A lane's run of N pairs of dwords in LDS, in 16-byte reads where it is a multiple of 16 bytes.
template <int N>
__device__ __forceinline__ void lds_pairs(u32x2 (&d)[N], const uint8_t* p) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const u32x4 x = reinterpret_cast<const u32x4*>(p)[i];
      d[2 * i] = u32x2{x[0], x[1]};
      d[2 * i + 1] = u32x2{x[2], x[3]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = reinterpret_cast<const u32x2*>(p)[i];
  }
}

// A wave's tiles on their way: each is copied into one of kDepth slots of LDS by loads that write LDS
// directly, 16 bytes a lane, and waited for when its turn comes. Four slots where they are within KB
// kilobytes (80: LDS holds two workgroups a CU), else two.
template <int NB, int W, int TILES = 1, int KB = 80>
struct TileRing {
  static constexpr uint32_t kBytes = TILES * kv4_tile_bytes(32 * NB);
  static constexpr uint32_t kLoads = (kBytes + 1023) / 1024;       // instructions per tile
  static constexpr uint32_t kDepth = W * 4 * kBytes <= KB * 1024 ? 4 : 2;
  static constexpr uint32_t kWaveBytes = kDepth * kBytes;

  const uint8_t* base;  // the head's first tile
  uint32_t lds;         // LDS address of the wave's slots
  uint32_t lane;

  // `bytes` of slot contents number `at` (zeros follow in the slot where there are fewer than kBytes).
  __device__ __forceinline__ void fetch(uint32_t at, uint32_t slot, uint32_t bytes = kBytes) const {
    const RsrcWords r = raw_buffer_words(base + static_cast<size_t>(at) * kBytes, bytes);
    const uint32_t to = lds + slot * kBytes;
#pragma unroll
    for (uint32_t i = 0; i < kBytes / 1024; ++i) lds_dma16(r, i * 1024 + lane * 16, to + i * 1024);
    if constexpr (kBytes % 1024 != 0) {
      if (lane < kBytes % 1024 / 16) lds_dma16(r, kBytes / 1024 * 1024 + lane * 16, to + kBytes / 1024 * 1024);
    }
  }
};

// Whether a wave keeps the queries' low terms in LDS, where registers would leave it alone on its SIMD (2000 rows
// behind none, 32 heads of size 128 over 8: 98 us, one tile of columns a wave 111; 4000 rows 324 and 386).
constexpr bool low_terms_in_lds(int nb, int ct) { return nb == 4 && ct == 2; }

// Whether a tile holds a value scale of 2 or more, or one that is not finite (the top bit of its exponent is set),
// among the positions below vis_hi: a lane takes the four of one block, a half-wave one of TILES tiles. The whole
// wave agrees on it.
template <int NB, int TILES, bool MASK>
__device__ __forceinline__ bool wide_scales(const uint8_t* tile, uint32_t lane, int32_t pos0, int32_t vis_hi) {
  const uint32_t which = TILES == 2 ? lane / 32 : 0, at = lane % (64 / TILES) % (8 * NB);  // (g 2 + s) NB + b
  u32x2 d = *reinterpret_cast<const u32x2*>(tile + which * kv4_tile_bytes(32 * NB) + 1088 * NB + at * 8);
  if constexpr (MASK) {
    const int32_t left = vis_hi - pos0 - static_cast<int32_t>(which * kKv4Tile + at / (2 * NB) * 4 + at / NB % 2 * 16);
    d[0] &= left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
    d[1] &= left >= 4 ? 0xffffffffu : left == 3 ? 0xffffu : 0u;
  }
  return __any(((d[0] | d[1]) & 0x40004000u) != 0);
}

// One wave's running softmax over its tiles, for 16 CT columns.
template <int NB, int CT>
struct WaveState {
  static constexpr bool kLowInLds = low_terms_in_lds(NB, CT);
  half8_t qhi[CT][NB], qlo[kLowInLds ? 1 : CT][kLowInLds ? 1 : NB];
  half8_t* low;            // the lane's of the first block, where they are in LDS: a block's are 64 apart
  float colf[CT];          // score in powers of two per unit of the integer product: a power of two
  float top[CT];           // the reference, in those units: the maximum when it last moved
  float limit[CT];         // scores above it move the reference
  float ref[CT];           // what is subtracted in the exponent
  float sum[CT];           // this lane's part of the sum
  f32x4 o[CT][NB][2];
};

// One tile. MASK: some column's row ends in it; WIDE: wide_scales.
template <int NB, int CT, bool MASK, bool WIDE>
__device__ __forceinline__ void tile_step(WaveState<NB, CT>& w, const CodeBits& bits, const uint8_t* tile, uint32_t lane,
                                          const int32_t (&vis)[CT], int32_t pos0) {
  const uint32_t g = lane / 16;
  u32x2 kc[NB], kd[2 * NB], vc[NB], vd[2 * NB];
  lds_pairs<NB>(kc, tile + lane * (8 * NB));
  lds_pairs<2 * NB>(kd, tile + 1024 * NB + g * (16 * NB));
  // Scores: S[s][r] of positions pos0 + 16 s + r (pos0 includes the lane's 4 g).
  float s[CT][8];
#pragma unroll
  for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int at = sub * NB + b;
      const uint32_t word = kc[at / 2][at % 2];
      const half8_t a = join8(codes_low(bits, word), codes_high(bits, word), codes_low(bits, word >> 8), codes_high(bits, word >> 8));
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        half8_t qlo;
        if constexpr (low_terms_in_lds(NB, CT)) qlo = w.low[(c * NB + b) * 64];
        else qlo = w.qlo[c][b];
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qlo, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, w.qhi[c][b], acc, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float d = half_of(kd[at], r);
          s[c][4 * sub + r] = __builtin_fmaf(acc[r], d, b == 0 ? 0.0f : s[c][4 * sub + r]);
        }
      }
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  lds_pairs<NB>(vc, tile + 512 * NB + lane * (8 * NB));
  lds_pairs<2 * NB>(vd, tile + 1088 * NB + g * (16 * NB));
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (MASK) {
        if (pos0 + 16 * (i / 4) + i % 4 >= vis[c]) s[c][i] = -__builtin_inff();
      }
      m = fmaxf(m, s[c][i]);
    }
    if (__builtin_expect(__any(m > w.limit[c]), 0)) {
      const float top = fmaxf(w.top[c], column_max(m));
      if (top != -__builtin_inff()) {
        const Reference to(top, w.colf[c]);
        const float scale = w.top[c] == -__builtin_inff() ? 1.0f : exp2_fast(w.ref[c] - to.ref);
        w.top[c] = top;
        w.limit[c] = to.limit;
        w.ref[c] = to.ref;
        w.sum[c] *= scale;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h) w.o[c][b][h] *= scale;
      }
    }
  }
  // Probabilities, and their sum.
  float p[CT][8];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[c][i] = exp2_fast(__builtin_fmaf(s[c][i], w.colf[c], -w.ref[c]));
      w.sum[c] += p[c][i];
    }
  }
  // Outputs. A register of value codes holds positions r 0..3 in its bytes: (0, 2) and (1, 3) mask out
  // as pairs, which is the order that probabilities and scales take too: pair i is positions e and e + 2.
  // With scales below 2, probabilities are split into two fp16 terms once, and a product with a
  // scale, again in two terms, is three packed instructions a pair: hi = fp16(ph d), ph d - hi (exact),
  // and pl d added to it (a quarter less than two mixed multiply-adds a value, which run at half rate; 2000
  // positions behind none, 32 heads of size 64 over 8, take 57 us, with those 7 more). With larger ones the products are
  // formed in 32 bits, and a block's are split where their own largest allows.
  uint32_t seen[CT][4];
  if constexpr (MASK) {
    // What lies past a row's own positions is not its, a NaN scale least of all.
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t at = pos0 + 16 * (i / 2) + i % 2;
        seen[c][i] = (at < vis[c] ? 0xffffu : 0u) | (at + 2 < vis[c] ? 0xffff0000u : 0u);
      }
  }
  // add(c, b, the block's scales, its codes): a column's part of a block.
  const auto each_block = [&](auto&& add) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t w0 = vc[b][0], w1 = vc[b][1];
      const half8_t lo16 = join8(codes_low(bits, w0), codes_low(bits, w0 >> 8), codes_low(bits, w1), codes_low(bits, w1 >> 8));
      const half8_t hi16 = join8(codes_high(bits, w0), codes_high(bits, w0 >> 8), codes_high(bits, w1), codes_high(bits, w1 >> 8));
      half2_t d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x2 dd = vd[i / 2 * NB + b];
        d[i] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(dd[1], dd[0], i % 2 != 0 ? 0x07060302u : 0x05040100u));
      }
#pragma unroll
      for (int c = 0; c < CT; ++c) add(c, b, d, lo16, hi16);
    }
  };
  if constexpr (!WIDE) {
    half2_t ph[CT][4], pl[CT][4];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) split2(p[c][i / 2 * 4 + i % 2], p[c][i / 2 * 4 + i % 2 + 2], ph[c][i], pl[c][i]);
    each_block([&](int c, int b, const half2_t (&d)[4], half8_t lo16, half8_t hi16) {
      half2_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hi[i] = ph[c][i] * d[i];
        lo[i] = __builtin_elementwise_fma(pl[c][i], d[i], __builtin_elementwise_fma(ph[c][i], d[i], -hi[i]));
        if constexpr (MASK) {
          hi[i] = __builtin_bit_cast(half2_t, __builtin_bit_cast(uint32_t, hi[i]) & seen[c][i]);
          lo[i] = __builtin_bit_cast(half2_t, __builtin_bit_cast(uint32_t, lo[i]) & seen[c][i]);
        }
      }
      const half8_t phi = join8(hi[0], hi[1], hi[2], hi[3]), plo = join8(lo[0], lo[1], lo[2], lo[3]);
      w.o[c][b][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo16, plo, w.o[c][b][0], 0, 0, 0);
      w.o[c][b][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi16, plo, w.o[c][b][1], 0, 0, 0);
      w.o[c][b][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo16, phi, w.o[c][b][0], 0, 0, 0);
      w.o[c][b][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi16, phi, w.o[c][b][1], 0, 0, 0);
    });
  } else {
    each_block([&](int c, int b, const half2_t (&d)[4], half8_t lo16, half8_t hi16) {
      float x[8], most = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = k / 2, at = i / 2 * 4 + i % 2 + k % 2 * 2;  // pair i's first and second
        x[k] = p[c][at] * static_cast<float>(d[i][k % 2]);
        if constexpr (MASK) x[k] = (seen[c][i] >> (16 * (k % 2)) & 1u) != 0 ? x[k] : 0.0f;
        most = fmaxf(most, fabsf(x[k]));
      }
      float inverse;
      const float by = to_fp16_range(column_max(most), inverse);
      half2_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) split2(x[2 * i] * by, x[2 * i + 1] * by, hi[i], lo[i]);
      const half8_t phi = join8(hi[0], hi[1], hi[2], hi[3]), plo = join8(lo[0], lo[1], lo[2], lo[3]);
      const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
      f32x4 even = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo16, plo, zero, 0, 0, 0);
      f32x4 odd = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi16, plo, zero, 0, 0, 0);
      even = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo16, phi, even, 0, 0, 0);
      odd = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi16, phi, odd, 0, 0, 0);
      w.o[c][b][0] += even * inverse;
      w.o[c][b][1] += odd * inverse;
      __builtin_amdgcn_sched_barrier(0);  // (one after another, in few registers)
    });
  }
}

// What a launch works on beside the arguments.
struct Kv4Plan {
  uint32_t row0;        // first row
  uint32_t n_rows;      // rows of this launch
  uint32_t block_rows;  // rows per workgroup (a chunk's rows share a sequence)
  uint32_t col_blocks;  // workgroups over a group's heads when one row's exceed the columns
  uint32_t splits;      // workgroups over a row's positions
  uint32_t split_tiles; // tiles per split
  uint32_t most_splits; // splits of any max_vis up to this one (rounding can make fewer of more)
  uint32_t waves;       // waves per workgroup
  uint32_t per_group;   // ceil(2^16 / group): column / group is (column * per_group) >> 16 (columns are below 64)
  uint32_t col_tiles;   // 16-column tiles a wave
  uint32_t shared_by;   // waves that share a set of columns and its positions
  bool by_row;          // the kernel for single rows
  bool chunk;           // the rows are one sequence's, the first row's
};

// Column `col` of a workgroup: its row behind the first and its head in the group.
__device__ __forceinline__ void row_head(const Kv4Plan& plan, uint32_t group, uint32_t head0, uint32_t col, uint32_t& row,
                                         uint32_t& head) {
  row = plan.block_rows > 1 ? (col * plan.per_group) >> 16 : 0;
  head = head0 + col - row * group;
}

__device__ __forceinline__ int32_t row_vis(const AttnKv4Args& a, uint32_t r) {
  const int32_t n = a.n_vis != nullptr ? a.n_vis[r] : a.n_past + static_cast<int32_t>(r) + 1;
  return min(max(n, 0), static_cast<int32_t>(a.max_vis));
}

// Floats of one part: the output of a (row, head) pair, then the exponent's reference and the sum.
constexpr uint32_t part_floats(uint32_t head_dim) { return head_dim + 2; }

// The waves' parts of eight consecutive outputs of a column, brought to their common reference: part k's at
// meet + k * meet_step, its reference and sum at refs[k * step], sums[k * step].
template <int PARTS>
__device__ __forceinline__ void join_parts(const float* meet, uint32_t meet_step, const float* refs, const float* sums,
                                           uint32_t step, float (&o)[8], float& ref, float& sum) {
  ref = -__builtin_inff();
#pragma unroll
  for (uint32_t k = 0; k < PARTS; ++k) ref = fmaxf(ref, refs[k * step]);
  sum = 0.0f;
#pragma unroll
  for (int t = 0; t < 8; ++t) o[t] = 0.0f;
#pragma unroll
  for (uint32_t k = 0; k < PARTS; ++k) {
    const float part = refs[k * step];
    if (part != -__builtin_inff()) {
      const float f = exp2_fast(part - ref);
      sum += f * sums[k * step];
      const f32x4 a = *reinterpret_cast<const f32x4*>(meet + k * meet_step), b = *reinterpret_cast<const f32x4*>(meet + k * meet_step + 4);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        o[t] += f * a[t];
        o[4 + t] += f * b[t];
      }
    }
  }
}

// Eight outputs of a (row, head) pair from value `at` on: into a part of the scratch, or divided by the sum
// into the output and its Q8_0 blocks, whose other quarters are in the three adjacent lanes. Every lane of
// a wave calls it.
__device__ __forceinline__ void put_outputs(const AttnKv4Args& a, const Kv4Plan& plan, uint32_t split, bool has, uint32_t r,
                                            uint32_t head, uint32_t at, float (&o)[8], float ref, float sum) {
  if (plan.splits > 1) {
    if (!has) return;
    float* part = a.scratch + ((static_cast<size_t>(r - plan.row0) * a.n_head + head) * plan.splits + split) * part_floats(a.head_dim);
    *reinterpret_cast<f32x4_a4*>(part + at) = f32x4{o[0], o[1], o[2], o[3]};
    *reinterpret_cast<f32x4_a4*>(part + at + 4) = f32x4{o[4], o[5], o[6], o[7]};
    if (at == 0) {
      part[a.head_dim] = ref;
      part[a.head_dim + 1] = sum;
    }
    return;
  }
  // A column that saw no position gives zeros.
  const float by = ref == -__builtin_inff() ? 0.0f : __builtin_amdgcn_rcpf(sum);
#pragma unroll
  for (int t = 0; t < 8; ++t) o[t] *= by;
  if (has) {
    float* out = a.out + static_cast<size_t>(r) * a.out_stride + head * a.head_dim + at;
    *reinterpret_cast<f32x4_a4*>(out) = f32x4{o[0], o[1], o[2], o[3]};
    *reinterpret_cast<f32x4_a4*>(out + 4) = f32x4{o[4], o[5], o[6], o[7]};
  }
  if (a.outq != nullptr)
    quantize8_store(o, has, static_cast<uint8_t*>(a.outq) +
                                ((static_cast<size_t>(r) * a.n_head + head) * (a.head_dim / kQK) + at / kQK) * kBytesQ8_0, at / 8 % 4);
}

// W waves: KS of them share 16 CT columns and take every KS-th tile each; W / KS such sets.
template <int NB, int CT, int KS, int W>
__global__ __launch_bounds__(W * 64, low_terms_in_lds(NB, CT) ? 2 : 1) void attention_kv4_kernel(AttnKv4Args a, Kv4Plan plan) {
  using Ring = TileRing<NB, W, 1, low_terms_in_lds(NB, CT) ? 40 : 80>;
  constexpr uint32_t kDim = 32 * NB;
  constexpr uint32_t kWaveCols = 16 * CT, kCols = kWaveCols * W / KS;
  constexpr uint32_t kStride = kDim + 4;  // floats between columns where the parts meet
  constexpr uint32_t kRingBytes = W * Ring::kWaveBytes, kMeetBytes = W * kWaveCols * kStride * 4;
  constexpr uint32_t kLowBytes = low_terms_in_lds(NB, CT) ? W * CT * NB * 1024 : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kRingBytes + kLowBytes > kMeetBytes ? kRingBytes + kLowBytes : kMeetBytes];
  __shared__ float lds_ref[W][kWaveCols], lds_sum[W][kWaveCols];
  // KV head fastest: workgroups go round the eight XCDs, so with eight heads each keeps to one L2.
  uint32_t id = blockIdx.x;
  const uint32_t h = id % a.n_kv;
  id /= a.n_kv;
  const uint32_t split = id % plan.splits;
  id /= plan.splits;
  const uint32_t cb = id % plan.col_blocks;
  // Later rows of a chunk see more positions: they start first.
  const uint32_t rb = gridDim.x / (a.n_kv * plan.splits * plan.col_blocks) - 1 - id / plan.col_blocks;
  const uint32_t r0 = plan.row0 + rb * plan.block_rows;
  const uint32_t rows = min(plan.block_rows, plan.row0 + plan.n_rows - r0);
  const uint32_t group = a.n_head / a.n_kv;
  const uint32_t cols = plan.block_rows > 1 ? rows * group : min(group - cb * kCols, kCols);
  const uint32_t lane = threadIdx.x & 63u, i = lane % 16, g = lane / 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), set = wave / KS, ks = wave % KS;

  // The queries and what their rows see.
  int32_t vis[CT];
  float seen_hi = 0.0f, seen_lo = -16777216.0f;  // the rows' largest and (negated) smallest
  f32x4 x[CT][NB][2];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const uint32_t col = set * kWaveCols + c * 16 + i;
    const bool has = col < cols;
    uint32_t r, head;
    row_head(plan, group, h * group + cb * kCols, col, r, head);
    r += r0;
    // A column without a row is computed along with the others and not stored.
    vis[c] = has ? row_vis(a, r) : 0x7fffffff;
    if (has) {
      seen_hi = fmaxf(seen_hi, static_cast<float>(vis[c]));
      seen_lo = fmaxf(seen_lo, -static_cast<float>(vis[c]));
    }
    const float* q = a.q + static_cast<size_t>(r) * a.q_stride + head * kDim + 8 * g;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        x[c][b][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (has) x[c][b][k] = *reinterpret_cast<const f32x4_a4*>(q + 32 * b + 4 * k);
      }
    }
  }
  const int32_t vis_hi = static_cast<int32_t>(wave_max(seen_hi));
  const int32_t vis_lo = static_cast<int32_t>(-wave_max(seen_lo));
  const uint32_t t0 = split * plan.split_tiles + ks;
  const uint32_t t1 = min(kv4_tiles(static_cast<uint32_t>(vis_hi)), (split + 1) * plan.split_tiles);
  // An empty part: the joining kernel knows which there are. (Splits go with one set of columns, where
  // every wave sees the same rows.)
  if (plan.splits > 1 && split * plan.split_tiles >= t1) return;
  const uint32_t n = __builtin_amdgcn_readfirstlane(t0 < t1 ? (t1 - t0 + KS - 1) / KS : 0);

  // The first tiles start while the queries are prepared.
  Ring ring;
  ring.base = static_cast<const uint8_t*>(a.cache) + (a.cache_off != nullptr ? a.cache_off[plan.chunk ? 0 : r0] : 0) + a.layer_off +
              static_cast<size_t>(h) * kv4_tiles(a.max_ctx) * Ring::kBytes;
  ring.lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(as_lds(lds))) + wave * Ring::kWaveBytes;
  ring.lane = lane;
  constexpr uint32_t kAhead = Ring::kDepth - 1;
#pragma unroll
  for (uint32_t j = 0; j < kAhead; ++j)
    if (j < n) ring.fetch(t0 + j * KS, j);

  WaveState<NB, CT> w;
  w.low = reinterpret_cast<half8_t*>(lds + kRingBytes) + wave * (CT * NB * 64) + lane;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int t = 0; t < 8; ++t) top = fmaxf(top, fabsf(x[c][b][t / 4][t % 4]));
    const QueryScale by = query_scale(column_max(top), a.scale);
    w.colf[c] = by.factor;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      half2_t hi[4], lo[4];
#pragma unroll
      for (int t = 0; t < 8; t += 2) split2(by(x[c][b][t / 4][t % 4]), by(x[c][b][t / 4][t % 4 + 1]), hi[t / 2], lo[t / 2]);
      w.qhi[c][b] = join8(hi[0], hi[1], hi[2], hi[3]);
      const half8_t qlo = join8(lo[0], lo[1], lo[2], lo[3]);
      if constexpr (low_terms_in_lds(NB, CT)) w.low[(c * NB + b) * 64] = qlo;
      else w.qlo[c][b] = qlo;
#pragma unroll
      for (int k = 0; k < 2; ++k) w.o[c][b][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    w.top[c] = w.limit[c] = -__builtin_inff();
    w.ref[c] = 0.0f;
    w.sum[c] = 0.0f;
  }

  const CodeBits bits;
  const uint8_t* slots = lds + wave * Ring::kWaveBytes;
  for (uint32_t j = 0; j < n; ++j) {
    // The slot that the next copy goes to was read in the step before: its reads have returned.
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    if (j + kAhead < n) {
      ring.fetch(t0 + (j + kAhead) * KS, (j + kAhead) % Ring::kDepth);
      wait_vm<kAhead * Ring::kLoads>();
    } else if (kAhead > 2 && j + 3 == n) {
      wait_vm<2 * Ring::kLoads>();
    } else if (kAhead > 1 && j + 2 == n) {
      wait_vm<Ring::kLoads>();
    } else {
      wait_vm<0>();
    }
    const uint32_t t = t0 + j * KS;
    const uint8_t* tile = slots + j % Ring::kDepth * Ring::kBytes;
    const int32_t first = static_cast<int32_t>(t * kKv4Tile), pos0 = first + static_cast<int32_t>(4 * g);
    const bool mask = first + static_cast<int32_t>(kKv4Tile) > vis_lo;
    const bool wide = mask ? wide_scales<NB, 1, true>(tile, lane, first, vis_hi) : wide_scales<NB, 1, false>(tile, lane, first, vis_hi);
    if (__builtin_expect(wide, 0)) {
      tile_step<NB, CT, true, true>(w, bits, tile, lane, vis, pos0);
    } else if (mask) {
      tile_step<NB, CT, true, false>(w, bits, tile, lane, vis, pos0);
    } else {
      tile_step<NB, CT, false, false>(w, bits, tile, lane, vis, pos0);
    }
  }

  // The waves' parts meet, where the tiles were: each brings its own to the common reference.
  __syncthreads();
  float* meet = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const float sum = column_sum(w.sum[c]);
    if (g == 0) {
      // A wave without a visible position takes no part.
      lds_ref[wave][c * 16 + i] = w.top[c] == -__builtin_inff() && sum == 0.0f ? -__builtin_inff() : w.ref[c];
      lds_sum[wave][c * 16 + i] = sum;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        *reinterpret_cast<f32x4*>(&meet[(wave * kWaveCols + c * 16 + i) * kStride + 32 * b + 16 * k + 4 * g]) = w.o[c][b][k];
    }
  }
  __syncthreads();
  constexpr uint32_t kUnits = kDim / 8;
  for (uint32_t u = threadIdx.x; u < kCols * kUnits; u += W * 64) {  // (whole waves)
    const uint32_t col = u / kUnits, at = u % kUnits * 8;
    const uint32_t first = col / kWaveCols * KS, c = col % kWaveCols;
    float o[8], ref, sum;
    join_parts<KS>(meet + (first * kWaveCols + c) * kStride + at, kWaveCols * kStride, &lds_ref[first][c], &lds_sum[first][c],
                   kWaveCols, o, ref, sum);
    uint32_t r, head;
    row_head(plan, group, h * group + cb * kCols, col, r, head);
    put_outputs(a, plan, split, col < cols, r0 + r, head, at, o, ref, sum);
  }
}

// ------------------------------------------------------------------------------------------
// Single rows, groups of up to 4 NS heads

// A wave's running softmax over its positions, 4 NS heads. Lane l is column l % 4 (a head of each set) of
// product l / 4; in the outputs it is dim l % 16 of a half block, over the positions of products
// 4 (l / 16) .. + 3, and its registers are the heads.
template <int NB, int NS>
struct RowState {
  // Queries: value 16 j + 4 m + t of the lane's head, m = l / 16: what the 2 NB registers hold in 16 lanes
  // is broadcast to all as the products need it.
  half4_t qhi[NS][2 * NB], qlo[NS][2 * NB];
  float colf[NS], top[NS], limit[NS], ref[NS], sum[NS];
  f32x4 o[NS][NB][2];
};

// The largest over the 16 lanes with one l % 4.
__device__ __forceinline__ float head_max(float x) {
  x = max_dpp<0x124>(x);  // row_ror 4
  x = max_dpp<0x128>(x);  // row_ror 8
  return column_max(x);
}

__device__ __forceinline__ half4_t join4(half2_t a, half2_t b) { return half4_t{a[0], a[1], b[0], b[1]}; }

// 64 positions: two tiles in LDS, in one of the slots. MASK: the row ends in them; WIDE: wide_scales.
template <int NB, int NS, bool MASK, bool WIDE>
__device__ __forceinline__ void row_step(RowState<NB, NS>& w, const CodeBits& bits, const uint8_t* slots, uint32_t slot,
                                         uint32_t lane, int32_t vis, int32_t pos0) {
  constexpr uint32_t kTileBytes = kv4_tile_bytes(32 * NB);
  // (Each form has its own beginning: what they share, ahead of the branch between them, holds a third more registers.)
  asm volatile("" : "+s"(slot));
  const uint8_t* tiles = slots + slot * (2 * kTileBytes);
  // The lane's position as a row of the first product: its codes.
  uint32_t kc[4][NB];
  {
    const uint8_t* t = tiles + lane / 32 * kTileBytes + ((lane % 16) * 2 + lane % 32 / 16) * (4 * NB);
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int b = 0; b < NB; ++b) kc[g][b] = reinterpret_cast<const uint32_t*>(t + g * (128 * NB))[b];
  }
  // The scales of product lane / 4's positions.
  u32x2 kd[NB], vd[NB];
  const uint32_t prod = lane / 4;
  const uint8_t* scales = tiles + prod / 8 * kTileBytes + 1024 * NB + (prod % 4 * 2 + prod % 8 / 4) * (8 * NB);
  lds_pairs<NB>(kd, scales);
  lds_pairs<NB>(vd, scales + 64 * NB);
  // Its codes of values as a column of the second product: half-block dim lane % 16, product 4 (l / 16) + k.
  uint32_t vc[4][NB];
  {
    const uint8_t* t = tiles + lane / 32 * kTileBytes + 512 * NB + (lane % 16) * (8 * NB) + lane % 32 / 16 * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int b = 0; b < NB; ++b) vc[k][b] = *reinterpret_cast<const uint32_t*>(t + k * (128 * NB) + b * 8);
  }
  float s[NS][4];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    f32x4 hi[NS], lo[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) hi[n] = lo[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for_each_index<0, 4>([&]<int G>() {
      const uint32_t word = kc[G][b];
      const half4_t a0 = join4(codes_low(bits, word), codes_high(bits, word));
      const half4_t a1 = join4(codes_low(bits, word >> 8), codes_high(bits, word >> 8));
      constexpr int kHalf = G % 2 * 2;  // values 32 b + 8 G .. are in lanes 16 kHalf .. of register 2 b + G / 2
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const half4_t qh = w.qhi[n][2 * b + G / 2], ql = w.qlo[n][2 * b + G / 2];
        hi[n] = __builtin_amdgcn_mfma_f32_4x4x4f16(a0, qh, hi[n], 0, 0, 4 + kHalf);
        lo[n] = __builtin_amdgcn_mfma_f32_4x4x4f16(a0, ql, lo[n], 0, 0, 4 + kHalf);
        hi[n] = __builtin_amdgcn_mfma_f32_4x4x4f16(a1, qh, hi[n], 0, 0, 5 + kHalf);
        lo[n] = __builtin_amdgcn_mfma_f32_4x4x4f16(a1, ql, lo[n], 0, 0, 5 + kHalf);
      }
    });
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[n][r] = __builtin_fmaf(hi[n][r] + lo[n][r], half_of(kd[b], r), b == 0 ? 0.0f : s[n][r]);
  }
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    if constexpr (MASK) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (pos0 + r >= vis) s[n][r] = -__builtin_inff();
    }
    const float m = fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3]));
    if (__builtin_expect(__any(m > w.limit[n]), 0)) {
      const float top = fmaxf(w.top[n], head_max(m));
      // (a head without a score so far stays as it is)
      const Reference to(top, w.colf[n]);
      const float ref = top == -__builtin_inff() ? w.ref[n] : to.ref;
      const float scale = w.top[n] == -__builtin_inff() ? 1.0f : exp2_fast(w.ref[n] - ref);
      w.top[n] = top;
      w.limit[n] = to.limit;
      w.ref[n] = ref;
      w.sum[n] *= scale;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float of_head = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scale), r));
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int k = 0; k < 2; ++k) w.o[n][b][k][r] *= of_head;
      }
    }
  }
  float p[NS][4];
#pragma unroll
  for (int n = 0; n < NS; ++n) {
#pragma unroll
    for (int r = 0; r < 4; ++r) p[n][r] = exp2_fast(__builtin_fmaf(s[n][r], w.colf[n], -w.ref[n]));
    w.sum[n] += (p[n][0] + p[n][1]) + (p[n][2] + p[n][3]);
  }
  constexpr int kOrder[4] = {0, 2, 1, 3};  // the order of a register of value codes
  // add(n, b, k, the codes): a set of heads' part of a block, over the k-th quarter of each 16 positions' products.
  const auto each_block = [&](int b, auto&& add) {
    for_each_index<0, 4>([&]<int K>() {
      const uint32_t word = vc[K][b];
      const half4_t lo16 = join4(codes_low(bits, word), codes_low(bits, word >> 8));
      const half4_t hi16 = join4(codes_high(bits, word), codes_high(bits, word >> 8));
      add.template operator()<K>(lo16, hi16);
    });
  };
  if constexpr (!WIDE) {
    half4_t ph[NS][NB], pl[NS][NB];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = kOrder[k];
          const float d = half_of(vd[b], r);
          _Float16 hi = static_cast<_Float16>(__builtin_fmaf(p[n][r], d, 0.0f));
          _Float16 lo = static_cast<_Float16>(__builtin_fmaf(p[n][r], d, -static_cast<float>(hi)));
          if constexpr (MASK) {
            if (pos0 + r >= vis) hi = lo = static_cast<_Float16>(0.0f);
          }
          ph[n][b][k] = hi;
          pl[n][b][k] = lo;
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      each_block(b, [&]<int K>(half4_t lo16, half4_t hi16) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          w.o[n][b][0] = __builtin_amdgcn_mfma_f32_4x4x4f16(pl[n][b], lo16, w.o[n][b][0], 2, K, 0);
          w.o[n][b][1] = __builtin_amdgcn_mfma_f32_4x4x4f16(pl[n][b], hi16, w.o[n][b][1], 2, K, 0);
          w.o[n][b][0] = __builtin_amdgcn_mfma_f32_4x4x4f16(ph[n][b], lo16, w.o[n][b][0], 2, K, 0);
          w.o[n][b][1] = __builtin_amdgcn_mfma_f32_4x4x4f16(ph[n][b], hi16, w.o[n][b][1], 2, K, 0);
        }
      });
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        float x[4], most = 0.0f, inverse;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = kOrder[k];
          x[k] = p[n][r] * half_of(vd[b], r);
          if constexpr (MASK) x[k] = pos0 + r < vis ? x[k] : 0.0f;
          most = fmaxf(most, fabsf(x[k]));
        }
        const float by = to_fp16_range(head_max(most), inverse);
        half2_t hi[2], lo[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) split2(x[2 * i] * by, x[2 * i + 1] * by, hi[i], lo[i]);
        const half4_t ph = join4(hi[0], hi[1]), pl = join4(lo[0], lo[1]);
        f32x4 even = {0.0f, 0.0f, 0.0f, 0.0f}, odd = {0.0f, 0.0f, 0.0f, 0.0f};
        each_block(b, [&]<int K>(half4_t lo16, half4_t hi16) {
          even = __builtin_amdgcn_mfma_f32_4x4x4f16(pl, lo16, even, 2, K, 0);
          odd = __builtin_amdgcn_mfma_f32_4x4x4f16(pl, hi16, odd, 2, K, 0);
          even = __builtin_amdgcn_mfma_f32_4x4x4f16(ph, lo16, even, 2, K, 0);
          odd = __builtin_amdgcn_mfma_f32_4x4x4f16(ph, hi16, odd, 2, K, 0);
        });
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float of_head = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(inverse), r));
          w.o[n][b][0][r] += even[r] * of_head;
          w.o[n][b][1][r] += odd[r] * of_head;
        }
        __builtin_amdgcn_sched_barrier(0);  // (one after another, in few registers)
      }
    }
  }
}

// One row of one KV head (and one run of positions): W waves take every W-th 64 positions each.
template <int NB, int NS, int W>
__global__ __launch_bounds__(W * 64) void attention_kv4_row_kernel(AttnKv4Args a, Kv4Plan plan) {
  using Ring = TileRing<NB, W, 2>;
  constexpr uint32_t kDim = 32 * NB, kHeads = 4 * NS, kTileBytes = kv4_tile_bytes(kDim);
  constexpr uint32_t kStride = kDim + 16;  // floats between heads where the parts meet
  constexpr uint32_t kRingBytes = W * Ring::kWaveBytes, kMeetBytes = W * kHeads * kStride * 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kRingBytes > kMeetBytes ? kRingBytes : kMeetBytes];
  __shared__ float lds_ref[W][kHeads], lds_sum[W][kHeads];
  uint32_t id = blockIdx.x;
  const uint32_t h = id % a.n_kv;
  id /= a.n_kv;
  const uint32_t split = id % plan.splits, r = plan.row0 + id / plan.splits;
  const uint32_t group = a.n_head / a.n_kv;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  // (both on their way before either is needed)
  const int64_t cache_off = a.cache_off != nullptr ? a.cache_off[r] : 0;
  const int32_t vis = row_vis(a, r);
  const uint32_t tiles = kv4_tiles(static_cast<uint32_t>(vis));
  const uint32_t first = split * plan.split_tiles;  // (splits are whole steps of two tiles)
  if (plan.splits > 1 && first >= tiles) return;    // an empty part: the joining kernel knows which there are
  const uint32_t last = min(tiles, first + plan.split_tiles);
  const uint32_t step0 = first / 2 + wave, steps = (last + 1) / 2;
  const uint32_t n = __builtin_amdgcn_readfirstlane(step0 < steps ? (steps - step0 + W - 1) / W : 0);

  Ring ring;
  ring.base = static_cast<const uint8_t*>(a.cache) + cache_off + a.layer_off +
              static_cast<size_t>(h) * kv4_tiles(a.max_ctx) * kTileBytes;
  ring.lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(as_lds(lds))) + wave * Ring::kWaveBytes;
  ring.lane = lane;
  // A last step of one tile: the copy ends with the tile.
  const auto bytes_of = [&](uint32_t step) { return min(2u, tiles - 2 * step) * kTileBytes; };
  constexpr uint32_t kAhead = Ring::kDepth - 1;
  // The queries come first, through the slot that is filled last (zeros for heads past the group: nothing is
  // read there), then the first steps; a step there is not reads nothing. The queries are then waited for alone,
  // and prepared while the first tiles are on their way (0.7 us less for a row of 1024 positions, now 5.9, than
  // with both waited for).
  static_assert(kHeads * kDim * 4 <= Ring::kBytes, "the queries fit a slot");
  const RsrcWords qr = raw_buffer_words(a.q + static_cast<size_t>(r) * a.q_stride + h * group * kDim, group * kDim * 4);
#pragma unroll
  for (uint32_t j = 0; j < kHeads * kDim; j += 64) lds_dma4(qr, (j + lane) * 4, ring.lds + kAhead * Ring::kBytes + j * 4);
#pragma unroll
  for (uint32_t j = 0; j < kAhead; ++j) ring.fetch(step0 + j * W, j, j < n ? bytes_of(step0 + j * W) : 0u);
  wait_vm<kAhead * Ring::kLoads>();
  f32x4 x[NS][2 * NB];
#pragma unroll
  for (int c = 0; c < NS; ++c)
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j)
      x[c][j] = *reinterpret_cast<const f32x4*>(lds + wave * Ring::kWaveBytes + kAhead * Ring::kBytes +
                                                ((4 * c + lane % 4) * kDim + 16 * j + 4 * (lane / 16)) * 4);

  RowState<NB, NS> w;
#pragma unroll
  for (int c = 0; c < NS; ++c) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t) top = fmaxf(top, fabsf(x[c][j][t]));
    const QueryScale by = query_scale(column_max(top), a.scale);
    w.colf[c] = by.factor;
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j) {
      half2_t hi[2], lo[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) split2(by(x[c][j][2 * t]), by(x[c][j][2 * t + 1]), hi[t], lo[t]);
      w.qhi[c][j] = join4(hi[0], hi[1]);
      w.qlo[c][j] = join4(lo[0], lo[1]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int k = 0; k < 2; ++k) w.o[c][b][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    w.top[c] = w.limit[c] = -__builtin_inff();
    w.ref[c] = 0.0f;
    w.sum[c] = 0.0f;
  }

  const CodeBits bits;
  const uint8_t* slots = lds + wave * Ring::kWaveBytes;
  for (uint32_t j = 0; j < n; ++j) {
    // The slot that the next copy goes to was read in the step before: its reads have returned.
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    if (j + kAhead < n) {
      ring.fetch(step0 + (j + kAhead) * W, (j + kAhead) % Ring::kDepth, bytes_of(step0 + (j + kAhead) * W));
      wait_vm<kAhead * Ring::kLoads>();
    } else if (kAhead > 2 && j + 3 == n) {
      wait_vm<2 * Ring::kLoads>();
    } else if (kAhead > 1 && j + 2 == n) {
      wait_vm<Ring::kLoads>();
    } else {
      wait_vm<0>();
    }
    const uint32_t step = step0 + j * W;
    const uint32_t slot = j % Ring::kDepth;
    const uint8_t* at = slots + slot * Ring::kBytes;
    const int32_t first = static_cast<int32_t>(step * 64), pos0 = first + static_cast<int32_t>(lane / 4 * 4);
    const bool mask = first + 64 > vis;
    const bool wide = mask ? wide_scales<NB, 2, true>(at, lane, first, vis) : wide_scales<NB, 2, false>(at, lane, first, vis);
    if (__builtin_expect(wide, 0)) {
      row_step<NB, NS, true, true>(w, bits, slots, slot, lane, vis, pos0);
    } else if (mask) {
      row_step<NB, NS, true, false>(w, bits, slots, slot, lane, vis, pos0);
    } else {
      row_step<NB, NS, false, false>(w, bits, slots, slot, lane, vis, pos0);
    }
  }

  // The waves' parts meet, where the tiles were: no copy is on its way any more, those of a wave without a step
  // (zeros) among them.
  wait_vm<0>();
  __syncthreads();
  float* meet = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int c = 0; c < NS; ++c) {
    float sum = w.sum[c];
    sum += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(sum), 0x124, 0xf, 0xf, true));  // row_ror 4
    sum += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(sum), 0x128, 0xf, 0xf, true));  // row_ror 8
    sum = column_sum(sum);
    if (lane < 4) {
      // A wave without a visible position takes no part.
      lds_ref[wave][4 * c + lane] = w.top[c] == -__builtin_inff() && sum == 0.0f ? -__builtin_inff() : w.ref[c];
      lds_sum[wave][4 * c + lane] = sum;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        meet[(wave * kHeads + 4 * c + lane / 16) * kStride + 32 * b + 16 * k + lane % 16] = row_sums(w.o[c][b][k]);
    }
  }
  __syncthreads();
  // A thread an output (whole waves), its parts one after another (0.4 us less for a row of 1024 positions than
  // eight outputs a thread, all of them one wave's).
  for (uint32_t u = threadIdx.x; u < kHeads * kDim; u += W * 64) {
    const uint32_t col = u / kDim, d = u % kDim;
    float ref = -__builtin_inff(), sum = 0.0f, o = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < W; ++k) ref = fmaxf(ref, lds_ref[k][col]);
#pragma unroll
    for (uint32_t k = 0; k < W; ++k) {
      const float part = lds_ref[k][col];
      const float f = part != -__builtin_inff() ? exp2_fast(part - ref) : 0.0f;
      sum += f * lds_sum[k][col];
      o += f * meet[(k * kHeads + col) * kStride + d];
    }
    if (col >= group) continue;  // (a whole block of 32 lanes, or more)
    const uint32_t head = h * group + col;
    if (plan.splits > 1) {
      float* part = a.scratch + ((static_cast<size_t>(r - plan.row0) * a.n_head + head) * plan.splits + split) * part_floats(kDim);
      part[d] = o;
      if (d == 0) {
        part[kDim] = ref;
        part[kDim + 1] = sum;
      }
      continue;
    }
    // A row that sees no position gives zeros.
    const float y = ref == -__builtin_inff() ? 0.0f : o * __builtin_amdgcn_rcpf(sum);
    a.out[static_cast<size_t>(r) * a.out_stride + head * kDim + d] = y;
    if (a.outq != nullptr)
      quantize_block_lanes(y, d % kQK, static_cast<uint8_t*>(a.outq) +
                                           ((static_cast<size_t>(r) * a.n_head + head) * NB + d / kQK) * kBytesQ8_0);
  }
}

// Joins the parts of a (row, head) pair: grid (heads, rows). Threads first bring every part's
// reference to its factor, then 256 / head_dim of them a value add the parts up. What a thread adds of the first
// parts is on its way before it is known which parts there are (1.2 us less for one row of 8192 positions, now
// 7.8, than with one load behind another).
constexpr uint32_t kMaxSplits = 128;
__global__ __launch_bounds__(256) void attention_kv4_join_kernel(AttnKv4Args a, Kv4Plan plan) {
  __shared__ float factor[kMaxSplits], red[4], sums[4], acc[256];
  const uint32_t head = blockIdx.x, r = plan.row0 + blockIdx.y, tid = threadIdx.x, lane = tid & 63u;
  const uint32_t stride = part_floats(a.head_dim);
  const float* part = a.scratch + (static_cast<size_t>(blockIdx.y) * a.n_head + head) * plan.splits * stride;
  const float none = -__builtin_inff();
  float ref = none, sum = 0.0f;
  if (tid < plan.splits) {
    ref = part[tid * stride + a.head_dim];
    sum = part[tid * stride + a.head_dim + 1];
  }
  const uint32_t per = 256 / a.head_dim, set = tid / a.head_dim, d = tid - set * a.head_dim;
  constexpr uint32_t kEarly = 4;
  float early[kEarly];
#pragma unroll
  for (uint32_t i = 0; i < kEarly; ++i) early[i] = set < per && set + i * per < plan.splits ? part[(set + i * per) * stride + d] : 0.0f;
  const uint32_t n = (kv4_tiles(static_cast<uint32_t>(row_vis(a, r))) + plan.split_tiles - 1) / plan.split_tiles;
  if (tid >= n) {  // (whatever was there)
    ref = none;
    sum = 0.0f;
  }
  const float top = wave_max(ref);
  if (lane == 0) red[tid / 64] = top;
  __syncthreads();
  const float all = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float f = ref == none ? 0.0f : exp2_fast(ref - all);
  if (tid < n) factor[tid] = f;
  float total = f * sum;  // (of a part too far below to count too: a NaN in it does)
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
  if (lane == 0) sums[tid / 64] = total;
  __syncthreads();
  float o = 0.0f;
  if (set < per) {
#pragma unroll
    for (uint32_t i = 0; i < kEarly; ++i)
      if (set + i * per < n) o += factor[set + i * per] * early[i];
#pragma unroll 4
    for (uint32_t s = set + kEarly * per; s < n; s += per) o += factor[s] * part[s * stride + d];
  }
  acc[tid] = o;
  __syncthreads();
  if (tid < a.head_dim) {
    for (uint32_t k = 1; k < per; ++k) o += acc[k * a.head_dim + tid];
    const float y = all == none ? 0.0f : o / ((sums[0] + sums[1]) + (sums[2] + sums[3]));
    a.out[static_cast<size_t>(r) * a.out_stride + head * a.head_dim + tid] = y;
    if (a.outq != nullptr)
      quantize_block_lanes(y, tid & 31u, static_cast<uint8_t*>(a.outq) +
                                             ((static_cast<size_t>(r) * a.n_head + head) * (a.head_dim / kQK) + tid / kQK) * kBytesQ8_0);
  }
}

// Column tiles of a wave at most, for rows of a chunk: two while the registers allow it.
constexpr uint32_t chunk_tiles(uint32_t nb) { return nb <= 4 ? 2 : 1; }

// Splits of rows' positions over workgroups of `waves` waves: for a workgroup a CU (two a CU cost more in
// the joining than they gained: 32 rows of 4096 positions 16.0 us with 256, 21.3 with 512) while each wave keeps
// two tiles, and none that does not spare every wave four tiles (one row of 1024 positions 5.9 us, in two parts
// 7.3; 16 rows of 1536 7.7 and 9.4; one row of 2048 8.6 and in four parts 7.4; of 8192 25.2 and in sixteen 7.8).
void split_positions(Kv4Plan& p, const AttnKv4Args& a, size_t items) {
  const uint32_t tiles = std::max(1u, kv4_tiles(a.max_vis));
  const uint32_t whole = p.by_row ? 2 * p.waves : p.waves;  // tiles of a step of all waves
  const size_t want = std::max<size_t>(1, 256 / std::max<size_t>(1, items));
  const size_t most = tiles <= 4 * p.waves ? 1 : ceil_div(tiles, 2 * p.waves);
  const size_t splits = std::min({want, most, static_cast<size_t>(kMaxSplits)});
  p.most_splits = static_cast<uint32_t>(splits);
  p.split_tiles = static_cast<uint32_t>(ceil_div(ceil_div(tiles, splits), whole) * whole);
  if (p.split_tiles + 4 * p.waves > tiles) p.split_tiles = tiles;
  p.splits = static_cast<uint32_t>(ceil_div(tiles, p.split_tiles));
}

// Rows of their own: the kernel for single rows where it has the head size and the group.
Kv4Plan decode_plan(const AttnKv4Args& a, uint32_t row0, uint32_t n_rows) {
  Kv4Plan p{};
  p.row0 = row0;
  p.n_rows = n_rows;
  p.block_rows = 1;
  const uint32_t group = a.n_head / a.n_kv;
  p.by_row = group <= 8 && a.head_dim <= 128;
  p.col_blocks = static_cast<uint32_t>(ceil_div(group, 16));
  const uint32_t tiles = kv4_tiles(a.max_vis);
  // Four waves up to two steps each (a step is a tile, of single rows two): 256 rows of 512 positions 22.0 us, with
  // eight 22.5; 64 rows 6.8 and 7.05; but one row 4.9 and 4.6.
  // (Eight waves of two sets of heads of size 128 would not have the registers.)
  p.waves = tiles <= (p.by_row ? 16u : 8u) || a.head_dim > 128 || (p.by_row && group > 4 && a.head_dim > 96) ? 4 : 8;
  split_positions(p, a, static_cast<size_t>(n_rows) * a.n_kv * p.col_blocks);
  return p;
}

// A chunk's rows. Two tiles of columns a wave share the codes' extraction, two waves on a set of columns
// read a tile half as often as four; both need the columns to fill the chip. One tile and four waves are split over
// positions, the others not. In us, from graph replays of 32 heads over 8 KV heads:
//   size, rows behind positions    one tile, 4 waves   one, 2    two, 4    two, 2
//   64, 128 behind 4000                         28.9     49.3      38.9      69.1
//   64, 512 behind 0                            11.2     10.9      11.8      14.6
//   64, 2000 behind 0                           73.8     67.1      61.7      60.4
//   64 (14 heads over 2), 2000 behind 0         37.1     38.7      33.0      39.2
//   128, 2000 behind 0                         124      111       105        97.8
Kv4Plan chunk_plan(const AttnKv4Args& a, uint32_t n_rows) {
  Kv4Plan p{};
  p.n_rows = n_rows;
  p.chunk = true;
  p.waves = 4;
  const uint32_t group = a.n_head / a.n_kv;
  p.per_group = 65536 / group + (65536 % group != 0);
  const auto sized = [&](uint32_t tiles, uint32_t shared_by) {
    const uint32_t cols = 16 * tiles * p.waves / shared_by;
    p.col_tiles = tiles;
    p.shared_by = shared_by;
    p.block_rows = std::max(1u, cols / group);
    p.col_blocks = static_cast<uint32_t>(ceil_div(group, cols));
    return ceil_div(n_rows, p.block_rows) * a.n_kv * p.col_blocks;
  };
  p.splits = 1;
  p.split_tiles = kv4_tiles(a.max_vis);
  if (chunk_tiles(a.head_dim / kQK) == 2 && (sized(2, 2) >= 512 || sized(2, 4) >= 768)) return p;
  if (sized(1, 2) < 512) split_positions(p, a, sized(1, 4));
  return p;
}

int launched(const AttnKv4Args& a, const Kv4Plan& p) {
  if (const int rc = check_launch("attention_kv4"); rc != kOk || p.splits == 1) return rc;
  hipLaunchKernelGGL(attention_kv4_join_kernel, dim3(a.n_head, p.n_rows), dim3(256), 0, stream(), a, p);
  return check_launch("attention_kv4 join");
}

size_t workgroups(const AttnKv4Args& a, const Kv4Plan& p) {
  return ceil_div(p.n_rows, p.block_rows) * a.n_kv * p.col_blocks * p.splits;
}

template <int NB, int CT, int KS, int W>
int run(const AttnKv4Args& a, const Kv4Plan& p) {
  hipLaunchKernelGGL((attention_kv4_kernel<NB, CT, KS, W>), dim3(static_cast<uint32_t>(workgroups(a, p))), dim3(W * 64), 0, stream(), a, p);
  return launched(a, p);
}

template <int NB, int NS, int W>
int run_rows(const AttnKv4Args& a, const Kv4Plan& p) {
  hipLaunchKernelGGL((attention_kv4_row_kernel<NB, NS, W>), dim3(static_cast<uint32_t>(workgroups(a, p))), dim3(W * 64), 0, stream(), a, p);
  return launched(a, p);
}

template <int NB>
int launch_nb(const AttnKv4Args& a, uint32_t n_rows) {
  if (a.chunk_rows != 0) {
    const Kv4Plan p = chunk_plan(a, a.chunk_rows);
    int rc = kOk;
    if constexpr (chunk_tiles(NB) == 2) {
      if (p.col_tiles == 2) rc = p.shared_by == 2 ? run<NB, 2, 2, 4>(a, p) : run<NB, 2, 4, 4>(a, p);
    }
    if (p.col_tiles == 1) rc = p.shared_by == 2 ? run<NB, 1, 2, 4>(a, p) : run<NB, 1, 4, 4>(a, p);
    if (rc != kOk) return rc;
  }
  if (n_rows == a.chunk_rows) return kOk;
  const Kv4Plan p = decode_plan(a, a.chunk_rows, n_rows - a.chunk_rows);
  if constexpr (NB <= 4) {
    if (p.by_row) {
      if (a.n_head / a.n_kv <= 4) return p.waves == 8 ? run_rows<NB, 1, 8>(a, p) : run_rows<NB, 1, 4>(a, p);
      if constexpr (NB <= 3)
        if (p.waves == 8) return run_rows<NB, 2, 8>(a, p);
      return run_rows<NB, 2, 4>(a, p);
    }
    if (p.waves == 8) return run<NB, 1, 8, 8>(a, p);
  }
  return run<NB, 1, 4, 4>(a, p);
}

size_t plan_floats(const AttnKv4Args& a, const Kv4Plan& p) {
  return p.most_splits <= 1 ? 0 : static_cast<size_t>(p.n_rows) * a.n_head * p.most_splits * part_floats(a.head_dim);
}

}  // namespace

// The chunk's rows and the others run one after the other, in the same scratch.
size_t attention_kv4_scratch_floats(const AttnKv4Args& a, uint32_t n_rows) {
  size_t floats = 0;
  if (a.chunk_rows != 0) floats = plan_floats(a, chunk_plan(a, std::min(a.chunk_rows, n_rows)));
  if (n_rows > a.chunk_rows) floats = std::max(floats, plan_floats(a, decode_plan(a, a.chunk_rows, n_rows - a.chunk_rows)));
  return floats;
}

// (Of either part, before the first is launched.)
int attention_kv4_check_size(const AttnKv4Args& a, uint32_t n_rows) {
  size_t most = 0;
  if (a.chunk_rows != 0) most = workgroups(a, chunk_plan(a, a.chunk_rows));
  if (n_rows > a.chunk_rows) most = std::max(most, workgroups(a, decode_plan(a, a.chunk_rows, n_rows - a.chunk_rows)));
  return launch_fits("attention_kv4", most, 512, 1);
}

int attention_kv4_launch(const AttnKv4Args& a, uint32_t n_rows) {
  switch (a.head_dim / kQK) {
  case 1: return launch_nb<1>(a, n_rows);
  case 2: return launch_nb<2>(a, n_rows);
  case 3: return launch_nb<3>(a, n_rows);
  case 4: return launch_nb<4>(a, n_rows);
  case 6: return launch_nb<6>(a, n_rows);
  default: return launch_nb<8>(a, n_rows);
  }
}

}  // namespace axon_hip
