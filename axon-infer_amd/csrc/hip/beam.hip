// Beam search: one step's selection over beams and vocabulary, and the beams' caches brought into the
// order of their survivors.
//
// Selection. The score of token v behind beam b is score_b + x_bv - lse_b, lse_b = log sum_v exp x_bv, so
// inside a row the order is that of the logits and lse_b only shifts it: one pass over the logits suffices
// for the sums, and finds where the best candidates can be. The first kernel reads every logit once and
// leaves each chunk's maximum and its sum of exponentials below it (a wave per chunk, up to 1024 logits in
// registers). The second, a workgroup per group of beams, joins the sums (in 64 bits) and takes the n_out
// chunks with the best maxima: a candidate of any other chunk has n_out better ones, those chunks' best. Of
// the chunk in place r no more than n_out - r candidates can be wanted, since r chunks have a better
// one, so what has to be kept is bounded however the logits lie. The chunks come from a bound near the
// n_out-th best of the lanes' (twice the best of 16 steps, counted by all waves), which hardly more than n_out
// reach as a rule; where too many do (equal maxima), from each beam's best one by one. An entry's place is
// its count of better ones, so the order in which waves arrive does not matter.
// The order is total: scores in 64 bits, then beam, then (in a beam) logit, then token.
// Bound: the logits' bytes, 4 a candidate; the second kernel's latency comes on top. 8 groups of 8 beams
// over 151936 tokens: 38.9 MB in 7.0 to 7.7 us (5.0 to 5.5 TB/s), then 6.9 us, of which about 1.8 read the parts and join
// the sums, 1.1 find the bound, 1.4 read the chosen chunks and 1.8 gather and rank.
//
// Reorder. A thread holds one 16-byte piece of every slot of a group that changes: it loads all of them
// from their parents before it stores any, and no other thread touches those bytes, so the exchange is in
// place without a copy of the pool and without waiting for others. Slots that are their own parents cost
// nothing. Bound by the bytes read (each parent once from HBM) and written.
#include "beam.h"
#include "common.h"

#include <algorithm>

namespace axon_hip {

namespace {

// ------------------------------------------------------------------------------------------
// Selection

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kScanThreads = 256;
constexpr uint32_t kPickThreads = 1024;

// Logits per lane of a chunk: few where a group's rows are short, so that they make 128 chunks and more
// (n_out of them are read again).
uint32_t chunk_lane_values(size_t n, size_t n_beams) {
  const size_t all = n * n_beams;
  return all >= 128 * 64 * 16 ? 16 : all >= 128 * 64 * 4 ? 4 : 1;
}

struct ChunkPart {
  float max, sum;  // the largest logit and sum of exp(x - max); -inf and 0 without a candidate
};

__device__ __forceinline__ float wave_sum_f(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// Where a chunk's value k of a lane is, loaded in runs of four: lanes next to each other read what is.
template <int E>
__device__ __forceinline__ uint32_t chunk_place(uint32_t lane, uint32_t k) {
  return E % 4 == 0 ? k / 4 * 256 + lane * 4 + k % 4 : k * 64 + lane;
}
// The chunk at x + at of a row of n; -inf past its end.
template <int E>
__device__ __forceinline__ void load_chunk(float (&v)[E], const float* x, size_t at, size_t n, uint32_t lane) {
  const float none = -__builtin_inff();
  if constexpr (E % 4 == 0) {
#pragma unroll
    for (int k = 0; k < E; k += 4) {
      const size_t i = at + chunk_place<E>(lane, k);
      if (i + 4 <= n) {
        const f32x4_a4 u = *reinterpret_cast<const f32x4_a4*>(x + i);
#pragma unroll
        for (int t = 0; t < 4; ++t) v[k + t] = u[t];
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) v[k + t] = i + t < n ? x[i + t] : none;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = at + chunk_place<E>(lane, k) < n ? x[at + chunk_place<E>(lane, k)] : none;
  }
}

// grid (workgroups of 4 chunks, rows).
template <int E>
__global__ __launch_bounds__(kScanThreads) void beam_scan_kernel(BeamSelectArgs a, uint32_t chunks, ChunkPart* __restrict__ part) {
  const uint32_t row = blockIdx.y;
  if (!(a.scores[row] > -__builtin_inff())) return;  // a dropped beam
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t chunk = blockIdx.x * (kScanThreads / 64) + threadIdx.x / 64;
  if (chunk >= chunks) return;
  const float* x = a.x + static_cast<size_t>(row) * a.stride;
  const float none = -__builtin_inff();
  float v[E];
  load_chunk<E>(v, x, static_cast<size_t>(chunk) * (64 * E), a.n, lane);
  float m = none;
#pragma unroll
  for (int k = 0; k < E; ++k) m = fmaxf(m, v[k]);  // (passes over NaN)
  m = wave_max(m);
  float sum = 0.0f;
  if (m != none) {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      // A NaN logit adds nothing; with an infinite one the sum is NaN, and the beam has no candidate.
      const float e = __builtin_amdgcn_exp2f((v[k] - m) * 1.4426950408889634f);
      sum += v[k] == v[k] ? e : 0.0f;
    }
  }
  sum = wave_sum_f(sum);
  if (lane == 0) part[static_cast<size_t>(row) * chunks + chunk] = ChunkPart{m, sum};
}

// The largest of v[0..N) over the wave, the lowest lane that holds it and, in that lane, its first place:
// taken out of v (NaN stands for a value that is gone; maxima pass over it). Returns -inf where nothing is
// left. `lane_of` and `place` are the same in every lane.
template <int N>
__device__ __forceinline__ float take_best(float (&v)[N], uint32_t lane, uint32_t& lane_of, uint32_t& place) {
  float best = v[0];
#pragma unroll
  for (int k = 1; k < N; ++k) best = fmaxf(best, v[k]);
  const float top = wave_max(best);
  lane_of = static_cast<uint32_t>(__ffsll(__ballot(best == top))) - 1;
  uint32_t at = 0;
#pragma unroll
  for (int k = N - 1; k >= 0; --k) at = v[k] == top ? k : at;
  place = __builtin_amdgcn_readlane(at, lane_of & 63u);
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = lane == lane_of && k == static_cast<int>(place) ? __builtin_nanf("") : v[k];
  return top;
}

// Candidates kept: of the chunk in place r = 0, 1, ... at most n_out - r.
constexpr uint32_t kListed = kMaxBeamOut * (kMaxBeamOut + 1) / 2;
constexpr uint32_t kSurvivors = 512;  // chunks at the bound; more of them take the lists

// A chunk by its best logit, or a candidate.
struct Scored {
  double s;
  float x;
  uint32_t beam, id;
};
// The order: score, beam, then in a beam logit and place.
__device__ __forceinline__ bool better(const Scored& a, const Scored& b) {
  const bool in_beam = (a.x > b.x) | ((a.x == b.x) & (a.id < b.id));
  return (a.s > b.s) | ((a.s == b.s) & ((a.beam < b.beam) | ((a.beam == b.beam) & in_beam)));
}

struct PickShared {
  double base[kMaxBeams];                      // score - lse
  uint32_t live[kMaxBeams];                    // whether the beam has candidates
  alignas(16) float best[kPickThreads * 2];    // each lane's best chunk of a beam, rounded down
  float top[kMaxBeams];                        // a beam's largest of them
  uint32_t reach[2][16];                       // how many reach each step of the bound's two rounds
  uint32_t chunks_of[kMaxBeams];               // the lists: entries of a beam's,
  float chunk_max[kMaxBeams * kMaxBeamOut];    // its best chunks, best first
  uint32_t chunk_id[kMaxBeams * kMaxBeamOut];
  Scored survivor[kSurvivors];
  uint32_t survivors;
  uint32_t chosen;                             // chunks taken, best first:
  uint32_t chosen_beam[kMaxBeamOut];
  uint32_t chosen_id[kMaxBeamOut];
  double chosen_score[kMaxBeamOut];
  uint32_t found;                              // candidates, in any order:
  Scored candidate[kListed];
};

// How many of best[0..64 per) reach `at` of the lanes with one lane % 16 (16 steps), added up over the waves in
// reach[lane % 16]: every lane takes `per`. (With 64 steps, every lane over its wave's all, it took four times
// as long.)
__device__ __forceinline__ void count_reaching(const float* best, uint32_t per, float at, uint32_t lane, uint32_t wave, uint32_t* reach) {
  uint32_t count = 0;
#pragma unroll 1
  for (uint32_t i = 0; i < per; i += 8) {
#pragma unroll
    for (uint32_t j = 0; j < 8; j += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(best + (wave * 4 + lane / 16) * per + i + j);
#pragma unroll
      for (int t = 0; t < 4; ++t) count += v[t] >= at ? 1u : 0u;
    }
  }
  if (count != 0) atomicAdd(&reach[lane % 16], count);
}

// A finite float that no finite x with base + x >= least is below, the sum rounded to 64 bits.
__device__ __forceinline__ float least_addend(double least, double base) {
  return fmaxf(__double2float_rd((least - base) - 0x1p-50 * fmax(fabs(least), fabs(base))), -3.40282347e38f);
}

// The places of entries by counting the better ones: calls put(entry, place) in one lane for each that has a
// place below n_out. A wave takes an entry at a time, a lane each of the others.
template <typename Put>
__device__ __forceinline__ void rank_entries(const Scored* all, uint32_t n, uint32_t n_out, uint32_t lane, uint32_t wave, Put put) {
  for (uint32_t e = wave; e < n; e += kPickThreads / 64) {
    const Scored me = all[e];
    uint32_t rank = 0;
    for (uint32_t j0 = 0; j0 < n && rank < n_out; j0 += 64) {
      const uint32_t j = j0 + lane;
      const Scored other = all[min(j, n - 1)];
      rank += static_cast<uint32_t>(__popcll(__ballot(j < n && better(other, me))));
    }
    if (lane == 0 && rank < n_out) put(me, rank);
  }
}

// The beam's chunk lists (where more chunks than kSurvivors reach the bound, as many equal maxima do): a
// beam's best chunks one by one, then their places among all by bisection of the other lists.
template <int L>
__device__ void choose_by_lists(PickShared& sh, const ChunkPart* part, uint32_t beams, uint32_t chunks, uint32_t n_out,
                                uint32_t lane, uint32_t wave) {
  constexpr uint32_t kPickWaves = kPickThreads / 64;
  const float none = -__builtin_inff();
  // Lane l holds chunks L l .. L l + L - 1, so the lowest lane with a maximum, and its first place, is the
  // first chunk with it.
  for (uint32_t b = wave; b < beams; b += kPickWaves) {
    uint32_t taken = 0;
    if (sh.live[b] != 0) {
      float m[L];
#pragma unroll
      for (int k = 0; k < L; ++k) m[k] = lane * L + k < chunks ? part[static_cast<size_t>(b) * chunks + lane * L + k].max : none;
      for (; taken < n_out; ++taken) {
        uint32_t l, k;
        const float best = take_best<L>(m, lane, l, k);
        if (!(best > none)) break;
        if (lane == 0) {
          sh.chunk_max[b * n_out + taken] = best;
          sh.chunk_id[b * n_out + taken] = l * L + k;
        }
      }
    }
    if (lane == 0) sh.chunks_of[b] = taken;
  }
  __syncthreads();
  for (uint32_t b = wave; b < beams; b += kPickWaves) {
    if (lane < sh.chunks_of[b]) {
      const double s = sh.base[b] + static_cast<double>(sh.chunk_max[b * n_out + lane]);
      uint32_t rank = lane;
      for (uint32_t o = 0; o < beams && rank < n_out; ++o) {
        if (o == b) continue;
        uint32_t lo = 0, hi = sh.chunks_of[o];  // the first entry of o that is not better
        while (lo < hi) {
          const uint32_t mid = (lo + hi) / 2;
          const double t = sh.base[o] + static_cast<double>(sh.chunk_max[o * n_out + mid]);
          if (t > s || (t == s && o < b)) lo = mid + 1;
          else hi = mid;
        }
        rank += lo;
      }
      if (rank < n_out) {
        sh.chosen_beam[rank] = b;
        sh.chosen_id[rank] = sh.chunk_id[b * n_out + lane];
        sh.chosen_score[rank] = s;
        atomicMax(&sh.chosen, rank + 1);  // (places have no gaps: the largest is the count)
      }
    }
  }
}

// E logits per lane of a chunk, L chunks per lane of a row.
template <int E, int L>
__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(BeamSelectArgs a, uint32_t chunks, const ChunkPart* __restrict__ all_parts) {
  __shared__ PickShared sh;
  constexpr uint32_t kPickWaves = kPickThreads / 64;
  const float none = -__builtin_inff();
  const uint32_t beams = static_cast<uint32_t>(a.n_beams), n_out = static_cast<uint32_t>(a.n_out);
  const uint32_t row0 = blockIdx.x * beams;
  const ChunkPart* part = all_parts + static_cast<size_t>(row0) * chunks;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  if (tid == 0) sh.survivors = sh.chosen = sh.found = 0;
  if (tid < 32) sh.reach[tid / 16][tid % 16] = 0;
  // A wave per beam (two at most): its lse, and each lane's chunks' scores.
  float best_of[2][L];
  double bases[2] = {0.0, 0.0};
#pragma unroll
  for (uint32_t turn = 0; turn < 2; ++turn) {
    const uint32_t b = wave + turn * kPickWaves;
    float best = none;
#pragma unroll
    for (int k = 0; k < L; ++k) best_of[turn][k] = none;
    if (b < beams) {
      // (a dropped beam's parts are whatever was there: they are loaded along and not used)
      const ChunkPart* p = part + static_cast<size_t>(b) * chunks;
      float m[L], sums[L];
#pragma unroll
      for (int k = 0; k < L; ++k) {
        const uint32_t c = lane * L + k;
        const ChunkPart q = p[min(c, chunks - 1)];
        m[k] = c < chunks ? q.max : none;
        sums[k] = q.sum;
      }
      const float score = a.scores[row0 + b];
      bool live = false;
      if (score > none) {
        float most = none;
#pragma unroll
        for (int k = 0; k < L; ++k) most = fmaxf(most, m[k]);
        const float top = wave_max(most);
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < L; ++k) {
          const float f = m[k] > none ? __builtin_amdgcn_exp2f((m[k] - top) * 1.4426950408889634f) : 0.0f;
          sum += static_cast<double>(sums[k]) * static_cast<double>(f);
        }
        sum = wave_sum(sum);
        const double base = static_cast<double>(score) - (static_cast<double>(top) + log(sum));
        // With an infinite logit, or without any, the sum is not a number or 0: no candidates.
        live = base == base && base > -__builtin_inf() && top > none;
        if (live) {
          if (lane == 0) sh.base[b] = base;
          bases[turn] = base;
#pragma unroll
          for (int k = 0; k < L; ++k) best_of[turn][k] = m[k];
          if (most > none) best = __double2float_rd(base + static_cast<double>(most));
        }
      }
      const float high = wave_max(best);
      if (lane == 0) {
        sh.live[b] = live ? 1 : 0;
        sh.top[b] = high;
      }
    }
    sh.best[turn * kPickThreads + tid] = best;
  }
  __syncthreads();
  // A bound that n_out chunks' best reach, near the n_out-th largest of the lanes': of 16 steps below the
  // largest, each 2.8 times as far (the last takes all), the first that so many reach, then of 16 equal ones
  // between the step before and it. Fewer than n_out: all that there are. The steps are compared as the numbers
  // they are, so how they were rounded does not matter.
  const uint32_t step = lane % 16;
  float hi = wave_max(lane < beams ? sh.top[lane] : none), bound = none;
  float at = step == 15 ? -3.40282347e38f : hi - __builtin_amdgcn_exp2f(1.5f * static_cast<float>(step) - 8.0f);
#pragma unroll 1
  for (uint32_t round = 0; round < 2; ++round) {
    count_reaching(sh.best, beams <= 8 ? 8 : beams <= 16 ? 16 : 32, at, lane, wave, sh.reach[round]);
    __syncthreads();
    const uint64_t enough = __ballot(sh.reach[round][step] >= n_out);
    if (enough == 0) break;
    const uint32_t first = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(enough))) - 1;
    bound = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(at), first));
    if (first != 0) hi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(at), first - 1));
    at = step == 15 ? bound : fmaxf(bound, hi - static_cast<float>(step) * ((hi - bound) * (1.0f / 15.0f)));
  }
#pragma unroll
  for (uint32_t turn = 0; turn < 2; ++turn) {
    const uint32_t b = wave + turn * kPickWaves;
    if (b >= beams) break;
    uint32_t in = 0;
#pragma unroll
    for (int k = 0; k < L; ++k)
      in |= best_of[turn][k] > none && bases[turn] + static_cast<double>(best_of[turn][k]) >= static_cast<double>(bound) ? 1u << k : 0u;
#pragma unroll 1
    for (; in != 0; in &= in - 1) {
      const uint32_t k = static_cast<uint32_t>(__ffs(in)) - 1;
      const uint32_t to = atomicAdd(&sh.survivors, 1u);
      const float m = part[static_cast<size_t>(b) * chunks + lane * L + k].max;
      if (to < kSurvivors) sh.survivor[to] = Scored{bases[turn] + static_cast<double>(m), m, b, lane * L + k};
    }
  }
  __syncthreads();
  const uint32_t survivors = sh.survivors;
  if (survivors <= kSurvivors) {
    rank_entries(sh.survivor, survivors, n_out, lane, wave, [&](const Scored& me, uint32_t rank) {
      sh.chosen_beam[rank] = me.beam;
      sh.chosen_id[rank] = me.id;
      sh.chosen_score[rank] = me.s;
    });
    if (tid == 0) sh.chosen = min(survivors, n_out);
  } else {
    choose_by_lists<L>(sh, part, beams, chunks, n_out, lane, wave);
  }
  __syncthreads();
  // A wave per chosen chunk: its candidates that reach the last chosen chunk's best, at most n_out - r.
  const uint32_t chosen = sh.chosen;
  const double least = chosen == n_out ? sh.chosen_score[n_out - 1] : -__builtin_inf();
  for (uint32_t r = wave; r < chosen; r += kPickWaves) {
    const uint32_t b = sh.chosen_beam[r], c = sh.chosen_id[r];
    const double base = sh.base[b];
    const float* x = a.x + static_cast<size_t>(row0 + b) * a.stride;
    const uint32_t i0 = c * (64 * E);
    float v[E];
    load_chunk<E>(v, x, i0, static_cast<uint32_t>(a.n), lane);
    // Those are rarely more: else one by one.
    const float from = least_addend(least, base);
    uint32_t in = 0;
#pragma unroll
    for (int k = 0; k < E; ++k) in |= v[k] >= from ? 1u << k : 0u;
    // (a lane with two or more is rarer still)
    const bool few = __ballot((in & (in - 1)) != 0) == 0 ? static_cast<uint32_t>(__popcll(__ballot(in != 0))) <= n_out - r
                                                         : wave_sum_f(static_cast<float>(__popc(in))) <= static_cast<float>(n_out - r);
    if (few) {
#pragma unroll 1
      for (; in != 0; in &= in - 1) {
        const uint32_t k = static_cast<uint32_t>(__ffs(in)) - 1;
        const uint32_t id = i0 + chunk_place<E>(lane, k);
        const float best = x[id];
        const double s = base + static_cast<double>(best);
        if (best > none && s >= least) sh.candidate[atomicAdd(&sh.found, 1u)] = Scored{s, best, b, id};
      }
      continue;
    }
    // Equal logits are taken in the tokens' order: a lane's are a run here.
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = i0 + lane * E + k < a.n ? x[i0 + lane * E + k] : none;
    for (uint32_t taken = 0; taken < n_out - r; ++taken) {
      uint32_t l, k;
      const float best = take_best<E>(v, lane, l, k);
      const double s = base + static_cast<double>(best);
      if (!(best > none) || s < least) break;
      if (lane == 0) sh.candidate[atomicAdd(&sh.found, 1u)] = Scored{s, best, b, i0 + l * E + k};
    }
  }
  __syncthreads();
  // Fewer candidates than wanted leave the rest saying so. (Then no bound cut any of them off.)
  const uint32_t found = sh.found;
  rank_entries(sh.candidate, found, n_out, lane, wave, [&](const Scored& me, uint32_t rank) {
    const size_t o = static_cast<size_t>(blockIdx.x) * n_out + rank;
    a.parent[o] = static_cast<int32_t>(me.beam);
    a.token[o] = static_cast<int32_t>(me.id);
    a.score[o] = static_cast<float>(me.s);
  });
  if (tid >= found && tid < n_out) {
    const size_t o = static_cast<size_t>(blockIdx.x) * n_out + tid;
    a.parent[o] = 0;
    a.token[o] = -1;
    a.score[o] = none;
  }
}

// ------------------------------------------------------------------------------------------
// Reorder

// grid (pieces of a region, regions, groups). Two pieces a thread while their registers allow it. What a
// slot needs is the same for every thread and is kept in scalar registers (the compiler cannot see that the
// tables do not lie in the pool).
template <typename V, int BEAMS>
__global__ __launch_bounds__(256) void cache_reorder_kernel(CacheReorderArgs a) {
  constexpr int kPieces = BEAMS <= 8 ? 2 : 1;
  const uint32_t byte0 = (blockIdx.x * 256 * kPieces + threadIdx.x) * static_cast<uint32_t>(sizeof(V));
  const uint32_t beams = static_cast<uint32_t>(a.n_beams);
  const size_t row0 = static_cast<size_t>(blockIdx.z) * beams;
  uint8_t* const region = static_cast<uint8_t*>(a.pool) + static_cast<size_t>(blockIdx.y) * a.region_stride;
  const auto slot = [&](uint32_t i) {
    const uint64_t off = static_cast<uint64_t>(a.slot_off[row0 + i]);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(off));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(off >> 32));
    return region + static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
  };
  V held[BEAMS][kPieces];
  uint32_t live[BEAMS];  // bytes of the region that the slot takes over
#pragma unroll
  for (int i = 0; i < BEAMS; ++i) {
    live[i] = 0;
    if (static_cast<uint32_t>(i) < beams) {
      const int32_t p = __builtin_amdgcn_readfirstlane(a.parent[row0 + i]);
      if (p != i && p >= 0 && static_cast<uint32_t>(p) < beams) {
        const uint32_t len = min(static_cast<uint32_t>(max(__builtin_amdgcn_readfirstlane(a.len[row0 + i]), 0)), static_cast<uint32_t>(a.max_len));
        const uint32_t unit = static_cast<uint32_t>(a.unit_positions);
        live[i] = (len + unit - 1) / unit * static_cast<uint32_t>(a.unit_bytes);
        const uint8_t* from = slot(p);
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const uint32_t byte = byte0 + k * 256 * sizeof(V);
          if (byte < live[i]) held[i][k] = *reinterpret_cast<const V*>(from + byte);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < BEAMS; ++i) {
    if (live[i] != 0) {
      uint8_t* to = slot(i);
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        const uint32_t byte = byte0 + k * 256 * sizeof(V);
        if (byte < live[i]) *reinterpret_cast<V*>(to + byte) = held[i][k];
      }
    }
  }
}

template <typename V>
int reorder(const CacheReorderArgs& a) {
  const size_t live = ceil_div(a.max_len, a.unit_positions) * a.unit_bytes;
  const size_t pieces = ceil_div(live, 256 * sizeof(V) * (a.n_beams <= 8 ? 2 : 1));
  const dim3 grid(static_cast<uint32_t>(pieces), static_cast<uint32_t>(a.n_regions), static_cast<uint32_t>(a.n_groups));
  if (a.n_beams <= 4) hipLaunchKernelGGL((cache_reorder_kernel<V, 4>), grid, dim3(256), 0, stream(), a);
  else if (a.n_beams <= 8) hipLaunchKernelGGL((cache_reorder_kernel<V, 8>), grid, dim3(256), 0, stream(), a);
  else if (a.n_beams <= 16) hipLaunchKernelGGL((cache_reorder_kernel<V, 16>), grid, dim3(256), 0, stream(), a);
  else hipLaunchKernelGGL((cache_reorder_kernel<V, 32>), grid, dim3(256), 0, stream(), a);
  return check_launch("cache_reorder");
}

template <int E, int L>
void pick(const BeamSelectArgs& a, uint32_t chunks, const ChunkPart* part) {
  hipLaunchKernelGGL((beam_pick_kernel<E, L>), dim3(static_cast<uint32_t>(a.n_groups)), dim3(kPickThreads), 0, stream(), a, chunks, part);
}

template <int E>
int select(const BeamSelectArgs& a) {
  const uint32_t chunks = static_cast<uint32_t>(ceil_div(a.n, 64 * E));
  ChunkPart* part = static_cast<ChunkPart*>(a.work);
  const uint32_t rows = static_cast<uint32_t>(a.n_groups * a.n_beams);
  hipLaunchKernelGGL((beam_scan_kernel<E>), dim3(static_cast<uint32_t>(ceil_div(chunks, kScanThreads / 64)), rows), dim3(kScanThreads), 0,
                     stream(), a, chunks, part);
  if (const int rc = check_launch("beam_select scan"); rc != kOk) return rc;
  // 64 L chunks cover a row: 4 a lane up to 262144 logits, 16 up to the most there can be.
  if (chunks <= 64 * 4) pick<E, 4>(a, chunks, part);
  else pick<E, 16>(a, chunks, part);
  return check_launch("beam_select pick");
}

}  // namespace

size_t beam_select_work_bytes(size_t n, size_t n_groups, size_t n_beams) {
  return n_groups * n_beams * ceil_div(n, 64 * chunk_lane_values(n, n_beams)) * sizeof(ChunkPart);
}

int beam_select_launch(const BeamSelectArgs& a) {
  if (a.n_groups == 0) return kOk;
  switch (chunk_lane_values(a.n, a.n_beams)) {
  case 16: return select<16>(a);
  case 4: return select<4>(a);
  default: return select<1>(a);
  }
}

int cache_reorder_launch(const CacheReorderArgs& a) {
  if (a.n_groups == 0 || a.n_regions == 0 || a.max_len == 0 || a.unit_bytes == 0) return kOk;
  const size_t grain = a.region_stride | a.unit_bytes;
  if (grain % 16 == 0) return reorder<u32x4>(a);
  if (grain % 4 == 0) return reorder<uint32_t>(a);
  return reorder<uint16_t>(a);
}

}  // namespace axon_hip
